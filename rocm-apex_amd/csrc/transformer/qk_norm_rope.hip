// RMS norm of every query / key head and the rotary position rotation, one pass each way, for gfx950.
//
//   forward : r = rsqrt(mean(x^2) + eps);  n = x r w;  (y1, y2) = (n1 c - n2 s, n2 c + n1 s)
//   backward: dn = R^T dy;  dw = sum_rows dn x r;  g = dn w;  dx = r (g - x r mean(g x r))
// with (c, s) the cosine / sine of the token's position and (1, 2) the two elements of a rotated
// pair: (i, i + rot/2), or (2i, 2i + 1) when interleaved.  Elements past rot are normed only.
// Everything between the one load and the one store of an element is fp32 in registers: the normed
// value is never rounded to the 16-bit type before it is rotated.
//
// Layout: a head of d elements belongs to a group of G lanes (one per PV pairs; a wave holds 64 / G
// groups); each lane holds PV pairs, as two PV-element vectors, so a rotation never leaves the lane and the
// mean is one sum over the group's lanes.  Half-split pairs load the vectors i and i + rot/2, interleaved ones
// 2 PV consecutive elements.  Where the rotated part or the rest is no multiple of PV pairs, its last lane
// starts earlier: the pairs it shares with its neighbour are computed (and stored) twice and counted
// once, which keeps every access a vector (head 80 with 34 rotated, 32768 x 16 heads bf16: 43-47 us forward and 75
// backward; one pair a lane and step took 103 and 215).
// A forward group takes two heads of its token (cosines and sines are loaded once for them, their loads are
// in flight together), a backward group one, and the registers stay within four waves a SIMD: 51 and 76 us at
// 32768 x 16 heads x 128 bf16, 5.2 and 5.3 TB/s (four heads and two: 56 and 90; a plain copy runs at 4.9).
// Neighbouring groups take neighbouring heads, so one load instruction of a wave covers whole cache lines.
// Blocks are dealt to q and k in proportion to their heads, so a lane's norm weights and dw sums belong to
// one tensor for the whole kernel.
// dw: fp32 per lane over the persistent loop, per block through LDS, then a fixed-order column sum
// over the blocks (no atomics: the same inputs give the same bits).
// Positions outside the table give NaN rows (the table is never read past its end).
#include "apex_amd/device.h"
#include "apex_amd/dispatch.h"
#include "apex_amd/qk_norm_rope_api.h"

namespace apex_amd {
namespace qkr {

constexpr int kThreads = 256;
constexpr int kHeads = 2;  // HB of the forward

// PV elements at p, any element alignment (gfx950 takes 16-byte accesses at 2-byte addresses)
template <typename T, int PV> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T e[PV]; };

template <typename T, int PV>
__device__ __forceinline__ void load(float (&r)[PV], const T* p) {
  const Pack<T, PV> v = *reinterpret_cast<const Pack<T, PV>*>(p);
#pragma unroll
  for (int i = 0; i < PV; ++i) r[i] = to_f(v.e[i]);
}
template <typename T, int PV>
__device__ __forceinline__ void store(T* p, const float (&r)[PV]) {
  Pack<T, PV> v;
#pragma unroll
  for (int i = 0; i < PV; ++i) v.e[i] = from_f<T>(r[i]);
  *reinterpret_cast<Pack<T, PV>*>(p) = v;
}

// A lane's PV pairs.  o1, o2: its two vectors in the head; p0: its first pair's index among the rotated (>=
// rot/2 for pairs that are not); skip: leading pairs that the lane before it counts.
struct Chunk { int o1, o2, p0, skip; };

template <int PV> __host__ __device__ inline int cdiv_pv(int n) { return (n + PV - 1) / PV; }

template <int PV, bool INTER>
__device__ __forceinline__ Chunk chunk_of(int c, int d, int rot) {
  const int half = rot >> 1, rest = (d - rot) >> 1;
  if constexpr (INTER) {
    const int p = min(PV * c, (d >> 1) - PV);
    return {2 * p, 2 * p + PV, p, PV * c - p};
  } else {
    const int c1 = cdiv_pv<PV>(half);
    if (c < c1) {
      const int p = min(PV * c, half - PV);
      return {p, half + p, p, PV * c - p};
    }
    const int p = min(PV * (c - c1), rest - PV);
    return {rot + p, rot + rest + p, half, PV * (c - c1) - p};
  }
}

// sum over a group's G lanes, the same bits in each of them
__device__ __forceinline__ float group_sum(float v, int G, bool pow2, int first) {
  if (pow2) {
    for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
  }
  float t = 0.f;
  for (int i = 0; i < G; ++i) t += __shfl(v, first + i, 64);
  return t;
}

// rotate the pairs held as (a, b); dir = -1 for the transposed rotation
template <int PV, bool INTER>
__device__ __forceinline__ void rotate(float (&a)[PV], float (&b)[PV], const float (&c)[PV], const float (&s)[PV],
                                       float dir) {
#pragma unroll
  for (int i = 0; i < PV; ++i) {
    const float sn = dir * s[i];
    if constexpr (INTER) {
      if constexpr (PV > 1) {
        // pair i sits at elements 2i, 2i + 1 of the 2 PV consecutive ones a | b
        float& x = 2 * i < PV ? a[2 * i < PV ? 2 * i : 0] : b[2 * i < PV ? 0 : 2 * i - PV];
        float& y = 2 * i + 1 < PV ? a[2 * i + 1 < PV ? 2 * i + 1 : 0] : b[2 * i + 1 < PV ? 0 : 2 * i + 1 - PV];
        const float nx = x * c[i] - y * sn, ny = y * c[i] + x * sn;
        x = nx;
        y = ny;
        continue;
      }
    }
    const float nx = a[i] * c[i] - b[i] * sn, ny = b[i] * c[i] + a[i] * sn;
    a[i] = nx;
    b[i] = ny;
  }
}

struct Side {  // q or k, as one block sees it
  const void* x;
  const void* g;
  void* o;
  const void* w;
  int64_t xs0, xs1, xsh, gs0, gs1, gsh, os0, os1, osh;
  int heads, sub;    // sub: groups per token
  int64_t tasks;     // tokens * sub
  int blocks, blk0;  // this side's blocks
};

struct Params {
  Side side[2];
  int64_t n1;
  int d, rot;
  const float* cos;
  const float* sin;
  int64_t table;
  const int64_t* pos;
  int64_t ps0, ps1;
  float eps;
  float* part;
};

// NJ chunks per lane; G = lanes per head; RAG: lanes may share pairs (Chunk::skip)
template <typename T, typename TW, int PV, int NJ, int HB, bool INTER, bool BWD, bool WEIGHT, bool RAG>
__global__ void __launch_bounds__(kThreads, BWD ? 4 : RAG ? 3 : 4) qk_kernel(const Params P, int G) {
  const int which = blockIdx.x >= P.side[1].blk0 ? 1 : 0;
  const Side S = P.side[which];
  const int wl = threadIdx.x & 63, gpw = 64 / G, lane = wl % G, first = wl - lane;
  const int group = (threadIdx.x >> 6) * gpw + wl / G, groups = kThreads / 64 * gpw;
  const bool pow2 = (G & (G - 1)) == 0, live = wl < gpw * G;  // the wave's last 64 % G lanes have no group
  const int d = P.d, half = P.rot >> 1;
  const int chunks = INTER ? cdiv_pv<PV>(d >> 1) : cdiv_pv<PV>(half) + cdiv_pv<PV>((d - P.rot) >> 1);
  const T* X = (const T*)S.x;
  const T* GY = (const T*)S.g;
  T* O = (T*)S.o;

  int o1[NJ], o2[NJ], p0[NJ], skip[NJ];
  bool on[NJ];
  float w1[NJ][PV], w2[NJ][PV];
  float dw1[BWD && WEIGHT ? NJ : 1][PV], dw2[BWD && WEIGHT ? NJ : 1][PV];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int c = lane + G * j;
    on[j] = live && c < chunks;
    const Chunk ch = chunk_of<PV, INTER>(on[j] ? c : 0, d, P.rot);
    o1[j] = ch.o1;
    o2[j] = ch.o2;
    p0[j] = ch.p0;
    skip[j] = RAG ? ch.skip : 0;
    if constexpr (WEIGHT) {
      load<TW, PV>(w1[j], (const TW*)S.w + o1[j]);
      load<TW, PV>(w2[j], (const TW*)S.w + o2[j]);
    }
    if constexpr (BWD && WEIGHT) {
#pragma unroll
      for (int i = 0; i < PV; ++i) dw1[j][i] = dw2[j][i] = 0.f;
    }
  }

  const float inv_d = 1.f / (float)d;
  const int64_t step = (int64_t)S.blocks * groups;
  for (int64_t t0 = (int64_t)(blockIdx.x - S.blk0) * groups; t0 < S.tasks; t0 += step) {
    // whole waves stay in the loop (the group sums shuffle); lanes past the tasks redo the last and store nothing
    const bool work = live && t0 + group < S.tasks;
    const int64_t task = min(t0 + group, S.tasks - 1);
    const int64_t tok = task / S.sub;
    const int sub = (int)(task - tok * S.sub);
    const int64_t i0 = tok / P.n1, i1 = tok - i0 * P.n1;
    const int64_t pos = P.pos[i0 * P.ps0 + i1 * P.ps1];
    const bool ok = pos >= 0 && pos < P.table;
    const float* cr = P.cos + (ok ? pos : 0) * half;
    const float* sr = P.sin + (ok ? pos : 0) * half;
    const T* xt = X + i0 * S.xs0 + i1 * S.xs1;
    const T* gt = BWD ? GY + i0 * S.gs0 + i1 * S.gs1 : nullptr;
    T* ot = O + i0 * S.os0 + i1 * S.os1;

    float a[HB][NJ][PV], b[HB][NJ][PV], ga[BWD ? HB : 1][NJ][PV], gb[BWD ? HB : 1][NJ][PV];
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const int head = sub + S.sub * h;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (on[j] && work && head < S.heads) {
          load<T, PV>(a[h][j], xt + head * S.xsh + o1[j]);
          load<T, PV>(b[h][j], xt + head * S.xsh + o2[j]);
          if constexpr (BWD) {
            load<T, PV>(ga[h][j], gt + head * S.gsh + o1[j]);
            load<T, PV>(gb[h][j], gt + head * S.gsh + o2[j]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < PV; ++i) {
            a[h][j][i] = b[h][j][i] = 0.f;
            if constexpr (BWD) ga[h][j][i] = gb[h][j][i] = 0.f;
          }
        }
      }
    }
    float cs[NJ][PV], sn[NJ][PV];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (p0[j] + PV <= half) {
        load<float, PV>(cs[j], cr + p0[j]);
        load<float, PV>(sn[j], sr + p0[j]);
      } else {
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          const bool in = p0[j] + i < half;
          cs[j][i] = in ? cr[p0[j] + i] : 1.f;
          sn[j][i] = in ? sr[p0[j] + i] : 0.f;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const int head = sub + S.sub * h;
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          // interleaved: entry i of a | b is element 2p + i, pair i / 2 and PV / 2 + i / 2
          const float qa = a[h][j][i] * a[h][j][i], qb = b[h][j][i] * b[h][j][i];
          if constexpr (!RAG) ss += qa + qb;
          else if constexpr (INTER) ss += (i / 2 >= skip[j] ? qa : 0.f) + (PV / 2 + i / 2 >= skip[j] ? qb : 0.f);
          else ss += i >= skip[j] ? qa + qb : 0.f;
        }
      ss = group_sum(ss, G, pow2, first);
      float r = rsqrtf(ss * inv_d + P.eps);
      r = ok ? r : __builtin_nanf("");
      if constexpr (!BWD) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
          for (int i = 0; i < PV; ++i) {
            a[h][j][i] *= r;
            b[h][j][i] *= r;
            if constexpr (WEIGHT) {
              a[h][j][i] *= w1[j][i];
              b[h][j][i] *= w2[j][i];
            }
          }
          rotate<PV, INTER>(a[h][j], b[h][j], cs[j], sn[j], 1.f);
          if (on[j] && work && head < S.heads) {
            store<T, PV>(ot + head * S.osh + o1[j], a[h][j]);
            store<T, PV>(ot + head * S.osh + o2[j], b[h][j]);
          }
        }
      } else {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          rotate<PV, INTER>(ga[h][j], gb[h][j], cs[j], sn[j], -1.f);
#pragma unroll
          for (int i = 0; i < PV; ++i) {
            a[h][j][i] *= r;
            b[h][j][i] *= r;
            if constexpr (WEIGHT) {
              // rows past the heads and lanes past the head size hold zeros (0 * NaN only where
              // the position itself is bad)
              if (on[j] && work && head < S.heads) {
                dw1[j][i] += ga[h][j][i] * a[h][j][i];
                dw2[j][i] += gb[h][j][i] * b[h][j][i];
              }
              ga[h][j][i] *= w1[j][i];
              gb[h][j][i] *= w2[j][i];
            }
            const float qa = ga[h][j][i] * a[h][j][i], qb = gb[h][j][i] * b[h][j][i];
            if constexpr (!RAG) dot += qa + qb;
            else if constexpr (INTER) dot += (i / 2 >= skip[j] ? qa : 0.f) + (PV / 2 + i / 2 >= skip[j] ? qb : 0.f);
            else dot += i >= skip[j] ? qa + qb : 0.f;
          }
        }
        dot = group_sum(dot, G, pow2, first) * inv_d;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
          for (int i = 0; i < PV; ++i) {
            a[h][j][i] = r * (ga[h][j][i] - a[h][j][i] * dot);
            b[h][j][i] = r * (gb[h][j][i] - b[h][j][i] * dot);
          }
          if (on[j] && work && head < S.heads) {
            store<T, PV>(ot + head * S.osh + o1[j], a[h][j]);
            store<T, PV>(ot + head * S.osh + o2[j], b[h][j]);
          }
        }
      }
    }
  }

  if constexpr (BWD && WEIGHT) {
    // [groups][d] image: at most 256 / G * 2 PV NJ G floats
    extern __shared__ __attribute__((aligned(16))) float red[];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (on[j]) {
#pragma unroll
        for (int i = 0; i < PV; ++i) {
          const bool own1 = !RAG || (INTER ? i / 2 : i) >= skip[j], own2 = !RAG || (INTER ? PV / 2 + i / 2 : i) >= skip[j];
          if (own1) red[group * d + o1[j] + i] = dw1[j][i];
          if (own2) red[group * d + o2[j] + i] = dw2[j][i];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += kThreads) {
      float t = 0.f;
      for (int g = 0; g < groups; ++g) t += red[g * d + c];
      P.part[(int64_t)blockIdx.x * d + c] = t;
    }
  }
}

// dw[c] = sum over a side's blocks, fixed order; blockIdx.y = 0: q, 1: k.  16 columns x 64 row groups a
// block: a column is a chain of parts / 64 / 4 loads (a thousand parts, 16 groups: 14 us, 64: 5)
template <typename TW>
__global__ void __launch_bounds__(1024) dw_finalize(const float* __restrict__ part, int bq, int bk, int d, TW* dq, TW* dk) {
  __shared__ float red[64][17];
  const bool isk = blockIdx.y != 0;
  const float* p = part + (isk ? (int64_t)bq * d : 0);
  const int parts = isk ? bk : bq, cl = threadIdx.x & 15, grp = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < d) {
    int j = grp;
    for (; j + 192 < parts; j += 256) {
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] += p[(int64_t)(j + 64 * u) * d + c];
    }
    for (; j < parts; j += 64) a[0] += p[(int64_t)j * d + c];
  }
  red[grp][cl] = (a[0] + a[1]) + (a[2] + a[3]);
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (grp < o) red[grp][cl] += red[grp + o][cl];
    __syncthreads();
  }
  if (grp == 0 && c < d) (isk ? dk : dq)[c] = from_f<TW>(red[0][cl]);
}

struct Plan {
  int pv, g, nj, hb;
  bool rag;
  int sub[2], blocks[2];
};

// PV = 8 (16-byte vectors of 16-bit types) wherever the rotated part and the rest hold a lane's 8 pairs or
// nothing (interleaved: the head does); smaller ones take one pair per lane and step (32768 x 32 heads bf16, us
// forward and backward: head 80 with 72 rotated 549 and 1257, with 80 rotated 71 and 106).
inline Plan make_plan(const QkRopeArgs& a, int cus, bool bwd) {
  Plan p{};
  const int pairs = a.d / 2, half = a.rot / 2, rest = pairs - half;
  const bool vec = a.interleaved ? pairs >= 8 : (half == 0 || half >= 8) && (rest == 0 || rest >= 8);
  p.pv = vec ? 8 : 1;
  const int chunks = !vec ? pairs : a.interleaved ? cdiv_pv<8>(pairs) : cdiv_pv<8>(half) + cdiv_pv<8>(rest);
  p.rag = vec && (a.interleaved ? pairs % 8 != 0 : half % 8 != 0 || rest % 8 != 0);
  p.g = chunks < 64 ? chunks : 64;
  p.nj = (chunks + p.g - 1) / p.g;
  if (p.nj == 3) p.nj = 4;
  const int64_t tokens = a.n0 * a.n1;
  const int groups = kThreads / 64 * (64 / p.g);
  // one head each when there are too few to fill the chip (single-token calls: latency counts, not loads)
  const int64_t rows = tokens * (a.hq + a.hk);
  p.hb = !bwd && rows >= (int64_t)cus * groups * 4 ? kHeads : 1;
  const int heads[2] = {a.hq, a.hk};
  const int64_t cap = (int64_t)cus * 8;  // persistent: the backward's blocks each leave a partial row
  for (int i = 0; i < 2; ++i) {
    p.sub[i] = (heads[i] + p.hb - 1) / p.hb;
    const int64_t need = (tokens * p.sub[i] + groups - 1) / groups;
    int64_t share = (cap * heads[i] + a.hq + a.hk - 1) / (a.hq + a.hk);
    if (share < 1) share = 1;
    p.blocks[i] = (int)(heads[i] == 0 ? 0 : (need < share ? need : share));
  }
  return p;
}

template <typename T, typename TW, int PV, int NJ, int HB, bool INTER, bool BWD, bool WEIGHT, bool RAG>
void launch(const QkRopeArgs& a, const Plan& p, hipStream_t s) {
  Params P{};
  const int64_t tokens = a.n0 * a.n1;
  auto side = [&](int i, const QkRopeView& x, const QkRopeView& g, const QkRopeView& o, const void* w, int heads) {
    Side& d = P.side[i];
    d = Side{x.p, g.p, o.p, w, x.s0, x.s1, x.sh, g.s0, g.s1, g.sh, o.s0, o.s1, o.sh, heads, p.sub[i],
             tokens * p.sub[i], p.blocks[i], i == 0 ? 0 : p.blocks[0]};
  };
  side(0, a.q, a.gq, a.qo, a.qw, a.hq);
  side(1, a.k, a.gk, a.ko, a.kw, a.hk);
  P.n1 = a.n1;
  P.d = a.d;
  P.rot = a.rot;
  P.cos = a.cos;
  P.sin = a.sin;
  P.table = a.table;
  P.pos = a.pos;
  P.ps0 = a.ps0;
  P.ps1 = a.ps1;
  P.eps = a.eps;
  P.part = a.part;
  const size_t lds = BWD && WEIGHT ? (size_t)(kThreads / 64 * (64 / p.g)) * a.d * sizeof(float) : 0;
  hipLaunchKernelGGL((qk_kernel<T, TW, PV, NJ, HB, INTER, BWD, WEIGHT, RAG>), dim3(p.blocks[0] + p.blocks[1]),
                     dim3(kThreads), lds, s, P, p.g);
  if (BWD && WEIGHT)
    hipLaunchKernelGGL((dw_finalize<TW>), dim3((a.d + 15) / 16, 2), dim3(1024), 0, s, a.part, p.blocks[0], p.blocks[1],
                       a.d, (TW*)a.dqw, (TW*)a.dkw);
}

template <typename T, typename TW, bool BWD, bool WEIGHT>
void dispatch_shape(const QkRopeArgs& a, const Plan& p, hipStream_t s) {
  auto inter = [&](auto pv, auto nj, auto hb, auto rag) {
    constexpr int PV = decltype(pv)::value, NJ = decltype(nj)::value, HB = decltype(hb)::value;
    constexpr bool RAG = decltype(rag)::value;
    if (a.interleaved) launch<T, TW, PV, NJ, HB, true, BWD, WEIGHT, RAG>(a, p, s);
    else launch<T, TW, PV, NJ, HB, false, BWD, WEIGHT, RAG>(a, p, s);
  };
  auto hb = [&](auto pv, auto nj, auto rag) {
    if constexpr (!BWD) {
      if (p.hb > 1) return inter(pv, nj, std::integral_constant<int, kHeads>{}, rag);
    }
    inter(pv, nj, std::integral_constant<int, 1>{}, rag);
  };
  using I1 = std::integral_constant<int, 1>;
  using I8 = std::integral_constant<int, 8>;
  if (p.pv == 8 && p.rag) hb(I8{}, I1{}, std::true_type{});
  else if (p.pv == 8) hb(I8{}, I1{}, std::false_type{});
  else if (p.nj == 1) hb(I1{}, I1{}, std::false_type{});
  else if (p.nj == 2) hb(I1{}, std::integral_constant<int, 2>{}, std::false_type{});
  else hb(I1{}, std::integral_constant<int, 4>{}, std::false_type{});
}

template <bool BWD>
void run(const QkRopeArgs& a, int cus, hipStream_t s) {
  if (a.n0 <= 0 || a.n1 <= 0 || a.hq + a.hk <= 0) return;
  if (a.d < 2 || a.d > kQkRopeMaxDim || a.d % 2 || a.rot < 0 || a.rot > a.d || a.rot % 2)
    throw std::runtime_error("qk_norm_rope: head size must be even and <= 512, the rotated part even and <= it");
  const Plan p = make_plan(a, cus, BWD);
  dispatch_float(a.dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    if (a.qw == nullptr) dispatch_shape<T, float, BWD, false>(a, p, s);
    else if (a.wdtype == kF32) dispatch_shape<T, float, BWD, true>(a, p, s);
    else if (a.wdtype == a.dtype) dispatch_shape<T, T, BWD, true>(a, p, s);
    else throw std::runtime_error("qk_norm_rope: weights must be fp32 or of the inputs' dtype");
  }, "qk_norm_rope");
  check_launch("qk_norm_rope");
}

}  // namespace qkr

int64_t qk_norm_rope_part_floats(const QkRopeArgs& a, int cus) {
  const qkr::Plan p = qkr::make_plan(a, cus, true);
  return (int64_t)(p.blocks[0] + p.blocks[1]) * a.d;
}
void qk_norm_rope_fwd(const QkRopeArgs& a, int cus, hipStream_t s) { qkr::run<false>(a, cus, s); }
void qk_norm_rope_bwd(const QkRopeArgs& a, int cus, hipStream_t s) { qkr::run<true>(a, cus, s); }

}  // namespace apex_amd
