// Gated feed-forward block for gfx950: both projections, the activation and the product in one
// GEMM kernel, and the products of its backward.
//
//   forward : a = x Wg^T + bg;  u = x Wu^T + bu;  h = act(a) u                (one kernel)
//             y = h W2^T + b2
//   backward: dh = dy W2;  da = dh u act'(a);  du = dh act(a)                  (one kernel)
//             dx = [da | du] W1;  dW1 = [da | du]^T x;  dW2 = dy^T h
//
// Every product is a 256 x BN x 64 MFMA tile of four waves (one per SIMD), 128 x BN/2 each, whose
// 256 (BN = 256) fp32 accumulators live in the AGPRs.  One wave per SIMD halves the LDS fragment traffic
// of eight 128 x 64 waves; the latency that a second wave would hide is hidden in the wave instead: the
// fragments of the next 16-deep k step are read while the current step's MFMAs run, and the next but one K
// tile is on its way by LDS-DMA.  One barrier per K tile:
//
//   k step 0..2 of tile t : read step + 1's fragments, 4 x NJ MFMAs
//   k step 3              : all reads of tile t are done, tile t + 1 has landed; barrier; start the DMA of
//                           tile t + 2 into tile t's buffer, read tile t + 1's step 0, MFMAs
//
// so a DMA has four k steps (about 2000 cycles) to land.  Operand tiles come through buffer loads whose
// range ends at the matrix: rows, k steps past an edge arrive as zeros, no K multiple is needed.
//
// The gate and up columns of a tile are dealt so that a wave holds both for the same outputs (its
// first BN/4 columns are rows of Wg, its last BN/4 the same rows of Wu): act(a) u is taken on the
// accumulators, in fp32, and rounded once.
// The MFMAs compute the transposed tile (the n operand first), which leaves four consecutive n of one
// row in a lane: the epilogue parks them in LDS with 8- / 16-byte writes and every global access of it
// is a 16-byte vector of consecutive columns.
#include <type_traits>

#include "apex_amd/device.h"
#include "apex_amd/dispatch.h"
#include "apex_amd/gated_ffn_api.h"
#include "apex_amd/mfma.h"

namespace apex_amd {
namespace ffn {

using mfma::f32x16;
using mfma::s16x4;
using mfma::s16x8;

constexpr int BM = 256, BK = 64, NT = 256;
constexpr int kOut = (int)0x80000000u;  // a buffer offset past every range: the load gives zeros

struct Params {
  const uint16_t* A;
  const uint16_t* B;
  void* C;
  int64_t lda, ldb, ldc;
  int M, N, K;
  const void* bias;
  const void* aux_in;
  void* aux_out;
  float* part;  // split-K partials [splits][M][N], or null
  int kchunk;
};

__device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t r, int voff, uint16_t* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const uint16_t* p, int64_t elems) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(elems * 2), 0x00027000);
}

// XCD-aware, bijective remap of the linear workgroup id (each XCD gets a contiguous band), then
// GROUP_M-grouped tile order
__device__ __forceinline__ void tile_coords(int tiles_m, int tiles_n, int& bm, int& bn) {
  const int nwg = tiles_m * tiles_n, orig = blockIdx.x;
  const int xcd = orig % 8, q = nwg / 8, r = nwg % 8;
  const int wgid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + orig / 8;
  constexpr int GROUP_M = 8;
  const int group = wgid / (GROUP_M * tiles_n);
  const int first_m = group * GROUP_M;
  const int gm = min(tiles_m - first_m, GROUP_M);
  bm = first_m + (wgid % (GROUP_M * tiles_n)) % gm;
  bn = (wgid % (GROUP_M * tiles_n)) / gm;
}

// One operand's tile of R rows x 64 k into LDS, 1 KB per wave instruction.
// k-major: image [R][64]; 16-byte chunk c of row r at c ^ ((r >> 1) & 7).
// m-major: image [64][R]; 16-byte chunk c of k row r at c ^ ((r & 3) << 1).
// Both swizzles spread the rows that one fragment read touches over all banks.
// GATED (k-major only): image row r is column r % (R/4) of group r / (R/4) = 2 wave + (0 gate, 1 up).
template <bool KMAJ, int R, bool GATED>
__device__ __forceinline__ void issue_tile(const uint16_t* __restrict__ X, int64_t ld, int rows, int K, int r0, int k0,
                                           uint16_t* dst, int wave, int lane) {
  const int kleft = K - k0;
  if constexpr (KMAJ) {
    const int row = 8 * wave + (lane >> 3);               // + 32 i
    const int c = (lane & 7) ^ ((row >> 1) & 7);
    const int lane_off = 8 * c < kleft ? (int)((row * ld + 8 * c) * 2) : kOut;
    if constexpr (!GATED) {
      const int nr = min(rows - r0, R);
      const auto rs = rsrc(X + r0 * ld + k0, (nr - 1) * ld + kleft);
#pragma unroll
      for (int i = 0; i < R / 32; ++i) dma(rs, lane_off + (int)(32 * i * ld * 2), dst + (4 * i + wave) * 512);
    } else {
      constexpr int GH = R / 4;
      const int nr = min(rows - r0, R / 2);
      const auto rg = rsrc(X + r0 * ld + k0, (nr - 1) * ld + kleft);
      const auto ru = rsrc(X + (rows + r0) * ld + k0, (nr - 1) * ld + kleft);
#pragma unroll
      for (int i = 0; i < R / 32; ++i) {
        const int grp = 32 * i / GH, at = (grp >> 1) * GH + 32 * i % GH;
        dma(grp & 1 ? ru : rg, lane_off + (int)(at * ld * 2), dst + (4 * i + wave) * 512);
      }
    }
  } else {
    constexpr int LPR = R / 8;              // lanes per k row
    constexpr int KPI = 64 / LPR;           // k rows per wave instruction
    const int kr = KPI * wave + lane / LPR;  // + 4 KPI i
    const int c = (lane % LPR) ^ ((kr & 3) << 1);
    const int nk = min(kleft, BK);
    const auto rs = rsrc(X + k0 * ld + r0, (nk - 1) * ld + (rows - r0));
    // a last tile narrower than R: chunks past its rows would run into the next k row; they are read as
    // zeros (their outputs are not stored)
    const int lane_off = 8 * c < rows - r0 ? (int)((kr * ld + 8 * c) * 2) : kOut;
#pragma unroll
    for (int i = 0; i < BK / (4 * KPI); ++i)
      dma(rs, lane_off + (int)(4 * KPI * i * ld * 2), dst + (4 * i + wave) * 512);
  }
}

// fragment of 32 rows at k step kk (16 deep): lane l holds row rowbase + (l & 31), k = 16 kk + 8 (l >> 5) + j
template <bool KMAJ, int R>
__device__ __forceinline__ s16x8 frag(const uint16_t* tile, int rowbase, int kk, int lane) {
  if constexpr (KMAJ) {
    const int row = rowbase + (lane & 31);
    const int c = (2 * kk + (lane >> 5)) ^ ((row >> 1) & 7);
    return *reinterpret_cast<const s16x8*>(tile + row * BK + 8 * c);
  } else {
    const int g = lane >> 4, li = lane & 15, q = li >> 2, p = li & 3;
    const int kb = 16 * kk + 8 * (g >> 1);
    const int col = rowbase + 16 * (g & 1) + 4 * p;
    const int ck = col >> 3, off = col & 7;
    const int k0 = kb + q, k1 = kb + 4 + q;
    const s16x4 lo = mfma::tr_read(tile + k0 * R + ((ck ^ ((k0 & 3) << 1)) << 3) + off);
    const s16x4 hi = mfma::tr_read(tile + k1 * R + ((ck ^ ((k1 & 3) << 1)) << 3) + off);
    return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

// act(x), and its derivative in d
template <int ACT>
__device__ __forceinline__ float activate(float x, float& d) {
  if constexpr (ACT == kGateSilu) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-x));
    d = s * (1.f + x * (1.f - s));
    return x * s;
  } else {
    // tanh-GeLU as x sigmoid(2 v), v = k0 (x + k1 x^3)
    const float k0 = 0.7978845608028654f, k1 = 0.044715f;
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-2.f * k0 * (x + k1 * x * x * x)));
    d = s + 2.f * x * s * (1.f - s) * k0 * (1.f + 3.f * k1 * x * x);
    return x * s;
  }
}

template <typename T>
__device__ __forceinline__ void load4(float (&r)[4], const T* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  r[0] = to_f(T{(uint16_t)w.x});
  r[1] = to_f(T{(uint16_t)(w.x >> 16)});
  r[2] = to_f(T{(uint16_t)w.y});
  r[3] = to_f(T{(uint16_t)(w.y >> 16)});
}
template <typename T>
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) {
  return make_uint2((uint32_t)from_f<T>(v[0]).x | (uint32_t)from_f<T>(v[1]).x << 16,
                    (uint32_t)from_f<T>(v[2]).x | (uint32_t)from_f<T>(v[3]).x << 16);
}

// 16-byte stores of a [256][W] 16-bit LDS image to rows row0.., columns col0.. of C
template <typename T, int W, int PITCH>
__device__ __forceinline__ void store_image(const uint16_t* img, T* C, int64_t ldc, int row0, int col0, int M, int N,
                                            int tid) {
  constexpr int V = W / 8;
  const int ch = tid % V, gc = col0 + 8 * ch;
  if (gc >= N) return;
#pragma unroll 4
  for (int r = tid / V; r < BM; r += NT / V) {
    if (row0 + r >= M) break;
    *reinterpret_cast<uint4*>(C + (int64_t)(row0 + r) * ldc + gc) = *reinterpret_cast<const uint4*>(img + r * PITCH + 8 * ch);
  }
}

template <int BN, int OP>
constexpr size_t lds_bytes() {
  const size_t ops = (size_t)2 * (BM + BN) * BK * 2;
  const size_t epi = OP == kFfnDGated ? (size_t)128 * (BN + 4) * 4 : (size_t)BM * (BN + 8) * 2;
  return ops > epi ? ops : epi;
}

template <typename T, bool AK, bool BKM, int OP, int BN, int ACT>
__global__ void __launch_bounds__(NT, 1) ffn_gemm_kernel(const Params P) {
  constexpr int NJ = BN / 64;                    // 32-column fragments per wave
  constexpr int HN = OP == kFfnGated ? BN / 2 : BN;  // output columns per tile
  constexpr int TA = BM * BK, TB = BN * BK;
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int tiles_m = (P.M + BM - 1) / BM, tiles_n = (P.N + HN - 1) / HN;
  int bm, bn;
  tile_coords(tiles_m, tiles_n, bm, bn);
  const int row0 = bm * BM, col0 = bn * HN;
  const int kbeg = (int)blockIdx.y * P.kchunk, kend = min(P.K, kbeg + P.kchunk);
  const int nk = (kend - kbeg + BK - 1) / BK;

  auto a_buf = [&](int b) { return lds + b * (TA + TB); };
  auto b_buf = [&](int b) { return lds + b * (TA + TB) + TA; };
  auto issue = [&](int kt, int b) {
    issue_tile<AK, BM, false>(P.A, P.lda, P.M, kend, row0, kbeg + kt * BK, a_buf(b), wave, lane);
    issue_tile<BKM, BN, OP == kFfnGated>(P.B, P.ldb, P.N, kend, col0, kbeg + kt * BK, b_buf(b), wave, lane);
  };

  f32x16 acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = mfma::zero16();
  s16x8 fa[2][4], fb[2][NJ];
  auto read = [&](int b, int kk, int set) {
#pragma unroll
    for (int i = 0; i < 4; ++i) fa[set][i] = frag<AK, BM>(a_buf(b), wm * 128 + 32 * i, kk, lane);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fb[set][j] = frag<BKM, BN>(b_buf(b), wn * (BN / 2) + 32 * j, kk, lane);
  };
  auto mma = [&](int set) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = mfma::mma<T>(fb[set][j], fa[set][i], acc[i][j]);
  };

  issue(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (nk > 1) issue(1, 1);
  read(0, 0, 0);
  for (int kt = 0; kt < nk; ++kt) {
    const int cur = kt & 1;
    read(cur, 1, 1);
    mma(0);
    read(cur, 2, 0);
    mma(1);
    read(cur, 3, 1);
    mma(0);
    if (kt + 1 < nk) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (kt + 2 < nk) issue(kt + 2, cur);
      read(cur ^ 1, 0, 0);
    }
    mma(1);
  }
  __syncthreads();

  // ---- epilogue; lane: row 32 i + (lane & 31) of the wave, columns 32 j + 8 q + 4 (lane >> 5) + 0..3 ----
  const int lrow = lane & 31, lcol = 4 * (lane >> 5);
  if (OP == kFfnPlain && P.part != nullptr) {
    float* dst = P.part + (int64_t)blockIdx.y * P.M * P.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int gr = row0 + wm * 128 + 32 * i + lrow;
      if (gr >= P.M) continue;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int gc = col0 + wn * (BN / 2) + 32 * j + 8 * q + lcol;
          if (gc < P.N)
            *reinterpret_cast<float4*>(dst + (int64_t)gr * P.N + gc) =
                make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
    }
    return;
  }
  if constexpr (OP == kFfnPlain) {
    constexpr int PITCH = BN + 8;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int lc = wn * (BN / 2) + 32 * j + 8 * q + lcol;
        float bv[4] = {0.f, 0.f, 0.f, 0.f};
        if (P.bias != nullptr && col0 + lc < P.N) load4<T>(bv, (const T*)P.bias + col0 + lc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v[4] = {acc[i][j][4 * q] + bv[0], acc[i][j][4 * q + 1] + bv[1], acc[i][j][4 * q + 2] + bv[2],
                              acc[i][j][4 * q + 3] + bv[3]};
          *reinterpret_cast<uint2*>(lds + (wm * 128 + 32 * i + lrow) * PITCH + lc) = pack4<T>(v);
        }
      }
    __syncthreads();
    store_image<T, BN, PITCH>(lds, (T*)P.C, P.ldc, row0, col0, P.M, P.N, tid);
  } else if constexpr (OP == kFfnGated) {
    // add the biases; the pre-activations (rounded to the 16-bit type: what the backward recomputes the
    // activation from) leave through one image [a | u], h through a second
    constexpr int PITCH = BN + 8, HP = HN + 8, NH = NJ / 2;
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int lc = wn * (HN / 2) + 32 * j + 8 * q + lcol;
        float ba[4] = {0.f, 0.f, 0.f, 0.f}, bu[4] = {0.f, 0.f, 0.f, 0.f};
        if (P.bias != nullptr && col0 + lc < P.N) {
          load4<T>(ba, (const T*)P.bias + col0 + lc);
          load4<T>(bu, (const T*)P.bias + P.N + col0 + lc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float a[4], u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = acc[i][j][4 * q + e] + ba[e];
            u[e] = acc[i][j + NH][4 * q + e] + bu[e];
          }
          if (P.aux_out != nullptr) {
            uint16_t* at = lds + (wm * 128 + 32 * i + lrow) * PITCH + lc;
            *reinterpret_cast<uint2*>(at) = pack4<T>(a);
            *reinterpret_cast<uint2*>(at + HN) = pack4<T>(u);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float d;
            acc[i][j][4 * q + e] = activate<ACT>(a[e], d) * u[e];
          }
        }
      }
    if (P.aux_out != nullptr) {
      __syncthreads();
      store_image<T, HN, PITCH>(lds, (T*)P.aux_out, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
      store_image<T, HN, PITCH>(lds + HN, (T*)P.aux_out + P.N, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          *reinterpret_cast<uint2*>(lds + (wm * 128 + 32 * i + lrow) * HP + wn * (HN / 2) + 32 * j + 8 * q + lcol) =
              pack4<T>(v);
        }
    __syncthreads();
    store_image<T, HN, HP>(lds, (T*)P.C, P.ldc, row0, col0, P.M, P.N, tid);
  } else {
    // dh stays fp32: 128 rows at a time through LDS, then 8 consecutive columns a thread with a and u
    constexpr int CST = BN + 4, V = BN / 8, RPP = NT / V;
    float* cs = reinterpret_cast<float*>(lds);
    const int ch = tid % V, gc = col0 + 8 * ch;
    const T* au = (const T*)P.aux_in;
    T* out = (T*)P.C;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (wm == half) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(cs + (32 * i + lrow) * CST + wn * (BN / 2) + 32 * j + 8 * q + lcol) =
                  make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
      }
      __syncthreads();
      if (gc < P.N) {
#pragma unroll 4
        for (int r = tid / V; r < 128; r += RPP) {
          const int gr = row0 + 128 * half + r;
          if (gr >= P.M) break;
          const int64_t at = (int64_t)gr * P.ldc + gc;
          float a[8], u[8], g[8], da[8], du[8];
          Vec8<T>::load(a, au + at);
          Vec8<T>::load(u, au + at + P.N);
          Vec8<float>::load(g, cs + r * CST + 8 * ch);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float d;
            du[e] = g[e] * activate<ACT>(a[e], d);
            da[e] = g[e] * u[e] * d;
          }
          Vec8<T>::store(out + at, da);
          Vec8<T>::store(out + at + P.N, du);
        }
      }
      __syncthreads();
    }
  }
}

// sum of the split-K partials (fixed order) + bias
template <typename T>
__global__ void __launch_bounds__(256) ffn_reduce(const float* __restrict__ part, int splits, int64_t M, int N,
                                                  const T* __restrict__ bias, T* __restrict__ C, int64_t ldc) {
  const int64_t nvec = M * N / 8, plane = M * N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * 256) {
    const int64_t e = i * 8, r = e / N;
    const int c = (int)(e - r * N);
    float v[8], t[8];
    Vec8<float>::load(v, part + e);
    for (int s = 1; s < splits; ++s) {
      Vec8<float>::load(t, part + s * plane + e);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += t[k];
    }
    if (bias != nullptr) {
      Vec8<T>::load(t, bias + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += t[k];
    }
    Vec8<T>::store(C + r * ldc + c, v);
  }
}

struct Plan {
  int bn;      // 256 or 128
  int splits, kchunk;
};

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile width and K splits by a count of K-tile steps of the busiest CU: rounds of workgroups x their K
// tiles x the tile's width (a 128-wide tile runs at about 0.8 of the wide one's rate: its A fragments feed
// half the MFMAs), plus the partials' traffic for splits.
inline Plan make_plan(const FfnArgs& g, int cus) {
  const int hn256 = g.op == kFfnGated ? 128 : 256;
  Plan best{256, 1, g.k};
  double cost = 1e300;
  for (int bn = 256; bn >= 128; bn /= 2) {
    const int64_t tiles = cdiv(g.m, BM) * cdiv(g.n, hn256 * bn / 256);
    for (int sp = 1; sp <= 16; ++sp) {
      if (sp > 1 && (g.op != kFfnPlain || tiles * sp > 2 * cus || g.k < sp * 512)) break;
      const int chunk = (int)(cdiv(cdiv(g.k, sp), BK) * BK);
      const int real = (int)cdiv(g.k, chunk);
      if (real != sp) continue;
      const double steps = (double)cdiv(tiles * sp, cus) * (chunk / BK + 6.0) * (bn == 256 ? 1.0 : 0.62);
      // a K-tile step of the wide tile is about 0.9 us; partials move 8 bytes an output and split at 4 TB/s
      const double extra = sp > 1 ? (double)g.m * g.n * sp * 8 / 4e6 / 0.9 + 5.0 : 0.0;
      if (steps + extra < cost) {
        cost = steps + extra;
        best = Plan{bn, sp, chunk};
      }
    }
  }
  return best;
}

template <typename T, bool AK, bool BKM, int OP, int BN, int ACT>
void launch(const FfnArgs& g, const Plan& p, int cus, hipStream_t s) {
  constexpr int HN = OP == kFfnGated ? BN / 2 : BN;
  Params P{(const uint16_t*)g.a, (const uint16_t*)g.b, g.c, g.lda, g.ldb, g.ldc, g.m, g.n, g.k, g.bias, g.aux_in,
           g.aux_out, p.splits > 1 ? g.ws : nullptr, p.kchunk};
  const unsigned tiles = (unsigned)(cdiv(g.m, BM) * cdiv(g.n, HN));
  hipLaunchKernelGGL((ffn_gemm_kernel<T, AK, BKM, OP, BN, ACT>), dim3(tiles, p.splits), dim3(NT),
                     (lds_bytes<BN, OP>()), s, P);
  if (p.splits > 1) {
    int64_t grid = cdiv((int64_t)g.m * g.n / 8, 256);
    if (grid > (int64_t)cus * 8) grid = (int64_t)cus * 8;
    hipLaunchKernelGGL((ffn_reduce<T>), dim3((unsigned)grid), dim3(256), 0, s, (const float*)g.ws, p.splits,
                       (int64_t)g.m, g.n, (const T*)g.bias, (T*)g.c, g.ldc);
  }
}

template <typename T, bool AK, bool BKM, int OP, int ACT>
void launch_bn(const FfnArgs& g, const Plan& p, int cus, hipStream_t s) {
  if (p.bn == 256) launch<T, AK, BKM, OP, 256, ACT>(g, p, cus, s);
  else launch<T, AK, BKM, OP, 128, ACT>(g, p, cus, s);
}

}  // namespace ffn

bool ffn_supported(const FfnArgs& g) {
  if (g.dtype != kF16 && g.dtype != kBF16) return false;
  if (g.m <= 0 || g.n <= 0 || g.k <= 0) return false;
  auto al = [](const void* p) { return ((uintptr_t)p & 15u) == 0; };
  if (!al(g.a) || !al(g.b) || !al(g.c) || !al(g.bias) || !al(g.aux_in) || !al(g.aux_out)) return false;
  if (g.n % 8 || g.lda % 8 || g.ldb % 8 || g.ldc % 8) return false;
  if ((g.a_kmajor || g.b_kmajor) && g.k % 8) return false;
  if (!g.a_kmajor && g.m % 8) return false;
  // a tile's buffer range (256 rows or 64 k rows) stays below 2 GiB
  if (g.lda >= (1 << 21) || g.ldb >= (1 << 21)) return false;
  if (ffn::cdiv(g.m, ffn::BM) * ffn::cdiv(g.n, 64) >= (1 << 24)) return false;
  switch (g.op) {
    case kFfnPlain: return !(!g.a_kmajor && g.b_kmajor);
    case kFfnGated: return g.a_kmajor && g.b_kmajor;
    case kFfnDGated: return g.a_kmajor && !g.b_kmajor && g.aux_in != nullptr && g.ldc == 2 * (int64_t)g.n;
    default: return false;
  }
}

int64_t ffn_workspace_floats(const FfnArgs& g, int cus) {
  const ffn::Plan p = ffn::make_plan(g, cus);
  return p.splits > 1 ? (int64_t)p.splits * g.m * g.n : 0;
}

void ffn_gemm(const FfnArgs& g, int cus, hipStream_t s) {
  if (!ffn_supported(g)) throw std::runtime_error("gated_ffn: unsupported shape, alignment or dtype");
  const ffn::Plan p = ffn::make_plan(g, cus);
  if (p.splits > 1 && g.ws == nullptr) throw std::runtime_error("gated_ffn: workspace missing");
  dispatch_16(g.dtype, [&](auto tag) {
    using T = typename decltype(tag)::type;
    if (g.op == kFfnGated) {
      if (g.act == kGateSilu) ffn::launch_bn<T, true, true, kFfnGated, kGateSilu>(g, p, cus, s);
      else ffn::launch_bn<T, true, true, kFfnGated, kGateGelu>(g, p, cus, s);
    } else if (g.op == kFfnDGated) {
      if (g.act == kGateSilu) ffn::launch_bn<T, true, false, kFfnDGated, kGateSilu>(g, p, cus, s);
      else ffn::launch_bn<T, true, false, kFfnDGated, kGateGelu>(g, p, cus, s);
    } else if (g.a_kmajor && g.b_kmajor) ffn::launch_bn<T, true, true, kFfnPlain, 0>(g, p, cus, s);
    else if (g.a_kmajor) ffn::launch_bn<T, true, false, kFfnPlain, 0>(g, p, cus, s);
    else ffn::launch_bn<T, false, false, kFfnPlain, 0>(g, p, cus, s);
  }, "gated_ffn");
  check_launch("gated_ffn");
}

}  // namespace apex_amd
