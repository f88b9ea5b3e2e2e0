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
//   k step 3              : all reads of tile t are done, tile t + 1 has landed; barrier; tile t's LDS goes
//                           to the DMA of later tiles (Ring), read tile t + 1's step 0, MFMAs
//
// Operand tiles come through buffer loads whose range ends at the matrix: rows and k steps past an edge
// arrive as zeros, no K multiple is needed.
//
// The gate and up columns of a tile are dealt so that a wave holds both for the same outputs (its
// first BN/4 columns are rows of Wg, its last BN/4 the same rows of Wu): act(a) u is taken on the
// accumulators, in fp32, and rounded once.
// Measured (bf16, us of kernel): 8192 x 4096 -> 11008: gated 1226-1310 (1.13-1.2 PFLOP/s, and 0.7 GB written);
// [da | du] 717-760; the plain products 541-660 (NT, NN, TN; 1.13-1.36 PFLOP/s, at the card's power limit:
// 1.3-1.7 GHz).  The 128 x 64 eight-wave tiles of gemm_mfma.hip take 1296, 855 and 617-871 there.
//
// The MFMAs compute the transposed tile (the n operand first), which leaves four consecutive n of one
// row in a lane: the epilogue parks them in LDS with 8- / 16-byte writes and every global access of it
// is a 16-byte vector of consecutive columns.
#include <type_traits>

#include "apex_amd/device.h"
#include "apex_amd/dispatch.h"
#include "apex_amd/gated_ffn_api.h"
#include "apex_amd/mfma.h"
#include "apex_amd/tile_order.h"

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
  uint16_t* au_hi;  // [M][2N] pre-activations a | u (gated: written unless null; dgated: read)
  uint8_t* au_lo;
  float* part;  // split-K partials [splits][M][N], or null
  int kchunk;
};

// LDS-DMA of 16 bytes a lane to dst + 16 lane.  Written in assembly: behind the builtin the compiler makes
// every transposing LDS read wait for all DMA in flight (it cannot tell their LDS ranges apart), and the
// tile that should land during the next four k steps would be waited out in the first.  The waits are
// the caller's: an s_waitcnt vmcnt before the barrier that opens a tile, counted so that only younger tiles'
// DMA stays in flight.  No register is written, and the compiler's own counts only become stricter.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void dma(i32x4 r, int voff, uint32_t dst) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass does not know the constraints
  // m0 is reserved: the compiler sets it right before an instruction that needs it, and this kernel has none
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(voff), "s"(r));
#endif
}

// raw buffer over `elems` 16-bit elements: loads past them give zeros
__device__ __forceinline__ i32x4 rsrc(const uint16_t* p, int64_t elems) {
  const uint64_t b = (uint64_t)p;
  return i32x4{(int)(uint32_t)b, (int)((uint32_t)(b >> 32) & 0xffffu), (int)(elems * 2), 0x00027000};
}

__device__ __forceinline__ uint32_t lds_addr(const uint16_t* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint16_t*)p;
}

// One operand's tile of R rows x 64 k on its way into LDS, R / 32 instructions of 1 KB a wave.
// k-major: image [R][64]; 16-byte chunk c of row r at c ^ ((r >> 1) & 7).
// m-major: image [64][R]; 16-byte chunk c of k row r at c ^ ((r & 3) << 1).
// Both swizzles spread the rows that one fragment read touches over all banks.
// GATED (k-major only): image row r is column r % (R/4) of group r / (R/4) = 2 wave + (0 gate, 1 up).
template <bool KMAJ, int R, bool GATED>
struct TileDma {
  i32x4 r0, r1;    // r1: the up rows
  int off, step;   // the lane's byte offset in instruction 0, bytes between instructions
  uint32_t dst;

  // the tile at row0, k0 of X; k0 >= K: an empty range, all zeros
  __device__ __forceinline__ void at(const uint16_t* __restrict__ X, int64_t ld, int rows, int K, int row0, int k0,
                                     uint32_t lds, int wave, int lane) {
    const int kleft = max(K - k0, 0);
    dst = lds + wave * 1024;
    if constexpr (KMAJ) {
      const int row = 8 * wave + (lane >> 3);  // + 32 i
      const int c = (lane & 7) ^ ((row >> 1) & 7);
      const int nr = min(rows - row0, GATED ? R / 2 : R);
      const int64_t range = kleft > 0 ? (nr - 1) * ld + kleft : 0;
      off = 8 * c < kleft ? (int)((row * ld + 8 * c) * 2) : kOut;
      r0 = rsrc(X + row0 * ld + k0, range);
      if constexpr (GATED) r1 = rsrc(X + (rows + row0) * ld + k0, range);
      step = (int)(64 * ld);
    } else {
      constexpr int LPR = R / 8, KPI = 64 / LPR;  // lanes per k row, k rows per instruction
      const int kr = KPI * wave + lane / LPR;      // + 4 KPI i
      const int c = (lane % LPR) ^ ((kr & 3) << 1);
      // chunks past the last row would run into the next k row; their outputs are not stored
      off = 8 * c < rows - row0 ? (int)((kr * ld + 8 * c) * 2) : kOut;
      r0 = rsrc(X + k0 * ld + row0, kleft > 0 ? (min(kleft, BK) - 1) * ld + (rows - row0) : 0);
      step = (int)(8 * KPI * ld);
    }
  }
  __device__ __forceinline__ void issue(int i) const {
    if constexpr (GATED) {
      constexpr int GH = R / 4;
      const int grp = 32 * i / GH, row = (grp >> 1) * GH + 32 * i % GH;
      dma(grp & 1 ? r1 : r0, off + row / 32 * step, dst + i * 4096);
    } else {
      dma(r0, off + i * step, dst + i * 4096);
    }
  }
};

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

// act(x) = x s, and its derivative in d; s = 1 / (1 + e^-y) with y = x for SiLU and 2 k0 (x + k1 x^3) for the
// tanh form of GeLU.  The epilogues' instructions count, since the matrix units are idle meanwhile: e^-y
// is one exp2 (of z) with log2(e) in y's constants, and d = s + x s (1 - s) y'.  x^2 stops at 1e4: s is 0 or 1
// long before, and an infinite y' would make 0 y' NaN.
template <int ACT>
__device__ __forceinline__ float activate(float x, float& d) {
  constexpr float kLog2e = 1.4426950408889634f, k0 = 0.7978845608028654f, k1 = 0.044715f;
  const float x2 = fminf(x * x, 1e4f);
  const float z = ACT == kGateSilu ? -kLog2e * x : x * fmaf(-2.f * k0 * k1 * kLog2e, x2, -2.f * k0 * kLog2e);
  const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z));
  const float p = x * s, q = p * (1.f - s);
  d = ACT == kGateSilu ? s + q : fmaf(q, fmaf(6.f * k0 * k1, x2, 2.f * k0), s);
  return p;
}

template <typename T>
__device__ __forceinline__ void load4(float (&r)[4], const T* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  r[0] = to_f(T{(uint16_t)w.x});
  r[1] = to_f(T{(uint16_t)(w.x >> 16)});
  r[2] = to_f(T{(uint16_t)w.y});
  r[3] = to_f(T{(uint16_t)(w.y >> 16)});
}
// rounded to nearest even, two at a time (one by one the compiler adds a shift and an or to each pair)
template <typename T>
__device__ __forceinline__ uint2 pack4(const float (&v)[4]) {
  using E = std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, _Float16>;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef E e16x2 __attribute__((ext_vector_type(2)));
  return make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), e16x2)),
                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), e16x2)));
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  const uint2 lo = pack4<T>({v[0], v[1], v[2], v[3]}), hi = pack4<T>({v[4], v[5], v[6], v[7]});
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// Pre-activations are kept for the backward as the upper 24 bits of their fp32 value (15 bits of
// mantissa) in a 16- and an 8-bit plane: rounded to bf16 / fp16 they would put two more roundings of the type
// into dx and dW1 (0.0030 instead of 0.0024 of their norm for bf16, where the result's own rounding is
// 0.0017), for 1 % of the time and 6 bytes a gate / up pair instead of 4.  The low bits are cut off, an error of
// one sign of up to 2^-15 of a value: a NaN stays one, nothing overflows.
__device__ __forceinline__ uint2 hi4(const float (&v)[4]) {
  return make_uint2(__builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302u),
                    __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302u));
}
__device__ __forceinline__ uint32_t lo4(const float (&v)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0501u);
  const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x0c0c0501u);
  return a | b << 16;
}
__device__ __forceinline__ void join8(float (&v)[8], uint4 hi, uint2 lo) {
  const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[2] = {lo.x, lo.y};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t h16 = e & 1 ? h[e >> 1] & 0xffff0000u : h[e >> 1] << 16;
    v[e] = __uint_as_float(h16 | ((l[e >> 2] >> (8 * (e & 3))) & 0xffu) << 8);
  }
}

// 8-byte stores of a [256][W] 8-bit LDS image
template <int W, int PITCH>
__device__ __forceinline__ void store_bytes(const uint8_t* img, uint8_t* C, int64_t ldc, int row0, int col0, int M, int N,
                                            int tid) {
  constexpr int V = W / 8;
  const int ch = tid % V, gc = col0 + 8 * ch;
  if (gc >= N) return;
#pragma unroll 4
  for (int r = tid / V; r < BM; r += NT / V) {
    if (row0 + r >= M) break;
    *reinterpret_cast<uint2*>(C + (int64_t)(row0 + r) * ldc + gc) = *reinterpret_cast<const uint2*>(img + r * PITCH + 8 * ch);
  }
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

// The LDS ring of operand tiles (byte offsets).
// BN = 256: five 32-KB slots, A and B tiles in turn (A(t) in slot 2t mod 5, B(t) in 2t + 1 mod 5).  When tile
// t has been read, B(t + 2) goes into A(t)'s slot and A(t + 3) into B(t)'s: B has three k steps to land,
// A seven.  Two buffers of both, the DMA of a whole tile in its predecessor's last step, left the
// MFMAs waiting 45 % of the time.
// BN = 128: three slots of A and B; tile t + 3 replaces tile t.
// kFirst of a round's instructions (B's, then A's) go out in the step after the barrier, the others in the
// next two steps.  kInFlight: instructions younger than tile t + 1's at the barrier that opens it.
template <int BN> struct Ring;
template <> struct Ring<256> {
  static constexpr int kSlot = 32768, kBytes = 5 * kSlot;
  static constexpr int kFirst = 8, kAheadB = 2, kInFlight = 8, kAfterPrologue = 16;
  static __device__ constexpr int first_a() { return 0; }
  static __device__ constexpr int first_b() { return kSlot; }
  static __device__ __forceinline__ int next_b_slot(int sa, int) { return sa; }
  static __device__ __forceinline__ int next_a_slot(int, int sb) { return sb; }
  static __device__ __forceinline__ void advance(int& sa, int& sb) {
    sa = sa + 2 * kSlot >= kBytes ? sa + 2 * kSlot - kBytes : sa + 2 * kSlot;
    sb = sa + kSlot >= kBytes ? sa + kSlot - kBytes : sa + kSlot;
  }
  // A0 B0 A1, and B1 of the round (B1, A2)
  template <int DA, int DB, typename AA, typename AB, typename IA, typename IB>
  static __device__ __forceinline__ void prologue(AA aim_a, AB aim_b, IA issue_a, IB issue_b) {
    aim_a(0, 0);
    for (int i = 0; i < DA; ++i) issue_a(i);
    aim_b(0, kSlot);
    for (int i = 0; i < DB; ++i) issue_b(i);
    aim_a(1, 2 * kSlot);
    for (int i = 0; i < DA; ++i) issue_a(i);
    aim_b(1, 3 * kSlot);
    for (int i = 0; i < DB; ++i) issue_b(i);
    aim_a(2, 4 * kSlot);
  }
};
template <> struct Ring<128> {
  static constexpr int kA = 32768, kSlot = 49152, kBytes = 3 * kSlot;
  static constexpr int kFirst = 4, kAheadB = 3, kInFlight = 12, kAfterPrologue = 16;
  static __device__ constexpr int first_a() { return 0; }
  static __device__ constexpr int first_b() { return kA; }
  static __device__ __forceinline__ int next_b_slot(int, int sb) { return sb; }
  static __device__ __forceinline__ int next_a_slot(int sa, int) { return sa; }
  static __device__ __forceinline__ void advance(int& sa, int& sb) {
    sa = sa + kSlot >= kBytes ? 0 : sa + kSlot;
    sb = sa + kA;
  }
  // tiles 0 and 1, and B2 of the round (B2, A2)
  template <int DA, int DB, typename AA, typename AB, typename IA, typename IB>
  static __device__ __forceinline__ void prologue(AA aim_a, AB aim_b, IA issue_a, IB issue_b) {
    for (int t = 0; t < 2; ++t) {
      aim_b(t, t * kSlot + kA);
      for (int i = 0; i < DB; ++i) issue_b(i);
      aim_a(t, t * kSlot);
      for (int i = 0; i < DA; ++i) issue_a(i);
    }
    aim_b(2, 2 * kSlot + kA);
    for (int i = 0; i < DB; ++i) issue_b(i);
    aim_a(2, 2 * kSlot);
  }
};

template <int BN, int OP>
constexpr size_t lds_bytes() {
  const size_t ops = Ring<BN>::kBytes;
  // gated: h beside the lower plane, or the upper plane alone
  const size_t epi = OP == kFfnDGated ? (size_t)128 * (BN + 4) * 4
                     : OP == kFfnGated ? (size_t)BM * (BN / 2 + 8) * 2 + (size_t)BM * (BN + 8)
                                       : (size_t)BM * (BN + 8) * 2;
  static_assert(Ring<256>::kBytes >= 256 * 264 * 2, "the upper plane's image");
  return ops > epi ? ops : epi;
}

template <typename T, bool AK, bool BKM, int OP, int BN, int ACT>
__global__ void __launch_bounds__(NT, 1) ffn_gemm_kernel(const Params P) {
  constexpr int NJ = BN / 64;                    // 32-column fragments per wave
  constexpr int HN = OP == kFfnGated ? BN / 2 : BN;  // output columns per tile
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int tiles_m = (P.M + BM - 1) / BM, tiles_n = (P.N + HN - 1) / HN;
  int bm, bn;
  tile_coords(tiles_m * tiles_n, tiles_m, tiles_n, bm, bn);
  // in scalar registers for certain (the divisions above run on the vector unit): the DMA's ranges need it
  const int row0 = __builtin_amdgcn_readfirstlane(bm * BM), col0 = __builtin_amdgcn_readfirstlane(bn * HN);
  const int kbeg = (int)blockIdx.y * P.kchunk, kend = min(P.K, kbeg + P.kchunk);
  const int nk = (kend - kbeg + BK - 1) / BK;

  using R = Ring<BN>;
  constexpr int DA = BM / 32, DB = BN / 32;  // DMA instructions of an A and a B tile
  const uint32_t lds0 = lds_addr(lds);
  TileDma<AK, BM, false> ta;
  TileDma<BKM, BN, OP == kFfnGated> tb;
  auto aim_a = [&](int kt, int slot) {
    ta.at(P.A, P.lda, P.M, kend, row0, kbeg + kt * BK, lds0 + slot, wave, lane);
  };
  auto aim_b = [&](int kt, int slot) {
    tb.at(P.B, P.ldb, P.N, kend, col0, kbeg + kt * BK, lds0 + slot, wave, lane);
  };
  // DMA of one round: B's instructions, then A's
  auto issue = [&](int i) {
    if (i < DB) tb.issue(i);
    else ta.issue(i - DB);
  };

  f32x16 acc[4][NJ];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = mfma::zero16();
  s16x8 fa[2][4], fb[2][NJ];
  constexpr int FRAGS = 4 + NJ, MFMAS = 4 * NJ;
  const uint16_t *at, *bt;  // the tile that is read
  auto read = [&](int f, int kk, int set) {  // fragment f of a step: B's, then A's
    if (f < NJ) fb[set][f] = frag<BKM, BN>(bt, wn * (BN / 2) + 32 * f, kk, lane);
    else fa[set][f - NJ] = frag<AK, BM>(at, wm * 128 + 32 * (f - NJ), kk, lane);
  };
  // One k step: MFMA by MFMA, each with its share of the reads of the next step's fragments (in the first
  // half of the step) and of DMA instructions D0 .. D1 - 1 (evenly: more at once than the CU's address
  // unit takes, 16 cycles each, would hold up the MFMAs behind them).  The order is pinned, since the
  // compiler sinks the reads to just before their MFMAs and the wave then waits out every one of them.
  auto step = [&](int set, int kk, auto d0, auto d1) {
    constexpr int H = MFMAS / 2, D0 = decltype(d0)::value, D1 = decltype(d1)::value;
#pragma unroll
    for (int m = 0; m < MFMAS; ++m) {
      acc[m / NJ][m % NJ] = mfma::mma<T>(fb[set][m % NJ], fa[set][m / NJ], acc[m / NJ][m % NJ]);
#pragma unroll
      for (int f = 0; f < FRAGS; ++f)
        if (f * H / FRAGS == m) read(f, kk, set ^ 1);
#pragma unroll
      for (int i = D0; i < D1; ++i)
        if ((i - D0) * MFMAS / (D1 - D0) == m) issue(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  using Zero = std::integral_constant<int, 0>;
  using First = std::integral_constant<int, R::kFirst>;
  using Half = std::integral_constant<int, (R::kFirst + DA + DB) / 2>;
  using All = std::integral_constant<int, DA + DB>;

  // Before tile 0: the tiles and the first part of the round that tile -1's last step would have issued
  int sa = R::first_a(), sb = R::first_b();  // slots of the current tile
  R::template prologue<DA, DB>(aim_a, aim_b, [&](int i) { ta.issue(i); }, [&](int i) { tb.issue(i); });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(R::kAfterPrologue) : "memory");
  __syncthreads();
  at = lds + sa / 2;
  bt = lds + sb / 2;
#pragma unroll
  for (int f = 0; f < FRAGS; ++f) read(f, 0, 0);
  __builtin_amdgcn_sched_barrier(0);
  // the DMA of tiles past the last one (empty range: zeros) and the last tile's read-ahead run like the
  // others: no branch splits the schedule
  for (int kt = 0; kt < nk; ++kt) {
    step(0, 1, First{}, Half{});
    step(1, 2, Half{}, All{});
    step(0, 3, Zero{}, Zero{});
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(R::kInFlight) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    aim_b(kt + R::kAheadB, R::next_b_slot(sa, sb));
    aim_a(kt + 3, R::next_a_slot(sa, sb));
    R::advance(sa, sb);
    at = lds + sa / 2;
    bt = lds + sb / 2;
    step(1, 0, Zero{}, First{});
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
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
    // biases; then the upper plane of the pre-activations leaves through one image [a | u], and their
    // lower plane with h through a second
    constexpr int PITCH = BN + 8, HP = HN + 8, NH = NJ / 2;
    uint8_t* low = reinterpret_cast<uint8_t*>(lds + BM * HP);
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
            a[e] = acc[i][j][4 * q + e] += ba[e];
            u[e] = acc[i][j + NH][4 * q + e] += bu[e];
          }
          if (P.au_hi != nullptr) {
            uint16_t* at = lds + (wm * 128 + 32 * i + lrow) * PITCH + lc;
            *reinterpret_cast<uint2*>(at) = hi4(a);
            *reinterpret_cast<uint2*>(at + HN) = hi4(u);
          }
        }
      }
    if (P.au_hi != nullptr) {
      __syncthreads();
      store_image<bf16_t, HN, PITCH>(lds, (bf16_t*)P.au_hi, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
      store_image<bf16_t, HN, PITCH>(lds + HN, (bf16_t*)P.au_hi + P.N, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = wm * 128 + 32 * i + lrow, lc = wn * (HN / 2) + 32 * j + 8 * q + lcol;
          float a[4], u[4], h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float d;
            a[e] = acc[i][j][4 * q + e];
            u[e] = acc[i][j + NH][4 * q + e];
            h[e] = activate<ACT>(a[e], d) * u[e];
          }
          if (P.au_hi != nullptr) {
            *reinterpret_cast<uint32_t*>(low + r * PITCH + lc) = lo4(a);
            *reinterpret_cast<uint32_t*>(low + r * PITCH + HN + lc) = lo4(u);
          }
          *reinterpret_cast<uint2*>(lds + r * HP + lc) = pack4<T>(h);
        }
    __syncthreads();
    store_image<T, HN, HP>(lds, (T*)P.C, P.ldc, row0, col0, P.M, P.N, tid);
    if (P.au_hi != nullptr) {
      store_bytes<HN, PITCH>(low, P.au_lo, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
      store_bytes<HN, PITCH>(low + HN, P.au_lo + P.N, 2 * (int64_t)P.N, row0, col0, P.M, P.N, tid);
    }
  } else {
    // dh stays fp32: 128 rows at a time through LDS, then 8 consecutive columns a thread with a and u.  These
    // are fetched AH rows ahead, the first of them before the staging (row by row, four at a time, their
    // latency was a third of the kernel at 1024-deep products).
    constexpr int CST = BN + 4, V = BN / 8, RPP = NT / V, IT = 128 / RPP, AH = 8;
    static_assert(IT % AH == 0, "the fetch ring's slots follow the row index");
    float* cs = reinterpret_cast<float*>(lds);
    const int ch = tid % V, gc = col0 + 8 * ch;
    const int64_t gcc = min(gc, P.N - 8);  // clamped: loads past the edges are not used
    T* out = (T*)P.C;
    uint4 pa[AH], pu[AH];
    uint2 la[AH], lu[AH];
    auto fetch = [&](int n) {  // row n of the thread's 2 IT
      const int64_t at = (int64_t)min(row0 + tid / V + RPP * n, P.M - 1) * P.ldc + gcc;
      pa[n % AH] = *reinterpret_cast<const uint4*>(P.au_hi + at);
      pu[n % AH] = *reinterpret_cast<const uint4*>(P.au_hi + at + P.N);
      la[n % AH] = *reinterpret_cast<const uint2*>(P.au_lo + at);
      lu[n % AH] = *reinterpret_cast<const uint2*>(P.au_lo + at + P.N);
    };
#pragma unroll
    for (int n = 0; n < AH; ++n) fetch(n);
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
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int r = tid / V + RPP * it, gr = row0 + 128 * half + r, n = half * IT + it;
        float a[8], u[8], g[8], da[8], du[8];
        join8(a, pa[n % AH], la[n % AH]);
        join8(u, pu[n % AH], lu[n % AH]);
        if (n + AH < 2 * IT) fetch(n + AH);
        Vec8<float>::load(g, cs + r * CST + 8 * ch);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float d;
          du[e] = g[e] * activate<ACT>(a[e], d);
          da[e] = g[e] * u[e] * d;
        }
        if (gr < P.M && gc < P.N) {
          T* o = out + (int64_t)gr * P.ldc + gc;
          *reinterpret_cast<uint4*>(o) = pack8<T>(da);
          *reinterpret_cast<uint4*>(o + P.N) = pack8<T>(du);
        }
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows (a token each of up to 32 sequences): the weights are read once and nothing else counts.
// A workgroup owns 16 outputs (16 rows of Wg and of Wu, or of W2) and its NW waves split K; the weights
// go straight from memory to the MFMA operand (16 rows x 32 k a load), U steps in flight per wave.  x goes
// through LDS by DMA, whole 64 U byte runs of a row at a time: read like the weights, 64 bytes of 16 rows a
// load, it kept the address unit as busy as they do (24 tokens at 2048 -> 5504 -> 2048: 32 us of kernels
// instead of 24, now 22).  The waves' partial tiles
// meet in LDS in a fixed order, where the block's epilogue (bias, activation, product) runs in fp32.
// One token at 4096 -> 11008 -> 4096: 32-33 + 16 us, 5.5-5.7 TB/s of weights (a plain read runs at 5.8).
// ---------------------------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ f32x4 mma16(i32x4 a, i32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma16<bf16_t>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mfma::bf16x8, a),
                                                 __builtin_bit_cast(mfma::bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<f16_t>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mfma::f16x8, a), __builtin_bit_cast(mfma::f16x8, b),
                                                c, 0, 0, 0);
}

constexpr int kFewRows = 32;

// floats of LDS: the waves' x tiles, then their partial tiles [NW][16 TM][16 or 32 outputs + 4]
template <bool GATED, int TM, int NW>
constexpr int few_lds() {
  return NW * (TM * 16 * (16 * (GATED ? 2 : 1) + 4) > 1024 ? TM * 16 * (16 * (GATED ? 2 : 1) + 4) : 1024);
}

template <typename T, bool GATED, int ACT, int TM, int NW>
__global__ void __launch_bounds__(NW * 64) ffn_few_kernel(const Params P) {
  constexpr int G = GATED ? 2 : 1, U = 4 / TM;  // 4 KB of x a wave and group of U steps
  constexpr int LPR = 4 * U, RPI = 64 / LPR;    // lanes (16-byte chunks) a row of x, rows a DMA instruction
  constexpr int TP = 16 * G + 4;  // floats a token takes in a wave's partial tile
  extern __shared__ __attribute__((aligned(16))) float part[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col0 = blockIdx.x * 16, l16 = lane & 15, g8 = 8 * (lane >> 4);
  const int chunk = ((P.K + NW - 1) / NW + 31) / 32 * 32;
  const int k1 = min(P.K, (wave + 1) * chunk);
  int k = wave * chunk;

  // buffer ranges end at the last row and K's end: loads past them give zeros
  const int rows = min(16, P.N - col0);
  __amdgpu_buffer_rsrc_t rw[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    rw[g] = __builtin_amdgcn_make_buffer_rsrc((void*)(P.B + ((int64_t)g * P.N + col0) * P.ldb), 0,
                                              (int)(((rows - 1) * P.ldb + P.K) * 2), 0x00027000);
  const int ow = (int)((l16 * P.ldb + g8) * 2);
  // x tile image [16 TM][32 U]: chunk c of row r at c ^ swz(r), so that a fragment's 16 rows hit all banks
  const auto swz = [](int r) { return U == 4 ? r & 15 : (r >> 1) & 7; };
  const i32x4 rx = rsrc(P.A, (P.M - 1) * P.lda + P.K);
  const uint16_t* xt = reinterpret_cast<const uint16_t*>(part) + wave * 2048;
  const uint32_t xdst = lds_addr(xt);
  const int xr = lane / LPR;
  f32x4 acc[G][TM];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int t = 0; t < TM; ++t) acc[g][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  // U steps of loads, all in flight, then their MFMAs; the last group's loads past the wave's chunk are zeros
  auto group = [&](auto last) {
    i32x4 wv[U][G];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = RPI * i + xr, kc = k + 8 * ((lane % LPR) ^ swz(r));
      dma(rx, !decltype(last)::value || kc < k1 ? (int)((r * P.lda + kc) * 2) : kOut, xdst + 1024 * i);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = !decltype(last)::value || k + 32 * u + g8 < k1;
#pragma unroll
      for (int g = 0; g < G; ++g)
        wv[u][g] = __builtin_bit_cast(
            i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw[g], in ? ow + 2 * (k + 32 * u) : kOut, 0, 0));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        const int r = 16 * t + l16, c = 4 * u + (lane >> 4);
        const i32x4 xv = *reinterpret_cast<const i32x4*>(xt + r * 32 * U + 8 * (c ^ swz(r)));
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g][t] = mma16<T>(wv[u][g], xv, acc[g][t]);
      }
    // the next group's DMA overwrites the tile
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  for (; k + 32 * U <= k1; k += 32 * U) group(std::false_type{});
  if (k < k1) group(std::true_type{});
  __syncthreads();
  // lane: token 16 t + (lane & 15), outputs 4 (lane >> 4) + 0..3
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int g = 0; g < G; ++g)
      *reinterpret_cast<f32x4*>(part + ((wave * TM + t) * 16 + l16) * TP + 16 * g + 4 * (lane >> 4)) = acc[g][t];
  __syncthreads();
  for (int i = tid; i < P.M * 16; i += NW * 64) {
    const int tok = i >> 4, c = i & 15, gc = col0 + c;
    if (gc >= P.N) continue;
    float v[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < NW; ++q) s += part[(q * TM * 16 + tok) * TP + 16 * g + c];
      v[g] = s + (P.bias != nullptr ? to_f(((const T*)P.bias)[(int64_t)g * P.N + gc]) : 0.f);
    }
    if constexpr (GATED) {
      if (P.au_hi != nullptr) {
        const int64_t at = (int64_t)tok * 2 * P.N + gc;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          P.au_hi[at + g * P.N] = (uint16_t)(__float_as_uint(v[g]) >> 16);
          P.au_lo[at + g * P.N] = (uint8_t)(__float_as_uint(v[g]) >> 8);
        }
      }
      float d;
      v[0] = activate<ACT>(v[0], d) * v[1];
    }
    ((T*)P.C)[(int64_t)tok * P.ldc + gc] = from_f<T>(v[0]);
  }
}

template <typename T, bool GATED, int ACT, int TM, int NW>
void launch_few(const FfnArgs& g, hipStream_t s) {
  Params P{(const uint16_t*)g.a, (const uint16_t*)g.b, g.c, g.lda, g.ldb, g.ldc, g.m, g.n, g.k, g.bias, g.au_hi,
           g.au_lo, nullptr, g.k};
  const size_t lds = (size_t)few_lds<GATED, TM, NW>() * sizeof(float);
  hipLaunchKernelGGL((ffn_few_kernel<T, GATED, ACT, TM, NW>), dim3((unsigned)((g.n + 15) / 16)), dim3(NW * 64), lds, s, P);
}

// Eight waves a workgroup; sixteen, with half the groups of steps one after the other, for a long second product
// of two token fragments.  us with 8 and 16 waves, K -> outputs: 24 rows 5504 -> 2048: 9.5, 11.1; 24 rows
// 8192 -> 4096: 17.6, 18.8; 32 rows 11008 -> 4096: 22.5, 20.0; 20 rows 16384 -> 8192: 76, 65.  One row 11008 ->
// 4096: 15.8, 17.0; gated, 24 rows 2048 -> 5504: 12.3, 12.9; 20 rows 8192 -> 16384: 101, 104.
template <typename T, bool GATED, int ACT>
void launch_few_tm(const FfnArgs& g, hipStream_t s) {
  if (g.m <= 16) return launch_few<T, GATED, ACT, 1, 8>(g, s);
  if constexpr (!GATED) {
    if (g.k > 8192) return launch_few<T, GATED, ACT, 2, 16>(g, s);
  }
  launch_few<T, GATED, ACT, 2, 8>(g, s);
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
// tiles (and six for fill and epilogue) x the tile's step, plus the partials' traffic for splits.  A step is
// about 1.5 us for the wide tile and 1.0-1.1 for the 128-wide one, whose A fragments feed half the MFMAs.
// Either side of the choices, us: 8192 x 1024 x 2736: 128-wide 54, wide 77, wide in two splits 70;
// 1024 x 2736 x 8192: 128-wide in two splits 69, unsplit 108, wide in four 69; 777 x 5504 x 2048 gated: wide
// 49 (bf16, SiLU; fp16, GeLU 52-53), 128-wide 56; 8192 x 2736 x 1024 gradient: 128-wide 87, wide 91.
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
      const double steps = (double)cdiv(tiles * sp, cus) * (chunk / BK + 6.0) * (bn == 256 ? 1.0 : 0.66);
      // partials move 8 bytes an output and split at 4 TB/s, the join is a launch
      const double extra = sp > 1 ? ((double)g.m * g.n * sp * 8 / 4e6 + 5.0) / 1.5 : 0.0;
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
  Params P{(const uint16_t*)g.a, (const uint16_t*)g.b, g.c, g.lda, g.ldb, g.ldc, g.m, g.n, g.k, g.bias, g.au_hi,
           g.au_lo, p.splits > 1 ? g.ws : nullptr, p.kchunk};
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
  if (!al(g.a) || !al(g.b) || !al(g.c) || !al(g.bias) || !al(g.au_hi) || !al(g.au_lo)) return false;
  if ((g.au_hi == nullptr) != (g.au_lo == nullptr)) return false;
  if (g.n % 8 || g.lda % 8 || g.ldb % 8 || g.ldc % 8) return false;
  if ((g.a_kmajor || g.b_kmajor) && g.k % 8) return false;
  if (!g.a_kmajor && g.m % 8) return false;
  // a tile's buffer range (256 rows or 64 k rows) stays below 2 GiB
  if (g.lda >= (1 << 21) || g.ldb >= (1 << 21)) return false;
  if (ffn::cdiv(g.m, ffn::BM) * ffn::cdiv(g.n, 64) >= (1 << 24)) return false;
  switch (g.op) {
    case kFfnPlain: return !(!g.a_kmajor && g.b_kmajor);
    case kFfnGated: return g.a_kmajor && g.b_kmajor;
    case kFfnDGated: return g.a_kmajor && !g.b_kmajor && g.au_hi != nullptr && g.ldc == 2 * (int64_t)g.n;
    default: return false;
  }
}

// Up to 32 rows of a k-major x k-major product.  us of kernels at 32 rows, and at 33 on the tiles (which 128 rows
// take too, within 5): 1024 -> 2736 -> 1024 12 and 29; 2048 -> 5504 -> 2048 30 and 41; 4096 -> 11008 -> 4096 72 and 84.
static bool ffn_few(const FfnArgs& g) { return g.m <= ffn::kFewRows && g.a_kmajor && g.b_kmajor; }

FfnPlan ffn_plan(const FfnArgs& g, int cus) {
  if (ffn_few(g)) return {0, 1};
  const ffn::Plan p = ffn::make_plan(g, cus);
  return {p.bn, p.splits};
}

int64_t ffn_workspace_floats(const FfnArgs& g, int cus) {
  const FfnPlan p = ffn_plan(g, cus);
  return p.splits > 1 ? (int64_t)p.splits * g.m * g.n : 0;
}

void ffn_gemm(const FfnArgs& g, int cus, hipStream_t s) {
  if (!ffn_supported(g)) throw std::runtime_error("gated_ffn: unsupported shape, alignment or dtype");
  if (ffn_few(g)) {
    dispatch_16(g.dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      if (g.op != kFfnGated) ffn::launch_few_tm<T, false, 0>(g, s);
      else if (g.act == kGateSilu) ffn::launch_few_tm<T, true, kGateSilu>(g, s);
      else ffn::launch_few_tm<T, true, kGateGelu>(g, s);
    }, "gated_ffn");
    check_launch("gated_ffn");
    return;
  }
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
