// Distillation loss against a teacher's top logits (forward + backward) for gfx950.
//
// Teacher: `top` logits z_k at classes j_k of a row (j_k < 0: no entry), t = softmax over the
// valid entries of z / T.  Student: q = softmax(x / T) over all classes.
//   loss = T^2 sum_k t_k (log t_k - log q_{j_k})          (T^2 KL(t || q); 0 for a row without entries)
//   dx_v = g T (q_v - sum_k t_k [j_k = v])
//
// Both passes are bound by the logits' bytes (8192 x 50304 bf16: 5.3 TB/s forward, 4.8-5.2 backward): the
// forward reads them once (running maximum and rescaled sum per lane over 8-element vectors, in base 2
// with 1/T folded into its scale), the backward reads them once and writes the gradient once.  Rows of
// any pitch and alignment (odd vocabularies) take the same 16-byte accesses at element-aligned addresses.
// A row is one workgroup when there are rows enough to fill the chip; fewer rows are split over
// workgroups, (maximum, sum) pairs of the parts joined in a fixed order by a second launch.
// In the backward the workgroup that wrote a class's dense value also writes the teacher's
// correction to it (after a barrier), so no atomics: entries naming one class twice are summed by
// the first of them.
// A class index past the vocabulary makes the row's loss and gradient NaN; nothing is read there.
// Row statistics, teacher weights and losses are fp32.  The backward gets the row's (maximum, sum)
// pair rather than their log-sum-exp: 2^((x - maximum) c) / sum keeps the digits that rounding
// maximum + log(sum) to 24 bits loses (about 1e-6 of q at logits of 30).
#include <climits>

#include "apex_amd/device.h"
#include "apex_amd/dispatch.h"
#include "apex_amd/topk_distill_api.h"

namespace apex_amd {
namespace kd {

constexpr int kThreads = 512;  // 8192 x 50304 bf16: 182 + 315 us, with 256 threads a row 188 + 338, with 1024 239 + 321
constexpr int kWaves = kThreads / 64;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kLastCache = 256ll << 20;  // bytes of the memory-side cache

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Pack8 { T e[8]; };

// a vector that nobody reads again before the caches have turned over
template <typename T>
__device__ __forceinline__ Pack8<T> stream8(const T* p) {
  typedef uint32_t vec __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
  return __builtin_bit_cast(Pack8<T>, __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)));
}

template <typename T>
__device__ __forceinline__ void load8(float (&r)[8], const T* p) {
  const Pack8<T> v = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = to_f(v.e[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&r)[8]) {
  Pack8<T> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.e[i] = from_f<T>(r[i]);
  *reinterpret_cast<Pack8<T>*>(p) = v;
}

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// (m, s): m the maximum so far, s = sum 2^((x - m) c), c = log2(e) / T.  The subtraction comes before
// the scale, so the error of an exponent is relative to x - m (exact at the maximum), not to x.  A maximum
// of -inf (nothing or only -inf so far) subtracts 0 instead, so -inf - -inf never appears; NaN reaches s.
__device__ __forceinline__ float base(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2, float c) {
  const float M = fmaxf(m, m2), b = base(M);
  s = s * exp2_((m - b) * c) + s2 * exp2_((m2 - b) * c);
  m = M;
}

template <int N>
__device__ __forceinline__ void accumulate(float& m, float& s, const float (&x)[N], float c) {
  float lm = x[0];
#pragma unroll
  for (int k = 1; k < N; ++k) lm = fmaxf(lm, x[k]);
  const float M = fmaxf(m, lm), b = base(M);
  float ls = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) ls += exp2_((x[k] - b) * c);
  s = s * exp2_((m - b) * c) + ls;
  m = M;
}

// The row's teacher entries into LDS: class (-1: none) and logit.  Returns the row's state in every thread:
// 0 no entries (or all -inf), 1 usable, 2 a class past the vocabulary.  All threads call it and the two
// below; `red` holds 2 * kWaves floats.
template <typename TI>
__device__ __forceinline__ int teacher_entries(const float* __restrict__ z, const TI* __restrict__ idx, int top,
                                               int classes, int* cls, float* t, float* red) {
  float state = 0.f;
  for (int k = threadIdx.x; k < top; k += kThreads) {
    const int64_t j = (int64_t)idx[k];
    const bool in = j >= 0 && j < classes;
    const float y = in ? z[k] : -INFINITY;
    cls[k] = in ? (int)j : -1;
    t[k] = y;
    state = fmaxf(state, j >= classes ? 2.f : y != -INFINITY ? 1.f : 0.f);
  }
  return (int)block_max(state, red);
}

// logits in t -> weights; T log of them in lt (forward)
__device__ __forceinline__ void teacher_weights(int top, float c, float temp, float* t, float* lt, float* red) {
  float m = -INFINITY;
  for (int k = threadIdx.x; k < top; k += kThreads) m = fmaxf(m, t[k]);
  m = block_max(m, red);
  const float b = base(m);
  float s = 0.f;
  for (int k = threadIdx.x; k < top; k += kThreads) s += exp2_((t[k] - b) * c);
  s = block_sum(s, red);
  const float inv = 1.f / s, ls = temp * kLn2 * __builtin_amdgcn_logf(s);
  for (int k = threadIdx.x; k < top; k += kThreads) {
    const float y = t[k] - b;
    if (lt != nullptr) lt[k] = y - ls;
    t[k] = exp2_(y * c) * inv;
  }
  __syncthreads();
}

// The row's loss and its (maximum, sum), from the latter (thread 0 writes).  Its terms are T t (T log t - T log q):
// log q of a logit at its type's lowest value overflows where its term does not.
template <typename T>
__device__ __forceinline__ void row_loss(const T* __restrict__ x, float m, float s, float temp, int state, int top,
                                         const int* cls, const float* t, const float* lt, float* red,
                                         float* __restrict__ loss, float2* __restrict__ stat) {
  const float ls = temp * kLn2 * __builtin_amdgcn_logf(s);
  float a = 0.f;
  if (state == 1)
    for (int k = threadIdx.x; k < top; k += kThreads)
      if (cls[k] >= 0 && t[k] != 0.f) a += t[k] * (lt[k] - (to_f(x[cls[k]]) - m - ls));
  a = block_sum(a, red);
  if (threadIdx.x == 0) {
    *loss = state == 2 ? __builtin_nanf("") : temp * a;
    *stat = make_float2(m, s);
  }
}

// One (row, part): the part's (maximum, sum); a row in one part also gets its loss here.  STREAM: logits that
// exceed the last cache are read past it: 155 us (5.3 TB/s) instead of 182 at 8192 x 50304 bf16 (0.8 GB), a
// backward behind it then takes 341 instead of 315; at 1021 x 50257 (0.1 GB) the pair would lose 8 of 61 us.
template <typename T, typename TI, bool STREAM>
__global__ void __launch_bounds__(kThreads)
kd_fwd_kernel(const T* __restrict__ logits, int64_t pitch, int classes, const float* __restrict__ tz,
              const TI* __restrict__ ti, int top, float c, float temp, float* __restrict__ losses,
              float2* __restrict__ stats, float2* __restrict__ parts, int chunk) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float red[2 * kWaves];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * pitch;
  const int c0 = blockIdx.y * chunk, c1 = min(classes, c0 + chunk);
  float m = -INFINITY, s = 0.f;
  int v = c0 + threadIdx.x * 8;
  for (; v + 24 * kThreads + 8 <= c1; v += 32 * kThreads) {  // four vectors in flight
    Pack8<T> w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T* p = x + v + 8 * kThreads * i;
      w[i] = STREAM ? stream8(p) : *reinterpret_cast<const Pack8<T>*>(p);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float r[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = to_f(w[i].e[k]);
      accumulate<8>(m, s, r, c);
    }
  }
  for (; v + 8 <= c1; v += 8 * kThreads) {
    float r0[8];
    load8<T>(r0, x + v);
    accumulate<8>(m, s, r0, c);
  }
  for (int e = c0 + ((c1 - c0) & ~7) + threadIdx.x; e < c1; e += kThreads) {
    const float r1[1] = {to_f(x[e])};
    accumulate<1>(m, s, r1, c);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) merge(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = m;
    red[kWaves + (threadIdx.x >> 6)] = s;
  }
  __syncthreads();
  m = red[0];
  s = red[kWaves];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) merge(m, s, red[w], red[kWaves + w], c);
  __syncthreads();
  if (parts != nullptr) {
    if (threadIdx.x == 0) parts[row * gridDim.y + blockIdx.y] = make_float2(m, s);
    return;
  }
  int* cls = (int*)lds;
  float *t = lds + top, *lt = lds + 2 * top;
  const int state = teacher_entries(tz + row * top, ti + row * top, top, classes, cls, t, red);
  if (state == 1) teacher_weights(top, c, temp, t, lt, red);
  row_loss(x, m, s, temp, state, top, cls, t, lt, red, losses + row, stats + row);
}

// join a row's parts (fixed order) and take its loss
template <typename T, typename TI>
__global__ void __launch_bounds__(kThreads)
kd_join_kernel(const T* __restrict__ logits, int64_t pitch, int classes, const float* __restrict__ tz,
               const TI* __restrict__ ti, int top, float c, float temp, float* __restrict__ losses,
               float2* __restrict__ stats, const float2* __restrict__ parts, int nparts) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float red[2 * kWaves];
  const int64_t row = blockIdx.x;
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x & 63; i < nparts; i += 64) {
    const float2 p = parts[row * nparts + i];
    merge(m, s, p.x, p.y, c);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) merge(m, s, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), c);
  int* cls = (int*)lds;
  float *t = lds + top, *lt = lds + 2 * top;
  const int state = teacher_entries(tz + row * top, ti + row * top, top, classes, cls, t, red);
  if (state == 1) teacher_weights(top, c, temp, t, lt, red);
  row_loss(logits + row * pitch, m, s, temp, state, top, cls, t, lt, red, losses + row, stats + row);
}

template <typename T, typename TI>
__global__ void __launch_bounds__(kThreads)
kd_bwd_kernel(const float* __restrict__ gl, int64_t gl_stride, const T* __restrict__ logits, int64_t pitch, int classes,
              const float* __restrict__ tz, const TI* __restrict__ ti, int top, float c, float temp,
              const float2* __restrict__ stats, T* __restrict__ grad, int chunk) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float red[2 * kWaves];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * pitch;
  T* gx = grad + row * classes;
  const int c0 = blockIdx.y * chunk, c1 = min(classes, c0 + chunk);
  // a lane's first vector is on its way while the teacher's entries are read
  int v = c0 + threadIdx.x * 8;
  Pack8<T> next;
  if (v + 8 <= c1) next = *reinterpret_cast<const Pack8<T>*>(x + v);
  int* cls = (int*)lds;
  float* t = lds + top;
  const int state = teacher_entries(tz + row * top, ti + row * top, top, classes, cls, t, red);
  const float2 st = stats[row];
  const float b = base(st.x);
  const float coef = state == 2 ? __builtin_nanf("") : gl[row * gl_stride] * temp;
  const float pc = coef / st.y;  // q_v = 2^((x - max) c) / sum
  const int tail = c0 + ((c1 - c0) & ~7);
  if (state == 0) {  // no teacher: a zero row whatever the logits and the incoming gradient hold
    const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (; v + 8 <= c1; v += 8 * kThreads) store8<T>(gx + v, zero);
    for (int e = tail + threadIdx.x; e < c1; e += kThreads) gx[e] = from_f<T>(0.f);
    return;
  }
  for (; v + 8 <= c1; v += 8 * kThreads) {
    const Pack8<T> w = next;
    if (v + 8 * kThreads + 8 <= c1) next = *reinterpret_cast<const Pack8<T>*>(x + v + 8 * kThreads);
    float r[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = to_f(w.e[k]);
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = pc * exp2_((r[k] - b) * c);
    store8<T>(gx + v, r);
  }
  for (int e = tail + threadIdx.x; e < c1; e += kThreads) gx[e] = from_f<T>(pc * exp2_((to_f(x[e]) - b) * c));
  if (state != 1) return;  // NaN everywhere already
  // the weights are taken while the stores above drain; its barriers also order them before the stores below
  teacher_weights(top, c, temp, t, nullptr, red);
  for (int k = threadIdx.x; k < top; k += kThreads) {
    const int j = cls[k];
    if (j < c0 || j >= c1) continue;
    float sum = 0.f;
    bool first = true;
    for (int i = 0; i < top; ++i)
      if (cls[i] == j) {
        first = first && i >= k;
        sum += t[i];
      }
    if (first) gx[j] = from_f<T>(pc * exp2_((to_f(x[j]) - b) * c) - coef * sum);
  }
}

// Parts of a row, of at least 4096 classes each.  Forward: one from two workgroups a CU on, else enough
// for four (1021 rows of 50257 fp16: 23 us in one part, 25 in two with the join).  Backward, where a part
// costs no join: enough for eight (the same rows: 51 us in one part, 38 in two).
inline int row_parts(int64_t rows, int classes, int cus, bool bwd, int* chunk) {
  const int64_t enough = (int64_t)cus * (bwd ? 8 : 2), target = (int64_t)cus * (bwd ? 8 : 4);
  int64_t p = rows >= enough ? 1 : (target + rows - 1) / rows;
  const int64_t most = classes / 4096 > 1 ? classes / 4096 : 1;
  if (p > most) p = most;
  const int64_t each = ((int64_t)classes + p - 1) / p;
  *chunk = (int)((each + 2047) / 2048 * 2048);
  return (int)(((int64_t)classes + *chunk - 1) / *chunk);
}

template <typename F>
void dispatch(const TopkDistillArgs& a, F&& f) {
  dispatch_float(a.dtype, [&](auto tag) {
    if (a.index64) f(tag, Tag<int64_t>{});
    else f(tag, Tag<int32_t>{});
  }, "topk_distill");
}

inline void check(const TopkDistillArgs& a) {
  if (a.rows < 0 || a.classes < 1 || a.classes > INT_MAX - (1 << 16) || a.top < 0 || a.top > kDistillMaxTop)
    throw std::runtime_error("topk_distill: sizes out of range");
}

// A launch has fewer than 2^32 threads an axis: more rows than these take another one.
constexpr int64_t kLaunchRows = ((int64_t(1) << 32) - 1) / kThreads;

// f(row0, rows) for each launch
template <typename F>
void launches(int64_t rows, F&& f) {
  for (int64_t r0 = 0; r0 < rows; r0 += kLaunchRows) f(r0, (unsigned)(rows - r0 < kLaunchRows ? rows - r0 : kLaunchRows));
}

}  // namespace kd

int64_t topk_distill_part_floats(const TopkDistillArgs& a, int cus) {
  int chunk;
  const int p = a.rows > 0 ? kd::row_parts(a.rows, a.classes, cus, false, &chunk) : 1;
  return p > 1 ? 2 * a.rows * p : 0;
}

void topk_distill_fwd(const TopkDistillArgs& a, float* losses, float* stats, float* parts, int cus, hipStream_t s) {
  kd::check(a);
  if (a.rows == 0) return;
  int chunk;
  const int p = kd::row_parts(a.rows, a.classes, cus, false, &chunk);
  const size_t lds = (size_t)3 * a.top * sizeof(float);
  const float c = 1.4426950408889634f / a.temperature;
  kd::dispatch(a, [&](auto tag, auto itag) {
    using T = typename decltype(tag)::type;
    using TI = typename decltype(itag)::type;
    kd::launches(a.rows, [&](int64_t r0, unsigned rows) {
      const T* x = (const T*)a.logits + r0 * a.pitch;
      const float* tz = a.teacher_logits + r0 * a.top;
      const TI* ti = (const TI*)a.teacher_indices + r0 * a.top;
      float2* st = (float2*)stats + r0;
      float2* pt = p > 1 ? (float2*)parts + r0 * p : nullptr;
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3(rows, p), dim3(kd::kThreads), p > 1 ? 0 : lds, s, x, a.pitch, a.classes, tz, ti,
                           a.top, c, a.temperature, losses + r0, st, pt, chunk);
      };
      if (a.rows * a.classes * (int64_t)sizeof(T) > kd::kLastCache) go(kd::kd_fwd_kernel<T, TI, true>);
      else go(kd::kd_fwd_kernel<T, TI, false>);
      if (p > 1)
        hipLaunchKernelGGL((kd::kd_join_kernel<T, TI>), dim3(rows), dim3(kd::kThreads), lds, s, x, a.pitch, a.classes,
                           tz, ti, a.top, c, a.temperature, losses + r0, st, (const float2*)pt, p);
    });
  });
  check_launch("topk_distill forward");
}

void topk_distill_bwd(const TopkDistillArgs& a, const float* grad_loss, int64_t grad_loss_stride, const float* stats,
                      void* grad, int cus, hipStream_t s) {
  kd::check(a);
  if (a.rows == 0) return;
  int chunk;
  const int p = kd::row_parts(a.rows, a.classes, cus, true, &chunk);
  const float c = 1.4426950408889634f / a.temperature;
  kd::dispatch(a, [&](auto tag, auto itag) {
    using T = typename decltype(tag)::type;
    using TI = typename decltype(itag)::type;
    kd::launches(a.rows, [&](int64_t r0, unsigned rows) {
      hipLaunchKernelGGL((kd::kd_bwd_kernel<T, TI>), dim3(rows, p), dim3(kd::kThreads),
                         (size_t)2 * a.top * sizeof(float), s, grad_loss + r0 * grad_loss_stride, grad_loss_stride,
                         (const T*)a.logits + r0 * a.pitch, a.pitch, a.classes, a.teacher_logits + r0 * a.top,
                         (const TI*)a.teacher_indices + r0 * a.top, a.top, c, a.temperature, (const float2*)stats + r0,
                         (T*)grad + r0 * a.classes, chunk);
    });
  });
  check_launch("topk_distill backward");
}

}  // namespace apex_amd
