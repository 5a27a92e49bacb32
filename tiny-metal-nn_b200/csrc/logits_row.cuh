// logits_row.cuh -- what the class-logit kernels (logits_wide.cuh,
// logits_narrow.cuh, logits.cu) have in common: a row's description, its
// logits in 16-byte granules, softmax statistics, keys that order logits, the
// teacher's entries and the terms of the gradients.
//
// For a row x[0..V) at temperature T, with m = max x and t_v = (x_v - m) / T:
//   s = sum e^{t_v},  p_v = e^{t_v} / s,  -log p_v = ln s - t_v
//   entropy = ln s - (sum e^{t_v} t_v) / s
// Differences are taken before the scale (x - m is exact or rounded once, and
// is -inf, never NaN, for any finite m), so rows of the type's lowest value
// and large offsets keep their accuracy.  ex2 of t_v log2(e) stands for the
// exponential.  Every sum and statistic is fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "logits.h"

namespace tmnn {
namespace logits {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

struct RowArgs {
  const void *x;
  int64_t stride;
  uint32_t rows;
  int32_t classes;
  float c;      // log2(e) / T
  float inv_t;  // 1 / T
  float t;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Order of a logit as an unsigned number: 0 for -inf (no alternative),
// otherwise growing with the value; +0 and -0 are one value.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (v == -kInf) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kLowestOrder = 0x00800000u;  // order of the lowest finite
// (value, lowest class first) as one key; 0 is none
__device__ __forceinline__ uint64_t key_of(float v, int32_t cls) {
  const uint32_t o = order_of(v);
  return o ? ((uint64_t)o << 32) | (0xFFFFFFFFu - (uint32_t)cls) : 0;
}
__device__ __forceinline__ int32_t class_of(uint64_t key) {
  return (int32_t)(0xFFFFFFFFu - (uint32_t)key);
}

__device__ __forceinline__ int64_t load_index(const void *p, int64_t i,
                                              int type) {
  return type == TMNN_INDEX_I64 ? static_cast<const int64_t *>(p)[i]
                                : static_cast<const int32_t *>(p)[i];
}
__device__ __forceinline__ float load_value(const void *p, int64_t i,
                                            int dtype) {
  if (dtype == TMNN_DTYPE_F32) return static_cast<const float *>(p)[i];
  if (dtype == TMNN_DTYPE_F16) return to_f(static_cast<const __half *>(p)[i]);
  return to_f(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// ------------------------------------------------------------ 16-byte granules
// Rows are read in granules of 16 bytes that lie on 16-byte boundaries; the
// first and the last one of a row may hold elements that are not the row's,
// which count as -inf.
template <class T>
constexpr int kElems = 16 / (int)sizeof(T);

__device__ __forceinline__ float2 f2(float a, float b) {
  return make_float2(a, b);
}
__device__ __forceinline__ void split(float2 v, float &a, float &b) {
  a = v.x;
  b = v.y;
}

__device__ __forceinline__ uint32_t word(const uint4 &g, int i) {
  return i == 0 ? g.x : i == 1 ? g.y : i == 2 ? g.z : g.w;
}
// the i-th pair of a granule's values
template <class T>
__device__ __forceinline__ float2 pair_of(const uint4 &g, int i);
template <>
__device__ __forceinline__ float2 pair_of<float>(const uint4 &g, int i) {
  return f2(__uint_as_float(word(g, 2 * i)), __uint_as_float(word(g, 2 * i + 1)));
}
template <>
__device__ __forceinline__ float2 pair_of<__half>(const uint4 &g, int i) {
  const uint32_t w = word(g, i);
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
  return f;
}
template <>
__device__ __forceinline__ float2 pair_of<__nv_bfloat16>(const uint4 &g,
                                                           int i) {
  const uint32_t w = word(g, i);
  return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
// two values rounded to T: one word of 16-bit values, two of fp32
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Running maximum (NaN wins) of granules, in T (a maximum is exact).
template <class T>
struct GranuleMax {
  uint32_t m[4];
  __device__ __forceinline__ static uint32_t two(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4)
      return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value)
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ void clear() {
    const uint32_t w = sizeof(T) == 4                      ? 0xFF800000u
                       : std::is_same<T, __half>::value ? 0xFC00FC00u
                                                           : 0xFF80FF80u;
    m[0] = m[1] = m[2] = m[3] = w;
  }
  __device__ __forceinline__ void add(const uint4 &g) {
    m[0] = two(m[0], g.x);
    m[1] = two(m[1], g.y);
    m[2] = two(m[2], g.z);
    m[3] = two(m[3], g.w);
  }
  __device__ __forceinline__ float get() const {
    const uint4 g{two(two(m[0], m[1]), two(m[2], m[3])), 0, 0, 0};
    if constexpr (sizeof(T) == 4) return __uint_as_float(g.x);
    float a, b;
    split(pair_of<T>(g, 0), a, b);
    return max_nan(a, b);
  }
};

// s += sum e^t and, if U, u += sum e^t t log2(e) over a granule, in two lanes;
// nm = -max and c = log2(e) / T twice
template <class T, bool U>
__device__ __forceinline__ void accumulate(const uint4 &g, float2 nm,
                                           float2 c, float2 &s,
                                           float2 &u) {
#pragma unroll
  for (int i = 0; i < kElems<T> / 2; ++i) {
    const float2 t = __fmul2_rn(__fadd2_rn(pair_of<T>(g, i), nm), c);
    float a, b;
    split(t, a, b);
    const float2 e = f2(ex2(a), ex2(b));
    s = __fadd2_rn(s, e);
    // where t is -inf e is 0: a finite t keeps 0 * t from being NaN
    if (U) u = __ffma2_rn(e, f2(fmaxf(a, -1e4f), fmaxf(b, -1e4f)), u);
  }
}

// Softmax statistics of a part of a row: the maximum m, s = sum e^{t} and
// u = sum e^{t} t log2(e), t = (x - m) / T.
struct Stat {
  float m, s, u;
};
// brings v to the maximum m
__device__ __forceinline__ void rescale(Stat &v, float m, float c) {
  const float d = (v.m - (m == -kInf ? 0.0f : m)) * c;
  const float f = ex2(d);
  v.s *= f;
  v.u = v.u * f + v.s * fmaxf(d, -1e4f);
  v.m = m;
}
__device__ __forceinline__ Stat warp_combine(Stat v, float c) {
  float m = v.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
  rescale(v, m, c);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    v.s += __shfl_xor_sync(~0u, v.s, o);
    v.u += __shfl_xor_sync(~0u, v.u, o);
  }
  return v;
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy16(void *smem, const void *global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(smem)),
               "l"(global)
               : "memory");
}
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
// Arrives without ordering memory, which costs a fence: by threads that have
// nothing to show to the other CTAs but that they came here.
__device__ __forceinline__ void cluster_arrive_started() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of `p` in the shared memory of another CTA of the cluster
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void peer_store(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

struct Teacher {
  const void *ids, *logits;
  int itype, dtype, k;
};

// the granule whose every element is -inf
template <class T>
__device__ __forceinline__ uint4 no_logits() {
  const uint32_t w = sizeof(T) == 4                   ? 0xFF800000u
                     : std::is_same<T, __half>::value ? 0xFC00FC00u
                                                      : 0xFF80FF80u;
  return uint4{w, w, w, w};
}
template <class T>
__device__ __forceinline__ uint4 pack_granule(const float *r) {
  if constexpr (sizeof(T) == 4)
    return uint4{__float_as_uint(r[0]), __float_as_uint(r[1]),
                 __float_as_uint(r[2]), __float_as_uint(r[3])};
  else
    return uint4{pack2<T>(r[0], r[1]), pack2<T>(r[2], r[3]),
                 pack2<T>(r[4], r[5]), pack2<T>(r[6], r[7])};
}

// What one row's reads give, from its statistics.
struct RowEnd {
  float m, s, u, inv_t, ln_s;
  bool bad, empty;
  __device__ __forceinline__ RowEnd(const Stat &v, float inv_t_)
      : m(v.m), s(v.s), u(v.u), inv_t(inv_t_), ln_s(logf(v.s)),
        bad(!(v.m < kInf)), empty(v.m == -kInf) {}
  __device__ __forceinline__ float logp(float x) const {
    return (x - m) * inv_t - ln_s;
  }
};
// T (log q - log p) of a teacher's entry: t_lq = T log q, x the logit of its
// class.  A loss is T times the mean of these; divided by T first, differences
// near the lowest fp32 value would leave its range.
__device__ __forceinline__ float entry_gap(const RowEnd &end, float t,
                                           float t_lq, float x) {
  return t_lq - ((x - end.m) - t * end.ln_s);
}
// An entry's part of a row's loss, q times its gap.  A class at -inf under an
// entry that counts (e^y > 0) makes the loss infinite, also where its share
// q = e^y / sum rounds to 0 and the product would be NaN.
__device__ __forceinline__ float entry_part(const RowEnd &end, float q,
                                            float gap) {
  return end.empty || gap == kInf ? kInf : q * gap;
}
__device__ __forceinline__ float not_a_number() {
  return __int_as_float(0x7FFFFFFF);
}
__device__ __forceinline__ void write_read(const LogprobOut &o, uint32_t row,
                                           const RowEnd &r, float tok_x,
                                           bool tok_ok) {
  const float nan = not_a_number();
  const float h = r.bad ? nan : r.empty ? 0.0f : r.ln_s - kLn2 * r.u / r.s;
  if (o.entropy) o.entropy[row] = h;
  if (o.logprob)
    o.logprob[row] = r.bad || !tok_ok ? nan : r.empty ? -kInf : r.logp(tok_x);
  if (o.stats) {
    float *so = o.stats + (int64_t)row * 3;
    so[0] = r.bad ? nan : r.m;
    so[1] = r.bad ? nan : r.empty ? 0.0f : r.s;
    so[2] = h;
  }
}
__device__ __forceinline__ void write_read_padding(const LogprobOut &o,
                                                   uint32_t row) {
  if (o.logprob) o.logprob[row] = 0.0f;
  if (o.entropy) o.entropy[row] = 0.0f;
  if (o.stats)
    for (int i = 0; i < 3; ++i) o.stats[(int64_t)row * 3 + i] = 0.0f;
}

// zeros in a row's gradient, in granules of its own alignment; by all threads
template <class T, int NT>
__device__ __forceinline__ void write_zeros(T *d, int n) {
  constexpr int E = kElems<T>;
  const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
  uint4 *base = reinterpret_cast<uint4 *>(d - dm);
  for (int g = threadIdx.x; g * E < dm + n; g += NT) {
    if (g * E >= dm && (g + 1) * E <= dm + n) {
      base[g] = uint4{0, 0, 0, 0};
    } else {
      for (int j = 0; j < E; ++j) {
        const int e = g * E + j - dm;
        if (e >= 0 && e < n) d[e] = from_f<T>(0.0f);
      }
    }
  }
}

// The granule that starts at any element: the two around it, shifted.  All of
// its elements are the caller's; the first granule begins up to 14 bytes before
// them and the second one ends up to 14 bytes behind them, so a row's first
// and last elements are not read this way.
template <class T>
__device__ __forceinline__ uint4 granule_at(const T *p) {
  const uint32_t at = (uint32_t)(uintptr_t)p & 15;
  const uint4 *base = reinterpret_cast<const uint4 *>(
      reinterpret_cast<const unsigned char *>(p) - at);
  const uint4 a = base[0], b = at ? base[1] : a;
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (at & 8)
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  if (at & 4)
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  const uint32_t bits = (at & 3) * 8;
  return uint4{
      __funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits)};
}

// The n elements of a row part x in memory as gradients to d, whose granules lie
// otherwise than those of x: thread `tid` of `threads` takes granules of d, body(granule
// of x, first element, its E results).  `lead`, `slack`: how near to the start
// and the end of x a granule of it may not be read whole, E at a row's start or
// end and 0 where the row goes on.
template <class T, class Body>
__device__ __forceinline__ void write_shifted(T *d, const T *x, int n, int tid,
                                              int threads, int lead, int slack,
                                              Body &&body) {
  constexpr int E = kElems<T>;
  const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
  uint4 *dst = reinterpret_cast<uint4 *>(d - dm);
  const int G = n > 0 ? (dm + n + E - 1) / E : 0;
  for (int g0 = tid; g0 < G; g0 += 4 * threads) {
    uint4 q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = (g0 + i * threads) * E - dm;
      if (e >= lead && e + E + slack <= n) q[i] = granule_at(x + e);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = g0 + i * threads, e = g * E - dm;
      float r[E];
      if (e >= lead && e + E + slack <= n) {
        body(q[i], e, r);
        dst[g] = pack_granule<T>(r);
      } else if (g < G) {  // the ends
        T v[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
          v[j] = e + j >= 0 && e + j < n ? x[e + j] : from_f<T>(-kInf);
        body(*reinterpret_cast<const uint4 *>(v), e, r);
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (e + j >= 0 && e + j < n) d[e + j] = from_f<T>(r[j]);
      }
    }
  }
}

// d[e] = e^((x[e] - m) / T) w for e < n, where d lies otherwise in its granules
// than x in shared memory: in words of 4 bytes, lanes side by side.  By all
// threads; nm, c, w: -m, log2(e) / T and w twice.
template <class T, int NT>
__device__ __forceinline__ void write_words(T *d, const T *x, int n, float2 nm,
                                            float2 c, float2 w) {
  auto two = [&](float a, float b) {
    const float2 t = __fmul2_rn(__fadd2_rn(f2(a, b), nm), c);
    return __fmul2_rn(f2(ex2(t.x), ex2(t.y)), w);
  };
  if constexpr (sizeof(T) == 2) {
    const int first = (int)((uintptr_t)d & 3) / 2;  // elements before a word
    const int pairs = (n - first) / 2;
    uint32_t *words = reinterpret_cast<uint32_t *>(d + first);
#pragma unroll 4
    for (int i = threadIdx.x; i < pairs; i += NT) {
      const float2 r = two(to_f(x[first + 2 * i]), to_f(x[first + 2 * i + 1]));
      words[i] = pack2<T>(r.x, r.y);
    }
    if (threadIdx.x == 0 && first && n > 0)
      d[0] = from_f<T>(two(to_f(x[0]), 0.0f).x);
    if (threadIdx.x == 1 && first + 2 * pairs < n)
      d[n - 1] = from_f<T>(two(to_f(x[n - 1]), 0.0f).x);
  } else {
#pragma unroll 4
    for (int e = threadIdx.x; e < n; e += NT)
      d[e] = from_f<T>(two(to_f(x[e]), 0.0f).x);
  }
}

// r = e^((x - m) / T) w of a granule; nm, c, w: -m, log2(e) / T and w twice
template <class T>
__device__ __forceinline__ void softmax_granule(const uint4 &g, float2 nm,
                                                float2 c, float2 w, float *r) {
#pragma unroll
  for (int i = 0; i < kElems<T> / 2; ++i) {
    const float2 t = __fmul2_rn(__fadd2_rn(pair_of<T>(g, i), nm), c);
    split(__fmul2_rn(f2(ex2(t.x), ex2(t.y)), w), r[2 * i], r[2 * i + 1]);
  }
}

// put(entry, q of all entries of its class) of every entry k that is the warp's:
// mine(class) says so of a class.  Entries of one class, which add up, so meet
// in one warp, where each lane holds entries lane + 32 i.
template <class Mine, class Put>
__device__ __forceinline__ void each_entry(const int32_t *ids, const float *qs,
                                           int K, Mine &&mine, Put &&put) {
  const int lane = threadIdx.x & 31;
  int32_t id[4];
  float q[4], both[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = lane + 32 * i;
    id[i] = k < K && ids[k] >= 0 && mine(ids[k]) ? ids[k] : -1;
    q[i] = k < K ? qs[k] : 0.0f;
    both[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (32 * i >= K) break;
    for (uint32_t has = __ballot_sync(~0u, id[i] >= 0); has; has &= has - 1) {
      const int from = __ffs(has) - 1;
      const int32_t of = __shfl_sync(~0u, id[i], from);
      const float add = __shfl_sync(~0u, q[i], from);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (id[j] == of) both[j] += add;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (id[i] >= 0) put(lane + 32 * i, both[i]);
}

// The last bit in which the orders of two values of T can differ and not by
// their sign alone: 7, 10 and 23 bits of fraction.
template <class T>
constexpr uint32_t kLastBit = sizeof(T) == 4                   ? 1u
                              : std::is_same<T, __half>::value ? 1u << 13
                                                               : 1u << 16;
// Whether a bound that `have` of the orders reach serves to find the K largest.
__device__ __forceinline__ bool hardly_more(uint32_t have, int K) {
  return have <= (uint32_t)(K + K / 4 + 8);
}

// A value that at least K of n <= N orders of T's reach, and hardly more: its
// first 16 bits are searched, and the others as long as too many reach it (fp32
// and fp16 logits that have much in common, like a large constant added to
// all); the order of the lowest logit if fewer than K are logits.  One warp,
// halving from the first bit in which the orders differ.
template <class T, int N>
__device__ __forceinline__ uint32_t reached_by(int K, const uint32_t *values,
                                               int n) {
  uint32_t v[N / 32], hi = 0, lo = ~0u, have = n;
#pragma unroll
  for (int i = 0; i < N / 32; ++i) {
    const int at = (threadIdx.x & 31) + 32 * i;
    v[i] = at < n ? values[at] : 0;
    hi = max(hi, v[i]);
    lo = at < n ? min(lo, v[i]) : lo;
  }
  hi = __reduce_max_sync(~0u, hi);
  lo = __reduce_min_sync(~0u, lo);
  const uint32_t same = (uint32_t)__clz(hi ^ lo);  // leading bits
  uint32_t t = same == 0 ? 0 : same == 32 ? hi : hi >> (32 - same) << (32 - same);
  auto raise = [&](uint32_t up) {  // to `up`, if K of them reach it
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < N / 32; ++i) c += v[i] >= up;
    c = __reduce_add_sync(~0u, c);
    if (c >= (uint32_t)K) {
      t = up;
      have = c;
    }
  };
  if (same < 16)
    for (uint32_t b = 1u << (31 - same); b >= 1u << 16; b >>= 1) raise(t | b);
  if (kLastBit<T> < 1u << 16 && same < 32)
    for (uint32_t b = 1u << (31 - max(same, 16u));
         b >= kLastBit<T> && !hardly_more(have, K); b >>= 1)
      raise(t | b);
  return max(t, kLowestOrder);
}

// What a kernel is made for: statistics (with alternatives), the distillation
// loss (with its gradient), the backward pass.
enum Mode { kRead = 0, kReadTop = 1, kLoss = 2, kLossGrad = 3, kBack = 4 };

// ------------------------------------------------------------ gradient terms
// d = -p (g + b (log p + H)) + g at the token
//   = e^t (k0 + k1 t log2(e)) with t = (x - m) / T
struct BackRow {
  float m, g, k0, k1;
  int tok;
  bool idle;
  __device__ __forceinline__ BackRow(const RowArgs &a, const void *tokens,
                                     int itype, const float *stats,
                                     const float *d_logprob,
                                     const float *d_entropy, uint32_t row) {
    const float *st = stats + (int64_t)row * 3;
    const int64_t t = tokens ? load_index(tokens, row, itype) : 0;
    m = st[0];
    const float s = st[1], h = st[2];
    g = d_logprob ? d_logprob[row] * a.inv_t : 0.0f;
    const float b = d_entropy ? d_entropy[row] * a.inv_t : 0.0f;
    idle = s == 0.0f || t < 0;
    if (t >= a.classes) g = not_a_number();
    tok = tokens && t < a.classes ? (int)t : -1;
    const float inv_s = 1.0f / s;
    k1 = -b * kLn2 * inv_s;
    k0 = -(b == 0.0f ? g : g + b * (h - logf(s))) * inv_s;
  }
  template <class T>
  __device__ __forceinline__ void granule(const uint4 &g, int e, float c,
                                          float *r) const {
#pragma unroll
    for (int i = 0; i < kElems<T> / 2; ++i) {
      const float2 v = pair_of<T>(g, i);
      r[2 * i] = at(v.x, e + 2 * i, c);
      r[2 * i + 1] = at(v.y, e + 2 * i + 1, c);
    }
  }
  // element e of value v
  __device__ __forceinline__ float at(float v, int e, float c) const {
    const float t = (v - m) * c;
    // where t is -inf e^t is 0: a finite t keeps 0 * t from being NaN
    const float r = ex2(t) * fmaf(k1, fmaxf(t, -1e4f), k0);
    return idle ? 0.0f : e == tok ? r + g : r;
  }
};

}  // namespace logits
}  // namespace tmnn
