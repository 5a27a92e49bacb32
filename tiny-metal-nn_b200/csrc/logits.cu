// logits.cu -- row-wise operators over class logits behind the C ABI
// (tmnn_cuda_token_logprobs, its backward pass, tmnn_cuda_distill).
//
// For a row x[0..V) at temperature T, with m = max x and t_v = (x_v - m) / T:
//   s = sum e^{t_v},  p_v = e^{t_v} / s,  -log p_v = ln s - t_v
//   entropy = ln s - (sum e^{t_v} t_v) / s
// Differences are taken before the scale (x - m is exact or rounded once, and
// is -inf, never NaN, for any finite m), so rows of the type's lowest value
// and large offsets keep their accuracy.  ex2 of t_v log2(e) stands for the
// exponential.  Every sum and statistic is fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "logits.h"

using namespace tmnn;

namespace {

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

// d[e] = e^((x(e) - m) / T) w for e < n in words of 4 bytes, lanes side by side:
// for gradients that lie otherwise in their granules than the logits.  By all
// threads; nm, c, w: -m, log2(e) / T and w twice.
template <class T, int NT, class X>
__device__ __forceinline__ void write_words(T *d, int n, X &&x, float2 nm,
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
      const float2 r = two(x(first + 2 * i), x(first + 2 * i + 1));
      words[i] = pack2<T>(r.x, r.y);
    }
    if (threadIdx.x == 0 && first && n > 0) d[0] = from_f<T>(two(x(0), 0.0f).x);
    if (threadIdx.x == 1 && first + 2 * pairs < n)
      d[n - 1] = from_f<T>(two(x(n - 1), 0.0f).x);
  } else {
#pragma unroll 4
    for (int e = threadIdx.x; e < n; e += NT) d[e] = from_f<T>(two(x(e), 0.0f).x);
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

// A value that at least K of n <= N orders reach, and hardly more: the largest
// one with the low 16 bits zero (all there is to a 16-bit logit), or what all n
// have in common; the order of the lowest logit if fewer than K are logits.
// One warp, halving from the first bit in which the orders differ.
template <int N>
__device__ __forceinline__ uint32_t reached_by(int K, const uint32_t *values,
                                               int n) {
  uint32_t v[N / 32], hi = 0, lo = ~0u;
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
  if (same < 16)
    for (uint32_t b = 1u << (31 - same); b >= 1u << 16; b >>= 1) {
      const uint32_t up = t | b;
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < N / 32; ++i) c += v[i] >= up;
      if (__reduce_add_sync(~0u, c) >= (uint32_t)K) t = up;
    }
  return max(t, kLowestOrder);
}

// ------------------------------------------------------------ a team a row
// A team -- a CTA, or a cluster of CTAs each holding a part ("slab") of the
// row in its shared memory -- reads a row once.  Every thread copies its own
// granules (cp.async) and sums over the same ones, so there is no barrier
// before the one exchange of (m, s, u) over the team; then the alternatives or
// the gradient come from the slab.  Memory traffic is that of the operator
// itself: the row once in, results or gradient once out.
//
// For a gradient three slabs of 64 KB lie on an SM (two load while one
// computes): 3687 rows of 131072 bf16 logits, in clusters of four, take 410 us,
// 5.0 TB/s.  What bounds it is a CTA's life, not the memory: load, exchange and
// two bursts of ex2 one after the other (without any ex2 it is 378 us, rows of
// one CTA each 345).  Measured and not kept: slabs of 32 KB (the same with 128
// threads), one CTA an SM that takes row after row and copies the next into
// its place (510 us), the second read out of the L2 (440 us and more; of
// 77 MB of rows in work a third is still there).
enum Mode { kRead = 0, kReadTop = 1, kLoss = 2, kLossGrad = 3, kBack = 4 };

constexpr int kMaxCluster = 16;
constexpr int kMaxGroups = 256;

// Shared memory of a CTA of a team, in bytes from its base: the slab, the
// exchange of statistics, and what the mode needs.
struct TeamLayout {
  int stats, teacher, misc, gmax, cand, total;
  int cap;     // candidates a CTA may hold
  int groups;  // groups of threads over the team, each with its maximum
};
__host__ __device__ inline TeamLayout team_layout(int mode, int threads,
                                                  int cluster, int k,
                                                  int granules) {
  TeamLayout l{};
  int off = granules * 16;
  l.stats = off;
  off += (threads / 32 + cluster) * 16;
  l.teacher = off;
  if (mode >= kLoss) off += (k * 8 + 4 + 15) / 16 * 16;
  l.misc = off;
  if (mode == kReadTop) {
    off += 16 + 2 * kMaxCluster * 4;  // count, threshold; counts of the CTAs
    l.gmax = off;
    l.groups = cluster * threads;
    while (l.groups > kMaxGroups) l.groups /= 2;
    off += l.groups * 4;
    l.cap = 2 * k > 128 ? 2 * k : 128;
    l.cand = off;
    off += cluster * l.cap * 8;  // in the first CTA those of all
  }
  l.total = (off + 15) / 16 * 16;
  return l;
}

struct TeamArgs {
  RowArgs a;
  const void *tokens;
  int itype, top_k;
  LogprobOut o;
  Teacher te;
  const float *row_weight;
  float weight;
  float *loss;
  void *dx;
  int64_t d_stride;
  int cluster;  // CTAs a row
  int slab;     // elements a CTA, a multiple of the granule
  int eager;    // copy the slab before it is known whether the row is padding
  TeamLayout l;
};

template <class T, int NT, int MODE>
__global__ void __launch_bounds__(NT) k_team(TeamArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int E = kElems<T>;
  constexpr int kWarps = NT / 32;
  constexpr bool kReads = MODE == kRead || MODE == kReadTop;
  const RowArgs &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t C = p.cluster, rank = blockIdx.x % C, row = blockIdx.x / C;
  const bool leader = rank == 0;
  const float nan = not_a_number();

  // ---- the slab: x[first .. first + n) of the row
  const int first = (int)rank * p.slab;
  const int n = max(0, min(p.slab, a.classes - first));
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride + first;
  const int mis = (int)((uintptr_t)x & 15) / (int)sizeof(T);
  const int G = n > 0 ? (mis + n + E - 1) / E : 0;
  uint4 *slab = reinterpret_cast<uint4 *>(smem);
  T *sx = reinterpret_cast<T *>(smem) + mis;  // sx[e] = x[e]
  // whole granules [lo, hi), the thread's from `mine0` on
  const int lo = mis ? 1 : 0, hi = (mis + n) / E;
  const int mine0 = lo && tid == 0 ? NT : tid;
  // the thread's elements outside whole granules: f(element)
  auto edges = [&](auto &&f) {
    if (lo && tid == 0)
      for (int j = 0; j < E; ++j) f(j - mis);
    if (G > hi && (hi || !lo) && tid == hi % NT)
      for (int j = 0; j < E; ++j) f(hi * E + j - mis);
  };
  auto load = [&] {
    const uint4 *src = reinterpret_cast<const uint4 *>(x - mis);
#pragma unroll 4
    for (int g = mine0; g < hi; g += NT) copy16(slab + g, src + g);
    edges([&](int e) { sx[e] = e >= 0 && e < n ? x[e] : from_f<T>(-kInf); });
  };
  if (p.eager) load();

  // ---- is the row padding?
  int64_t tok = 0;
  float *sq = reinterpret_cast<float *>(smem + p.l.teacher);
  int32_t *sid = reinterpret_cast<int32_t *>(sq + p.te.k);
  [[maybe_unused]] int32_t *bad_entries = sid + p.te.k;
  [[maybe_unused]] float ty[4], tq[4], ln_ys = 0.0f, ym = 0.0f;
  [[maybe_unused]] int32_t tid_[4];
  bool idle;
  if constexpr (kReads) {
    if (p.tokens) tok = load_index(p.tokens, row, p.itype);
    idle = tok < 0;
    if (idle && leader) {
      if (tid == 0) write_read_padding(p.o, row);
      if constexpr (MODE == kReadTop)
        for (int k = tid; k < p.top_k; k += NT) {
          p.o.top_ids[(int64_t)row * p.top_k + k] = -1;
          p.o.top_logprobs[(int64_t)row * p.top_k + k] = -kInf;
        }
    }
  } else {
    // Entry lane + 32 i in register i of the first warp; the others only look
    // whether there is any.
    ym = -kInf;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ty[i] = -kInf;
      tid_[i] = -1;
      const int k = lane + 32 * i;
      if (k < p.te.k && (warp == 0 || ym == -kInf)) {
        const int64_t at = (int64_t)row * p.te.k + k;
        const int64_t id = load_index(p.te.ids, at, p.te.itype);
        const float y = load_value(p.te.logits, at, p.te.dtype);
        if (id >= 0 && y != -kInf) {  // not left out
          tid_[i] = id < a.classes ? (int32_t)id : 0;
          ty[i] = id < a.classes ? y : nan;
          ym = max_nan(ym, ty[i]);
        }
      }
      if (warp && __any_sync(~0u, ym != -kInf)) {
        ym = 0.0f;
        break;
      }
    }
    if (warp == 0)
      for (int o = 16; o; o >>= 1) ym = max_nan(ym, __shfl_xor_sync(~0u, ym, o));
    idle = ym == -kInf;
    if (idle && leader && tid == 0) p.loss[row] = 0.0f;
  }
  T *d = MODE == kLossGrad
             ? static_cast<T *>(p.dx) + (int64_t)row * p.d_stride + first
             : nullptr;
  if (idle) {
    if constexpr (MODE == kLossGrad) write_zeros<T, NT>(d, n);
    copies_done();
    return;  // all CTAs of the cluster alike
  }
  if (C > 1) cluster_arrive_started();
  if (!p.eager) load();

  [[maybe_unused]] float xk[4], tok_x = 0.0f;
  if constexpr (!kReads) {
    // meanwhile the first warp: the teacher's softmax, and the logits of its
    // entries (read before any CTA of the row writes its gradient: the exchange
    // below is a barrier of them all)
    if (warp == 0) {
      float ys = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xk[i] = 0.0f;
        ty[i] = tid_[i] >= 0 ? (ty[i] - ym) * a.inv_t : -kInf;
        tq[i] = expf(ty[i]);
        ys += tq[i];
        if (leader && tid_[i] >= 0) xk[i] = to_f((x - first)[tid_[i]]);
      }
      for (int o = 16; o; o >>= 1) ys += __shfl_xor_sync(~0u, ys, o);
      ln_ys = logf(ys);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tq[i] = tq[i] / ys;
        const int k = lane + 32 * i;
        if (MODE == kLossGrad && k < p.te.k) {
          sq[k] = tq[i];
          sid[k] = tid_[i];
        }
      }
      if (lane == 0) *bad_entries = !(ym < kInf);
    }
  } else {
    if (leader && tid == 0 && p.o.logprob && tok < a.classes)
      tok_x = to_f(x[tok]);
  }
  copies_done();

  // ---- statistics of the thread's granules, four at a time: their maximum,
  // the sums brought to it, their terms
  constexpr int kBatch = 4;
  float mine = -kInf;
  Stat st;
  {
    const float2 c2 = f2(a.c, a.c);
    float2 s2 = f2(0.0f, 0.0f), u2 = s2;
    auto add = [&](const uint4 *q) {
      GranuleMax<T> gm;
      gm.clear();
#pragma unroll
      for (int i = 0; i < kBatch; ++i) gm.add(q[i]);
      const float m = max_nan(mine, gm.get());
      const float m0 = m == -kInf ? 0.0f : m;
      const float dm = (mine - m0) * a.c, f = ex2(dm);
      mine = m;
      s2 = __fmul2_rn(s2, f2(f, f));
      if (kReads) {
        const float dd = fmaxf(dm, -1e4f);
        u2 = __ffma2_rn(u2, f2(f, f), __fmul2_rn(s2, f2(dd, dd)));
      }
      const float2 nm = f2(-m0, -m0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        accumulate<T, kReads>(q[i], nm, c2, s2, u2);
    };
    int g = tid;
    uint4 q[kBatch];
    for (; g - tid + kBatch * NT <= G; g += kBatch * NT) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) q[i] = slab[g + i * NT];
      add(q);
    }
    if (g - tid < G) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        q[i] = g + i * NT < G ? slab[g + i * NT] : no_logits<T>();
      add(q);
    }
    float s0, s1, u0, u1;
    split(s2, s0, s1);
    split(u2, u0, u1);
    st = Stat{mine, s0 + s1, u0 + u1};
  }
  st = warp_combine(st, a.c);
  uint32_t *gmax = reinterpret_cast<uint32_t *>(smem + p.l.gmax);
  uint32_t *misc = reinterpret_cast<uint32_t *>(smem + p.l.misc);
  if constexpr (MODE == kReadTop) {
    // the largest logits of groups of neighbouring threads, to all CTAs
    uint32_t o = order_of(mine);
    const int size = (int)C * NT / p.l.groups;
    for (int i = 1; i < size; i *= 2)
      o = max(o, __shfl_xor_sync(~0u, o, i));
    if (C > 1) cluster_wait();
    if (tid % size == 0) {
      uint32_t *to = gmax + ((int)rank * NT + tid) / size;
      if (C > 1) {
        for (uint32_t r = 0; r < C; ++r)
          peer_store(peer_addr(to, r), __uint_as_float(o));
      } else {
        *to = o;
      }
    }
    if (tid == 0) misc[0] = 0;  // candidates
  }
  {
    // the warps' parts, then the CTAs'; all add the same parts in one order
    float *part = reinterpret_cast<float *>(smem + p.l.stats);
    float *whole = part + kWarps * 4;
    if (lane == 0) {
      part[warp * 4] = st.m;
      part[warp * 4 + 1] = st.s;
      part[warp * 4 + 2] = st.u;
    }
    __syncthreads();
    auto combine = [&](const float *of, int parts) {
      st = Stat{-kInf, 0.0f, 0.0f};
      if (lane < parts)
        st = Stat{of[lane * 4], of[lane * 4 + 1], of[lane * 4 + 2]};
      st = warp_combine(st, a.c);
    };
    if (C == 1) {
      combine(part, kWarps);
    } else {
      if (MODE != kReadTop) cluster_wait();
      if (warp == 0) {
        combine(part, kWarps);
        if (lane < (int)C) {
          const uint32_t to = peer_addr(whole + rank * 4, lane);
          peer_store(to, st.m);
          peer_store(to + 4, st.s);
          peer_store(to + 8, st.u);
        }
      }
      // Whoever wrote to a peer orders that before the barrier (a fence, which
      // costs); the others have nothing to order.
      if (warp == 0 || MODE == kReadTop)
        cluster_arrive();
      else
        cluster_arrive_started();
      cluster_wait();
      combine(whole, (int)C);
    }
  }
  RowEnd end(st, a.inv_t);
  if (!kReads) end.bad |= *bad_entries != 0;
  const float m = end.m, s = end.s;
  const bool bad = end.bad, empty = end.empty;

  if constexpr (kReads)
    if (leader && tid == 0) write_read(p.o, row, end, tok_x, tok < a.classes);

  if constexpr (MODE == kReadTop) {
    // ---- alternatives.  A value that at least K groups' maxima reach is a
    // lower bound of the K-th largest logit, and few logits lie above it.
    const int K = p.top_k;
    int32_t *ids = p.o.top_ids + (int64_t)row * K;
    float *lps = p.o.top_logprobs + (int64_t)row * K;
    auto put = [&](int at, uint64_t key) {
      ids[at] = key ? class_of(key) : -1;
      lps[at] = bad ? nan : key ? end.logp(value_of((uint32_t)(key >> 32))) : -kInf;
    };
    if (bad || empty) {  // the same in all CTAs of the row
      if (leader)
        for (int k = tid; k < K; k += NT) put(k, 0);
      return;
    }
    if (warp == 0) {
      const uint32_t t = reached_by<kMaxGroups>(K, gmax, p.l.groups);
      if (lane == 0) misc[1] = t;
    }
    __syncthreads();
    const uint32_t tau = misc[1];
    uint64_t *cand = reinterpret_cast<uint64_t *>(smem + p.l.cand);
    uint32_t *counts = misc + 4;
    const uint32_t my_order = order_of(mine);
    // Keys at or above `least`: those that fit go to this CTA's part of the
    // first CTA's buffer; returns their number over the team, or a large number
    // if a part overflowed.
    int round = 0;
    auto collect = [&](uint64_t least) {
      const float floor = value_of((uint32_t)(least >> 32));
      uint64_t *part = cand + (int)rank * p.l.cap;
      const uint32_t to = C > 1 ? peer_addr(part, 0) : smem_addr(part);
      // The warp goes together through the granules of each thread that has
      // such a key: lanes 2 i and 2 i + 1 take the halves of granule i.
      uint32_t have = __ballot_sync(
          ~0u, (((uint64_t)my_order << 32) | 0xFFFFFFFFu) >= least);
      while (have) {
        const int src = __ffs(have) - 1;
        have &= have - 1;
        for (int g = warp * 32 + src + NT * (lane >> 1); g < G; g += NT * 16) {
          const uint2 q = reinterpret_cast<const uint2 *>(slab + g)[lane & 1];
          const uint4 q4{q.x, q.y, 0, 0};
#pragma unroll
          for (int i = 0; i < E / 2; ++i) {
            float f[2];
            split(pair_of<T>(q4, i >> 1), f[0], f[1]);
            const float v = f[i & 1];
            if (v >= floor) {
              const uint64_t key =
                  key_of(v, first + g * E + (lane & 1) * (E / 2) + i - mis);
              if (key >= least) {
                const uint32_t at = atomicAdd(misc, 1u);
                if (at < (uint32_t)p.l.cap) {
                  if (C > 1)
                    peer_store(to + at * 8, key);
                  else
                    part[at] = key;
                }
              }
            }
          }
        }
      }
      __syncthreads();
      if (C == 1) {
        const int M = (int)misc[0];
        counts[0] = M;
        __syncthreads();
        if (tid == 0) misc[0] = 0;
        return M;
      }
      // two sets of counts in turn: one is written while the other is read
      uint32_t *now = counts + (round++ & 1) * kMaxCluster;
      if (tid < (int)C)
        peer_store(peer_addr(now + rank, tid), __uint_as_float(misc[0]));
      cluster_arrive();
      cluster_wait();
      if (tid == 0) misc[0] = 0;
      int M = 0, most = 0;
      for (uint32_t r = 0; r < C; ++r) {
        M += (int)now[r];
        most = max(most, (int)now[r]);
      }
      return most > p.l.cap ? 0x7FFFFFFF : M;
    };
    const int limit = C > 1 ? p.l.cap * 2 : p.l.cap;  // the first CTA ranks them
    int M = collect((uint64_t)tau << 32);
    // Rows with many equal or regularly placed values overflow the buffers:
    // halve the interval of keys (which are distinct) until few enough, but K
    // at least, are left.  64 halvings use the interval up.
    uint64_t lo = (uint64_t)tau << 32, hi = ~0ull;
    for (int i = 0; i < 64 && M > limit; ++i) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      __syncthreads();
      const int c = collect(mid);
      (c < K ? hi : lo) = mid;
      if (c >= K) M = c;
    }
    if (!leader) return;  // nothing of this CTA is read from here on
    const uint32_t *now = counts + ((round - 1) & 1) * kMaxCluster;
    if (C == 1) now = counts;
    auto held = [&](uint32_t r) { return min((int)now[r], p.l.cap); };
    int all = 0;
    for (uint32_t r = 0; r < C; ++r) all += held(r);
    for (int i = tid; i < all; i += NT) {
      int at = i;
      uint32_t r = 0;
      for (; at >= held(r); ++r) at -= held(r);
      const uint64_t key = cand[(int)r * p.l.cap + at];
      int above = 0;
      for (uint32_t q = 0; q < C; ++q) {
        const uint64_t *of = cand + (int)q * p.l.cap;
        const int many = held(q);
        for (int j = 0; j < many; ++j) above += of[j] > key;
      }
      if (above < K) put(above, key);
    }
    for (int k = all + tid; k < K; k += NT) put(k, 0);
  }

  if constexpr (!kReads) {
    if (leader && warp == 0) {
      float l = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tq[i] > 0.0f)
          l += empty ? kInf : tq[i] * ((ty[i] - ln_ys) - end.logp(xk[i]));
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
      if (lane == 0) p.loss[row] = bad ? nan : a.t * a.t * l;
    }
  }
  if constexpr (MODE == kLossGrad) {
    const float w = (p.row_weight ? p.row_weight[row] : p.weight) * a.t;
    const float ws = bad ? nan : empty ? 0.0f : w / s;
    // an empty row: 0 * 0 (its logits at -inf give e = 0 against m = 0)
    const float m0 = empty ? 0.0f : m;
    const float2 nm = f2(-m0, -m0), c2 = f2(a.c, a.c), w2 = f2(ws, ws);
    const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
    if (dm == mis) {
      uint4 *dst = reinterpret_cast<uint4 *>(d - dm);
#pragma unroll 4
      for (int g = mine0; g < hi; g += NT) {
        const uint4 q = slab[g];
        float r[E];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const float2 t = __fmul2_rn(__fadd2_rn(pair_of<T>(q, i), nm), c2);
          split(__fmul2_rn(f2(ex2(t.x), ex2(t.y)), w2), r[2 * i], r[2 * i + 1]);
        }
        dst[g] = pack_granule<T>(r);
      }
      edges([&](int e) {
        if (e >= 0 && e < n)
          d[e] = from_f<T>(ex2((to_f(sx[e]) - m0) * a.c) * ws);
      });
    } else {
      // rows of another alignment (the copies of other threads are visible
      // since the exchange)
      write_words<T, NT>(d, n, [&](int e) { return to_f(sx[e]); }, nm, c2, w2);
    }
    // An entry's element is written again, after its first value: by the warp
    // that wrote that (of another alignment: by any one, after all have).
    const bool aligned = dm == mis;
    if (aligned)
      __syncwarp();
    else
      __syncthreads();
    if (!bad && !empty)
      each_entry(
          sid, sq, p.te.k,
          [&](int32_t id) {
            const int e = id - first;
            return e >= 0 && e < n &&
                   (aligned ? (e + mis) / E % NT / 32 : e % kWarps) == warp;
          },
          [&](int k, float q) {
            const int e = sid[k] - first;
            d[e] = from_f<T>(w * (ex2((to_f(sx[e]) - m) * a.c) / s - q));
          });
  }
}

// ------------------------------------------------------------ a CTA a row
// Short rows, and wide ones without a gradient that are enough to fill the SMs:
// a CTA streams its row through registers, four granules a thread at a time,
// and nothing of the row is kept.  One exchange at the end; a gradient reads
// the row again.  Without alternatives the next four granules are on their way
// while four are worked on; with them (more registers) more CTAs do as well.
//
// Bound by the memory: 3687 rows of 131072 bf16 logits take 141 us, 6.9 TB/s
// (measured with alternatives: 2048 rows and 64 of them 109 us, 83 without --
// the search after a row's end is what is left over).  One ex2 a logit keeps
// the special-function unit busy for two thirds of that time.
//
// For the alternatives each thread notes the maximum of every run of granules
// it read.  The K-th largest of the threads' maxima is a lower bound of the
// row's K-th largest logit; the few runs that reach it are read once more (out
// of the L2) and their logits above it ranked.
constexpr int kRuns = 16;             // runs a thread
constexpr int kPicked = 4 * kMaxTop;  // runs read again, logits ranked

struct StreamArgs {
  RowArgs a;
  const void *tokens;
  int itype, top_k;
  LogprobOut o;
  Teacher te;
  const float *row_weight;
  float weight;
  float *loss;
  void *dx;
  int64_t d_stride;
};

template <class T, int NT, int MODE>
__global__ void __launch_bounds__(NT) k_stream(StreamArgs p) {
  constexpr int E = kElems<T>, kBatch = 4, kWarps = NT / 32;
  constexpr bool kReads = MODE == kRead || MODE == kReadTop;
  constexpr bool kTop = MODE == kReadTop;
  __shared__ float part[kWarps * 3];
  __shared__ float run_max[kTop ? (kRuns + 1) * NT : 1];
  __shared__ uint32_t gmax[kTop ? NT : 1], runs[kTop ? kPicked : 1];
  __shared__ uint64_t picked[kTop ? kPicked : 1];
  __shared__ uint32_t misc[4];  // runs to read, tau, logits picked
  constexpr bool kGrad = MODE == kLossGrad;
  __shared__ float sq[kGrad ? kMaxTop : 1], sxk[kGrad ? kMaxTop : 1];
  __shared__ int32_t sid[kGrad ? kMaxTop : 1];
  const RowArgs &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t row = blockIdx.x;
  const int V = a.classes;
  const float nan = not_a_number();

  // ---- `head` elements up to a 16-byte boundary, whole granules, the rest
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
  const int mis = (int)((uintptr_t)x & 15) / (int)sizeof(T);
  const int head = min(mis ? E - mis : 0, V), F = (V - head) / E;
  const uint4 *src = reinterpret_cast<const uint4 *>(x + head);
  T *d = kGrad ? static_cast<T *>(p.dx) + (int64_t)row * p.d_stride : nullptr;
  // The row in batches, body(granules, first one): the last, short one first,
  // then the whole ones, each loaded while the one before is worked on.
  constexpr bool kAhead = MODE == kRead && NT > 128;
  const int whole = F / (kBatch * NT);
  const bool rest = F > whole * kBatch * NT;
  auto load = [&](uint4 *to, int b) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) to[i] = src[(b * kBatch + i) * NT + tid];
  };
  auto load_last = [&](uint4 *to) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int f = (whole * kBatch + i) * NT + tid;
      to[i] = f < F ? src[f] : no_logits<T>();
    }
  };
  auto sweep = [&](uint4 *one, auto &&body) {  // one: the last batch
    if constexpr (!kAhead) {
      if (rest) body(one, whole);
      for (int b = 0; b < whole; ++b) {
        load(one, b);
        body(one, b);
      }
      return;
    }
    uint4 two[kBatch];
    if (whole) load(two, 0);
    if (rest) body(one, whole);
    for (int b = 0; b < whole;) {
      if (b + 1 < whole) load(one, b + 1);
      body(two, b++);
      if (b == whole) break;
      if (b + 1 < whole) load(two, b + 1);
      body(one, b++);
    }
  };
  uint4 q[kBatch];
  if (rest) load_last(q);
  // the elements outside whole granules, one a lane of the first warp
  float odd = -kInf;
  int odd_class = 0;
  if (warp == 0 && lane < 16) {
    odd_class = lane < 8 ? lane : head + F * E + lane - 8;
    if (lane < 8 ? lane < head : odd_class < V) odd = to_f(x[odd_class]);
  }

  // ---- is the row padding?
  int64_t tok = 0;
  float tok_x = 0.0f;
  [[maybe_unused]] float ty[4], xk[4], ym = -kInf;
  [[maybe_unused]] int32_t tid_[4];
  if constexpr (kReads) {
    if (p.tokens) tok = load_index(p.tokens, row, p.itype);
    if (tok < 0) {
      if (tid == 0) write_read_padding(p.o, row);
      if constexpr (kTop)
        for (int k = tid; k < p.top_k; k += NT) {
          p.o.top_ids[(int64_t)row * p.top_k + k] = -1;
          p.o.top_logprobs[(int64_t)row * p.top_k + k] = -kInf;
        }
      return;
    }
    if (tid == 0 && p.o.logprob && tok < V) tok_x = to_f(x[tok]);
  } else {
    // entry lane + 32 i in register i (every warp: all of them must know)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ty[i] = -kInf;
      xk[i] = 0.0f;
      tid_[i] = -1;
      const int k = lane + 32 * i;
      if (k >= p.te.k) continue;
      const int64_t at = (int64_t)row * p.te.k + k;
      const int64_t id = load_index(p.te.ids, at, p.te.itype);
      const float y = load_value(p.te.logits, at, p.te.dtype);
      if (id < 0 || y == -kInf) continue;  // left out
      ty[i] = id < V ? y : nan;
      tid_[i] = id < V ? (int32_t)id : 0;
      if (warp == 0 && id < V) xk[i] = to_f(x[id]);
      ym = max_nan(ym, ty[i]);
    }
    for (int o = 16; o; o >>= 1) ym = max_nan(ym, __shfl_xor_sync(~0u, ym, o));
    if (ym == -kInf) {
      if (tid == 0) p.loss[row] = 0.0f;
      if constexpr (kGrad) write_zeros<T, NT>(d, V);
      return;
    }
  }
  if (kTop && tid == 0) misc[0] = misc[2] = 0;

  // ---- the stream
  Stat st{-kInf, 0.0f, 0.0f};
  float2 s2 = f2(0.0f, 0.0f), u2 = s2;
  const float2 c2 = f2(a.c, a.c);
  // a run is `per` batches, the last batch one of its own
  const int per = max(1, (whole + kRuns - 1) / kRuns);
  int run = 0, in_run = 0;
  float run_of = -kInf;
  // the logits outside whole granules, first of all
  if (warp == 0) {
    const float m0 = odd == -kInf ? 0.0f : odd;
    const float t = (odd - m0) * a.c, e = ex2(t);
    st.m = odd;
    s2 = f2(e, 0.0f);
  }
  sweep(q, [&](const uint4 *g, int b) {
    GranuleMax<T> gm;
    gm.clear();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) gm.add(g[i]);
    const float batch = gm.get();
    const float m = max_nan(st.m, batch), m0 = m == -kInf ? 0.0f : m;
    const float dm = (st.m - m0) * a.c, f = ex2(dm);
    st.m = m;
    s2 = __fmul2_rn(s2, f2(f, f));
    if (kReads) {
      const float dd = fmaxf(dm, -1e4f);
      u2 = __ffma2_rn(u2, f2(f, f), __fmul2_rn(s2, f2(dd, dd)));
    }
    const float2 nm = f2(-m0, -m0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) accumulate<T, kReads>(g[i], nm, c2, s2, u2);
    if constexpr (kTop) {
      if (b == whole) {
        run_max[kRuns * NT + tid] = batch;
      } else {
        run_of = fmaxf(run_of, batch);
        if (++in_run == per) {
          run_max[run++ * NT + tid] = run_of;
          run_of = -kInf;
          in_run = 0;
        }
      }
    }
  });
  {
    float s0, s1, u0, u1;
    split(s2, s0, s1);
    split(u2, u0, u1);
    st.s = s0 + s1;
    st.u = u0 + u1;
  }
  if constexpr (kTop) {
    if (in_run) run_max[run++ * NT + tid] = run_of;
    gmax[tid] = order_of(st.m);
  }
  st = warp_combine(st, a.c);
  if (lane == 0) {
    part[warp * 3] = st.m;
    part[warp * 3 + 1] = st.s;
    part[warp * 3 + 2] = st.u;
  }
  __syncthreads();
  if (!kTop && !kGrad && warp) return;
  st = Stat{-kInf, 0.0f, 0.0f};
  if (lane < kWarps)
    st = Stat{part[lane * 3], part[lane * 3 + 1], part[lane * 3 + 2]};
  st = warp_combine(st, a.c);
  RowEnd end(st, a.inv_t);

  if constexpr (kReads) {
    if (tid == 0) write_read(p.o, row, end, tok_x, tok < V);
  } else {
    end.bad |= !(ym < kInf);
  }
  if (!kReads && warp == 0) {
    float tq[4], ys = 0.0f, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = !(ty[i] == -kInf);
      ty[i] = (ty[i] - ym) * a.inv_t;
      tq[i] = in ? expf(ty[i]) : 0.0f;
      ys += tq[i];
    }
    for (int o = 16; o; o >>= 1) ys += __shfl_xor_sync(~0u, ys, o);
    const float ln_ys = logf(ys);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (tq[i] > 0.0f)
        l += end.empty ? kInf
                       : tq[i] / ys * ((ty[i] - ln_ys) - end.logp(xk[i]));
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    if (lane == 0) p.loss[row] = end.bad ? nan : a.t * a.t * l;
    if constexpr (kGrad) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = lane + 32 * i;
        if (k < p.te.k) {
          sq[k] = tq[i] / ys;
          sxk[k] = xk[i];
          sid[k] = tid_[i];
        }
      }
    }
  }
  if constexpr (kGrad) {
    const float w = (p.row_weight ? p.row_weight[row] : p.weight) * a.t;
    const float ws = end.bad ? nan : end.empty ? 0.0f : w / end.s;
    // an empty row: 0 * 0 (its logits at -inf give e = 0 against m = 0)
    const float m0 = end.empty ? 0.0f : end.m;
    const float2 nm = f2(-m0, -m0), w2 = f2(ws, ws);
    if ((int)((uintptr_t)d & 15) == mis * (int)sizeof(T)) {
      uint4 *dst = reinterpret_cast<uint4 *>(d + head);
      if (rest) load_last(q);
      sweep(q, [&](const uint4 *g, int b) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          float r[E];
#pragma unroll
          for (int j = 0; j < E / 2; ++j) {
            const float2 t = __fmul2_rn(__fadd2_rn(pair_of<T>(g[i], j), nm), c2);
            split(__fmul2_rn(f2(ex2(t.x), ex2(t.y)), w2), r[2 * j], r[2 * j + 1]);
          }
          const int f = (b * kBatch + i) * NT + tid;
          if (b < whole || f < F) dst[f] = pack_granule<T>(r);
        }
      });
      if (warp == 0 && lane < 16 && (lane < 8 ? lane < head : odd_class < V))
        d[odd_class] = from_f<T>(ex2((odd - m0) * a.c) * ws);
    } else {
      // rows of another alignment
      write_words<T, NT>(d, V, [&](int e) { return to_f(x[e]); }, nm, c2, w2);
    }
    __syncthreads();  // an entry's element is written again, after its first value
    if (!end.bad && !end.empty)
      each_entry(
          sid, sq, p.te.k, [&](int32_t id) { return id % kWarps == warp; },
          [&](int k, float q) {
            d[sid[k]] =
                from_f<T>(w * (ex2((sxk[k] - end.m) * a.c) / end.s - q));
          });
  }
  if constexpr (kTop) {
    const int K = p.top_k;
    int32_t *ids = p.o.top_ids + (int64_t)row * K;
    float *lps = p.o.top_logprobs + (int64_t)row * K;
    auto put = [&](int at, uint64_t key) {
      ids[at] = key ? class_of(key) : -1;
      lps[at] =
          end.bad ? nan : key ? end.logp(value_of((uint32_t)(key >> 32))) : -kInf;
    };
    if (end.bad || end.empty) {
      for (int k = tid; k < K; k += NT) put(k, 0);
      return;
    }
    if (warp == 0) {
      const uint32_t t = reached_by<NT>(K, gmax, NT);
      if (lane == 0) misc[1] = t;
    }
    __syncthreads();
    const uint32_t tau = misc[1];
    const float floor = value_of(tau);
    for (int r = 0; r <= kRuns; ++r)
      if ((r < run || (r == kRuns && rest)) && run_max[r * NT + tid] >= floor) {
        const uint32_t at = atomicAdd(misc, 1u);
        if (at < kPicked) runs[at] = (uint32_t)(r << 16 | tid);
      }
    __syncthreads();
    const bool over = misc[0] > kPicked;
    const int todo = over ? 0 : (int)misc[0], of = per * kBatch;
    // f(key, place) of every logit of those runs, or of the row if there were
    // too many, and of the logits outside whole granules
    auto each = [&](auto &&f) {
      auto granule = [&](int g) {
        const uint4 w = src[g];
#pragma unroll
        for (int j = 0; j < E; ++j) {
          float v[2];
          split(pair_of<T>(w, j >> 1), v[0], v[1]);
          if (v[j & 1] >= floor) f(key_of(v[j & 1], head + g * E + j));
        }
      };
      for (int i = tid; i < todo * of; i += NT) {
        const uint32_t r = runs[i / of];
        const bool end_run = r >> 16 == kRuns;
        const int at = (end_run ? whole * kBatch : (int)(r >> 16) * of) + i % of;
        const int g = at * NT + (int)(r & 0xFFFF);
        if (end_run ? g < F : at < whole * kBatch) granule(g);
      }
      if (over)
        for (int g = tid; g < F; g += NT) granule(g);
      if (odd >= floor) f(key_of(odd, odd_class));
    };
    auto pick = [&](uint64_t least) {
      each([&](uint64_t key) {
        if (key >= least) {
          const uint32_t at = atomicAdd(misc + 2, 1u);
          if (at < kPicked) picked[at] = key;
        }
      });
      __syncthreads();
      return (int)misc[2];
    };
    uint64_t lo = (uint64_t)tau << 32, hi = ((uint64_t)order_of(end.m) + 1) << 32;
    int M = over ? kPicked + 1 : pick(lo);
    if (M > kPicked) {
      // Many equal logits: halve the interval of keys, which are distinct,
      // until K of them at least are left, but few enough.  64 halvings use
      // the interval up.
      for (int i = 0; i < 64; ++i) {
        const uint64_t mid = lo + ((hi - lo) >> 1);
        int c = 0;
        each([&](uint64_t key) { c += key >= mid; });
        c = __reduce_add_sync(~0u, c);
        __syncthreads();
        if (lane == 0) gmax[warp] = (uint32_t)c;
        if (tid == 0) misc[2] = 0;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all += (int)gmax[w];
        (all >= K ? lo : hi) = mid;
        if (all >= K && all <= kPicked) break;
      }
      M = min(pick(lo), kPicked);
    }
    for (int i = tid; i < M; i += NT) {
      const uint64_t key = picked[i];
      int above = 0;
      for (int j = 0; j < M; ++j) above += picked[j] > key;
      if (above < K) put(above, key);
    }
    for (int k = M + tid; k < K; k += NT) put(k, 0);
  }
}

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
  // element e of value v
  __device__ __forceinline__ float at(float v, int e, float c) const {
    const float t = (v - m) * c;
    // where t is -inf e^t is 0: a finite t keeps 0 * t from being NaN
    const float r = ex2(t) * fmaf(k1, fmaxf(t, -1e4f), k0);
    return idle ? 0.0f : e == tok ? r + g : r;
  }
};

// ------------------------------------------------------------ a thread a row
// Rows of up to 128 classes (a field has up to 64 outputs): a warp brings 32 of them into
// shared memory as fp32, side by side as they lie in memory, and each thread
// works through one row there.  No lane idles on a row's odd end and nothing
// is reduced over lanes.  Rows of whole quads lie `pitch` apart, an odd number
// of quads, so that the lanes' 16-byte reads meet different banks; other rows
// keep their distance V (odd, or twice an odd number).
constexpr int kTinyClasses = 128;

struct TinyArgs {
  RowArgs a;
  const void *tokens;
  int itype, top_k;
  LogprobOut o;
  const float *stats, *d_logprob, *d_entropy;  // backward
  Teacher te;
  const float *row_weight;
  float weight;
  float *loss;
  void *dx;
  int64_t d_stride;
  int pitch;            // floats between rows in shared memory
  int packed, d_packed; // rows without gaps from a 16-byte boundary on
};

// EIGHTS: eights of classes a row may have
template <class T, int MODE, bool QUADS, int EIGHTS>
__global__ void __launch_bounds__(128) k_tiny(TinyArgs p) {
  extern __shared__ __align__(16) float image_all[];
  constexpr bool kReads = MODE == kRead || MODE == kReadTop;
  constexpr bool kTeacher = MODE == kLoss || MODE == kLossGrad;
  const RowArgs &a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int V = a.classes, P = p.pitch;
  const uint32_t row0 = (blockIdx.x * 4 + warp) * 32;
  if (row0 >= a.rows) return;
  const int rows = min(32u, a.rows - row0);
  float *image = image_all + warp * ((32 * P + 3) / 4 * 4);
  const float nan = not_a_number();

  // use(row, i, load(row, i)) of every i < N of every row, lanes side by side,
  // four loads in flight
  auto each_of = [&](int N, auto &&load, auto &&use) {
    int r = 0, c = lane;
    while (c >= N) c -= N, ++r;
    const int dr = 32 / N, dc = 32 - dr * N;
    while (__any_sync(~0u, r < rows)) {
      int rs[4], cs[4];
      decltype(load(0, 0)) v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rs[i] = r;
        cs[i] = c;
        if (r < rows) v[i] = load(r, c);
        r += dr;
        c += dc;
        if (c >= N) c -= N, ++r;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (rs[i] < rows) use(rs[i], cs[i], v[i]);
    }
  };
  // The same of every quad of packed rows: load(quad), then use(first of its
  // four places in the image, quad, value).
  auto each_quad = [&](int end, auto &&load, auto &&use) {
    const int R = QUADS ? V / 4 : 1;  // quads a row
    int r = lane / R, c = lane - r * R;
    const int dr = 32 / R, dc = 32 - dr * R;
    for (int i0 = lane; i0 - lane < end; i0 += 128) {
      int at[4];
      decltype(load(0, 0)) v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at[i] = QUADS ? r * P + c * 4 : (i0 + 32 * i) * 4;
        if (i0 + 32 * i < end) v[i] = load(at[i], i0 + 32 * i);
        if (QUADS) {
          r += dr;
          c += dc;
          if (c >= R) c -= R, ++r;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + 32 * i < end) use(at[i], i0 + 32 * i, v[i]);
    }
  };

  // ---- in
  const T *x = static_cast<const T *>(a.x) + (int64_t)row0 * a.stride;
  const int quads = rows * V / 4;  // whole ones
  const bool on = lane < rows;
  const uint32_t row = row0 + (on ? lane : 0);
  int64_t tok = 0;
  float weight = p.weight;
  if (kReads && p.tokens) tok = load_index(p.tokens, row, p.itype);
  if (MODE == kLossGrad && p.row_weight) weight = p.row_weight[row];
  if (p.packed) {
    if constexpr (sizeof(T) == 4) {
      each_quad(
          quads,
          [&](int at, int i) {
            copy16(image + at, reinterpret_cast<const uint4 *>(x) + i);
            return 0;
          },
          [](int, int, int) {});
    } else {
      each_quad(
          quads,
          [&](int, int i) { return reinterpret_cast<const uint2 *>(x)[i]; },
          [&](int at, int, const uint2 &w) {
            const uint4 g{w.x, w.y, 0, 0};
            float4 v;
            split(pair_of<T>(g, 0), v.x, v.y);
            split(pair_of<T>(g, 1), v.z, v.w);
            *reinterpret_cast<float4 *>(image + at) = v;
          });
    }
    const int e = quads * 4 + lane;
    if (!QUADS && e < rows * V) image[e] = to_f(x[e]);
  } else {
    each_of(
        V, [&](int r, int c) { return x[(int64_t)r * a.stride + c]; },
        [&](int r, int c, T v) { image[r * P + c] = to_f(v); });
  }
  // the teacher's entries: id (-1 if left out) and logit, rows an odd number
  // apart
  const int K = kTeacher ? p.te.k : 0, KP = K | 1;
  float *ey = image_all + 4 * ((32 * P + 3) / 4 * 4) + warp * 64 * KP;
  int32_t *eid = reinterpret_cast<int32_t *>(ey + 32 * KP);
  if constexpr (kTeacher) {
    struct Entry {
      int64_t id;
      float y;
    };
    const int64_t first = (int64_t)row0 * K;
    each_of(
        K,
        [&](int r, int k) {
          return Entry{load_index(p.te.ids, first + r * K + k, p.te.itype),
                       load_value(p.te.logits, first + r * K + k, p.te.dtype)};
        },
        [&](int r, int k, const Entry &t) {
          const bool out = t.id < 0 || t.y == -kInf;  // left out
          ey[r * KP + k] = out ? -kInf : t.id < V ? t.y : nan;
          eid[r * KP + k] = out ? -1 : t.id < V ? (int32_t)t.id : 0;
        });
    ey += lane * KP;
    eid += lane * KP;
  }
  if (p.packed && sizeof(T) == 4) copies_done();
  __syncwarp();

  float *mine = image + lane * P;
  // the j-th eight of the thread's row, -inf behind its end
  auto eight = [&](int j, float *v) {
    const int c = j * 8;
    if (QUADS) {
      const float4 lo = *reinterpret_cast<const float4 *>(mine + c);
      float4 hi{-kInf, -kInf, -kInf, -kInf};
      if (c + 4 < V) hi = *reinterpret_cast<const float4 *>(mine + c + 4);
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w;
      v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    } else if (c + 8 <= V) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mine[c + i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < V ? mine[c + i] : -kInf;
    }
  };
  auto write_eight = [&](int j, const float *v) {
    const int c = j * 8;
    if (QUADS) {
      *reinterpret_cast<float4 *>(mine + c) = float4{v[0], v[1], v[2], v[3]};
      if (c + 4 < V)
        *reinterpret_cast<float4 *>(mine + c + 4) = float4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < V) mine[c + i] = v[i];
    }
  };
  auto max8 = [](const float *v) {
    return max_nan(max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])),
                   max_nan(max_nan(v[4], v[5]), max_nan(v[6], v[7])));
  };
  const int eights = (V + 7) / 8;

  if (on) {
    if constexpr (MODE == kBack) {
      const BackRow b(a, p.tokens, p.itype, p.stats, p.d_logprob, p.d_entropy,
                      row);
#pragma unroll 2
      for (int j = 0; j < eights; ++j) {
        float v[8];
        eight(j, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = b.at(v[i], j * 8 + i, a.c);
        write_eight(j, v);
      }
    } else {
      float ym = -kInf;
      bool idle = tok < 0;
      if constexpr (kTeacher) {
        for (int k = 0; k < K; ++k) ym = max_nan(ym, ey[k]);
        idle = ym == -kInf;
      }
      float best[EIGHTS];  // maxima of the eights
#pragma unroll
      for (int j = 0; j < EIGHTS; ++j) {
        best[j] = -kInf;
        if (j < eights) {
          float v[8];
          eight(j, v);
          best[j] = max8(v);
        }
      }
      float top = max8(best);
#pragma unroll
      for (int j = 8; j < EIGHTS; j += 8) top = max_nan(top, max8(best + j));
      Stat st{top, 0.0f, 0.0f};
      const float m0 = st.m == -kInf ? 0.0f : st.m;
      const float2 nm = f2(-m0, -m0), c2 = f2(a.c, a.c);
      {
        float2 s2 = f2(0.0f, 0.0f), u2 = s2;
#pragma unroll 2
        for (int j = 0; j < eights; ++j) {
          float v[8];
          eight(j, v);
#pragma unroll
          for (int i = 0; i < 8; i += 4)
            accumulate<float, kReads>(
                uint4{__float_as_uint(v[i]), __float_as_uint(v[i + 1]),
                      __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])},
                nm, c2, s2, u2);
        }
        float s0, s1, u0, u1;
        split(s2, s0, s1);
        split(u2, u0, u1);
        st.s = s0 + s1;
        st.u = u0 + u1;
      }
      RowEnd end(st, a.inv_t);
      if (kTeacher) end.bad |= !(ym < kInf);
      if constexpr (kReads) {
        if (idle)
          write_read_padding(p.o, row);
        else
          write_read(p.o, row, end, tok < V ? mine[tok] : 0.0f, tok < V);
      }
      if constexpr (MODE == kReadTop) {
        // the largest of the eights' maxima, its class, and that eight without
        // it, again and again; four alternatives are written together
        const bool none = end.bad || idle;
        int32_t *ids = p.o.top_ids + (int64_t)row * p.top_k;
        float *lps = p.o.top_logprobs + (int64_t)row * p.top_k;
        const bool fours = p.top_k % 4 == 0 && (uintptr_t)p.o.top_ids % 16 == 0 &&
                           (uintptr_t)p.o.top_logprobs % 16 == 0;
        for (int k0 = 0; k0 < p.top_k; k0 += 4) {
          int32_t id[4];
          float lp[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v = best[0];
            int at = 0;
#pragma unroll
            for (int j = 1; j < EIGHTS; ++j)
              if (best[j] > v) {
                v = best[j];
                at = j;
              }
            const bool some = v > -kInf && !none && k0 + k < p.top_k;
            id[k] = -1;
            lp[k] = end.bad && !idle ? nan : -kInf;
            if (some) {
              float w[8];
              eight(at, w);
              int i = 7;
#pragma unroll
              for (int e = 6; e >= 0; --e)
                if (w[e] == v) i = e;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e == i) w[e] = -kInf;
              const float rest = max8(w);
              id[k] = at * 8 + i;
              lp[k] = end.logp(v);
              mine[id[k]] = -kInf;
#pragma unroll
              for (int j = 0; j < EIGHTS; ++j)
                if (j == at) best[j] = rest;
            }
          }
          if (fours) {
            *reinterpret_cast<int4 *>(ids + k0) = int4{id[0], id[1], id[2], id[3]};
            *reinterpret_cast<float4 *>(lps + k0) =
                float4{lp[0], lp[1], lp[2], lp[3]};
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k0 + k < p.top_k) {
                ids[k0 + k] = id[k];
                lps[k0 + k] = lp[k];
              }
          }
        }
      }
      if constexpr (kTeacher) {
        // loss = sum q (log q - log p) = (sum e (y - log p)) / sum e
        //        - log sum e  with e = e^y, y = (teacher - max) / T
        const float w = weight * a.t;
        const bool zero = idle || (end.empty && !end.bad);
        float ys = 0.0f, loss = 0.0f;
        for (int k = 0; k < K; ++k) {
          const float y = (ey[k] - ym) * a.inv_t, e = eid[k] >= 0 ? expf(y) : 0.0f;
          ys += e;
          if (e > 0.0f)
            loss += end.empty ? kInf : e * (y - end.logp(mine[eid[k]]));
          if (MODE == kLossGrad) ey[k] = e;
        }
        const float inv_ys = 1.0f / ys;
        p.loss[row] = idle      ? 0.0f
                      : end.bad ? nan
                                : a.t * a.t * (loss * inv_ys - logf(ys));
        if constexpr (MODE == kLossGrad) {
          const float ws = zero ? 0.0f : end.bad ? nan : w / end.s;
          const float2 w2 = f2(ws, ws);
#pragma unroll 2
          for (int j = 0; j < eights; ++j) {
            float v[8];
            eight(j, v);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
              float t, u;
              split(__fmul2_rn(__fadd2_rn(f2(v[i], v[i + 1]), nm), c2), t, u);
              split(__fmul2_rn(f2(ex2(t), ex2(u)), w2), v[i], v[i + 1]);
              if (zero) v[i] = v[i + 1] = 0.0f;
            }
            write_eight(j, v);
          }
          if (!zero && !end.bad) {
            const float wq = w * inv_ys;
            for (int k = 0; k < K; ++k)
              if (eid[k] >= 0) mine[eid[k]] -= wq * ey[k];
          }
        }
      }
    }
  }

  // ---- out
  if constexpr (MODE == kLossGrad || MODE == kBack) {
    __syncwarp();
    T *d = static_cast<T *>(p.dx) + (int64_t)row0 * p.d_stride;
    if (p.d_packed) {
      each_quad(
          quads,
          [&](int at, int) { return *reinterpret_cast<const float4 *>(image + at); },
          [&](int, int i, const float4 &v) {
            if constexpr (sizeof(T) == 4)
              reinterpret_cast<float4 *>(d)[i] = v;
            else
              reinterpret_cast<uint2 *>(d)[i] =
                  uint2{pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)};
          });
      const int e = quads * 4 + lane;
      if (!QUADS && e < rows * V) d[e] = from_f<T>(image[e]);
    } else {
      each_of(
          V, [&](int r, int c) { return image[r * P + c]; },
          [&](int r, int c, float v) {
            d[(int64_t)r * p.d_stride + c] = from_f<T>(v);
          });
    }
  }
}

// ------------------------------------------------------------ lanes a row
// Narrow rows: 1 to 32 neighbouring lanes hold a row in registers, NG granules
// each (granule lane + lanes * j), and reduce over one another with shuffles.
// There is no shared memory but for a teacher's entries, and nothing is read
// or written twice.
struct NarrowArgs {
  RowArgs a;
  const void *tokens;
  int itype, top_k;
  LogprobOut o;
  const float *stats, *d_logprob, *d_entropy;  // backward
  Teacher te;
  const float *row_weight;
  float weight;
  float *loss;
  void *dx;
  int64_t d_stride;
  int lanes;
  int cap;  // logits listed for a row's alternatives, 0: no list
  // the logits' memory, inside which a whole granule may be read although it
  // holds elements of other rows (null where those may be written meanwhile)
  const void *lo, *hi;
};

template <class T, int NG, int MODE>
__global__ void __launch_bounds__(128) k_narrow(NarrowArgs p) {
  extern __shared__ __align__(16) float entries[];
  constexpr int E = kElems<T>;
  constexpr bool kReads = MODE == kRead || MODE == kReadTop;
  constexpr bool kTeacher = MODE == kLoss || MODE == kLossGrad;
  const RowArgs &a = p.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = p.lanes, l = lane & (L - 1), V = a.classes;
  const uint32_t want = (blockIdx.x * 4 + warp) * (32 / L) + lane / L;
  const bool on = want < a.rows;  // lanes of no row repeat the last one
  const uint32_t row = on ? want : a.rows - 1;
  const float nan = not_a_number();
  auto group_max = [&](float v) {
    for (int o = 1; o < L; o *= 2) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
    return v;
  };
  auto group_sum = [&](float v) {
    for (int o = 1; o < L; o *= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
  };

  // ---- the row
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
  const int mis = (int)((uintptr_t)x & 15) / (int)sizeof(T);
  const int G = (mis + V + E - 1) / E, whole = (mis + V) / E;
  uint4 q[NG];
  {
    const uint4 *src = reinterpret_cast<const uint4 *>(x - mis);
    // the granules that may be read as a whole
    const int from = mis && !(p.lo && src >= p.lo) ? 1 : 0;
    const int to = p.lo && src + G <= p.hi ? G : whole;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int g = l + L * j;
      q[j] = no_logits<T>();
      if (g >= from && g < to) {
        q[j] = src[g];
      } else if (g < G) {
        T v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int e = g * E - mis + i;
          v[i] = e >= 0 && e < V ? x[e] : from_f<T>(-kInf);
        }
        q[j] = *reinterpret_cast<const uint4 *>(v);
      }
    }
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int g = l + L * j;
      if (!(mis && g == 0) && !(g == whole && g < G)) continue;
      T v[E];
      *reinterpret_cast<uint4 *>(v) = q[j];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = g * E - mis + i;
        if (e < 0 || e >= V) v[i] = from_f<T>(-kInf);
      }
      q[j] = *reinterpret_cast<const uint4 *>(v);
    }
  }
  T *d = MODE == kLossGrad || MODE == kBack
             ? static_cast<T *>(p.dx) + (int64_t)row * p.d_stride
             : nullptr;
  // writes what f(value, next value, element, to, next to) gives of every pair
  auto write_rows = [&](auto &&f) {
    const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
    uint4 *dst = reinterpret_cast<uint4 *>(d - dm);
    if (!on) return;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int g = l + L * j, e0 = g * E - mis;
      if (g >= G) continue;
      float r[E];
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float u, v;
        split(pair_of<T>(q[j], i), u, v);
        f(u, v, e0 + 2 * i, r[2 * i], r[2 * i + 1]);
      }
      if (dm == mis && !(mis && g == 0) && g < whole) {
        dst[g] = pack_granule<T>(r);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (e0 + i >= 0 && e0 + i < V) d[e0 + i] = from_f<T>(r[i]);
      }
    }
  };

  if constexpr (MODE == kBack) {
    const BackRow b(a, p.tokens, p.itype, p.stats, p.d_logprob, p.d_entropy, row);
    write_rows([&](float u, float v, int e, float &ru, float &rv) {
      ru = b.at(u, e, a.c);
      rv = b.at(v, e + 1, a.c);
    });
    return;
  }

  // ---- the teacher's entries, entry l + lanes * i of a row by lane l
  const int K = kTeacher ? p.te.k : 0;
  float *sq = entries + (warp * (32 / L) + lane / L) * K * 3;  // e^(y - max)
  float *sy = sq + K;                                          // y, then own d
  int32_t *sid = reinterpret_cast<int32_t *>(sy + K);
  float ym = 0.0f, ys = 1.0f;
  int64_t tok = 0;
  bool idle = false;
  float tok_x = 0.0f;
  if constexpr (kTeacher) {
    ym = -kInf;
    for (int k = l; k < K; k += L) {
      const int64_t at = (int64_t)row * K + k;
      const int64_t id = load_index(p.te.ids, at, p.te.itype);
      float y = load_value(p.te.logits, at, p.te.dtype);
      const bool out = id < 0 || y == -kInf;  // left out
      if (!out && id >= V) y = nan;
      sid[k] = out ? -1 : id < V ? (int32_t)id : 0;
      sy[k] = out ? -kInf : y;
      ym = max_nan(ym, sy[k]);
    }
    ym = group_max(ym);
    idle = ym == -kInf;
    ys = 0.0f;
    for (int k = l; k < K; k += L) {
      const float y = sid[k] >= 0 ? (sy[k] - ym) * a.inv_t : -kInf;
      sy[k] = y;
      sq[k] = expf(y);
      ys += sq[k];
    }
    ys = group_sum(ys);
  } else {
    if (p.tokens) tok = load_index(p.tokens, row, p.itype);
    idle = tok < 0;
    if (l == 0 && p.o.logprob && !idle && tok < V) tok_x = to_f(x[tok]);
  }

  // ---- statistics
  GranuleMax<T> gm;
  gm.clear();
#pragma unroll
  for (int j = 0; j < NG; ++j) gm.add(q[j]);
  Stat st;
  st.m = group_max(gm.get());
  {
    const float m0 = st.m == -kInf ? 0.0f : st.m;
    const float2 nm = f2(-m0, -m0), c2 = f2(a.c, a.c);
    float2 s2 = f2(0.0f, 0.0f), u2 = s2;
#pragma unroll
    for (int j = 0; j < NG; ++j)
      if (l + L * j < G)
        accumulate<T, kReads>(q[j], nm, c2, s2, u2);
    float s0, s1, u0, u1;
    split(s2, s0, s1);
    split(u2, u0, u1);
    st.s = group_sum(s0 + s1);
    st.u = kReads ? group_sum(u0 + u1) : 0.0f;
  }
  RowEnd end(st, a.inv_t);
  if (kTeacher) end.bad |= !(ym < kInf);

  if constexpr (kReads) {
    if (l == 0 && on) {
      if (idle)
        write_read_padding(p.o, row);
      else
        write_read(p.o, row, end, tok_x, tok < V);
    }
  }
  if constexpr (MODE == kReadTop) {
    int32_t *ids = p.o.top_ids + (int64_t)row * p.top_k;
    float *lps = p.o.top_logprobs + (int64_t)row * p.top_k;
    const int K = p.top_k;
    const bool none = end.bad || idle;
    float best[NG];  // maximum of each granule
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      GranuleMax<T> t;
      t.clear();
      t.add(q[j]);
      best[j] = none ? -kInf : t.get();
    }
    // A value (16 bits of it) that K granules of the row reach is a lower bound
    // of its K-th largest logit: the granules that reach it are listed, then
    // their logits above it, which are ranked.  For a few alternatives the loop
    // below is the shorter way.
    bool open = true;  // the row's alternatives are still to be found
    if (p.cap) {
      uint32_t o[NG], t = 0;
#pragma unroll
      for (int j = 0; j < NG; ++j) o[j] = order_of(best[j]);
      for (uint32_t b = 1u << 31; b >= 1u << 16; b >>= 1) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < NG; ++j) c += o[j] >= (t | b);
        if (L == 32)
          c = __reduce_add_sync(~0u, c);
        else
          for (int i = 1; i < L; i *= 2) c += __shfl_xor_sync(~0u, c, i);
        if (c >= K) t |= b;
      }
      const float floor = value_of(max(t, kLowestOrder));
      // a row's part of the shared memory: granules, keys, the granules'
      // classes, two counts
      const int of = warp * (32 / L) + lane / L;
      uint4 *kept = reinterpret_cast<uint4 *>(entries) + of * (p.cap * 7 / 4 + 1);
      uint64_t *list = reinterpret_cast<uint64_t *>(kept + p.cap);
      int *kept_at = reinterpret_cast<int *>(list + p.cap);
      int *count = kept_at + p.cap;
      if (l < 2) count[l] = 0;
      if (L == 1) count[1] = 0;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < NG; ++j)
        if (best[j] >= floor) {
          const int at = atomicAdd(count, 1);
          if (at < p.cap) {
            kept[at] = q[j];
            kept_at[at] = (l + L * j) * E - mis;
          }
        }
      __syncwarp();
      const int granules = count[0];
      if (granules <= p.cap)
        for (int i = l; i < granules * E; i += L) {
          const float v = to_f(reinterpret_cast<const T *>(kept)[i]);
          if (v >= floor) {
            const int at = atomicAdd(count + 1, 1);
            if (at < p.cap) list[at] = key_of(v, kept_at[i / E] + i % E);
          }
        }
      __syncwarp();
      const int M = count[1];
      open = granules > p.cap || M > p.cap;
      if (!open && on) {
        for (int i = l; i < M; i += L) {
          const uint64_t key = list[i];
          int above = 0;
          for (int j = 0; j < M; ++j) above += list[j] > key;
          if (above < K) {
            ids[above] = class_of(key);
            lps[above] = end.logp(value_of((uint32_t)(key >> 32)));
          }
        }
        for (int k = M + l; k < K; k += L) {
          ids[k] = -1;
          lps[k] = end.bad && !idle ? nan : -kInf;
        }
      }
    }
    // one alternative after the other: the largest value, of the lowest class
    if (__any_sync(~0u, open))
    for (int k = 0; k < p.top_k; ++k) {
      float v = best[0];
      uint4 w = q[0];
      int at = 0;
#pragma unroll
      for (int j = 1; j < NG; ++j)
        if (best[j] > v) {
          v = best[j];
          w = q[j];
          at = j;
        }
      const float top = group_max(v);
      int cls = 0x7FFFFFFF, where = 0;
      if (v == top && top > -kInf) {
#pragma unroll
        for (int i = E - 1; i >= 0; --i) {
          float f[2];
          split(pair_of<T>(w, i >> 1), f[0], f[1]);
          if (f[i & 1] == v) where = i;
        }
        cls = (l + L * at) * E + where - mis;
      }
      int first = cls;
      for (int o = 1; o < L; o *= 2)
        first = min(first, __shfl_xor_sync(~0u, first, o));
      if (cls == first && top > -kInf) {  // taken: the granule without it
        T t[E];
        *reinterpret_cast<uint4 *>(t) = w;
        float rest = -kInf;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          if (i == where) t[i] = from_f<T>(-kInf);
          rest = fmaxf(rest, to_f(t[i]));
        }
        w = *reinterpret_cast<const uint4 *>(t);
#pragma unroll
        for (int j = 0; j < NG; ++j)
          if (j == at) {
            q[j] = w;
            best[j] = rest;
          }
      }
      if (l == 0 && on && open) {
        const bool some = top > -kInf;
        ids[k] = some ? first : -1;
        lps[k] = some ? end.logp(top) : end.bad && !idle ? nan : -kInf;
      }
    }
  }
  if constexpr (kTeacher) {
    const float ln_ys = logf(ys), inv_ys = 1.0f / ys;
    const float w = (p.row_weight ? p.row_weight[row] : p.weight) * a.t;
    float loss = 0.0f;
    __syncwarp();
    if (!idle)
      for (int k = l; k < K; k += L) {
        const float e = sq[k];
        if (sid[k] < 0) continue;
        const float xv = to_f(x[sid[k]]);
        if (e > 0.0f)
          loss += end.empty ? kInf
                            : e / ys * ((sy[k] - ln_ys) - end.logp(xv));
        if constexpr (MODE == kLossGrad) {
          float both = 0.0f;  // entries of one class add up
          for (int j = 0; j < K; ++j) both += sid[j] == sid[k] ? sq[j] : 0.0f;
          sy[k] = w * (ex2((xv - end.m) * a.c) / end.s - both * inv_ys);
        }
      }
    loss = group_sum(loss);
    if (l == 0 && on)
      p.loss[row] = idle ? 0.0f : end.bad ? nan : a.t * a.t * loss;
    if constexpr (MODE == kLossGrad) {
      const bool zero = idle || (end.empty && !end.bad);
      const float ws = zero ? 0.0f : end.bad ? nan : w / end.s;
      const float m0 = zero ? 0.0f : end.m;
      __syncwarp();  // every lane has read what the row's lanes now write
      const float2 nm = f2(-m0, -m0), c2 = f2(a.c, a.c), w2 = f2(ws, ws);
      write_rows([&](float u, float v, int, float &ru, float &rv) {
        const float2 t = __fmul2_rn(__fadd2_rn(f2(u, v), nm), c2);
        split(__fmul2_rn(f2(ex2(t.x), ex2(t.y)), w2), ru, rv);
        if (zero) ru = rv = 0.0f;
      });
      __syncwarp();  // an entry's element is written again
      if (on && !zero && !end.bad)
        for (int k = l; k < K; k += L)
          if (sid[k] >= 0) d[sid[k]] = from_f<T>(sy[k]);
    }
  }
}

// ------------------------------------------------------------ backward
// Wide rows, element by element from the saved statistics; a warp takes a run
// of 32 x kRun granules of one row.  Bound by the memory: the logits in, the
// gradient out.
constexpr int kRun = 8;

template <class T>
__global__ void __launch_bounds__(256)
    k_backward(RowArgs a, const void *tokens, int itype, const float *stats,
               const float *d_logprob, const float *d_entropy, T *dx,
               int64_t d_stride, uint32_t runs) {
  constexpr int E = kElems<T>;
  const int lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t row = unit / runs;
  if (row >= a.rows) return;
  const int run = (int)(unit - row * runs);
  const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
  T *d = dx + (int64_t)row * d_stride;
  const BackRow b(a, tokens, itype, stats, d_logprob, d_entropy, row);
  const int mis = (int)((uintptr_t)x & 15) / (int)sizeof(T);
  const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
  const int V = a.classes;
  if (mis == dm) {
    const uint4 *src = reinterpret_cast<const uint4 *>(x - mis);
    uint4 *dst = reinterpret_cast<uint4 *>(d - dm);
    const int g0 = run * 32 * kRun + lane;
    uint4 q[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int g = g0 + 32 * i;
      q[i] = uint4{0, 0, 0, 0};
      if (!b.idle && g * E >= mis && (g + 1) * E <= mis + V) q[i] = src[g];
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int g = g0 + 32 * i, e0 = g * E - mis;
      if (e0 >= 0 && e0 + E <= V) {
        float r[E];
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          float u, v;
          split(pair_of<T>(q[i], j), u, v);
          r[2 * j] = b.at(u, e0 + 2 * j, a.c);
          r[2 * j + 1] = b.at(v, e0 + 2 * j + 1, a.c);
        }
        dst[g] = pack_granule<T>(r);
      } else {
        for (int j = 0; j < E; ++j) {
          const int e = e0 + j;
          if (e >= 0 && e < V)
            d[e] = from_f<T>(b.idle ? 0.0f : b.at(to_f(x[e]), e, a.c));
        }
      }
    }
  } else {
    const int e0 = run * 32 * kRun * E + lane;
#pragma unroll 8
    for (int i = 0; i < kRun * E; ++i) {
      const int e = e0 + 32 * i;
      if (e < V) d[e] = from_f<T>(b.idle ? 0.0f : b.at(to_f(x[e]), e, a.c));
    }
  }
}

__global__ void __launch_bounds__(1024)
    k_row_sum(const float *v, uint32_t n, double *sum) {
  __shared__ double buf[32];
  double a = 0.0;
  for (uint64_t i = threadIdx.x; i < n; i += 1024) a += (double)v[i];
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) a += buf[w];
    *sum = a;
  }
}

// --------------------------------------------------------------- host side
[[noreturn]] void bad(const std::string &m) { throw std::invalid_argument(m); }

void launched(const char *who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    throw std::runtime_error(std::string(who) + ": " + cudaGetErrorString(e));
}

int elem_size(int dtype) { return dtype == TMNN_DTYPE_F32 ? 4 : 2; }

void check_dtype(const char *who, const char *what, int dtype) {
  if (dtype != TMNN_DTYPE_F32 && dtype != TMNN_DTYPE_F16 &&
      dtype != TMNN_DTYPE_BF16)
    bad(std::string(who) + ": " + what + " must be F32, F16 or BF16");
}

void check_ptr(const char *who, const char *what, const void *p, size_t align) {
  if (!p) bad(std::string(who) + ": " + what + " is null");
  if ((uintptr_t)p % align)
    bad(std::string(who) + ": " + what + " is not aligned to its element");
}
void check_opt(const char *who, const char *what, const void *p, size_t align) {
  if (p) check_ptr(who, what, p, align);
}

RowArgs check_logits(const char *who, const tmnn_logits &x) {
  check_dtype(who, "logits", x.dtype);
  if (x.classes < 1 || x.classes > kMaxClasses)
    bad(std::string(who) + ": classes must be in [1, 524288]");
  if (!(x.temperature >= 1e-4f && x.temperature <= 1e4f))
    bad(std::string(who) + ": temperature must be in [1e-4, 1e4]");
  if (x.row_stride < 0 || x.row_stride > (int64_t)1 << 40)
    bad(std::string(who) + ": row_stride must be in [0, 2^40]");
  if (x.rows > 1 && x.row_stride > ((int64_t)1 << 56) / (int64_t)x.rows)
    bad(std::string(who) + ": the rows span more than memory");
  if (x.rows) check_ptr(who, "logits", x.data, elem_size(x.dtype));
  RowArgs a;
  a.x = x.data;
  a.stride = x.row_stride;
  a.rows = x.rows;
  a.classes = (int32_t)x.classes;
  a.t = x.temperature;
  a.c = (float)(1.4426950408889634 / (double)x.temperature);
  a.inv_t = (float)(1.0 / (double)x.temperature);
  return a;
}

void check_index(const char *who, int type) {
  if (type != TMNN_INDEX_I32 && type != TMNN_INDEX_I64)
    bad(std::string(who) + ": index_type must be I32 or I64");
}
size_t index_size(int type) { return type == TMNN_INDEX_I64 ? 8 : 4; }

// The bytes from a first to behind a last one.
struct Span {
  uintptr_t from, to;
  Span(const void *p, uint64_t bytes)
      : from((uintptr_t)p), to(p ? (uintptr_t)p + bytes : (uintptr_t)p) {}
  bool meets(const Span &o) const { return from < o.to && o.from < to; }
};
Span rows_of(const void *p, uint64_t rows, int64_t stride, uint64_t classes,
             int size) {
  return Span(p, ((rows - 1) * (uint64_t)stride + classes) * size);
}
Span logits_of(const tmnn_logits &x) {
  return rows_of(x.data, x.rows, x.row_stride, x.classes, elem_size(x.dtype));
}
void check_apart(const char *who, const char *what, const Span &out,
                 std::initializer_list<Span> others) {
  for (const Span &o : others)
    if (out.meets(o))
      bad(std::string(who) + ": " + what + " overlaps another argument");
}

// The gradient's rows: as wide as the classes, and either the logits' own
// memory or apart from it.
Span check_grad(const char *who, const tmnn_logits &x, const void *d,
                int64_t stride) {
  check_ptr(who, "d_logits", d, elem_size(x.dtype));
  if (stride < (int64_t)x.classes || stride > (int64_t)1 << 40 ||
      (x.rows > 1 && stride > ((int64_t)1 << 56) / (int64_t)x.rows))
    bad(std::string(who) + ": d_row_stride must be in [classes, 2^40]");
  const Span span = rows_of(d, x.rows, stride, x.classes, elem_size(x.dtype));
  const bool same = d == x.data && (stride == x.row_stride || x.rows == 1);
  if (!same && span.meets(logits_of(x)))
    bad(std::string(who) + ": d_logits overlaps the logits in part");
  return span;
}

#define BY_DTYPE(dtype, ...)                 \
  do {                                       \
    if ((dtype) == TMNN_DTYPE_F32) {         \
      using T = float;                       \
      __VA_ARGS__;                           \
    } else if ((dtype) == TMNN_DTYPE_F16) {  \
      using T = __half;                      \
      __VA_ARGS__;                           \
    } else {                                 \
      using T = __nv_bfloat16;               \
      __VA_ARGS__;                           \
    }                                        \
  } while (0)

constexpr int kMaxDevices = 64;
int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) !=
        cudaSuccess)
      return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Shared memory above 48 KB and clusters above 8 CTAs are asked for once a
// kernel and device.
constexpr int kMostShared = 227 * 1024;  // a CTA's, static and dynamic
template <class K>
void allow(K kernel, std::atomic<uint64_t> &done, int dynamic = kMostShared) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return;
  cudaError_t e = cudaFuncSetAttribute(
      kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dynamic);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("class-logit kernel: ") +
                             cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
}

void check_launch(cudaError_t e) {
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("class-logit kernel: ") +
                             cudaGetErrorString(e));
}

template <class T, int NT, int MODE>
void launch_team_of(TeamArgs &p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto kernel = k_team<T, NT, MODE>;
  allow(kernel, done);
  const int granules = p.slab / kElems<T> + 1;
  p.l = team_layout(MODE, NT, p.cluster, MODE >= kLoss ? p.te.k : p.top_k,
                    granules);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.a.rows * (uint32_t)p.cluster);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)p.l.total;
  cfg.stream = st;
  cudaLaunchAttribute at;
  if (p.cluster > 1) {
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
  }
  check_launch(cudaLaunchKernelEx(&cfg, kernel, p));
}

// Threads and CTAs of a row.  Slabs of up to 64 KB leave three CTAs on an SM,
// so that two of them load while one computes; with too few rows to fill the
// SMs a row is split further.
template <class T, int MODE>
void launch_team(TeamArgs &p, cudaStream_t st) {
  constexpr int E = kElems<T>;
  const int64_t bytes = (int64_t)p.a.classes * (int)sizeof(T);
  const int sms = sm_count();
  int c = 1;
  while (c < 8 && bytes > (int64_t)c * 64 * 1024) c *= 2;
  while (c < 8 && bytes >= (int64_t)c * 16 * 1024 &&
         (int64_t)p.a.rows * c < 2 * sms)
    c *= 2;
  if (bytes > 8 * 128 * 1024) c = 16;
  p.cluster = c;
  p.slab = ((p.a.classes + c - 1) / c + E - 1) / E * E;
  p.eager = (int64_t)p.a.rows * c <= 2 * sms;
  const int granules = p.slab / E + 1;
  if (granules <= 1024 && (MODE != kReadTop || p.top_k <= 64))
    launch_team_of<T, 128, MODE>(p, st);
  else
    launch_team_of<T, 256, MODE>(p, st);
}

// Bytes of a row that a second read finds in the L2 while all SMs stream.
constexpr int64_t kReread = 48 * 1024;
// Whether rows are streamed by one CTA each: short rows always (one of 20 KB
// with 20 alternatives takes 6.4 us, a cluster 7.5; of 64 KB 8.4 and 6.9),
// others when there are enough of them to keep every SM loading (150 rows of
// 256 KB: 14.4 us, clusters 16.4; 100 rows: 13.1 and 10.0).  A gradient takes
// a second read of the row.
bool streams(const RowArgs &a, int size, bool grad) {
  const int64_t bytes = (int64_t)a.classes * size;
  if (grad) return bytes <= kReread;
  return bytes <= 40 * 1024 || (int64_t)a.rows >= (int64_t)sm_count();
}
template <class T, int MODE>
void launch_stream(const TeamArgs &p, cudaStream_t st) {
  const StreamArgs q{p.a,  p.tokens,     p.itype,  p.top_k, p.o,       p.te,
                     p.row_weight, p.weight, p.loss, p.dx, p.d_stride};
  // With many rows a few batches a thread at least, and maxima well above the
  // alternatives in number; few rows are over sooner with more threads.
  if (p.a.classes <= 4 * 4 * 256 * kElems<T> &&
      (int64_t)p.a.rows >= (int64_t)sm_count() &&
      (MODE != kReadTop || p.top_k <= 32))
    k_stream<T, 128, MODE><<<p.a.rows, 128, 0, st>>>(q);
  else
    k_stream<T, 256, MODE><<<p.a.rows, 256, 0, st>>>(q);
  check_launch(cudaGetLastError());
}

template <class T, int MODE, bool QUADS, int EIGHTS>
void launch_tiny_of(const TinyArgs &p, size_t smem, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto kernel = k_tiny<T, MODE, QUADS, EIGHTS>;
  allow(kernel, done);
  kernel<<<(p.a.rows + 127) / 128, 128, smem, st>>>(p);
  check_launch(cudaGetLastError());
}
template <class T, int MODE>
void launch_tiny(TinyArgs &p, cudaStream_t st) {
  const int V = p.a.classes;
  const bool quads = V % 4 == 0;
  p.pitch = quads ? (V / 4 | 1) * 4 : V;
  auto packed = [&](const void *at, int64_t stride) {
    return (uintptr_t)at % 16 == 0 && (stride == V || p.a.rows == 1);
  };
  p.packed = packed(p.a.x, p.a.stride);
  p.d_packed = packed(p.dx, p.d_stride);
  size_t smem = (size_t)((32 * p.pitch + 3) / 4 * 4) * 4 * sizeof(float);
  if (MODE == kLoss || MODE == kLossGrad)
    smem += (size_t)4 * 64 * (p.te.k | 1) * sizeof(float);
  if (V <= 64)
    quads ? launch_tiny_of<T, MODE, true, 8>(p, smem, st)
          : launch_tiny_of<T, MODE, false, 8>(p, smem, st);
  else
    quads ? launch_tiny_of<T, MODE, true, 16>(p, smem, st)
          : launch_tiny_of<T, MODE, false, 16>(p, smem, st);
}

// Granules of the widest row when rows may start anywhere inside one.
int granules_of(const RowArgs &a, int dtype) {
  const int size = elem_size(dtype), e = 16 / size;
  const bool aligned =
      (uintptr_t)a.x % 16 == 0 && (a.rows == 1 || a.stride % e == 0);
  return (a.classes + (aligned ? 0 : e - 1) + e - 1) / e;
}
constexpr int kNarrow = 256;  // granules of a narrow row

template <class T, int NG, int MODE>
void launch_narrow_of(NarrowArgs &p, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  auto kernel = k_narrow<T, NG, MODE>;
  size_t smem = 0;
  if (MODE == kLoss || MODE == kLossGrad) {
    allow(kernel, done);
    smem = (size_t)(128 / p.lanes) * p.te.k * 12;
  }
  // (four rounds of the loop over the alternatives cost about a list)
  p.cap = MODE == kReadTop && p.top_k > 4 ? (32 + 2 * p.top_k) / 4 * 4 : 0;
  if (p.cap) {
    allow(kernel, done);
    smem = (size_t)(128 / p.lanes) * (p.cap * 7 / 4 + 1) * 16;
  }
  const uint32_t rows = 128 / p.lanes;
  kernel<<<(p.a.rows + rows - 1) / rows, 128, smem, st>>>(p);
  check_launch(cudaGetLastError());
}

// Four granules a lane keep enough loads in flight and few lanes idle; eight
// only where 32 lanes are not enough.
template <class T, int MODE>
void launch_narrow(NarrowArgs &p, int dtype, cudaStream_t st) {
  const int g = granules_of(p.a, dtype);
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes * 4 < g) p.lanes *= 2;
  const bool in_place = p.dx == p.a.x;
  p.lo = in_place ? nullptr : p.a.x;
  p.hi = static_cast<const T *>(p.a.x) +
         ((int64_t)(p.a.rows - 1) * p.a.stride + p.a.classes);
  if (p.lanes * 4 >= g)
    launch_narrow_of<T, 4, MODE>(p, st);
  else
    launch_narrow_of<T, 8, MODE>(p, st);
}

// Launches for rows [i, i + n) of all, n small enough for a grid.
template <class F>
int in_parts(uint32_t rows, F &&f) {
  constexpr uint32_t most = 1u << 26;
  int launches = 0;
  for (uint64_t i = 0; i < rows; i += most, ++launches)
    f((uint32_t)i, (uint32_t)(rows - i < most ? rows - i : most));
  return launches;
}
const void *at(const void *p, int64_t bytes) {
  return p ? static_cast<const unsigned char *>(p) + bytes : nullptr;
}

}  // namespace

namespace tmnn {

int launch_token_logprobs(const tmnn_logits &x, const void *tokens,
                          int index_type, uint32_t top_k, const LogprobOut &o,
                          cudaStream_t st) {
  const char *who = "token_logprobs";
  RowArgs a = check_logits(who, x);
  if (top_k > kMaxTop || top_k > x.classes)
    bad("token_logprobs: top_k must be at most min(classes, 128)");
  if (o.logprob && !tokens && x.rows)
    bad("token_logprobs: logprob needs tokens");
  if (tokens) check_index(who, index_type);
  if (!x.rows) return 0;
  check_opt(who, "tokens", tokens, index_size(index_type));
  check_opt(who, "logprob", o.logprob, 4);
  check_opt(who, "entropy", o.entropy, 4);
  check_opt(who, "stats", o.stats, 4);
  if (top_k) {
    check_ptr(who, "top_ids", o.top_ids, 4);
    check_ptr(who, "top_logprobs", o.top_logprobs, 4);
  }
  const uint64_t n = x.rows;
  const Span in = logits_of(x), toks(tokens, n * index_size(index_type));
  const Span out[] = {{o.logprob, n * 4},
                      {o.entropy, n * 4},
                      {top_k ? o.top_ids : nullptr, n * top_k * 4},
                      {top_k ? o.top_logprobs : nullptr, n * top_k * 4},
                      {o.stats, n * 12}};
  for (int i = 0; i < 5; ++i) {
    check_apart(who, "an output", out[i], {in, toks});
    for (int j = 0; j < i; ++j) check_apart(who, "an output", out[i], {out[j]});
  }
  return in_parts(x.rows, [&](uint32_t i, uint32_t n) {
    TeamArgs p{};
    p.a = a;
    p.a.x = at(x.data, (int64_t)i * x.row_stride * elem_size(x.dtype));
    p.a.rows = n;
    p.tokens = at(tokens, (int64_t)i * index_size(index_type));
    p.itype = index_type;
    p.top_k = (int)top_k;
    p.o.logprob = o.logprob ? o.logprob + i : nullptr;
    p.o.entropy = o.entropy ? o.entropy + i : nullptr;
    p.o.top_ids = top_k ? o.top_ids + (int64_t)i * top_k : nullptr;
    p.o.top_logprobs = top_k ? o.top_logprobs + (int64_t)i * top_k : nullptr;
    p.o.stats = o.stats ? o.stats + (int64_t)i * 3 : nullptr;
    if (x.classes <= kTinyClasses) {
      TinyArgs q{};
      q.a = p.a;
      q.tokens = p.tokens;
      q.itype = p.itype;
      q.top_k = p.top_k;
      q.o = p.o;
      if (top_k)
        BY_DTYPE(x.dtype, (launch_tiny<T, kReadTop>(q, st)));
      else
        BY_DTYPE(x.dtype, (launch_tiny<T, kRead>(q, st)));
    } else if (granules_of(p.a, x.dtype) <= kNarrow) {
      NarrowArgs q{};
      q.a = p.a;
      q.tokens = p.tokens;
      q.itype = p.itype;
      q.top_k = p.top_k;
      q.o = p.o;
      if (top_k)
        BY_DTYPE(x.dtype, (launch_narrow<T, kReadTop>(q, x.dtype, st)));
      else
        BY_DTYPE(x.dtype, (launch_narrow<T, kRead>(q, x.dtype, st)));
    } else if (streams(p.a, elem_size(x.dtype), false)) {
      if (top_k)
        BY_DTYPE(x.dtype, (launch_stream<T, kReadTop>(p, st)));
      else
        BY_DTYPE(x.dtype, (launch_stream<T, kRead>(p, st)));
    } else if (top_k) {
      BY_DTYPE(x.dtype, (launch_team<T, kReadTop>(p, st)));
    } else {
      BY_DTYPE(x.dtype, (launch_team<T, kRead>(p, st)));
    }
  });
}

int launch_token_logprobs_backward(const tmnn_logits &x, const void *tokens,
                                   int index_type, const float *stats,
                                   const float *d_logprob,
                                   const float *d_entropy, void *d_logits,
                                   int64_t d_stride, cudaStream_t st) {
  const char *who = "token_logprobs_backward";
  RowArgs a = check_logits(who, x);
  if (d_logprob && !tokens && x.rows)
    bad("token_logprobs_backward: d_logprob needs tokens");
  if (tokens) check_index(who, index_type);
  if (!x.rows) return 0;
  check_opt(who, "tokens", tokens, index_size(index_type));
  check_ptr(who, "stats", stats, 4);
  check_opt(who, "d_logprob", d_logprob, 4);
  check_opt(who, "d_entropy", d_entropy, 4);
  const uint64_t rows = x.rows;
  check_apart(who, "d_logits", check_grad(who, x, d_logits, d_stride),
              {{tokens, rows * index_size(index_type)},
               {stats, rows * 12},
               {d_logprob, rows * 4},
               {d_entropy, rows * 4}});
  const int size = elem_size(x.dtype), per_run = 32 * kRun * (16 / size);
  // one granule more than the row's bytes hold: rows may start inside one
  const uint32_t runs = (x.classes + 16 / size + per_run - 1) / per_run;
  return in_parts(x.rows, [&](uint32_t i, uint32_t n) {
    RowArgs b = a;
    b.x = at(x.data, (int64_t)i * x.row_stride * size);
    b.rows = n;
    const void *d = at(d_logits, (int64_t)i * d_stride * size);
    if (x.classes <= kTinyClasses / 2) {
      TinyArgs q{};
      q.a = b;
      q.tokens = at(tokens, (int64_t)i * index_size(index_type));
      q.itype = index_type;
      q.stats = stats + (int64_t)i * 3;
      q.d_logprob = d_logprob ? d_logprob + i : nullptr;
      q.d_entropy = d_entropy ? d_entropy + i : nullptr;
      q.dx = const_cast<void *>(d);
      q.d_stride = d_stride;
      BY_DTYPE(x.dtype, (launch_tiny<T, kBack>(q, st)));
      return;
    }
    if (granules_of(b, x.dtype) <= kNarrow) {
      NarrowArgs q{};
      q.a = b;
      q.tokens = at(tokens, (int64_t)i * index_size(index_type));
      q.itype = index_type;
      q.stats = stats + (int64_t)i * 3;
      q.d_logprob = d_logprob ? d_logprob + i : nullptr;
      q.d_entropy = d_entropy ? d_entropy + i : nullptr;
      q.dx = const_cast<void *>(d);
      q.d_stride = d_stride;
      BY_DTYPE(x.dtype, (launch_narrow<T, kBack>(q, x.dtype, st)));
      return;
    }
    const uint32_t grid = (uint32_t)(((uint64_t)n * runs + 7) / 8);
    BY_DTYPE(x.dtype,
             (k_backward<T><<<grid, 256, 0, st>>>(
                 b, at(tokens, (int64_t)i * index_size(index_type)), index_type,
                 stats + (int64_t)i * 3, d_logprob ? d_logprob + i : nullptr,
                 d_entropy ? d_entropy + i : nullptr,
                 static_cast<T *>(const_cast<void *>(d)), d_stride, runs)));
    launched(who);
  });
}

int launch_distill(const tmnn_logits &x, const void *ids, int index_type,
                   const void *teacher, int teacher_dtype, uint32_t k,
                   const float *row_weight, float weight, float *loss,
                   void *d_logits, int64_t d_stride, cudaStream_t st) {
  const char *who = "distill";
  RowArgs a = check_logits(who, x);
  check_index(who, index_type);
  check_dtype(who, "teacher_logits", teacher_dtype);
  if (k < 1 || k > kMaxTop) bad("distill: k must be in [1, 128]");
  if (!x.rows) return 0;
  check_ptr(who, "teacher_ids", ids, index_size(index_type));
  check_ptr(who, "teacher_logits", teacher, elem_size(teacher_dtype));
  check_opt(who, "row_weight", row_weight, 4);
  check_ptr(who, "loss", loss, 4);
  const uint64_t rows = x.rows;
  const Span id_span(ids, rows * k * index_size(index_type)),
      teacher_span(teacher, rows * k * elem_size(teacher_dtype)),
      weights(d_logits ? row_weight : nullptr, rows * 4), losses(loss, rows * 4);
  check_apart(who, "loss", losses,
              {logits_of(x), id_span, teacher_span, weights});
  if (d_logits)
    check_apart(who, "d_logits", check_grad(who, x, d_logits, d_stride),
                {id_span, teacher_span, weights, losses});
  const int size = elem_size(x.dtype);
  return in_parts(x.rows, [&](uint32_t i, uint32_t n) {
    TeamArgs p{};
    p.a = a;
    p.a.x = at(x.data, (int64_t)i * x.row_stride * size);
    p.a.rows = n;
    p.te = {at(ids, (int64_t)i * k * index_size(index_type)),
            at(teacher, (int64_t)i * k * elem_size(teacher_dtype)), index_type,
            teacher_dtype, (int)k};
    p.row_weight = row_weight ? row_weight + i : nullptr;
    p.weight = weight;
    p.loss = loss + i;
    p.dx = const_cast<void *>(at(d_logits, (int64_t)i * d_stride * size));
    p.d_stride = d_stride;
    if (x.classes <= kTinyClasses) {
      TinyArgs q{};
      q.a = p.a;
      q.te = p.te;
      q.row_weight = p.row_weight;
      q.weight = weight;
      q.loss = p.loss;
      q.dx = p.dx;
      q.d_stride = d_stride;
      if (d_logits)
        BY_DTYPE(x.dtype, (launch_tiny<T, kLossGrad>(q, st)));
      else
        BY_DTYPE(x.dtype, (launch_tiny<T, kLoss>(q, st)));
    } else if (granules_of(p.a, x.dtype) <= kNarrow) {
      NarrowArgs q{};
      q.a = p.a;
      q.te = p.te;
      q.row_weight = p.row_weight;
      q.weight = weight;
      q.loss = p.loss;
      q.dx = p.dx;
      q.d_stride = d_stride;
      if (d_logits)
        BY_DTYPE(x.dtype, (launch_narrow<T, kLossGrad>(q, x.dtype, st)));
      else
        BY_DTYPE(x.dtype, (launch_narrow<T, kLoss>(q, x.dtype, st)));
    } else if (!d_logits && streams(p.a, size, false)) {
      BY_DTYPE(x.dtype, (launch_stream<T, kLoss>(p, st)));
    } else if (d_logits && streams(p.a, size, true)) {
      BY_DTYPE(x.dtype, (launch_stream<T, kLossGrad>(p, st)));
    } else if (d_logits) {
      BY_DTYPE(x.dtype, (launch_team<T, kLossGrad>(p, st)));
    } else {
      BY_DTYPE(x.dtype, (launch_team<T, kLoss>(p, st)));
    }
  });
}

void launch_row_sum(const float *values, uint32_t n, double *sum,
                    cudaStream_t st) {
  k_row_sum<<<1, 1024, 0, st>>>(values, n, sum);
  launched("row_sum");
}

}  // namespace tmnn

namespace {
thread_local std::string g_logits_err;

// Runs f with `device` current and puts the caller's device back.
template <class F>
tmnn_status on_device(int device, F &&f) {
  try {
    g_logits_err.clear();
    int before = device;
    const bool known = cudaGetDevice(&before) == cudaSuccess;
    if (!known) cudaGetLastError();
    if (known && before != device) {
      const cudaError_t e = cudaSetDevice(device);
      if (e != cudaSuccess)
        throw std::runtime_error(std::string("cudaSetDevice: ") +
                                 cudaGetErrorString(e));
    }
    struct Back {
      int device;
      bool on;
      ~Back() {
        if (on) cudaSetDevice(device);
      }
    } back{before, known && before != device};
    f();
    return TMNN_OK;
  } catch (const std::invalid_argument &e) {
    g_logits_err = e.what();
    return TMNN_ERR_INVALID_ARGUMENT;
  } catch (const std::exception &e) {
    g_logits_err = e.what();
    return TMNN_ERR_OPERATION_FAILED;
  } catch (...) {
    g_logits_err = "unknown error";
    return TMNN_ERR_OPERATION_FAILED;
  }
}

tmnn_status null_logits() {
  g_logits_err = "null logits";
  return TMNN_ERR_NULL_OBJECT;
}
}  // namespace

extern "C" {

tmnn_status tmnn_cuda_token_logprobs(int device, void *stream,
                                     const tmnn_logits *logits,
                                     const void *tokens, int32_t index_type,
                                     uint32_t top_k, float *logprob,
                                     float *entropy, int32_t *top_ids,
                                     float *top_logprobs, float *stats) {
  if (!logits) return null_logits();
  return on_device(device, [&] {
    launch_token_logprobs(*logits, tokens, index_type, top_k,
                          {logprob, entropy, top_ids, top_logprobs, stats},
                          static_cast<cudaStream_t>(stream));
  });
}

tmnn_status tmnn_cuda_token_logprobs_backward(
    int device, void *stream, const tmnn_logits *logits, const void *tokens,
    int32_t index_type, const float *stats, const float *d_logprob,
    const float *d_entropy, void *d_logits, int64_t d_row_stride) {
  if (!logits) return null_logits();
  return on_device(device, [&] {
    launch_token_logprobs_backward(*logits, tokens, index_type, stats,
                                   d_logprob, d_entropy, d_logits,
                                   d_row_stride,
                                   static_cast<cudaStream_t>(stream));
  });
}

tmnn_status tmnn_cuda_distill(int device, void *stream,
                              const tmnn_logits *logits,
                              const void *teacher_ids, int32_t index_type,
                              const void *teacher_logits,
                              int32_t teacher_dtype, uint32_t k,
                              const float *row_weight, float *loss,
                              void *d_logits, int64_t d_row_stride) {
  if (!logits) return null_logits();
  return on_device(device, [&] {
    const float mean = logits->rows ? 1.0f / (float)logits->rows : 0.0f;
    launch_distill(*logits, teacher_ids, index_type, teacher_logits,
                   teacher_dtype, k, row_weight, mean, loss, d_logits,
                   d_row_stride, static_cast<cudaStream_t>(stream));
  });
}

const char *tmnn_cuda_logits_last_error(void) { return g_logits_err.c_str(); }

}  // extern "C"
