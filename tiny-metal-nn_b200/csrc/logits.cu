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

#include <cmath>
#include <stdexcept>
#include <string>

#include "logits.h"

using namespace tmnn;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
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

// ------------------------------------------------------------ one CTA a row
constexpr int kThreads = 256;

struct OpAdd {
  __device__ static float f(float a, float b) { return a + b; }
};
struct OpMax {
  __device__ static float f(float a, float b) { return max_nan(a, b); }
};
template <class Op>
__device__ float block_reduce(float v, float *buf) {
  for (int o = 16; o; o >>= 1) v = Op::f(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < kThreads / 32; ++w) v = Op::f(v, buf[w]);
  return v;
}
__device__ uint64_t block_max_key(uint64_t v, uint64_t *buf) {
  for (int o = 16; o; o >>= 1) {
    const uint64_t u = __shfl_xor_sync(~0u, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < kThreads / 32; ++w) v = buf[w] > v ? buf[w] : v;
  return v;
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    k_logprobs(RowArgs a, const void *tokens, int itype, int top_k,
               LogprobOut o) {
  __shared__ float buf[kThreads / 32];
  __shared__ uint64_t kbuf[kThreads / 32];
  const int tid = threadIdx.x;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
    const int64_t tok = tokens ? load_index(tokens, row, itype) : 0;
    int32_t *tid_out = top_k ? o.top_ids + (int64_t)row * top_k : nullptr;
    float *tlp = top_k ? o.top_logprobs + (int64_t)row * top_k : nullptr;
    if (tok < 0) {
      if (tid == 0) {
        if (o.logprob) o.logprob[row] = 0.0f;
        if (o.entropy) o.entropy[row] = 0.0f;
        if (o.stats)
          for (int i = 0; i < 3; ++i) o.stats[(int64_t)row * 3 + i] = 0.0f;
      }
      for (int k = tid; k < top_k; k += kThreads) {
        tid_out[k] = -1;
        tlp[k] = -kInf;
      }
      continue;
    }
    float m = -kInf;
    for (int v = tid; v < a.classes; v += kThreads) m = max_nan(m, to_f(x[v]));
    m = block_reduce<OpMax>(m, buf);
    const bool bad = !(m < kInf);  // NaN or +inf
    const bool empty = m == -kInf;
    float s = 0.0f, u = 0.0f;
    if (!bad && !empty)
      for (int v = tid; v < a.classes; v += kThreads) {
        const float t = (to_f(x[v]) - m) * a.c;
        const float e = ex2(t);
        s += e;
        u += e * fmaxf(t, -1e4f);  // e is 0 there: no 0 * inf
      }
    s = block_reduce<OpAdd>(s, buf);
    u = block_reduce<OpAdd>(u, buf);
    const float ln_s = logf(s);
    const float nan = __int_as_float(0x7FFFFFFF);
    if (tid == 0) {
      const float h = bad ? nan : empty ? 0.0f : ln_s - kLn2 * u / s;
      if (o.entropy) o.entropy[row] = h;
      if (o.logprob) {
        float lp = nan;
        if (!bad && tok < a.classes)
          lp = empty ? -kInf : (to_f(x[tok]) - m) * a.inv_t - ln_s;
        o.logprob[row] = lp;
      }
      if (o.stats) {
        float *st = o.stats + (int64_t)row * 3;
        st[0] = bad ? nan : m;
        st[1] = bad ? nan : s;
        st[2] = h;
      }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < top_k; ++k) {
      uint64_t best = 0;
      if (!bad && last)
        for (int v = tid; v < a.classes; v += kThreads) {
          const uint64_t key = key_of(to_f(x[v]), v);
          if (key < last && key > best) best = key;
        }
      last = block_max_key(best, kbuf);
      if (tid == 0) {
        tid_out[k] = last ? class_of(last) : -1;
        tlp[k] = bad    ? nan
                 : last ? (value_of(last >> 32) - m) * a.inv_t - ln_s
                        : -kInf;
      }
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    k_logprobs_backward(RowArgs a, const void *tokens, int itype,
                        const float *stats, const float *d_logprob,
                        const float *d_entropy, T *dx, int64_t d_stride) {
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
    T *d = dx + (int64_t)row * d_stride;
    const int64_t tok = tokens ? load_index(tokens, row, itype) : -1;
    const float m = stats[(int64_t)row * 3], s = stats[(int64_t)row * 3 + 1],
                h = stats[(int64_t)row * 3 + 2];
    float g = d_logprob ? d_logprob[row] * a.inv_t : 0.0f;
    const float b = d_entropy ? d_entropy[row] * a.inv_t : 0.0f;
    if (tokens && tok >= a.classes) g = __int_as_float(0x7FFFFFFF);
    const bool idle = s == 0.0f || (tokens && tok < 0);
    const float ln_s = logf(s), inv_s = 1.0f / s;
    for (int v = threadIdx.x; v < a.classes; v += kThreads) {
      float r = 0.0f;
      if (!idle) {
        const float t = (to_f(x[v]) - m) * a.c;
        const float p = ex2(t) * inv_s;
        const float lp = fmaxf(t, -1e4f) * kLn2 - ln_s;
        r = -p * (g + b * (lp + h));
        if (v == tok) r += g;
      }
      d[v] = from_f<T>(r);
    }
  }
}

struct Teacher {
  const void *ids, *logits;
  int itype, dtype, k;
};

template <class T>
__global__ void __launch_bounds__(kThreads)
    k_distill(RowArgs a, Teacher te, const float *row_weight, float weight,
              float *loss, T *dx, int64_t d_stride) {
  __shared__ float buf[kThreads / 32];
  __shared__ float sq[kMaxTop];
  __shared__ int32_t sid[kMaxTop];
  const int tid = threadIdx.x;
  const float nan = __int_as_float(0x7FFFFFFF);
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.stride;
    T *d = dx ? dx + (int64_t)row * d_stride : nullptr;
    // the teacher's entry of this thread: id -1 when left out
    float y = -kInf;
    int32_t id = -1;
    if (tid < te.k) {
      const int64_t i = (int64_t)row * te.k + tid;
      const int64_t q = load_index(te.ids, i, te.itype);
      y = load_value(te.logits, i, te.dtype);
      if (q >= 0 && y != -kInf) {
        id = (int32_t)q;
        if (q >= a.classes) y = nan, id = 0;
      } else {
        y = -kInf;
      }
    }
    const float ym = block_reduce<OpMax>(y, buf);
    if (ym == -kInf) {  // no entries: a padded row
      if (tid == 0) loss[row] = 0.0f;
      if (d)
        for (int v = tid; v < a.classes; v += kThreads) d[v] = from_f<T>(0.0f);
      continue;
    }
    const float ty = (y - ym) * a.inv_t;
    const float ey = id >= 0 ? expf(ty) : 0.0f;
    const float ys = block_reduce<OpAdd>(ey, buf);
    float m = -kInf;
    for (int v = tid; v < a.classes; v += kThreads) m = max_nan(m, to_f(x[v]));
    m = block_reduce<OpMax>(m, buf);
    const bool bad = !(m < kInf) || !(ym < kInf);
    const bool empty = m == -kInf;
    float s = 0.0f;
    if (!bad && !empty)
      for (int v = tid; v < a.classes; v += kThreads)
        s += ex2((to_f(x[v]) - m) * a.c);
    s = block_reduce<OpAdd>(s, buf);
    const float ln_s = logf(s), q = ey / ys;
    float l = 0.0f;
    if (q > 0.0f)
      l = empty ? kInf
                : q * ((ty - logf(ys)) - ((to_f(x[id]) - m) * a.inv_t - ln_s));
    l = block_reduce<OpAdd>(l, buf);
    if (tid == 0) loss[row] = bad ? nan : a.t * a.t * l;
    if (!d) continue;
    const float w = (row_weight ? row_weight[row] : weight) * a.t;
    if (tid < te.k) {
      sq[tid] = q;
      sid[tid] = id;
    }
    __syncthreads();
    // x is read before dx of the same element is written (they may be one)
    float own = 0.0f;
    if (!bad && !empty && tid < te.k && id >= 0) {
      float both = 0.0f;  // entries of one class add up
      for (int j = 0; j < te.k; ++j) both += sid[j] == id ? sq[j] : 0.0f;
      own = w * (ex2((to_f(x[id]) - m) * a.c) / s - both);
    }
    __syncthreads();
    const float ws = w / s;
    for (int v = tid; v < a.classes; v += kThreads) {
      const float r =
          bad ? nan : empty ? 0.0f : ex2((to_f(x[v]) - m) * a.c) * ws;
      d[v] = from_f<T>(r);
    }
    __syncthreads();
    if (!bad && !empty && tid < te.k && id >= 0) d[id] = from_f<T>(own);
    __syncthreads();
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

// The gradient's rows: as wide as the classes, and either the logits' own
// memory or apart from it.
void check_grad(const char *who, const tmnn_logits &x, const void *d,
                int64_t stride) {
  check_ptr(who, "d_logits", d, elem_size(x.dtype));
  if (stride < (int64_t)x.classes || stride > (int64_t)1 << 40)
    bad(std::string(who) + ": d_row_stride must be in [classes, 2^40]");
  if (d == x.data && stride == x.row_stride) return;
  const uintptr_t size = elem_size(x.dtype), n = x.rows;
  const uintptr_t xb = (uintptr_t)x.data, db = (uintptr_t)d;
  const uintptr_t xe = xb + ((n - 1) * x.row_stride + x.classes) * size;
  const uintptr_t de = db + ((n - 1) * stride + x.classes) * size;
  if (db < xe && xb < de)
    bad(std::string(who) + ": d_logits overlaps the logits in part");
}

uint32_t row_grid(uint32_t rows) { return rows < (1u << 20) ? rows : 1u << 20; }

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
  BY_DTYPE(x.dtype, (k_logprobs<T><<<row_grid(x.rows), kThreads, 0, st>>>(
                        a, tokens, index_type, (int)top_k, o)));
  launched(who);
  return 1;
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
  check_grad(who, x, d_logits, d_stride);
  BY_DTYPE(x.dtype,
           (k_logprobs_backward<T><<<row_grid(x.rows), kThreads, 0, st>>>(
               a, tokens, index_type, stats, d_logprob, d_entropy,
               static_cast<T *>(d_logits), d_stride)));
  launched(who);
  return 1;
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
  if (d_logits) check_grad(who, x, d_logits, d_stride);
  const Teacher te{ids, teacher, index_type, teacher_dtype, (int)k};
  BY_DTYPE(x.dtype, (k_distill<T><<<row_grid(x.rows), kThreads, 0, st>>>(
                        a, te, row_weight, weight, loss,
                        static_cast<T *>(d_logits), d_stride)));
  launched(who);
  return 1;
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
