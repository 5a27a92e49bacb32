// logits.cu -- row-wise operators over class logits behind the C ABI
// (tmnn_cuda_token_logprobs, its backward pass, tmnn_cuda_distill): the checks
// of their arguments, the choice of a kernel by the rows' width and number, and
// the kernels that need neither.
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "logits.h"
#include "logits_narrow.cuh"
#include "logits_wide.cuh"

using namespace tmnn;
using namespace tmnn::logits;

namespace {

// ------------------------------------------------------------ backward
// Wide rows, element by element from the saved statistics; a warp takes a run
// of 32 x kRun granules of one row.  Bound by the memory, the logits in and the
// gradient out: 4096 rows of 131072 bf16 logits, a tenth of them padding, take
// 316 us, 6.5 TB/s, 1021 of 32003 fp32 ones 41 us, 6.4 TB/s.
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
        b.granule<T>(q[i], e0, a.c, r);
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
    // rows of another alignment: the run's part of the row, in granules of d
    const int e0 = max(0, run * 32 * kRun * E - dm);
    const int e1 = min(V, (run + 1) * 32 * kRun * E - dm);
    if (b.idle) {
      for (int e = e0 + lane; e < e1; e += 32) d[e] = from_f<T>(0.0f);
    } else {
      write_shifted<T>(d + e0, x + e0, e1 - e0, lane, 32, e0 ? 0 : E,
                       e1 + E <= V ? 0 : E,
                       [&](const uint4 &q, int e, float *r) {
                         b.granule<T>(q, e0 + e, a.c, r);
                       });
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

void check_logits(const char *who, const tmnn_logits &x) {
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
}

RowArgs row_args(const tmnn_logits &x) {
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
// SMs a row is split further (64 rows of 131072 bf16 logits, 20 alternatives:
// 11.7 us in clusters of 8, 15.6 streamed).
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
  if (MODE == kReadTop && c < 2) c = 2;  // written for clusters
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
  // With many rows a few batches a thread, so that little of its time goes into
  // a row's start and end (70130 rows of 2215 bf16 logits, distilled: 239 us
  // with 64 threads, 303 with 128; 16384 of 8192 fp32: 236 and 185); few rows
  // are over sooner with more threads.  For alternatives the threads' maxima
  // must be well above them in number.
  const int granules = p.a.classes / kElems<T>;
  const bool many = (int64_t)p.a.rows >= (int64_t)sm_count() &&
                    (MODE != kReadTop || p.top_k <= 32);
  if (many && granules <= 1024)
    k_stream<T, 64, MODE><<<p.a.rows, 64, 0, st>>>(q);
  else if (many && granules <= 4096)
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
    return (uintptr_t)at % 16 == 0 &&
           (stride == V || p.a.rows == 1 ||
            (quads && stride % 4 == 0 && stride < 1 << 25));
  };
  p.packed = packed(p.a.x, p.a.stride);
  p.d_packed = packed(p.dx, p.d_stride);
  size_t smem = (size_t)((32 * p.pitch + 3) / 4 * 4) * 4 * sizeof(float);
  if (MODE == kLoss || MODE == kLossGrad)
    smem += (size_t)4 * 64 * (p.te.k | 1) * sizeof(float);
  if constexpr (MODE != kBack)
    if (V > 64) {
      quads ? launch_tiny_of<T, MODE, true, 16>(p, smem, st)
            : launch_tiny_of<T, MODE, false, 16>(p, smem, st);
      return;
    }
  quads ? launch_tiny_of<T, MODE, true, 8>(p, smem, st)
        : launch_tiny_of<T, MODE, false, 8>(p, smem, st);
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

void check_token_logprobs(const tmnn_logits &x, const void *tokens,
                          int index_type, uint32_t top_k, const LogprobOut &o) {
  const char *who = "token_logprobs";
  check_logits(who, x);
  if (top_k > kMaxTop || top_k > x.classes)
    bad("token_logprobs: top_k must be at most min(classes, 128)");
  if (o.logprob && !tokens && x.rows)
    bad("token_logprobs: logprob needs tokens");
  if (tokens) check_index(who, index_type);
  if (!x.rows) return;
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
}

int launch_token_logprobs(const tmnn_logits &x, const void *tokens,
                          int index_type, uint32_t top_k, const LogprobOut &o,
                          cudaStream_t st) {
  check_token_logprobs(x, tokens, index_type, top_k, o);
  const RowArgs a = row_args(x);
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
  check_logits(who, x);
  const RowArgs a = row_args(x);
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

void check_distill(const tmnn_logits &x, const void *ids, int index_type,
                   const void *teacher, int teacher_dtype, uint32_t k,
                   const float *row_weight, const float *loss,
                   const void *d_logits, int64_t d_stride) {
  const char *who = "distill";
  check_logits(who, x);
  check_index(who, index_type);
  check_dtype(who, "teacher_logits", teacher_dtype);
  if (k < 1 || k > kMaxTop) bad("distill: k must be in [1, 128]");
  if (!x.rows) return;
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
}

int launch_distill(const tmnn_logits &x, const void *ids, int index_type,
                   const void *teacher, int teacher_dtype, uint32_t k,
                   const float *row_weight, float weight, float *loss,
                   void *d_logits, int64_t d_stride, cudaStream_t st) {
  check_distill(x, ids, index_type, teacher, teacher_dtype, k, row_weight, loss,
                d_logits, d_stride);
  const RowArgs a = row_args(x);
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
