// logits_wide.cuh -- class-logit kernels for rows of more than some 2000
// classes: a team of CTAs a row, and a CTA a row.
#pragma once
#include "logits_row.cuh"

namespace tmnn {
namespace logits {

// ------------------------------------------------------------ a team a row
// A team -- a CTA, or a cluster of CTAs each holding a part ("slab") of the
// row in its shared memory -- reads a row once.  Every thread copies its own
// granules (cp.async) and sums over the same ones, so there is no barrier
// before the one exchange of (m, s, u) over the team; then the alternatives or
// the gradient come from the slab.  Memory traffic is that of the operator
// itself: the row once in, results or gradient once out.
//
// For a gradient three slabs of 64 KB lie on an SM (two load while one
// computes): 4096 rows of 131072 bf16 logits, 409 of them padding (zeros, not
// read), in clusters of four, take 413 us for 2.04 GB, 4.9 TB/s.  What bounds it is a CTA's life, not the memory: load, exchange and
// two bursts of ex2 one after the other (without any ex2 it is 378 us, rows of
// one CTA each 345).  Measured and not kept: slabs of 32 KB (the same with 128
// threads), one CTA an SM that takes row after row and copies the next into
// its place (510 us), the second read out of the L2 (440 us and more; of
// 77 MB of rows in work a third is still there).
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
  [[maybe_unused]] int32_t tid_[4], counted = 0;  // entries with e^y > 0
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
        ty[i] = tid_[i] >= 0 ? ty[i] - ym : -kInf;
        tq[i] = expf(ty[i] * a.inv_t);
        ys += tq[i];
        counted |= (tq[i] > 0.0f) << i;
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
    cluster_wait();
    if (tid % size == 0) {
      uint32_t *to = gmax + ((int)rank * NT + tid) / size;
      for (uint32_t r = 0; r < C; ++r)
        peer_store(peer_addr(to, r), __uint_as_float(o));
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
    // ---- alternatives (of clusters only: what one CTA could hold is streamed).
    // A value that at least K groups' maxima reach is a lower bound of the K-th
    // largest logit, and few logits lie above it.
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
      const uint32_t t = reached_by<T, kMaxGroups>(K, gmax, p.l.groups);
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
      const uint32_t to = peer_addr(cand + (int)rank * p.l.cap, 0);
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
                if (at < (uint32_t)p.l.cap) peer_store(to + at * 8, key);
              }
            }
          }
        }
      }
      __syncthreads();
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
    const int limit = p.l.cap * 2;  // the first CTA ranks them
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
        if (counted >> i & 1)
          l += entry_part(end, tq[i],
                          entry_gap(end, a.t, ty[i] - a.t * ln_ys, xk[i]));
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
      if (lane == 0) p.loss[row] = bad ? nan : a.t * l;
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
        softmax_granule<T>(q, nm, c2, w2, r);
        dst[g] = pack_granule<T>(r);
      }
      edges([&](int e) {
        if (e >= 0 && e < n)
          d[e] = from_f<T>(ex2((to_f(sx[e]) - m0) * a.c) * ws);
      });
    } else {
      // rows of another alignment (the copies of other threads are visible
      // since the exchange)
      write_words<T, NT>(d, sx, n, nm, c2, w2);
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
// Bound by the memory: 3687 rows of 131072 bf16 logits take 142 us in a row of
// calls, 6.8 TB/s, and 159 us each by itself (162 for 155 without the loads
// ahead, 170 with eight granules at a time, when measured side by side).  One ex2 a
// logit keeps the special-function unit busy for two thirds of that time.
// With alternatives, 2048 rows and 64 of them: 110 us, 82 without; the search
// after a row's end is what is left over.  Rows whose bound many equal logits
// reach are read again for each halving of the keys' interval: 1024 rows of
// 131072 equal bf16 logits take 3.2 ms with 64 alternatives, 65 us without ties.
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
      ty[i] -= ym;
      tq[i] = in ? expf(ty[i] * a.inv_t) : 0.0f;
      ys += tq[i];
    }
    for (int o = 16; o; o >>= 1) ys += __shfl_xor_sync(~0u, ys, o);
    const float ln_ys = logf(ys);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (tq[i] > 0.0f)
        l += entry_part(end, tq[i] / ys,
                        entry_gap(end, a.t, ty[i] - a.t * ln_ys, xk[i]));
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    if (lane == 0) p.loss[row] = end.bad ? nan : a.t * l;
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
          softmax_granule<T>(g[i], nm, c2, w2, r);
          const int f = (b * kBatch + i) * NT + tid;
          if (b < whole || f < F) dst[f] = pack_granule<T>(r);
        }
      });
      if (warp == 0 && lane < 16 && (lane < 8 ? lane < head : odd_class < V))
        d[odd_class] = from_f<T>(ex2((odd - m0) * a.c) * ws);
    } else {
      // rows of another alignment
      write_shifted<T>(d, x, V, tid, NT, E, E, [&](const uint4 &g, int, float *r) {
        softmax_granule<T>(g, nm, c2, w2, r);
      });
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
      const uint32_t t = reached_by<T, NT>(K, gmax, NT);
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

}  // namespace logits
}  // namespace tmnn
