// logits_narrow.cuh -- class-logit kernels for rows of up to 256 granules, which
// is 2048 classes (1024 fp32 ones) where rows start on 16-byte boundaries and
// 2041 (1021) elsewhere: a thread a row, and 1 to 32 lanes a row.
#pragma once
#include "logits_row.cuh"

namespace tmnn {
namespace logits {

// ------------------------------------------------------------ a thread a row
// Rows of up to 128 classes (a field has up to 64 outputs): a warp brings 32 of them into
// shared memory as fp32, side by side as they lie in memory, and each thread
// works through one row there.  No lane idles on a row's odd end and nothing
// is reduced over lanes.  Rows of whole quads lie `pitch` apart, an odd number
// of quads, so that the lanes' 16-byte reads meet different banks; other rows
// keep their distance V (odd, or twice an odd number).
//
// 262144 rows of 64 fp32 logits with 4 alternatives take 22 us, 3.6 TB/s (lanes
// side by side: 43 us), of 19 classes, distilled from 4 entries, 16.7 us, 3.0
// TB/s (27 us).  Their 55 and 45 instructions of a warp a row would be 12 and 10
// us of all issue slots, of which half are used: a warp loads, computes and
// stores its 32 rows one after the other, and the images leave room for 24 and
// 40 of 64 warps on an SM (a third and half of them active over the kernel), too
// few to cover each other's waits.
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
  int packed, d_packed; // rows from a 16-byte boundary on that have no gaps, or
                        // whose quads lie on boundaries of their size
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
  // The same of every quad of packed rows `stride` apart: load(its first place in
  // the image, in memory), then use(both, value); four in flight.
  auto each_quad = [&](int end, int stride, auto &&load, auto &&use) {
    const int R = QUADS ? V / 4 : 1;  // quads a row
    int r = lane / R, c = lane - r * R;
    const int dr = 32 / R, dc = 32 - dr * R;
    for (int i0 = lane; i0 - lane < end; i0 += 128) {
      int at[4], from[4];
      decltype(load(0, 0)) v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at[i] = QUADS ? r * P + c * 4 : (i0 + 32 * i) * 4;
        from[i] = QUADS ? r * stride + c * 4 : at[i];
        if (i0 + 32 * i < end) v[i] = load(at[i], from[i]);
        if (QUADS) {
          r += dr;
          c += dc;
          if (c >= R) c -= R, ++r;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + 32 * i < end) use(at[i], from[i], v[i]);
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
          quads, (int)a.stride,
          [&](int at, int from) {
            copy16(image + at, x + from);
            return 0;
          },
          [](int, int, int) {});
    } else {
      each_quad(
          quads, (int)a.stride,
          [&](int, int from) { return *reinterpret_cast<const uint2 *>(x + from); },
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
        // loss / T = sum q T (log q - log p) = (sum e T (y - log p)) / sum e
        //            - T log sum e  with e = e^y, y = (teacher - max) / T;
        // the sum is kept in units of 2^8 > K, so that it stays in range.  A
        // class at -inf under an e > 0 makes it infinite; in a row without a
        // distribution (all at -inf) the terms are no numbers.
        const float w = weight * a.t;
        const bool zero = idle || (end.empty && !end.bad);
        float ys = 0.0f, loss = 0.0f;
        // (not unrolled: 262144 rows of 19 classes with 4 entries take 13.8 us,
        // 15.0 as the compiler unrolls it)
#pragma unroll 1
        for (int k = 0; k < K; ++k) {
          const float dy = ey[k] - ym;
          const float e = eid[k] >= 0 ? expf(dy * a.inv_t) : 0.0f;
          ys += e;
          if (e > 0.0f)
            loss += e * (0x1p-8f * entry_gap(end, a.t, dy, mine[eid[k]]));
          if (MODE == kLossGrad) ey[k] = e;
        }
        const float inv_ys = 1.0f / ys;
        p.loss[row] = idle        ? 0.0f
                      : end.bad   ? nan
                      : end.empty ? kInf
                                  : a.t * (loss * (0x1p8f * inv_ys) - a.t * logf(ys));
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
          quads, (int)p.d_stride,
          [&](int at, int) { return *reinterpret_cast<const float4 *>(image + at); },
          [&](int, int to, const float4 &v) {
            if constexpr (sizeof(T) == 4)
              *reinterpret_cast<float4 *>(d + to) = v;
            else
              *reinterpret_cast<uint2 *>(d + to) =
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
// There is no shared memory but for a teacher's entries and the listed
// alternatives, and nothing is read or written twice.
//
// 65536 rows of 1000 bf16 logits: backward 53 us, 4.9 TB/s; distilled from 10
// entries 90 us; with 10 alternatives 96 us, bound by the instructions (1440 of
// a warp a row; 193 us with one search through the row an alternative).  Two
// granules more a lane than 8 cost more registers than they save (rows of 4039
// fp16 logits: 190 us, streamed 144).
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
  // A warp without a row ends here: the last one may be another warp's, which
  // writes it in place.  Lanes of no row in a warp that has one repeat its last.
  if ((blockIdx.x * 4 + warp) * (32 / L) >= a.rows) return;
  const bool on = want < a.rows;
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
  // writes what f(granule, first element, to) gives
  auto write_rows = [&](auto &&f) {
    const int dm = (int)((uintptr_t)d & 15) / (int)sizeof(T);
    if (!on) return;
    uint4 *dst = reinterpret_cast<uint4 *>(d - dm);
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int g = l + L * j, e0 = g * E - mis;
      if (g >= G) continue;
      float r[E];
      f(q[j], e0, r);
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
    __syncwarp();  // every lane has read what the row's lanes now write
    write_rows([&](const uint4 &g, int e, float *r) { b.granule<T>(g, e, a.c, r); });
    return;
  }

  // ---- the teacher's entries, entry l + lanes * i of a row by lane l
  const int K = kTeacher ? p.te.k : 0;
  float *sq = entries + (warp * (32 / L) + lane / L) * K * 3;  // e^(y - max)
  float *sy = sq + K;                                          // y - max, then own d
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
      const float dy = sid[k] >= 0 ? sy[k] - ym : -kInf;
      sy[k] = dy;
      sq[k] = expf(dy * a.inv_t);
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
    // A value (16 bits of it, and more where too many reach it) that K granules of
    // the row reach is a lower bound of its K-th largest logit: the granules that
    // reach it are listed, then their logits above it, which are ranked.  For a
    // few alternatives the loop below is the shorter way.
    bool open = true;  // the row's alternatives are still to be found
    if (p.cap) {
      uint32_t o[NG], t = 0, have = 0;
#pragma unroll
      for (int j = 0; j < NG; ++j) o[j] = order_of(best[j]);
      auto raise = [&](uint32_t up) {  // to `up`, if K granules reach it
        int c = 0;
#pragma unroll
        for (int j = 0; j < NG; ++j) c += o[j] >= up;
        if (L == 32)
          c = __reduce_add_sync(~0u, c);
        else
          for (int i = 1; i < L; i *= 2) c += __shfl_xor_sync(~0u, c, i);
        if (c >= K) {
          t = up;
          have = c;
        }
      };
      for (uint32_t b = 1u << 31; b >= 1u << 16; b >>= 1) raise(t | b);
      if (kLastBit<T> < 1u << 16 && !__all_sync(~0u, hardly_more(have, K))) {
        const uint32_t most = order_of(end.m);
        raise(most);  // many equal ones
        for (uint32_t b = 1u << 15; b >= kLastBit<T>; b >>= 1) {
          if (__all_sync(~0u, t == most || hardly_more(have, K))) break;
          raise(t == most ? most : t | b);
        }
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
          loss += entry_part(end, e / ys,
                             entry_gap(end, a.t, sy[k] - a.t * ln_ys, xv));
        if constexpr (MODE == kLossGrad) {
          float both = 0.0f;  // entries of one class add up
          for (int j = 0; j < K; ++j) both += sid[j] == sid[k] ? sq[j] : 0.0f;
          sy[k] = w * (ex2((xv - end.m) * a.c) / end.s - both * inv_ys);
        }
      }
    loss = group_sum(loss);
    if (l == 0 && on)
      p.loss[row] = idle ? 0.0f : end.bad ? nan : a.t * loss;
    if constexpr (MODE == kLossGrad) {
      const bool zero = idle || (end.empty && !end.bad);
      const float ws = zero ? 0.0f : end.bad ? nan : w / end.s;
      const float m0 = zero ? 0.0f : end.m;
      __syncwarp();  // every lane has read what the row's lanes now write
      const float2 nm = f2(-m0, -m0), c2 = f2(a.c, a.c), w2 = f2(ws, ws);
      write_rows([&](const uint4 &g, int, float *r) {
        softmax_granule<T>(g, nm, c2, w2, r);
        if (zero)
#pragma unroll
          for (int i = 0; i < E; ++i) r[i] = 0.0f;
      });
      __syncwarp();  // an entry's element is written again
      if (on && !zero && !end.bad)
        for (int k = l; k < K; k += L)
          if (sid[k] >= 0) d[sid[k]] = from_f<T>(sy[k]);
    }
  }
}

}  // namespace logits
}  // namespace tmnn
