// attendgrad.hip -- attention over packs, backward.  With p = softmax, D_i = do[i] . o[i] and
// ds_ij = p_ij (do[i] . v[j] - D_i):  dq[i] = scale sum_j ds_ij k[j],  dk[j] = scale sum_i ds_ij q[i],
// dv[j] = sum_i p_ij do[i], the sums of dk and dv over the heads that share the key head as well.
//
// Two kernels compute the scores again instead of one with atomics on dq: five products become seven, and
// every sum has a fixed order.  dq: as the forward, the wave's 32 columns are rows of q.  dk / dv: the
// columns are keys, and the rows of the group's heads stream past.  Both feed their second products from the
// accumulators of the first in place (seqcommon.h, acc_frag); the streamed tiles are read from LDS along
// rows for the first products and along columns for the second.
// Rounding: p and ds are rounded to the inputs' type for the second products, half a step each; sums stay
// in 32 bits.  float16 has few exponents: there ds, and p for dv, are multiplied by a power of two of their column
// (fit_column), and the result by its inverse, both exact.
// Masked places that hold infinities or NaN: as in attend.hip.
// Bound by issue and by the longest rows: 8191 rows in 4 packs, causal, 16 / 4 heads of 64, bf16: dq 165 us, dk and dv
// in four splits of the rows 243 and 14 for their join (f16: 188, 273 and 14), with the matrix units busy in 35 to 40 % of
// the cycles.
#include "attend32.h"

namespace kl {

struct Grad {
  const float2 *ld;    // (lse, D) of each (row, head)
  const int2 *range;   // keys of each row
};

// D and the key ranges: LANES lanes per (row, head), kItems of those a group at once.  (float with heads up to 32: the
// kernel of dq does it, which has do at hand: attend_rays_train 60 + 352 us, now 392.)
constexpr int kItems = 4;
template <typename T, int LANES>
__global__ void __launch_bounds__(256) attend_prep_kernel(Attend a, const T *__restrict__ o, const T *__restrict__ low,
                                                        const T *__restrict__ go, const float *__restrict__ lse,
                                                        float2 *__restrict__ ld, int2 *__restrict__ range) {
  constexpr int E = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  union Piece {
    u32x4 w;
    T v[E];
  };
  const int64_t rows = (int64_t)a.nq * a.kv_heads * a.group;
  const int sub = threadIdx.x % LANES, c = sub * E;
  for (int64_t at0 = ((int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES) * kItems; at0 < rows;
       at0 += (int64_t)gridDim.x * GROUPS * kItems) {
    Piece x[kItems], y[kItems], z[kItems];
    float ls[kItems];
#pragma unroll
    for (int i = 0; i < kItems; i++) {
      x[i].w = y[i].w = z[i].w = u32x4{0, 0, 0, 0};
      ls[i] = 0;
      if (at0 + i < rows && c < a.dim) {
        x[i].w = *reinterpret_cast<const u32x4 *>(o + (at0 + i) * a.dim + c);
        y[i].w = *reinterpret_cast<const u32x4 *>(go + (at0 + i) * a.dim + c);
        if (low) z[i].w = *reinterpret_cast<const u32x4 *>(low + (at0 + i) * a.dim + c);
        ls[i] = lse[at0 + i];
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; i++) {
      float d = 0;
#pragma unroll
      for (int e = 0; e < E; e++) d = fmaf((float)x[i].v[e] + (float)z[i].v[e], (float)y[i].v[e], d);
#pragma unroll
      for (int s = LANES / 2; s > 0; s >>= 1) d += __shfl_xor(d, s);
      if (sub == 0 && at0 + i < rows) ld[at0 + i] = make_float2(ls[i], d);
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.nq; row += (int64_t)gridDim.x * 256) {
    const Range r = key_range(a, (int)row);
    range[row] = make_int2(r.lo, r.hi);
  }
}

// What is rounded to float16 for a second product is first multiplied by a power of two of its column (this lane and the
// other half's; a row of q in dq, a key in dk and dv), `up`, and the product divided by it in the end, both exact.  It
// starts at kMostUp and falls, the sums so far with it, where a column's largest number would pass 2^15: that one
// then lies in [2^11, 2^12), and smaller ones keep their bits down to 2^-25 of it.  So neither overflows, nor do large
// numbers of another row, key or pack cost bits here, nor long packs those of the weights.  (One power for all, from the
// largest |do|: ds overflowed where v is large, and a pack of small gradients lost its bits to one of large ones.  Weights
// as they are: under 2^-14 dv lost bits, at 2^-25 all.  Forward and backward of 8191 rows in 4 packs, causal, 16 / 4
// heads: 611 us with those, 631 now, for heads of 64; 1333 and 1321 for 128; 458 and 492 for 32.)
template <typename T>
constexpr bool kFitted = std::is_same<T, f16_t>::value;
constexpr float kMostUp = 0x1p60f;  // leaves room for sums of 2^31 products of two of the largest float16 numbers

template <int N>
__device__ __forceinline__ void fit_column(f32x16 &x, float &up, f32x16 (&acc)[N]) {
  float top = 0;
#pragma unroll
  for (int r = 0; r < 16; r++) top = fmaxf(top, fabsf(x[r]));
  top = half_max(top);
  const bool over = top * up > 0x1p15f;
  if (__any(over)) {
    // top = m 2^e, m in [0.5, 1).  An infinity stays one.
    const float fit = over && finite(top) ? __builtin_amdgcn_ldexpf(1.f, 12 - __builtin_amdgcn_frexp_expf(top)) : up;
    const float keep = fit / up;
    up = fit;
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][r] *= keep;
    }
  }
#pragma unroll
  for (int r = 0; r < 16; r++) x[r] *= up;
}

template <typename T, int DP>
struct DqTile {
  static constexpr int BN = sizeof(T) == 4 || DP == 128 ? 32 : 64;
};

template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void dq_walk(const Attend &a, const T *__restrict__ k, const T *__restrict__ v, int first,
                                        int end, int2 mine, float2 ld, float &up, int wlo, int whi, int full_lo,
                                        int full_hi, const V8<T> (&qf)[DP / 16], const V8<T> (&gf)[DP / 16], T *ks,
                                        T *vs, uint32_t *bad, f32x16 (&acc)[DP / 32]) {
  constexpr int BN = DqTile<T, DP>::BN;
  constexpr int SIZE = Stage<T, DP, BN>::SIZE;
  using L = Tile<T, DP>;
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  stream<T, DP, BN, CAREFUL>(
      0, end > first ? (end - first + BN - 1) / BN : 0, ks, vs, bad,
      [&](auto &x, auto &y, int t) {
        const int kt = first + t * BN;
        x.load(k, a.k.row, kt, end, a.dim);
        y.load(v, a.v.row, kt, end, a.dim);
      },
      [](int) {},
      [&](int t, int buffer) {
        const int kt = first + t * BN;
        if (kt >= whi || kt + BN <= wlo) return;
        T *kb = ks + buffer * SIZE, *vb = vs + buffer * SIZE;
        const bool whole = !CAREFUL && kt >= full_lo && kt + BN <= full_hi;
#pragma unroll
        for (int b = 0; b < BN / 32; b++) {
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < DP / 16; i++) {
            s = mma(L::row_frag(kb, 32 * b + col, 16 * i + 8 * h), qf[i], s);
            dp = mma(L::row_frag(vb, 32 * b + col, 16 * i + 8 * h), gf[i], dp);
          }
#pragma unroll
          for (int r = 0; r < 16; r++) s[r] = exp2_fast(fmaf(s[r], a.c, -ld.x)) * (dp[r] - ld.y);
          if (!whole) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int key = kt + 32 * b + acc_row(r, h);
              bool in = (key >= mine.x) & (key < mine.y);
              if constexpr (CAREFUL) in = in & !(bad[b] >> acc_row(r, h) & 1);
              s[r] = in ? s[r] : 0.f;
            }
          }
          if constexpr (kFitted<T>) fit_column(s, up, acc);
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const V8<T> ds = acc_frag<T>(s, i);
#pragma unroll
            for (int db = 0; db < DP / 32; db++) acc[db] = mma(L::col_frag(kb, 32 * b + 16 * i, 32 * db), ds, acc[db]);
          }
        }
        if constexpr (CAREFUL) {
          for (int r = 0; r < BN; r++) {
            const int key = kt + r;
            if (!(bad[r / 32] >> (r % 32) & 1) || key >= whi || key < wlo) continue;
            const float t = frag_dot<T, DP>(qf, ks + SIZE, r, h) * a.c;
            const float dp = frag_dot<T, DP>(gf, vs + SIZE, r, h);
            if (key >= mine.x && key < mine.y)
              add_row<T, DP>(acc, exp2_fast(t - ld.x) * (dp - ld.y) * up, ks + SIZE, r, h);
          }
        }
      });
}

struct GradArgs {
  const void *q, *k, *v, *go;
  void *dq, *dk, *dv;
  float *part;  // dk, dv: the splits' sums (NULL without splits)
  const void *out;  // dq, kDirect: what the first kernel takes and writes
  const float *lse;
  float2 *ld;
  int2 *range;
  int *used;        // dq: splits of each tile that have keys
};

// This workgroup's split of the keys [begin, end) of its tile; false: none are left for it, and nobody asks for it.  The
// first leaves the number of those that have some.
__device__ __forceinline__ bool dq_split(const GradArgs &p, int &begin, int &end, int step) {
  const int steps = (end - begin + step - 1) / step, share = (steps + (int)gridDim.y - 1) / (int)gridDim.y;
  if (blockIdx.y == 0 && threadIdx.x == 0)
    p.used[blockIdx.z * gridDim.x + blockIdx.x] = share ? (steps + share - 1) / share : 0;
  take_split(begin, end, blockIdx.y, gridDim.y, step);
  return begin < end;
}

template <typename T, int DP>
struct DqLds {
  static constexpr int N = (kDirect<T, DP> ? 1 : 2) * Stage<T, DP, DqTile<T, DP>::BN>::SIZE;
  alignas(16) T ks[N];
  alignas(16) T vs[N];
  uint32_t bad[2];
  int lo[4], hi[4], redo;
};

// One workgroup's rows.  True: something was not finite, and nothing was stored.
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ bool dq_rows(const Attend &a, const Grad &g, const GradArgs &p, DqLds<T, DP> &lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const Place at_place = place(a, p.part != nullptr);
  const int head = at_place.head, heads = a.kv_heads * a.group, total = a.nq * a.group;  // virtual rows: under 2^31
  const int m = (at_place.tiles - 1 - at_place.tile) * (32 * kWaves<T, DP>) + wave * 32 + col;
  const bool live = m < total;
  const Row at_row = virtual_row(a, live ? m : 0);
  const int row = at_row.row, qhead = head * a.group + at_row.sub;
  const Range none = no_keys();
  const int64_t at = (int64_t)row * heads + qhead;
  int2 mine = make_int2(none.lo, none.hi);
  float2 ld = make_float2(0, 0);
  V8<T> qf[DP / 16], gf[DP / 16];
  const T *qrow = (const T *)p.q + row * a.q.row + qhead * a.q.head, *grow = (const T *)p.go + at * a.dim;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
    qf[i] = global_frag(qrow, live, 16 * i + 8 * h, a.dim);
    gf[i] = global_frag(grow, live, 16 * i + 8 * h, a.dim);
  }
  if constexpr (kDirect<T, DP>) {  // the first kernel's work, where do is in registers anyway
    const T *orow = (const T *)p.out + at * a.dim;
    float sum[2] = {0, 0};  // in that kernel's order: pieces of four, then pieces 4, 2 and 1 apart
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
      const V8<T> x = global_frag(orow, live, 16 * i + 8 * h, a.dim);
#pragma unroll
      for (int b = 0; b < 2; b++) {
        float d = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) d = fmaf(x[4 * b + e], gf[i][4 * b + e], d);
        sum[b] += d;
      }
    }
    const float d = half_sum(sum[0]) + half_sum(sum[1]);
    if (live) {
      const Range r = key_range(a, row);
      mine = make_int2(r.lo, r.hi);
      ld = make_float2(p.lse[at], d);
      if (h == 0 && blockIdx.y == 0) {
        p.ld[at] = ld;
        if (qhead == 0) p.range[row] = mine;
      }
    }
  } else if (live) {
    mine = g.range[row];
    ld = g.ld[at];
  }
  const int wlo = min_over(mine.x), whi = max_over(mine.y);
  const int full_lo = max_over(mine.x), full_hi = min_over(mine.y);
  const T *kh = (const T *)p.k + head * a.k.head, *vh = (const T *)p.v + head * a.v.head;
  f32x16 acc[DP / 32] = {};
  float up = kFitted<T> ? kMostUp : 1.f;
  if constexpr (kDirect<T, DP>) {
    int begin = wlo, end = whi;
    if (begin >= end) begin = end = 0;
    if (p.part && !dq_split(p, begin, end, DqTile<T, DP>::BN)) return false;
    dq_walk32<DP, CAREFUL>(a, kh, vh, begin, end, mine, ld, full_lo, full_hi, qf, gf, lds.ks, lds.vs, acc);
    if (!CAREFUL && __any(!all_finite(acc))) return true;
  } else {
    if (lane == 0) {
      lds.lo[wave] = wlo;
      lds.hi[wave] = whi;
    }
    if (CAREFUL) __syncthreads();  // everyone has read lds.redo
    if (threadIdx.x == 0) lds.redo = 0;
    __syncthreads();
    int begin = uniform(min(min(lds.lo[0], lds.lo[1]), min(lds.lo[2], lds.lo[3])));
    int end = uniform(max(max(lds.hi[0], lds.hi[1]), max(lds.hi[2], lds.hi[3])));
    if (begin >= end) begin = end = 0;
    if (p.part && !dq_split(p, begin, end, DqTile<T, DP>::BN)) return false;
    dq_walk<T, DP, CAREFUL>(a, kh, vh, begin, end, mine, ld, up, wlo, whi, full_lo, full_hi, qf, gf, lds.ks, lds.vs,
                            lds.bad, acc);
    if (!CAREFUL) {
      if (!all_finite(acc)) lds.redo = 1;
      __syncthreads();
      if (lds.redo) return true;
    }
  }
  if (!live) return false;
  if (p.part) {
    const int64_t all = (int64_t)a.nq * heads;
    store_cols<float, DP>(p.part + (blockIdx.y * all + at) * a.dim, acc, a.scale / up, h, a.dim);
  } else {
    store_cols<T, DP>((T *)p.dq + at * a.dim, acc, a.scale / up, h, a.dim);
  }
  return false;
}

// grid: places(tiles, splits of the keys)
template <typename T, int DP>
__global__ void __launch_bounds__((64 * kWaves<T, DP>), (kDirect<T, DP> ? 3 : sizeof(T) == 4 && DP == 128 ? 1 : 2))
    attend_dq_kernel(Attend a, Grad g, GradArgs p) {
  __shared__ DqLds<T, DP> lds;
  if (dq_rows<T, DP, false>(a, g, p, lds)) dq_rows<T, DP, true>(a, g, p, lds);
}

// The splits of dq added in their order: four elements a thread.
template <typename T>
__global__ void __launch_bounds__(256) attend_dq_join_kernel(Attend a, int tile_rows, int tiles, const int *__restrict__ used,
                                                           const float *__restrict__ part, T *__restrict__ dq) {
  const int64_t all = (int64_t)a.nq * a.kv_heads * a.group * a.dim, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= all) return;
  const int heads = a.kv_heads * a.group;
  const int64_t line = at / a.dim;
  const int row = (int)(line / heads), qhead = (int)(line % heads);
  const int tile = tiles - 1 - (row * a.group + qhead % a.group) / tile_rows;  // as the workgroups were numbered
  const int splits = used[tile * a.kv_heads + qhead / a.group];
  f32x4 sum = {};
#pragma unroll 4
  for (int s = 0; s < splits; s++) sum += *reinterpret_cast<const f32x4 *>(part + s * all + at);
  *reinterpret_cast<V4<T> *>(dq + at) = __builtin_convertvector(sum, V4<T>);
}

template <typename T, int DP>
struct DkvTile {
  static constexpr int KEYS = 32 * kWaves<T, DP>;
  static constexpr int BQ = sizeof(T) == 4 || DP == 128 ? 32 : 64;  // virtual rows per step
};

template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void dkv_walk(const Attend &a, const Grad &g, const T *__restrict__ q, Heads gst,
                                         const T *__restrict__ go, int head, int begin, int end, Range rows,
                                         int tiles, int key0, float &up_k, float &up_v,
                                         const V8<T> (&kf)[DP / 16], const V8<T> (&vf)[DP / 16], T *qs, T *os,
                                         float2 *s_ld, int2 *s_range, uint32_t *bad, f32x16 (&dk)[DP / 32],
                                         f32x16 (&dv)[DP / 32]) {
  constexpr int BQ = DkvTile<T, DP>::BQ;
  constexpr int SIZE = Stage<T, DP, BQ>::SIZE;
  using L = Tile<T, DP>;
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int heads = a.kv_heads * a.group, key = key0 + col;
  const Range none = no_keys();
  float2 ld = make_float2(0, 0);
  int2 range = make_int2(none.lo, none.hi);
  stream<T, DP, BQ, CAREFUL>(
      begin, end, qs, os, bad,
      [&](auto &x, auto &y, int t) {
        const int sub = t / tiles, row0 = rows.lo + (t - sub * tiles) * BQ;
        x.load(q + sub * a.q.head, a.q.row, row0, rows.hi, a.dim);
        y.load(go + sub * gst.head, gst.row, row0, rows.hi, a.dim);
        if (threadIdx.x < BQ) {
          const int row = row0 + (int)threadIdx.x;
          const bool live = row < rows.hi;
          ld = live ? g.ld[(int64_t)row * heads + head * a.group + sub] : make_float2(0, 0);
          range = live ? g.range[row] : make_int2(none.lo, none.hi);
        }
      },
      [&](int buffer) {
        if (threadIdx.x < BQ) {
          s_ld[buffer * BQ + threadIdx.x] = ld;
          s_range[buffer * BQ + threadIdx.x] = range;
        }
      },
      [&](int, int buffer) {
        const int slot = buffer * BQ;
        const int2 mine = s_range[slot + lane % BQ];
        if (!__any(mine.x < key0 + 32 && mine.y > key0)) return;
        const bool whole = !CAREFUL && __all(mine.x <= key0 && mine.y >= key0 + 32);
        T *qb = qs + buffer * SIZE, *ob = os + buffer * SIZE;
#pragma unroll
        for (int b = 0; b < BQ / 32; b++) {
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < DP / 16; i++) {
            s = mma(L::row_frag(qb, 32 * b + col, 16 * i + 8 * h), kf[i], s);
            dp = mma(L::row_frag(ob, 32 * b + col, 16 * i + 8 * h), vf[i], dp);
          }
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const float2 x = s_ld[slot + 32 * b + acc_row(r, h)];
            s[r] = exp2_fast(fmaf(s[r], a.c, -x.x));
            dp[r] = s[r] * (dp[r] - x.y);
          }
          if (!whole) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int2 kr = s_range[slot + 32 * b + acc_row(r, h)];
              bool in = (key >= kr.x) & (key < kr.y);
              if constexpr (CAREFUL) in = in & !(bad[b] >> acc_row(r, h) & 1);
              s[r] = in ? s[r] : 0.f;
              dp[r] = in ? dp[r] : 0.f;
            }
          }
          if constexpr (kFitted<T>) {
            fit_column(dp, up_k, dk);
            fit_column(s, up_v, dv);
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const V8<T> p = acc_frag<T>(s, i), ds = acc_frag<T>(dp, i);
#pragma unroll
            for (int db = 0; db < DP / 32; db++) {
              dv[db] = mma(L::col_frag(ob, 32 * b + 16 * i, 32 * db), p, dv[db]);
              dk[db] = mma(L::col_frag(qb, 32 * b + 16 * i, 32 * db), ds, dk[db]);
            }
          }
        }
        if constexpr (CAREFUL) {
          for (int r = 0; r < BQ; r++) {
            const int2 kr = s_range[slot + r];
            if (!(bad[r / 32] >> (r % 32) & 1) || kr.x >= key0 + 32 || kr.y <= key0) continue;
            const float2 x = s_ld[slot + r];
            const float t = frag_dot<T, DP>(kf, qs + SIZE, r, h) * a.c, dpx = frag_dot<T, DP>(vf, os + SIZE, r, h);
            if (key >= kr.x && key < kr.y) {
              const float p = exp2_fast(t - x.x);
              add_row<T, DP>(dv, p * up_v, os + SIZE, r, h);
              add_row<T, DP>(dk, p * (dpx - x.y) * up_k, qs + SIZE, r, h);
            }
          }
        }
      });
}

// The query rows that see any of keys [j0, j1).  They stream past as steps, the rows of the group's first head,
// then of its second, ...
__device__ __forceinline__ Range row_range(const Attend &a, int j0, int j1) {
  const int first = a.kid[j0], last = a.kid[j1 - 1];
  if (last < 0) return {0, 0};
  int r0 = a.qstart[min(max(first, 0), a.nq)];
  const int r1 = a.qstart[min(last + 1, a.nq)];
  if (a.causal && first >= 0) {
    const int ke = a.kstart[min(first + 1, a.nk)], qe = a.qstart[min(first + 1, a.nq)];
    r0 = max(r0, j0 - ke + qe);
  }
  return {min(r0, r1), r1};
}

template <typename T, int DP>
struct DkvLds {
  static constexpr int BQ = DkvTile<T, DP>::BQ, N = (kDirect<T, DP> ? 1 : 2) * Stage<T, DP, BQ>::SIZE;
  alignas(16) T qs[N];
  alignas(16) T os[N];
  RowSums rows[32];                 // kDirect
  float2 ld[2 * BQ];
  int2 range[2 * BQ];
  uint32_t bad[2];
  int redo;
};

// One workgroup's keys.  True: something was not finite, and nothing was stored.
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ bool dkv_keys(const Attend &a, const Grad &g, const GradArgs &p, DkvLds<T, DP> &lds) {
  constexpr int BQ = DkvTile<T, DP>::BQ, KEYS = DkvTile<T, DP>::KEYS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const Place at_place = place(a, p.part != nullptr);
  const int head = at_place.head, heads = a.kv_heads * a.group;
  const int j0 = at_place.tile * KEYS, key0 = j0 + wave * 32, key = key0 + col;
  const bool live = key < a.nk;
  Range rows = row_range(a, j0, min(j0 + KEYS, a.nk));
  rows = {uniform(rows.lo), uniform(rows.hi)};
  const int tiles = max(1, (rows.hi - rows.lo + BQ - 1) / BQ);
  int begin = 0, end = rows.hi > rows.lo ? tiles * a.group : 0;
  if (p.part) {
    const int share = (end + (int)gridDim.y - 1) / (int)gridDim.y;
    begin = min(end, share * (int)blockIdx.y);
    end = min(end, begin + share);
    if (begin >= end) return false;  // the join does not ask for it
  }
  const T *qh = (const T *)p.q + (int64_t)head * a.group * a.q.head;
  const Heads gst = {(int64_t)heads * a.dim, a.dim};
  const T *gh = (const T *)p.go + (int64_t)head * a.group * a.dim;
  V8<T> kf[DP / 16], vf[DP / 16];
  const T *krow = (const T *)p.k + (live ? key : 0) * a.k.row + head * a.k.head;
  const T *vrow = (const T *)p.v + (live ? key : 0) * a.v.row + head * a.v.head;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
    kf[i] = global_frag(krow, live, 16 * i + 8 * h, a.dim);
    vf[i] = global_frag(vrow, live, 16 * i + 8 * h, a.dim);
  }
  f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
  float up_k = kFitted<T> ? kMostUp : 1.f, up_v = up_k;
  if constexpr (kDirect<T, DP>) {
    const float2 *ld = g.ld + head * a.group;
    dkv_walk32<DP, CAREFUL>(a, qh, gst, gh, ld, heads, g.range, begin, end, rows, tiles, key0, kf, vf, lds.qs, lds.os,
                            lds.rows, dk, dv);
    if (!CAREFUL && __any(!(all_finite(dk) && all_finite(dv)))) return true;
  } else {
    if (CAREFUL) __syncthreads();  // everyone has read lds.redo
    if (threadIdx.x == 0) lds.redo = 0;
    __syncthreads();
    dkv_walk<T, DP, CAREFUL>(a, g, qh, gst, gh, head, begin, end, rows, tiles, key0, up_k, up_v, kf, vf, lds.qs, lds.os,
                             lds.ld, lds.range, lds.bad, dk, dv);
    if (!CAREFUL) {
      if (!(all_finite(dk) && all_finite(dv))) lds.redo = 1;
      __syncthreads();
      if (lds.redo) return true;
    }
  }
  if (!live) return false;
  const int64_t at = ((int64_t)key * a.kv_heads + head) * a.dim;
  if (p.part) {
    const int64_t all = (int64_t)a.nk * a.kv_heads * a.dim;
    store_cols<float, DP>(p.part + 2 * blockIdx.y * all + at, dk, a.scale / up_k, h, a.dim);
    store_cols<float, DP>(p.part + (2 * blockIdx.y + 1) * all + at, dv, 1.f / up_v, h, a.dim);
    return false;
  }
  store_cols<T, DP>((T *)p.dk + at, dk, a.scale / up_k, h, a.dim);
  store_cols<T, DP>((T *)p.dv + at, dv, 1.f / up_v, h, a.dim);
  return false;
}

// grid: places(tiles of keys, splits of the rows)
template <typename T, int DP>
__global__ void __launch_bounds__((64 * kWaves<T, DP>), (DP == 128 ? 1 : kDirect<T, DP> ? 3 : 2))
    attend_dkv_kernel(Attend a, Grad g, GradArgs p) {
  __shared__ DkvLds<T, DP> lds;
  if (dkv_keys<T, DP, false>(a, g, p, lds)) dkv_keys<T, DP, true>(a, g, p, lds);
}

// The splits of dk and dv added in their order: four elements a thread.
template <typename T>
__global__ void __launch_bounds__(256) attend_dkv_join_kernel(Attend a, int splits, int step,
                                                            int keys, const float *__restrict__ part, T *__restrict__ dk,
                                                            T *__restrict__ dv) {
  const int64_t all = (int64_t)a.nk * a.kv_heads * a.dim;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= all) return;
  const int j0 = (int)(at / ((int64_t)a.kv_heads * a.dim)) / keys * keys;
  const Range rows = row_range(a, j0, min(j0 + keys, a.nk));
  const int steps = rows.hi > rows.lo ? (rows.hi - rows.lo + step - 1) / step * a.group : 0;
  const int share = max(1, (steps + splits - 1) / splits), used = (steps + share - 1) / share;
  f32x4 k = {}, v = {};
#pragma unroll 4
  for (int s = 0; s < used; s++) {
    k += *reinterpret_cast<const f32x4 *>(part + 2 * s * all + at);
    v += *reinterpret_cast<const f32x4 *>(part + (2 * s + 1) * all + at);
  }
  *reinterpret_cast<V4<T> *>(dk + at) = __builtin_convertvector(k, V4<T>);
  *reinterpret_cast<V4<T> *>(dv + at) = __builtin_convertvector(v, V4<T>);
}

// Splits of the keys that a tile of rows walks for dq: two waves for each of the 1024 SIMDs (forward and backward of
// 2264 rows in 4 packs, 3 heads of 32 that share one key head, float: 171 us without, 111 with)
static int dq_splits(kl_dtype dtype, int64_t nq, int64_t nk, int kv_heads, int group, int dim) {
  const int waves = is_direct(dtype, dim) ? 1 : 4, step = dtype == KL_F32 ? 32 : 64;
  const int64_t all = cdiv(nq * group, 32 * waves) * kv_heads * waves;
  return (int)std::max<int64_t>(1, std::min<int64_t>({2048 / std::max<int64_t>(all, 1), cdiv(nk, 2 * step), 16}));
}

// Splits of the rows that stream past a tile of keys: up to four waves for each of the 1024 SIMDs, so that tiles of long
// packs do not come last; two where heads are over 64, whose registers let only one run and whose partial sums are long
// (one pack of 4935 rows, 2 heads of 80, f16, training: 219 us with four, 195 with two).
static int dkv_splits(kl_dtype dtype, int64_t nq, int64_t nk, int kv_heads, int group, int dim) {
  const int waves = is_direct(dtype, dim) ? 1 : 4, step = dtype == KL_F32 ? 32 : 64;
  const int64_t all = cdiv(nk, 32 * waves) * kv_heads * waves;
  const int64_t most = dim > 64 ? 2048 : 4096;
  return (int)std::max<int64_t>(
      1, std::min<int64_t>({most / std::max<int64_t>(all, 1), cdiv(nq, 2 * step) * group, 16}));
}

// lanes per (row, head) of the first kernel: 16 bytes each
static int prep_lanes(kl_dtype dtype, int dim) { return dim * (dtype == KL_F32 ? 4 : 2) / 16; }

// Its workgroups: one per kItems * groups (row, head)s
static unsigned prep_blocks(kl_dtype dtype, int64_t num_q, int heads, int dim) {
  const int lanes = prep_lanes(dtype, dim), pow2 = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
  return (unsigned)std::max<int64_t>(1, cdiv(num_q * heads, (int64_t)kItems * (256 / pow2)));
}

template <typename F>
static int with_prep_lanes(int lanes, F f) {
  if (lanes <= 4) return f(std::integral_constant<int, 4>());
  if (lanes <= 8) return f(std::integral_constant<int, 8>());
  if (lanes <= 16) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}

template <typename T, int DP>
static int attend_backward(const Attend &a, const Grad &g, const void *q, const void *k, const void *v, const void *go,
                           void *dq, void *dk, void *dv, float *part, const void *out, const float *lse, hipStream_t st) {
  if (a.nq > 0 && dq) {
    const int splits = dq_splits(sizeof(T) == 4 ? KL_F32 : KL_F16, a.nq, a.nk, a.kv_heads, a.group, a.dim);
    constexpr int ROWS = 32 * kWaves<T, DP>;
    const int64_t tiles = cdiv((int64_t)a.nq * a.group, ROWS), all = (int64_t)a.nq * a.kv_heads * a.group * a.dim;
    int *used = (int *)(part + splits * all);
    hipLaunchKernelGGL((attend_dq_kernel<T, DP>), places(a, tiles, splits), dim3(64 * kWaves<T, DP>), 0, st, a, g,
                       GradArgs{q, k, v, go, dq, nullptr, nullptr, splits > 1 ? part : nullptr, out, lse,
                                (float2 *)g.ld, (int2 *)g.range, used});
    KL_CHECK_LAUNCH();
    if (splits > 1) {
      hipLaunchKernelGGL(attend_dq_join_kernel<T>, dim3((unsigned)cdiv(all / 4, 256)), dim3(256), 0, st, a, ROWS,
                         (int)tiles, used, part, (T *)dq);
      KL_CHECK_LAUNCH();
    }
  }
  if (a.nk > 0 && dk) {
    constexpr int KEYS = DkvTile<T, DP>::KEYS, step = DkvTile<T, DP>::BQ;
    const int splits = dkv_splits(sizeof(T) == 4 ? KL_F32 : KL_F16, a.nq, a.nk, a.kv_heads, a.group, a.dim);
    hipLaunchKernelGGL((attend_dkv_kernel<T, DP>), places(a, cdiv(a.nk, KEYS), splits), dim3(64 * kWaves<T, DP>), 0, st,
                       a, g,
                       GradArgs{q, k, v, go, nullptr, dk, dv, splits > 1 ? part : nullptr, nullptr, nullptr, nullptr,
                                nullptr, nullptr});
    KL_CHECK_LAUNCH();
    if (splits > 1) {
      const int64_t pieces = (int64_t)a.nk * a.kv_heads * a.dim / 4;
      hipLaunchKernelGGL(attend_dkv_join_kernel<T>, dim3((unsigned)cdiv(pieces, 256)), dim3(256), 0, st, a, splits, step,
                         KEYS, part, (T *)dk, (T *)dv);
      KL_CHECK_LAUNCH();
    }
  }
  return KL_OK;
}

}  // namespace kl

using namespace kl;

extern "C" size_t kl_pack_attention_bwd_workspace_bytes(kl_dtype dtype, int64_t num_q, int64_t num_k, int heads,
                                                        int kv_heads, int dim) {
  if (num_q < 0 || num_k < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0) return 256;
  const int splits = dkv_splits(dtype, num_q, num_k, kv_heads, heads / kv_heads, dim);
  const int dq = dq_splits(dtype, num_q, num_k, kv_heads, heads / kv_heads, dim);
  return al256((size_t)num_q * heads * 8) + al256((size_t)num_q * 8) +
         std::max(splits > 1 ? (size_t)2 * splits * num_k * kv_heads * dim * 4 : 0,
                  dq > 1 ? (size_t)dq * num_q * heads * dim * 4 + (size_t)cdiv(num_q * (heads / kv_heads), 32) * kv_heads * 4 : 0);
}

extern "C" int kl_pack_attention_backward(kl_dtype dtype, int64_t num_q, int64_t num_k, int heads, int kv_heads,
                                          int dim, const void *grad_out, const void *q, const void *k, const void *v,
                                          const int64_t *strides_host, const int32_t *q_ids, const int32_t *q_starts,
                                          const int32_t *k_ids, const int32_t *k_starts, const void *out,
                                          const void *out_low, const float *lse, float scale, int causal, void *grad_q,
                                          void *grad_k, void *grad_v, void *ws, size_t ws_bytes, kl_stream stream) {
  Attend a;
  KL_CHECK_RC(fill_attend(a, "pack_attention", dtype, num_q, num_k, heads, kv_heads, dim, q, k, v, strides_host, q_ids,
                          q_starts, k_ids, k_starts, scale, causal));
  KL_REQUIRE(ws_bytes >= kl_pack_attention_bwd_workspace_bytes(dtype, num_q, num_k, heads, kv_heads, dim),
             "pack_attention: the workspace is too small");
  KL_REQUIRE((grad_k == nullptr) == (grad_v == nullptr), "pack_attention: grad_k and grad_v go together");
  float2 *ld = (float2 *)ws;
  int2 *range = (int2 *)((char *)ws + al256((size_t)num_q * heads * 8));
  float *part = (float *)((char *)range + al256((size_t)num_q * 8));
  const Grad g = {ld, range};
  return with_type(dtype, "pack_attention", [&](auto t) -> int {
    using T = decltype(t);
    if (num_q > 0 && !(is_direct(dtype, dim) && grad_q)) {
      KL_CHECK_RC(with_prep_lanes(prep_lanes(dtype, dim), [&](auto lanes) -> int {
        hipLaunchKernelGGL((attend_prep_kernel<T, decltype(lanes)::value>),
                           dim3(prep_blocks(dtype, num_q, heads, dim)), dim3(256), 0, S(stream), a, (const T *)out,
                           sizeof(T) == 2 ? (const T *)out_low : (const T *)nullptr, (const T *)grad_out, lse, ld, range);
        KL_CHECK_LAUNCH();
        return KL_OK;
      }));
    }
    return with_dim(dim, [&](auto dp) {
      return attend_backward<T, decltype(dp)::value>(a, g, q, k, v, grad_out, grad_q, grad_k, grad_v, part, out, lse,
                                                     S(stream));
    });
  });
}
