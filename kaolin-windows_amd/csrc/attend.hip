// attend.hip -- attention over packs, forward: o[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j] over the
// keys j of row i's pack, with grouped heads (attend.h).
//
// One workgroup of four waves takes 128 virtual rows of one key head and walks the keys that any of them sees, a
// tile at a time (float with heads up to 32: attend32.h), keeping the running maximum and sum of the softmax in 32
// bits.  Scores are computed transposed, S^T = K Q^T, so a lane holds one row's scores: the softmax is lane-local but
// for one exchange with the other half, and the weights are the second product's operand (O^T = V^T P^T) where
// they lie, without a trip through LDS (seqcommon.h, acc_frag).
// Bound by issue where rows are many: 16,385 rows in 6 packs, causal, 32 / 8 heads of 128, bf16: 526 us a call among others,
// 819 TFLOP/s (565 to 614 us a kernel under a profiler, which lets each end before the next), with the matrix units busy
// in 41 % of the cycles, the vector units in 43 % and LDS in 31 %, without bank conflicts.
// Bound by memory where they are few: one row for each of 96 sequences (205,153 keys of 8 heads of 128, f16, 842 MB):
// 175 us, 4.8 TB/s, and 5 us for the join.
// low (training, 16-bit types): what the rounding of o left out, so that the backward's sums over do . o,
// which cancel against other terms, have o to twice its bits.
// Rounding: weights, at most 2^kLag (float16: times 2^kLift), are rounded to the inputs' type for the second product (each
// off by half a step at most, whatever their size; float stays float); the sum they are divided by is taken before the
// rounding, in 32 bits.
//
// A key outside a row's range has weight 0, but 0 * inf and 0 * NaN would still reach the row through the
// product.  Nothing in the main walk guards against that: if an accumulator ends up not finite, the
// workgroup walks its keys again with the rows of k and v that hold such values taken out of the tiles and
// added one by one to just the rows that see them.
#include "attend32.h"

namespace kl {

template <typename T, int DP>
struct FwdTile {
  static constexpr int BM = 32 * kWaves<T, DP>;                  // virtual rows
  static constexpr int BN = sizeof(T) == 4 ? 32 : 64;    // keys
};

template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void fwd_walk(const Attend &a, const T *__restrict__ k, const T *__restrict__ v, int first,
                                         int end, Range mine, int wlo, int whi, int full_lo, int full_hi,
                                         const V8<T> (&qf)[DP / 16], T *ks, T *vs, uint32_t *bad,
                                         f32x16 (&acc)[DP / 32], RowState &st) {
  constexpr int BN = FwdTile<T, DP>::BN;
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
        f32x16 s[BN / 32];
#pragma unroll
        for (int b = 0; b < BN / 32; b++) s[b] = f32x16{};
#pragma unroll
        for (int i = 0; i < DP / 16; i++) {
#pragma unroll
          for (int b = 0; b < BN / 32; b++) s[b] = mma(L::row_frag(kb, 32 * b + col, 16 * i + 8 * h), qf[i], s[b]);
        }
        if (CAREFUL || kt < full_lo || kt + BN > full_hi) {
#pragma unroll
          for (int b = 0; b < BN / 32; b++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
              const int key = kt + 32 * b + acc_row(r, h);
              bool in = (key >= mine.lo) & (key < mine.hi);
              if constexpr (CAREFUL) in = in & !(bad[b] >> acc_row(r, h) & 1);
              s[b][r] = in ? s[b][r] : -INFINITY;
            }
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < BN / 32; b++) {
#pragma unroll
          for (int r = 0; r < 16; r++) top = fmaxf(top, s[b][r]);
        }
        top = half_max(top) * a.c;
        if (__any(top > st.m + kLag)) rescale(st, fmaxf(st.m, top), acc);
        const float base = st.base() - kLift<T>;
#pragma unroll
        for (int b = 0; b < BN / 32; b++) {
#pragma unroll
          for (int r = 0; r < 16; r++) {
            s[b][r] = exp2_fast(fmaf(s[b][r], a.c, -base));
            st.l += s[b][r];
          }
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const V8<T> p = acc_frag<T>(s[b], i);
#pragma unroll
            for (int db = 0; db < DP / 32; db++) acc[db] = mma(L::col_frag(vb, 32 * b + 16 * i, 32 * db), p, acc[db]);
          }
        }
        if constexpr (CAREFUL) {
          for (int r = 0; r < BN; r++) {
            const int key = kt + r;
            if (!(bad[r / 32] >> (r % 32) & 1) || key >= whi || key < wlo) continue;
            const float t = frag_dot<T, DP>(qf, ks + SIZE, r, h) * a.c;
            if (key >= mine.lo && key < mine.hi) {
              rescale(st, fmaxf(st.m, t), acc);
              const float p = exp2_fast(t - (st.base() - kLift<T>));
              st.l += h == 0 ? p : 0.f;
              add_row<T, DP>(acc, p, vs + SIZE, r, h);
            }
          }
        }
      });
}

// What a workgroup keeps in LDS
template <typename T, int DP>
struct FwdLds {
  static constexpr int BN = FwdTile<T, DP>::BN;
  alignas(16) T ks[(kDirect<T, DP> ? 1 : 2) * Stage<T, DP, BN>::SIZE];
  alignas(16) T vs[kDirect<T, DP> ? 1 : 2 * Stage<T, DP, BN>::SIZE];
  uint32_t bad[2];
  int lo[4], hi[4], redo;
};

struct FwdArgs {
  const void *q, *k, *v;
  void *o, *low;
  float *lse, *part;  // part, stat: the splits' unfinished sums (NULL without splits)
  float2 *stat;
};

// One workgroup's rows.  True: something was not finite, and nothing was stored.
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ bool fwd_rows(const Attend &a, const FwdArgs &p, FwdLds<T, DP> &lds) {
  constexpr int BM = FwdTile<T, DP>::BM, BN = FwdTile<T, DP>::BN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5, col = lane & 31;
  const Place at_place = place(a, p.part != nullptr);
  const int head = at_place.head, total = a.nq * a.group;  // virtual rows: under 2^31
  const int m = (at_place.tiles - 1 - at_place.tile) * BM + wave * 32 + col;  // the last rows see most keys
  const bool live = m < total;
  const Row at_row = virtual_row(a, live ? m : 0);
  const int row = at_row.row, qhead = head * a.group + at_row.sub;
  const Range mine = live ? key_range(a, row) : no_keys();
  const int wlo = min_over(mine.lo), whi = max_over(mine.hi);
  const int full_lo = max_over(mine.lo), full_hi = min_over(mine.hi);
  V8<T> qf[DP / 16];
  const T *qrow = (const T *)p.q + row * a.q.row + qhead * a.q.head;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) qf[i] = global_frag(qrow, live, 16 * i + 8 * h, a.dim);
  const T *kh = (const T *)p.k + head * a.k.head, *vh = (const T *)p.v + head * a.v.head;
  f32x16 acc[DP / 32] = {};
  RowState st;
  if constexpr (kDirect<T, DP>) {
    int begin = wlo, end = whi;
    if (begin >= end) begin = end = 0;
    if (p.part) take_split(begin, end, blockIdx.y, gridDim.y, BN);
    fwd_walk32<DP, CAREFUL>(a, kh, vh, begin, end, mine, full_lo, full_hi, qf, lds.ks, acc, st);
    if (!CAREFUL && __any(!(all_finite(acc) && finite(st.l)))) return true;
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
    if (p.part) take_split(begin, end, blockIdx.y, gridDim.y, BN);
    fwd_walk<T, DP, CAREFUL>(a, kh, vh, begin, end, mine, wlo, whi, full_lo, full_hi, qf, lds.ks, lds.vs, lds.bad, acc,
                             st);
    if (!CAREFUL) {
      if (!(all_finite(acc) && finite(st.l))) lds.redo = 1;
      __syncthreads();
      if (lds.redo) return true;
    }
  }
  const float l = half_sum(st.l);
  if (!live) return false;
  if (p.part) {
    const int64_t at = ((int64_t)blockIdx.y * a.kv_heads + head) * total + m;
    if (h == 0) p.stat[at] = make_float2(st.m, l);
    if (st.m != -INFINITY || l != 0) store_cols<float, DP>(p.part + at * a.dim, acc, 1.f, h, a.dim);
    return false;
  }
  const int64_t at = (int64_t)row * a.kv_heads * a.group + qhead;
  const bool blind = mine.lo >= mine.hi;   // a row that sees no key: 0; one whose scores are all -inf: NaN
  const float w = blind ? 0.f : 1.f / l;
  store_cols<T, DP>((T *)p.o + at * a.dim, acc, w, h, a.dim);
  if constexpr (sizeof(T) == 2) {
    if (p.low) {
#pragma unroll
      for (int db = 0; db < DP / 32; db++) {
#pragma unroll
        for (int r = 0; r < 16; r++) acc[db][r] = acc[db][r] * w - (float)(T)(acc[db][r] * w);
      }
      store_cols<T, DP>((T *)p.low + at * a.dim, acc, 1.f, h, a.dim);
    }
  }
  if (p.lse && h == 0) p.lse[at] = blind ? 0.f : st.m - kLift<T> + log2_fast(l);
  return false;
}

// grid: places(tiles, splits)
template <typename T, int DP>
__global__ void __launch_bounds__((64 * kWaves<T, DP>), (kDirect<T, DP> ? 3 : sizeof(T) == 4 && DP == 128 ? 1 : 2))
    attend_fwd_kernel(Attend a, FwdArgs p) {
  __shared__ FwdLds<T, DP> lds;
  if (fwd_rows<T, DP, false>(a, p, lds)) fwd_rows<T, DP, true>(a, p, lds);
}

// The splits of one (key head, virtual row) joined: `lanes` threads of eight elements (a power of two), and
// `shares` of them that take every shares-th split, for each of 256 / (lanes * shares) rows.  Every share has sums of
// its own maximum; they are joined two by two, in an order that the sizes alone give.
constexpr int kMaxSplits = 256, kJoinEach = kMaxSplits * 16 / 256;  // splits of a share: 16 lanes, 16 shares
template <typename T>
__global__ void __launch_bounds__(256) attend_join_kernel(Attend a, int splits, int lanes, int shares,
                                                        const float *__restrict__ part, const float2 *__restrict__ stat,
                                                        T *__restrict__ o, T *__restrict__ low,
                                                        float *__restrict__ lse) {
  __shared__ float2 s_stat[64];
  __shared__ float s_sum[64 * 8];
  const int64_t total = (int64_t)a.nq * a.group, rows = total * a.kv_heads;
  const int per = lanes * shares, here = 256 / per;
  const int mine = threadIdx.x / per, lane = threadIdx.x % lanes, share = threadIdx.x / lanes % shares;
  const int64_t at = (int64_t)blockIdx.x * here + mine;
  const int d = lane * 8;
  const bool live = at < rows;
  float2 x[kJoinEach];
  float top = -INFINITY, l = 0;
#pragma unroll
  for (int i = 0; i < kJoinEach; i++) {
    const int s = share + i * shares;
    x[i] = i * shares < splits && live && s < splits ? stat[s * rows + at] : make_float2(-INFINITY, 0);
    top = fmaxf(top, x[i].x);
  }
  f32x8 sum = {};
  constexpr int kAhead = 4;  // splits whose loads are in flight together
#pragma unroll
  for (int i0 = 0; i0 < kJoinEach; i0 += kAhead) {
    if (i0 * shares >= splits) break;
    f32x4 u0[kAhead], u1[kAhead];
    bool full[kAhead];  // the row has keys in this split
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int i = i0 + j;
      full[j] = x[i].x != -INFINITY || x[i].y != 0;
      u0[j] = u1[j] = f32x4{0, 0, 0, 0};
      if (full[j] && d < a.dim) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(part + ((share + i * shares) * rows + at) * a.dim + d);
        u0[j] = p[0];
        u1[j] = p[1];
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const float w = full[j] ? exp2_fast(x[i0 + j].x - (top == -INFINITY ? 0.f : top)) : 0.f;
      l = fmaf(w, x[i0 + j].y, l);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        sum[e] = fmaf(w, u0[j][e], sum[e]);
        sum[4 + e] = fmaf(w, u1[j][e], sum[4 + e]);
      }
    }
  }
  auto join = [&](float m, float n, const f32x8 &u) {
    const float both = fmaxf(top, m), base = both == -INFINITY ? 0.f : both;
    const float w = exp2_fast(top - base), v = exp2_fast(m - base);
    top = both;
    l = fmaf(l, w, n * v);
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] = fmaf(sum[e], w, u[e] * v);
  };
  for (int off = lanes; off < 64 && off < per; off *= 2) {
    f32x8 u;
#pragma unroll
    for (int e = 0; e < 8; e++) u[e] = __shfl_xor(sum[e], off);
    const float m = __shfl_xor(top, off), n = __shfl_xor(l, off);
    join(m, n, u);
  }
  if (per > 64) {  // then the waves'
    const int wave = threadIdx.x >> 6, in = threadIdx.x & 63;
    if (in < lanes) {
      s_stat[wave * lanes + in] = make_float2(top, l);
#pragma unroll
      for (int e = 0; e < 8; e++) s_sum[(wave * lanes + in) * 8 + e] = sum[e];
    }
    __syncthreads();
    if (share > 0) return;
    for (int w = 1; w < per / 64; w++) {
      const int from = (wave + w) * lanes + in;
      f32x8 u;
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] = s_sum[from * 8 + e];
      join(s_stat[from].x, s_stat[from].y, u);
    }
  }
  if (!live || share > 0) return;
  if (d >= a.dim) return;
  const int head = (int)(at / total);
  const int64_t m = at % total;
  const int64_t out = m / a.group * a.kv_heads * a.group + head * a.group + m % a.group;
  bool blind = false;
  if (l == 0) {
    const Range r = key_range(a, (int)(m / a.group));
    blind = r.lo >= r.hi;
  }
  const float inv = blind ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 8; e++) sum[e] *= inv;
  const V8<T> y = __builtin_convertvector(sum, V8<T>);
  *reinterpret_cast<V8<T> *>(o + out * a.dim + d) = y;
  if (low) {
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] -= (float)y[e];
    *reinterpret_cast<V8<T> *>(low + out * a.dim + d) = __builtin_convertvector(sum, V8<T>);
  }
  if (lse && d == 0) lse[out] = blind ? 0.f : top - kLift<T> + log2_fast(l);
}

// Splits of the keys: two waves for each of the chip's 1024 SIMDs and no more, which is what runs at once (one more
// workgroup waits for a whole round: attend_step with 43 splits 209 us, with 42 or 21 178), and at least two tiles of
// keys for each of them if one pack held all keys.
static int attend_splits(kl_dtype dtype, int64_t nq, int64_t nk, int kv_heads, int group, int dim) {
  const int waves = is_direct(dtype, dim) ? 1 : 4, step = dtype == KL_F32 ? 32 : 64;
  const int64_t all = cdiv(nq * group, 32 * waves) * kv_heads * waves;
  return (int)std::max<int64_t>(
      1, std::min<int64_t>({2048 / std::max<int64_t>(all, 1), cdiv(nk, 2 * step), kMaxSplits}));
}

int fill_attend(Attend &a, const char *func, kl_dtype dtype, int64_t nq, int64_t nk, int heads, int kv_heads, int dim,
                const void *q, const void *k, const void *v, const int64_t *strides, const int32_t *qid, const int32_t *qstart, const int32_t *kid,
                const int32_t *kstart, float scale, int causal) {
  const std::string f = std::string(func) + ": ";
  KL_REQUIRE(nq >= 0 && nk >= 0 && nq < (int64_t)1 << 31 && nk < (int64_t)1 << 31, f + "rows out of range");
  KL_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 4096,
             f + "the query heads must be a multiple of the key heads");
  KL_REQUIRE(dim > 0 && dim <= 128 && dim % 8 == 0, f + "the head size must be a multiple of 8 up to 128");
  KL_REQUIRE(scale > 0 && scale < INFINITY, f + "the scale must be positive and finite");
  // virtual rows and workgroups are counted in 31 bits
  KL_REQUIRE(nq * (heads / kv_heads) <= ((int64_t)1 << 31) - 256 &&
                 cdiv(std::max(nq * (heads / kv_heads), nk), 32) * kv_heads < (int64_t)1 << 31,
             f + "too many rows and heads");
  KL_REQUIRE(nk <= ((int64_t)1 << 31) - 256, f + "rows out of range");
  for (int i = 0; i < 6; i++) KL_REQUIRE(strides[i] >= 0, f + "negative stride");
  for (int i = 0; i < 6; i += 2) KL_REQUIRE(strides[i] < kMaxStride, f + "rows lie too far apart");
  KL_REQUIRE((int64_t)heads * dim < kMaxStride, f + "rows lie too far apart");
  a.q = {strides[0], strides[1]};
  a.k = {strides[2], strides[3]};
  a.v = {strides[4], strides[5]};
  const size_t esize = dtype == KL_F32 ? 4 : 2;
  KL_REQUIRE(whole_pieces(q, nq, heads, a.q, esize) && whole_pieces(k, nk, kv_heads, a.k, esize) &&
                 whole_pieces(v, nk, kv_heads, a.v, esize),
             f + "rows do not start at multiples of 16 bytes");
  a.qid = qid;
  a.qstart = qstart;
  a.kid = kid;
  a.kstart = kstart;
  a.nq = (int)nq;
  a.nk = (int)nk;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.dim = dim;
  a.causal = causal ? 1 : 0;
  a.scale = scale;
  a.c = scale * kLog2e;
  return KL_OK;
}

template <typename T, int DP>
static int attend_forward(const Attend &a, const void *q, const void *k, const void *v, void *o, void *low, float *lse,
                          void *ws, hipStream_t st) {
  const int splits = attend_splits(sizeof(T) == 4 ? KL_F32 : KL_F16, a.nq, a.nk, a.kv_heads, a.group, a.dim);
  const int64_t total = (int64_t)a.nq * a.group, rows = total * a.kv_heads;
  const int64_t tiles = cdiv(total, FwdTile<T, DP>::BM);
  float2 *stat = splits > 1 ? (float2 *)ws : nullptr;
  float *part = splits > 1 ? (float *)((char *)ws + al256((size_t)splits * rows * 8)) : nullptr;
  hipLaunchKernelGGL((attend_fwd_kernel<T, DP>), places(a, tiles, splits), dim3(64 * kWaves<T, DP>), 0, st, a,
                     FwdArgs{q, k, v, o, low, lse, part, stat});
  KL_CHECK_LAUNCH();
  if (splits > 1) {
    int lanes = 1, shares = 1;
    while (lanes * 8 < a.dim) lanes *= 2;
    // many rows: a wave each (attend_step, 96 rows of 32 heads in 21 splits: a workgroup each took 10.4 us, now 5.5)
    while (shares < splits && (lanes * shares < (rows > 1024 ? 64 : 256) || shares * kJoinEach < splits)) shares *= 2;
    hipLaunchKernelGGL(attend_join_kernel<T>, dim3((unsigned)cdiv(rows, 256 / (lanes * shares))), dim3(256), 0, st, a,
                       splits, lanes, shares, part, stat, (T *)o, (T *)low, lse);
    KL_CHECK_LAUNCH();
  }
  return KL_OK;
}

}  // namespace kl

using namespace kl;

extern "C" size_t kl_pack_attention_workspace_bytes(kl_dtype dtype, int64_t num_q, int64_t num_k, int heads,
                                                    int kv_heads, int dim) {
  if (num_q <= 0 || kv_heads <= 0 || heads % kv_heads) return 256;
  const int splits = attend_splits(dtype, num_q, num_k, kv_heads, heads / kv_heads, dim);
  if (splits == 1) return 256;
  const size_t rows = (size_t)num_q * heads;
  return al256((size_t)splits * rows * 8) + al256((size_t)splits * rows * dim * 4);
}

extern "C" int kl_pack_attention_forward(kl_dtype dtype, int64_t num_q, int64_t num_k, int heads, int kv_heads, int dim,
                                         const void *q, const void *k, const void *v, const int64_t *strides_host,
                                         const int32_t *q_ids, const int32_t *q_starts, const int32_t *k_ids,
                                         const int32_t *k_starts, float scale, int causal, void *out, void *out_low,
                                         float *lse, void *ws, size_t ws_bytes, kl_stream stream) {
  Attend a;
  KL_CHECK_RC(fill_attend(a, "pack_attention", dtype, num_q, num_k, heads, kv_heads, dim, q, k, v, strides_host, q_ids,
                          q_starts, k_ids, k_starts, scale, causal));
  KL_REQUIRE(ws_bytes >= kl_pack_attention_workspace_bytes(dtype, num_q, num_k, heads, kv_heads, dim),
             "pack_attention: the workspace is too small");
  if (num_q == 0) return KL_OK;
  return with_type(dtype, "pack_attention", [&](auto t) {
    return with_dim(dim, [&](auto dp) {
      return attend_forward<decltype(t), decltype(dp)::value>(a, q, k, v, out, sizeof(t) == 2 ? out_low : nullptr, lse, ws,
                                                              S(stream));
    });
  });
}
