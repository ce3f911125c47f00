// attend32.h -- the walks of attention over packs for float with heads up to 32 (attend.hip, attendgrad.hip).
//
// A 32 x 32 x 16 product of floats takes the matrix cores 16 times as long as one of a 16-bit type, so
// feeding them is easy and idle waves are what costs.  Every wave walks by itself, without a barrier: 32 virtual
// rows (or keys) against just the keys (rows) that they see, so that packs of a few dozen rows, where a
// workgroup's waves see different keys, do not wait for each other.  A tile of 32 rows goes from memory through
// registers to LDS of the wave's own, 128 bytes of a row by 8 neighbouring lanes (row fragments straight from
// memory took the L1 cache one line for each lane).
//
// Bound by the matrix units and waits for them, 45 to 49 % busy: tiles of 32 rows meet 1.8 times the keys that their
// rows see.  311,094 rows in 8192 packs of 38 on average, 4 heads of 32: forward 258 us, dq with the sums of do . o 341,
// dk and dv 428 (kernels under a profiler), where the bytes alone take 379 us.  Three waves a SIMD: with two, 303, 347
// (without the sums) and 549; with four, whose registers spill, 315, 402 and 797, where three took 260, 346 and 496.
//
// Rows past the end are copies of the last one: their scores are masked.  Rows with infinities or NaN: as in
// attend.hip; the careful walk finds a tile's bad rows in its registers, zeroes them and adds them one by one.
#pragma once

#include "attend.h"

namespace kl {

// 32 rows of a matrix whose rows are `stride` bytes apart (under 2^27: the rows of a tile span less than 2^32),
// on their way to LDS: lane l holds the pieces l % 8 of rows l / 8 + 8 i.  base is the same for the whole wave.
struct Rows32 {
  static_assert(Tile<float, 32>::E == 4, "8 pieces a row");
  const char *base;
  uint32_t stride;
  bool in;  // this lane's piece is one of the row's
  u32x4 w[4];
  __device__ __forceinline__ Rows32(const float *p, int64_t row_stride, int dim)
      : base((const char *)p), stride((uint32_t)row_stride * 4), in((int)(threadIdx.x & 7) * 4 < dim) {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load(int row0, int end) {
    const char *p = base + (int64_t)row0 * stride;
    const uint32_t row = (threadIdx.x & 63) / 8, col = (threadIdx.x & 7) * 16;
    const uint32_t last = (uint32_t)(end - 1 - row0);
    if (in) {
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const u32x4 *>(p + (min(row + 8 * i, last) * stride + col));
    }
  }
  // to LDS, rows of `bad` as zeros
  __device__ __forceinline__ void store(float *tile, uint32_t bad) const {
    const int row = (threadIdx.x & 63) / 8, p = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < 4; i++)
      *reinterpret_cast<u32x4 *>(tile + Tile<float, 32>::piece(row + 8 * i, p)) =
          bad >> (row + 8 * i) & 1 ? u32x4{0, 0, 0, 0} : w[i];
  }
  // bit r: row r has an infinity or a NaN
  __device__ __forceinline__ uint32_t bad_rows() const {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint64_t b = ballot(in && piece_bad<float>(w[i]));
      for (int r = 0; r < 8; r++) out |= (b >> (8 * r) & 0xff) ? 1u << (8 * i + r) : 0u;
    }
    return out;
  }
};

// One wave writes its tile and reads it: LDS keeps the order of a wave's accesses, the compiler has to as well
__device__ __forceinline__ void own_lds() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Column fragments straight from memory, where 32 lanes read 128 bytes of a row: element e of f[i] =
// M[row0 + 16 i + acc_row(e, h)][l % 32]
struct Cols32 {
  const char *base;
  uint32_t stride, row[8], col;  // this lane's places in the first 16 rows of a tile, bytes
  __device__ __forceinline__ Cols32(const float *p, int64_t row_stride, int h, int dim)
      : base((const char *)p), stride((uint32_t)row_stride * 4), col(4 * min((int)(threadIdx.x & 31), dim - 1)) {
#pragma unroll
    for (int e = 0; e < 8; e++) row[e] = (uint32_t)acc_row(e, h) * stride + col;
  }
  __device__ __forceinline__ void load(f32x8 (&f)[2], int row0, int end, int h) const {
    const char *p = base + (int64_t)row0 * stride;
    if (row0 + 32 <= end) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) f[i][e] = *reinterpret_cast<const float *>(p + (int64_t)(16 * i) * stride + row[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          f[i][e] = *reinterpret_cast<const float *>(
              p + ((uint32_t)min(16 * i + acc_row(e, h), end - 1 - row0) * stride + col));
      }
    }
  }
  __device__ static __forceinline__ uint32_t bad_rows(const f32x8 (&f)[2]) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint64_t b = ballot(!finite(f[i][e]));
        if ((uint32_t)b) out |= 1u << (16 * i + acc_row(e, 0));
        if (b >> 32) out |= 1u << (16 * i + acc_row(e, 1));
      }
    }
    return out;
  }
};

// sum over dim of this lane's stationary row (fragments f) times another row in memory
template <int DP>
__device__ __forceinline__ float dot32(const f32x8 (&f)[DP / 16], const float *__restrict__ other, int h, int dim) {
  float s = 0;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
    const int c = 16 * i + 8 * h;
    for (int e = 0; e < 8 && c < dim; e++) s = fmaf(f[i][e], other[c + e], s);
  }
  return half_sum(s);
}
template <int DP>
__device__ __forceinline__ void add_row32(f32x16 (&acc)[DP / 32], float w, const float *__restrict__ row, int h,
                                          int dim) {
#pragma unroll
  for (int db = 0; db < DP / 32; db++) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const f32x4 x = *reinterpret_cast<const f32x4 *>(row + min(32 * db + 8 * b + 4 * h, dim - 4));
#pragma unroll
      for (int i = 0; i < 4; i++) acc[db][4 * b + i] = fmaf(w, x[i], acc[db][4 * b + i]);
    }
  }
}

// Forward: the wave's 32 virtual rows against keys [begin, end)
template <int DP, bool CAREFUL>
__device__ __forceinline__ void fwd_walk32(const Attend &a, const float *__restrict__ k, const float *__restrict__ v,
                                           int begin, int end, Range mine, int full_lo, int full_hi,
                                           const f32x8 (&qf)[DP / 16], float *ks, f32x16 (&acc)[DP / 32],
                                           RowState &st) {
  using L = Tile<float, DP>;
  const int h = threadIdx.x >> 5 & 1, col = threadIdx.x & 31;
  if (begin >= end) return;
  Rows32 km(k, a.k.row, a.dim);
  const Cols32 vm(v, a.v.row, h, a.dim);
  f32x8 vf[2], next[2];
  km.load(begin, end);
  vm.load(next, begin, end, h);
  for (int kt = begin; kt < end; kt += 32) {
    vf[0] = next[0];
    vf[1] = next[1];
    uint32_t bad = 0;
    if constexpr (CAREFUL) {
      bad = km.bad_rows() | Cols32::bad_rows(vf);
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) vf[i][e] = bad >> (16 * i + acc_row(e, h)) & 1 ? 0.f : vf[i][e];
      }
    }
    km.store(ks, bad);
    own_lds();
    if (kt + 32 < end) {
      km.load(kt + 32, end);
      vm.load(next, kt + 32, end, h);
    }
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) s = mma(L::row_frag(ks, col, 16 * i + 8 * h), qf[i], s);
    if (CAREFUL || kt < full_lo || kt + 32 > full_hi) {
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int key = kt + acc_row(r, h);
        bool in = (key >= mine.lo) & (key < mine.hi);
        if constexpr (CAREFUL) in = in & !(bad >> acc_row(r, h) & 1);
        s[r] = in ? s[r] : -INFINITY;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; r++) top = fmaxf(top, s[r]);
    top = half_max(top) * a.c;
    if (__any(top > st.m + kLag)) rescale(st, fmaxf(st.m, top), acc);
    const float base = st.base();
#pragma unroll
    for (int r = 0; r < 16; r++) {
      s[r] = exp2_fast(fmaf(s[r], a.c, -base));
      st.l += s[r];
    }
#pragma unroll
    for (int i = 0; i < 2; i++) acc[0] = mma(vf[i], acc_frag<float>(s, i), acc[0]);
    own_lds();
    if constexpr (CAREFUL) {
      for (; bad; bad &= bad - 1) {
        const int key = kt + __builtin_ctz(bad);
        if (key >= end) break;  // copies of the last row
        const float t = dot32<DP>(qf, k + key * a.k.row, h, a.dim) * a.c;
        if (key >= mine.lo && key < mine.hi) {
          rescale(st, fmaxf(st.m, t), acc);
          const float p = exp2_fast(t - st.base());
          st.l += h == 0 ? p : 0.f;
          add_row32<DP>(acc, p, v + key * a.v.row, h, a.dim);
        }
      }
    }
  }
}

// dq: the wave's 32 virtual rows against keys [begin, end)
template <int DP, bool CAREFUL>
__device__ __forceinline__ void dq_walk32(const Attend &a, const float *__restrict__ k, const float *__restrict__ v,
                                          int begin, int end, int2 mine, float2 ld, int full_lo, int full_hi,
                                          const f32x8 (&qf)[DP / 16], const f32x8 (&gf)[DP / 16], float *ks, float *vs,
                                          f32x16 (&acc)[DP / 32]) {
  using L = Tile<float, DP>;
  const int h = threadIdx.x >> 5 & 1, col = threadIdx.x & 31;
  if (begin >= end) return;
  Rows32 km(k, a.k.row, a.dim), vm(v, a.v.row, a.dim);
  km.load(begin, end);
  vm.load(begin, end);
  for (int kt = begin; kt < end; kt += 32) {
    uint32_t bad = 0;
    if constexpr (CAREFUL) bad = km.bad_rows() | vm.bad_rows();
    km.store(ks, bad);
    vm.store(vs, bad);
    own_lds();
    if (kt + 32 < end) {
      km.load(kt + 32, end);
      vm.load(kt + 32, end);
    }
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
      s = mma(L::row_frag(ks, col, 16 * i + 8 * h), qf[i], s);
      dp = mma(L::row_frag(vs, col, 16 * i + 8 * h), gf[i], dp);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = exp2_fast(fmaf(s[r], a.c, -ld.x)) * (dp[r] - ld.y);
    if (CAREFUL || kt < full_lo || kt + 32 > full_hi) {
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int key = kt + acc_row(r, h);
        bool in = (key >= mine.x) & (key < mine.y);
        if constexpr (CAREFUL) in = in & !(bad >> acc_row(r, h) & 1);
        s[r] = in ? s[r] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) acc[0] = mma(L::col_frag(ks, 16 * i, 0), acc_frag<float>(s, i), acc[0]);
    own_lds();
    if constexpr (CAREFUL) {
      for (; bad; bad &= bad - 1) {
        const int key = kt + __builtin_ctz(bad);
        if (key >= end) break;
        const float t = dot32<DP>(qf, k + key * a.k.row, h, a.dim) * a.c;
        const float dpx = dot32<DP>(gf, v + key * a.v.row, h, a.dim);
        if (key >= mine.x && key < mine.y)
          add_row32<DP>(acc, exp2_fast(t - ld.x) * (dpx - ld.y), k + key * a.k.row, h, a.dim);
      }
    }
  }
}

// dk, dv: the wave's 32 keys against steps [begin, end) of the query rows that see any of them: step t is the
// 32 rows from rows.lo + t % tiles * 32 of head t / tiles of the key head's group (rows of one head lie a
// constant stride apart).  q, go, ld: of the key head's first head.  qs, os, s_row: LDS of this wave, the tiles of q
// and of do and the sums and ranges of their rows.
struct RowSums {
  float lse, d;
  int lo, hi;
};
template <int DP, bool CAREFUL>
__device__ __forceinline__ void dkv_walk32(const Attend &a, const float *__restrict__ q, Heads gst,
                                           const float *__restrict__ go, const float2 *__restrict__ ld, int ld_row,
                                           const int2 *__restrict__ range, int begin, int end, Range rows, int tiles,
                                           int key0, const f32x8 (&kf)[DP / 16], const f32x8 (&vf)[DP / 16], float *qs,
                                           float *os, RowSums *s_row, f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32]) {
  using L = Tile<float, DP>;
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31, key = key0 + col;
  if (begin >= end) return;
  Rows32 qm(q, a.q.row, a.dim), gm(go, gst.row, a.dim);
  RowSums mine;
  int head = begin / tiles, row0 = rows.lo + begin % tiles * 32;  // of the step whose loads come next
  auto load = [&]() {
    qm.base = (const char *)(q + head * a.q.head);
    gm.base = (const char *)(go + head * gst.head);
    qm.load(row0, rows.hi);
    gm.load(row0, rows.hi);
    const int row = min(row0 + col, rows.hi - 1);
    const float2 l = ld[(int64_t)row * ld_row + head];
    const int2 r = range[row];
    const bool live = row0 + col < rows.hi;
    mine = {l.x, l.y, live ? r.x : 0x7fffffff, live ? r.y : (int)0x80000000};
  };
  load();
  for (int t = begin; t < end; t++) {
    const int here = row0;
    const char *qbase = qm.base, *gbase = gm.base;
    const bool some = __any(mine.lo < key0 + 32 && mine.hi > key0);
    const bool whole = !CAREFUL && __all(mine.lo <= key0 && mine.hi >= key0 + 32);
    uint32_t bad = 0;
    if (some) {
      if constexpr (CAREFUL) bad = qm.bad_rows() | gm.bad_rows();
      qm.store(qs, bad);
      gm.store(os, bad);
      if (h == 0) s_row[col] = mine;
    }
    own_lds();
    if (t + 1 < end) {
      row0 += 32;
      if (row0 >= rows.hi) {
        row0 = rows.lo;
        head++;
      }
      load();
    }
    if (!some) continue;
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
      s = mma(L::row_frag(qs, col, 16 * i + 8 * h), kf[i], s);
      dp = mma(L::row_frag(os, col, 16 * i + 8 * h), vf[i], dp);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const RowSums x = s_row[acc_row(r, h)];
      s[r] = exp2_fast(fmaf(s[r], a.c, -x.lse));
      dp[r] = s[r] * (dp[r] - x.d);
      if (!whole) {
        bool in = (key >= x.lo) & (key < x.hi);
        if constexpr (CAREFUL) in = in & !(bad >> acc_row(r, h) & 1);
        s[r] = in ? s[r] : 0.f;
        dp[r] = in ? dp[r] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      dv[0] = mma(L::col_frag(os, 16 * i, 0), acc_frag<float>(s, i), dv[0]);
      dk[0] = mma(L::col_frag(qs, 16 * i, 0), acc_frag<float>(dp, i), dk[0]);
    }
    if constexpr (CAREFUL) {
      for (; bad; bad &= bad - 1) {
        const int r = __builtin_ctz(bad);
        if (here + r >= rows.hi) break;
        const RowSums x = s_row[r];
        const float *qrow = (const float *)(qbase + (int64_t)(here + r) * qm.stride);
        const float *grow = (const float *)(gbase + (int64_t)(here + r) * gm.stride);
        const float tt = dot32<DP>(kf, qrow, h, a.dim) * a.c, dpx = dot32<DP>(vf, grow, h, a.dim);
        if (key >= x.lo && key < x.hi) {
          const float p = exp2_fast(tt - x.lse);
          add_row32<DP>(dv, p, grow, h, a.dim);
          add_row32<DP>(dk, p * (dpx - x.d), qrow, h, a.dim);
        }
      }
    }
    own_lds();
  }
}

}  // namespace kl
