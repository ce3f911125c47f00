// attend32.h -- the walks of attention over packs for float with heads up to 32 (attend.hip, attendgrad.hip).
//
// A 32 x 32 x 16 product of floats takes the matrix cores 16 times as long as one of a 16-bit type, so
// feeding them is easy and idle waves are what costs.  Every wave walks by itself: 32 virtual rows (or keys)
// against just the keys (rows) that they see, operands straight from memory to registers.  Along rows, a
// lane's fragment is 32 bytes of its row; along columns, the 32 lanes of a half read 128 bytes of one row.  No
// LDS, no barrier: packs of a few dozen rows, where a workgroup's waves see different keys, do not wait for
// each other.  attend_rays_train's shapes (311,000 rows, 4 heads of 32): forward 354 -> TBD us against tiles in
// LDS shared by four waves.
//
// Rows past the end and columns past dim are read from the last ones that exist: their scores are masked and
// their outputs not stored.  Rows with infinities or NaN: as in attend.hip; the careful walk finds a tile's bad
// rows from the registers, zeroes them and adds them one by one.
#pragma once

#include "attend.h"

namespace kl {

// A matrix whose rows are `stride` bytes apart (under 2^27, so 32 rows span less than 2^32), read 32 rows at a
// time: the tile's address is the same for the whole wave, and a lane's offsets into it stay in registers.
template <int DP>
struct Rows32 {
  const char *base;
  uint32_t stride, col[DP / 16];  // col: this lane's fragments within its row, bytes
  __device__ __forceinline__ Rows32(const float *p, int64_t row_stride, int h, int dim)
      : base((const char *)p), stride((uint32_t)row_stride * 4) {
#pragma unroll
    for (int i = 0; i < DP / 16; i++) col[i] = 4 * min(16 * i + 8 * h, dim - 8);
  }
  __device__ __forceinline__ const char *tile(int row0) const { return base + (int64_t)row0 * stride; }

  // along rows: element e of f[i] = M[row0 + l % 32][16 i + 8 h + e]
  __device__ __forceinline__ void load(f32x8 (&f)[DP / 16], int row0, int end) const {
    const char *p = tile(row0);
    const uint32_t row = (uint32_t)min((int)(threadIdx.x & 31), end - 1 - row0) * stride;
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
      const f32x4 *q = reinterpret_cast<const f32x4 *>(p + (row + col[i]));
      const f32x4 a = q[0], b = q[1];
      f[i] = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
};

template <int DP>
struct Cols32 {
  uint32_t row[8], col[DP / 32];  // this lane's places in the first 16 rows of a tile, bytes
  __device__ __forceinline__ Cols32(uint32_t stride, int h, int dim) {
#pragma unroll
    for (int e = 0; e < 8; e++) row[e] = (uint32_t)acc_row(e, h) * stride;
#pragma unroll
    for (int db = 0; db < DP / 32; db++) col[db] = 4 * min(32 * db + (int)(threadIdx.x & 31), dim - 1);
  }
  // along columns: element e of f[i][db] = M[row0 + 16 i + acc_row(e, h)][32 db + l % 32]
  __device__ __forceinline__ void load(f32x8 (&f)[2][DP / 32], const Rows32<DP> &m, int row0, int end, int h) const {
    const char *p = m.tile(row0);
    if (row0 + 32 <= end) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
#pragma unroll
          for (int db = 0; db < DP / 32; db++)
            f[i][db][e] = *reinterpret_cast<const float *>(p + (int64_t)(16 * i) * m.stride + (row[e] + col[db]));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t r = (uint32_t)min(16 * i + acc_row(e, h), end - 1 - row0) * m.stride;
#pragma unroll
          for (int db = 0; db < DP / 32; db++) f[i][db][e] = *reinterpret_cast<const float *>(p + (r + col[db]));
        }
      }
    }
  }
};

// bit r: row r of the tile has an infinity or a NaN among its fragments along rows
template <int DP>
__device__ __forceinline__ uint32_t bad_rows32(const f32x8 (&f)[DP / 16]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
#pragma unroll
    for (int e = 0; e < 8; e++) bad |= !finite(f[i][e]);
  }
  const uint64_t b = ballot(bad);
  return (uint32_t)b | (uint32_t)(b >> 32);
}
// the same for fragments along columns
template <int DP>
__device__ __forceinline__ uint32_t bad_cols32(const f32x8 (&f)[2][DP / 32]) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      bool bad = false;
#pragma unroll
      for (int db = 0; db < DP / 32; db++) bad |= !finite(f[i][db][e]);
      const uint64_t b = ballot(bad);
      if ((uint32_t)b) out |= 1u << (16 * i + acc_row(e, 0));
      if (b >> 32) out |= 1u << (16 * i + acc_row(e, 1));
    }
  }
  return out;
}
template <int DP>
__device__ __forceinline__ void zero_rows32(f32x8 (&f)[DP / 16], uint32_t bad) {
  const bool b = bad >> (threadIdx.x & 31) & 1;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
#pragma unroll
    for (int e = 0; e < 8; e++) f[i][e] = b ? 0.f : f[i][e];
  }
}
template <int DP>
__device__ __forceinline__ void zero_cols32(f32x8 (&f)[2][DP / 32], uint32_t bad, int h) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool b = bad >> (16 * i + acc_row(e, h)) & 1;
#pragma unroll
      for (int db = 0; db < DP / 32; db++) f[i][db][e] = b ? 0.f : f[i][db][e];
    }
  }
}

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

__device__ __forceinline__ f32x8 frag32(const f32x16 &acc, int i) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = acc[8 * i + e];
  return v;
}

// Forward: the wave's 32 virtual rows against keys [begin, end)
template <int DP, bool CAREFUL>
__device__ __forceinline__ void fwd_walk32(const Attend &a, const float *__restrict__ k, const float *__restrict__ v,
                                           int begin, int end, Range mine, int full_lo, int full_hi,
                                           const f32x8 (&qf)[DP / 16], f32x16 (&acc)[DP / 32], RowState &st) {
  const int h = threadIdx.x >> 5 & 1;
  if (begin >= end) return;
  const Rows32<DP> km(k, a.k.row, h, a.dim), vm(v, a.v.row, h, a.dim);
  const Cols32<DP> vc(vm.stride, h, a.dim);
  f32x8 kf[DP / 16], vf[2][DP / 32];
  km.load(kf, begin, end);
  for (int kt = begin; kt < end; kt += 32) {
    vc.load(vf, vm, kt, end, h);
    uint32_t bad = 0;
    if constexpr (CAREFUL) {
      bad = bad_rows32<DP>(kf) | bad_cols32<DP>(vf);
      zero_rows32<DP>(kf, bad);
      zero_cols32<DP>(vf, bad, h);
    }
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) s = mma(kf[i], qf[i], s);
    if (kt + 32 < end) km.load(kf, kt + 32, end);
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
    for (int i = 0; i < 2; i++) {
      const f32x8 p = frag32(s, i);
#pragma unroll
      for (int db = 0; db < DP / 32; db++) acc[db] = mma(vf[i][db], p, acc[db]);
    }
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
                                          const f32x8 (&qf)[DP / 16], const f32x8 (&gf)[DP / 16],
                                          f32x16 (&acc)[DP / 32]) {
  const int h = threadIdx.x >> 5 & 1;
  if (begin >= end) return;
  const Rows32<DP> km(k, a.k.row, h, a.dim), vm(v, a.v.row, h, a.dim);
  const Cols32<DP> cols(km.stride, h, a.dim);
  f32x8 kf[DP / 16], vf[DP / 16], kc[2][DP / 32];
  km.load(kf, begin, end);
  vm.load(vf, begin, end);
  for (int kt = begin; kt < end; kt += 32) {
    cols.load(kc, km, kt, end, h);
    uint32_t bad = 0;
    if constexpr (CAREFUL) {
      bad = bad_rows32<DP>(kf) | bad_rows32<DP>(vf);
      zero_rows32<DP>(kf, bad);
      zero_rows32<DP>(vf, bad);
      zero_cols32<DP>(kc, bad, h);
    }
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < DP / 16; i++) {
      s = mma(kf[i], qf[i], s);
      dp = mma(vf[i], gf[i], dp);
    }
    if (kt + 32 < end) {
      km.load(kf, kt + 32, end);
      vm.load(vf, kt + 32, end);
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
    for (int i = 0; i < 2; i++) {
      const f32x8 ds = frag32(s, i);
#pragma unroll
      for (int db = 0; db < DP / 32; db++) acc[db] = mma(kc[i][db], ds, acc[db]);
    }
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
// constant stride apart).  q, go, ld: of the key head's first head.  s_row: LDS of this wave, the sums and
// ranges of 32 rows.
struct RowSums {
  float lse, d;
  int lo, hi;
};
template <int DP, bool CAREFUL>
__device__ __forceinline__ void dkv_walk32(const Attend &a, const float *__restrict__ q, Heads gst,
                                           const float *__restrict__ go, const float2 *__restrict__ ld, int ld_row,
                                           const int2 *__restrict__ range, int begin, int end, Range rows, int tiles,
                                           int key0, const f32x8 (&kf)[DP / 16], const f32x8 (&vf)[DP / 16],
                                           RowSums *s_row, f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32]) {
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31, key = key0 + col;
  if (begin >= end) return;
  Rows32<DP> qm(q, a.q.row, h, a.dim), gm(go, gst.row, h, a.dim);
  const Cols32<DP> qcols(qm.stride, h, a.dim), gcols(gm.stride, h, a.dim);
  f32x8 qf[DP / 16], gf[DP / 16], qc[2][DP / 32], gc[2][DP / 32];
  RowSums mine;
  int head = begin / tiles, row0 = rows.lo + begin % tiles * 32;  // of the step whose loads come next
  auto at_head = [&]() {
    qm.base = (const char *)(q + head * a.q.head);
    gm.base = (const char *)(go + head * gst.head);
  };
  at_head();
  auto load = [&]() {
    qm.load(qf, row0, rows.hi);
    gm.load(gf, row0, rows.hi);
    const int row = min(row0 + col, rows.hi - 1);
    const float2 l = ld[(int64_t)row * ld_row + head];
    const int2 r = range[row];
    const bool live = row0 + col < rows.hi;
    mine = {l.x, l.y, live ? r.x : 0x7fffffff, live ? r.y : (int)0x80000000};
  };
  load();
  for (int t = begin; t < end; t++) {
    const int here = row0;
    const bool some = __any(mine.lo < key0 + 32 && mine.hi > key0);
    const bool whole = !CAREFUL && __all(mine.lo <= key0 && mine.hi >= key0 + 32);
    uint32_t bad = 0;
    const char *qbase = qm.base, *gbase = gm.base;
    f32x16 s = {}, dp = {};
    if (some) {
      qcols.load(qc, qm, here, rows.hi, h);
      gcols.load(gc, gm, here, rows.hi, h);
      if constexpr (CAREFUL) {
        bad = bad_rows32<DP>(qf) | bad_rows32<DP>(gf);
        zero_rows32<DP>(qf, bad);
        zero_rows32<DP>(gf, bad);
        zero_cols32<DP>(qc, bad, h);
        zero_cols32<DP>(gc, bad, h);
      }
      // this wave alone writes and reads s_row, and LDS keeps its order
      if (h == 0) s_row[col] = mine;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < DP / 16; i++) {
        s = mma(qf[i], kf[i], s);
        dp = mma(gf[i], vf[i], dp);
      }
    }
    if (t + 1 < end) {
      row0 += 32;
      if (row0 >= rows.hi) {
        row0 = rows.lo;
        head++;
        at_head();
      }
      load();
    }
    if (!some) continue;
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
      const f32x8 p = frag32(s, i), ds = frag32(dp, i);
#pragma unroll
      for (int db = 0; db < DP / 32; db++) {
        dv[db] = mma(gc[i][db], p, dv[db]);
        dk[db] = mma(qc[i][db], ds, dk[db]);
      }
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
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace kl
