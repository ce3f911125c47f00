// attend.h -- the geometry that the attention kernels over packs share (attend.hip, attendgrad.hip).
#pragma once

#include "seqcommon.h"

namespace kl {

constexpr int64_t kMaxStride = 1 << 25;  // elements from row to row: 32 rows of floats span under 2^32 bytes

// One attention call.  The query heads g = 0 .. group - 1 of key head m are its heads m * group + g, and
// the (row, g) of one key head are numbered as virtual rows row * group + g: they share keys and values,
// so one tile of virtual rows serves a whole group, and a single query row with its group still fills
// part of a tile.
struct Attend {
  Heads q, k, v;
  const int32_t *qid, *qstart, *kid, *kstart;
  int nq, nk;         // rows
  int kv_heads, group, dim, causal;
  float scale, c;     // c = scale * log2(e): exponentials are base 2
};

// Whether waves walk by themselves (attend32.h): float with small heads, whose
// registers allow it.  Waves of a workgroup.
template <typename T, int DP>
constexpr bool kDirect = sizeof(T) == 4 && DP == 32;
template <typename T, int DP>
constexpr int kWaves = kDirect<T, DP> ? 1 : 4;
inline bool is_direct(kl_dtype dtype, int dim) { return dtype == KL_F32 && dim <= 32; }

// The keys [lo, hi) that query row `row` sees: those of its pack; causal: the pack's last query sees all,
// and each query before it one key fewer.  No key: lo = INT_MAX, hi = INT_MIN.
struct Range {
  int lo, hi;
};
__device__ __forceinline__ Range no_keys() { return {0x7fffffff, (int)0x80000000}; }
__device__ __forceinline__ Range key_range(const Attend &a, int row) {
  const int p = a.qid[row];
  if (p < 0) return no_keys();
  const int lo = a.kstart[min(p, a.nk)];
  int hi = a.kstart[min(p + 1, a.nk)];
  if (a.causal) hi -= a.qstart[p + 1] - 1 - row;
  return hi > lo ? Range{lo, hi} : no_keys();
}

// The part of keys [begin, end) that split `y` of `n` takes, in whole steps
__device__ __forceinline__ void take_split(int &begin, int &end, int y, int n, int step) {
  const int steps = (end - begin + step - 1) / step, share = (steps + n - 1) / n * step;
  begin = (int)min((int64_t)end, begin + (int64_t)share * y);
  end = (int)min((int64_t)end, (int64_t)begin + share);
}

// Where a workgroup is.  Splits of one tile run side by side, so that tiles with much to do start first whichever
// their splits are (a split of all tiles after the other: attend_long_train's dk and dv 322 us, now 263).
struct Place {
  int head, tile, tiles;
};
__device__ __forceinline__ Place place(const Attend &a, bool split) {
  if (split) return {(int)blockIdx.x, (int)blockIdx.z, (int)gridDim.z};
  const int tile = (int)blockIdx.x / a.kv_heads;
  return {(int)blockIdx.x - tile * a.kv_heads, tile, (int)gridDim.x / a.kv_heads};
}
inline dim3 places(const Attend &a, int64_t tiles, int splits) {  // splits > 1: there are few tiles
  return splits > 1 ? dim3(a.kv_heads, splits, (unsigned)tiles) : dim3((unsigned)(tiles * a.kv_heads));
}

// A tile of ROWS rows on its way from memory through the registers of a workgroup's 256 threads to LDS
template <typename T, int DP, int ROWS>
struct Stage {
  static constexpr int CH = DP * (int)sizeof(T) / 16;  // pieces per row
  static constexpr int PER = ROWS * CH / 256;
  static constexpr int E = 16 / (int)sizeof(T);
  static constexpr int SIZE = ROWS * Tile<T, DP>::LD;
  static_assert(ROWS * CH % 256 == 0, "whole pieces per thread");
  u32x4 w[PER];

  // Columns at or past `dim` become zeros, rows at or past `end` zeros or, where rows overlap, some row's finite or
  // other elements: nobody sees them.  The buffer ends with row end - 1, so no lane has to ask; base, row0 and end
  // are the same for the whole workgroup.
  __device__ __forceinline__ void load(const T *__restrict__ base, int64_t stride, int row0, int end, int dim) {
    static_assert(ROWS <= 64 && ROWS * sizeof(T) <= 128, "a tile's rows span less than 2^32 bytes (kMaxStride)");
    constexpr uint32_t kNowhere = 0xfffffff0u;
    const uint64_t bytes = ((uint64_t)(end - 1 - row0) * (uint64_t)stride + (uint64_t)dim) * sizeof(T);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(base + row0 * stride), (short)0, (int)(uint32_t)min(bytes, (uint64_t)kNowhere), 0x00020000);
    const uint32_t row = (uint32_t)stride * (uint32_t)sizeof(T), col = threadIdx.x % CH * E;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const uint32_t at = (threadIdx.x / CH + 256 / CH * i) * row + col * (uint32_t)sizeof(T);
      w[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)((int)col < dim ? at : kNowhere), 0, 0);
    }
  }
  __device__ __forceinline__ void store(T *tile) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int at = threadIdx.x + 256 * i;
      *reinterpret_cast<u32x4 *>(tile + Tile<T, DP>::piece(at / CH, at % CH)) = w[i];
    }
  }
  // bit r of bad[r / 32] for every row r that holds an infinity or a NaN
  __device__ __forceinline__ void mark_bad(uint32_t *bad) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int r = (threadIdx.x + 256 * i) / CH;
      if (piece_bad<T>(w[i])) atomicOr(&bad[r / 32], 1u << (r % 32));
    }
  }
  // bad rows as zeros
  __device__ __forceinline__ void store_good(T *tile, const uint32_t *bad) const {
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int at = threadIdx.x + 256 * i, r = at / CH;
      const bool b = bad[r / 32] >> (r % 32) & 1;
      *reinterpret_cast<u32x4 *>(tile + Tile<T, DP>::piece(r, at % CH)) = b ? u32x4{0, 0, 0, 0} : w[i];
    }
  }
};

// Two tiles of ROWS rows streaming past a workgroup, x and y, in two LDS buffers each, steps [begin, end).
// While one pair is computed on, the next is on its way from memory to registers; one barrier a step.
// load(x, y, t) starts the loads of step t, commit(buffer) stores what it kept besides the tiles.
// CAREFUL (rows that hold infinities or NaN are taken out): buffer 0 has the rows with the bad ones as
// zeros, buffer 1 all of them as they are, `bad` says which.
template <typename T, int DP, int ROWS, bool CAREFUL, typename LOAD, typename COMMIT, typename STEP>
__device__ __forceinline__ void stream(int begin, int end, T *xs, T *ys, uint32_t *bad, LOAD load, COMMIT commit,
                                       STEP step) {
  using St = Stage<T, DP, ROWS>;
  if (begin >= end) return;
  St x, y;
  load(x, y, begin);
  if constexpr (CAREFUL) {
    for (int t = begin; t < end; t++) {
      __syncthreads();  // the step before is done with the buffers
      if (threadIdx.x < ROWS / 32) bad[threadIdx.x] = 0;
      __syncthreads();
      x.mark_bad(bad);
      y.mark_bad(bad);
      __syncthreads();
      x.store_good(xs, bad);
      y.store_good(ys, bad);
      x.store(xs + St::SIZE);
      y.store(ys + St::SIZE);
      commit(0);
      __syncthreads();
      if (t + 1 < end) load(x, y, t + 1);
      step(t, 0);
    }
  } else {
    __syncthreads();
    x.store(xs);
    y.store(ys);
    commit(0);
    if (begin + 1 < end) load(x, y, begin + 1);
    __syncthreads();
    int buffer = 0;
    for (int t = begin; t < end; t++) {
      const int other = buffer ^ 1;
      if (t + 1 < end) {
        x.store(xs + other * St::SIZE);
        y.store(ys + other * St::SIZE);
        commit(other);
        if (t + 2 < end) load(x, y, t + 2);
      }
      step(t, buffer);
      __syncthreads();
      buffer = other;
    }
  }
}

// The stationary operand: the 32 columns of a wave are 32 rows of a (rows, dim) matrix; element e of
// fragment s is row[16 * s + 8 * h + e].
template <typename T>
__device__ __forceinline__ V8<T> global_frag(const T *row, bool valid, int col, int dim) {
  union {
    u32x4 w[sizeof(T) / 2];
    V8<T> v;
  } x;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++)
    x.w[i] = valid && col < dim ? reinterpret_cast<const u32x4 *>(row + col)[i] : u32x4{0, 0, 0, 0};
  return x.v;
}

// sum over a column's stationary row (fragments f) times row r of a tile
template <typename T, int DP>
__device__ __forceinline__ float frag_dot(const V8<T> (&f)[DP / 16], const T *tile, int r, int h) {
  float s = 0;
#pragma unroll
  for (int i = 0; i < DP / 16; i++) {
    const V8<T> x = Tile<T, DP>::row_frag(tile, r, 16 * i + 8 * h);
#pragma unroll
    for (int e = 0; e < 8; e++) s = fmaf((float)f[i][e], (float)x[e], s);
  }
  return half_sum(s);
}

// acc[db][r] += w * tile[row][32 * db + acc_row(r, h)]: one inner index of the transposed product by itself
template <typename T, int DP>
__device__ __forceinline__ void add_row(f32x16 (&acc)[DP / 32], float w, const T *tile, int row, int h) {
#pragma unroll
  for (int db = 0; db < DP / 32; db++) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const V4<T> x = *reinterpret_cast<const V4<T> *>(tile + Tile<T, DP>::at(row, 32 * db + 8 * b + 4 * h));
#pragma unroll
      for (int i = 0; i < 4; i++) acc[db][4 * b + i] = fmaf(w, (float)x[i], acc[db][4 * b + i]);
    }
  }
}

// Minimum and maximum over the wave (all lanes active), the same in every lane: rows of 16 lanes, then across
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int dpp_imax(int v) {
  return max(v, __builtin_amdgcn_update_dpp(v, v, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ int max_over(int v) {
  v = dpp_imax<0x111, 0xf>(v);
  v = dpp_imax<0x112, 0xf>(v);
  v = dpp_imax<0x114, 0xf>(v);
  v = dpp_imax<0x118, 0xf>(v);
  v = dpp_imax<0x142, 0xa>(v);
  v = dpp_imax<0x143, 0xc>(v);
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int min_over(int v) { return ~max_over(~v); }

// Virtual row m of a key head
struct Row {
  int row, sub;
};
__device__ __forceinline__ Row virtual_row(const Attend &a, int m) {
  if (a.group == 1) return {m, 0};
  const int row = (int)((unsigned)m / (unsigned)a.group);
  return {row, m - row * a.group};
}

// Rows of the transposed accumulators (columns = rows of the output) to memory, four at a time
template <typename T, int DP>
__device__ __forceinline__ void store_cols(T *row, const f32x16 (&acc)[DP / 32], float w, int h, int dim) {
#pragma unroll
  for (int db = 0; db < DP / 32; db++) {
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const int d = 32 * db + 8 * b + 4 * h;
      if (d < dim) {
        const f32x4 x = {acc[db][4 * b] * w, acc[db][4 * b + 1] * w, acc[db][4 * b + 2] * w, acc[db][4 * b + 3] * w};
        *reinterpret_cast<V4<T> *>(row + d) = __builtin_convertvector(x, V4<T>);
      }
    }
  }
}

template <int N>
__device__ __forceinline__ bool all_finite(const f32x16 (&acc)[N]) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < N; i++) {
#pragma unroll
    for (int r = 0; r < 16; r++) ok = ok && finite(acc[i][r]);
  }
  return ok;
}

// The running maximum (in the scores' base-2 scale) and sum of a row.  The maximum lags: sums are
// rescaled only when a score passes it by kLag, for which weights grow to 2^kLag at most (rescaling at every
// new maximum cost 64 multiplications a tile, a quarter of the arithmetic).
struct RowState {
  float m = -INFINITY, l = 0;
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
};
constexpr float kLag = 8;
// float16's weights are 2^kLift times larger, so that 2^kLag * 2^kLift = 2^15 is in its range and those down to 2^-32
// of the largest are: without it 131,072 keys of weights 2^-25 of another's, a 256th of it together, were lost.  A
// row's sum is of the same weights, so the result has no factor.
template <typename T>
constexpr float kLift = std::is_same<T, f16_t>::value ? 7.f : 0.f;

template <int N>
__device__ __forceinline__ void rescale(RowState &st, float m, f32x16 (&acc)[N]) {
  const float keep = exp2_fast(st.m - (m == -INFINITY ? 0.f : m));
  st.m = m;
  st.l *= keep;
#pragma unroll
  for (int i = 0; i < N; i++) {
#pragma unroll
    for (int r = 0; r < 16; r++) acc[i][r] *= keep;
  }
}

template <typename F>
int with_dim(int dim, F f) {
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}
// Checks an Attend's sizes and addresses and fills it.  dim: a multiple of 8 up to 128, so rows are whole 16-byte
// pieces.
int fill_attend(Attend &a, const char *func, kl_dtype dtype, int64_t nq, int64_t nk, int heads, int kv_heads, int dim,
                const void *q, const void *k, const void *v, const int64_t *strides, const int32_t *qid, const int32_t *qstart, const int32_t *kid,
                const int32_t *kstart, float scale, int causal);

}  // namespace kl
