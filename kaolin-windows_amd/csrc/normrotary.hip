// normrotary.hip -- RMS norm of each head of queries and keys and the rotation of its first elements by the
// row's position, in one pass: y = x * rsqrt(mean(x^2) + eps) * w, then each pair (a, b) of the first
// `turn` elements becomes (a cos - b sin, a sin + b cos), angle = position * freqs[pair].
//
// Bound by memory: every element is read once and written once.  A workgroup first writes the cosines and
// sines of its rows to LDS, one thread a (row, pair), and all heads of both tensors use them; then groups of
// `lanes` lanes take one head each, 16 bytes a lane.  Angles are formed in 64 bits (a position of 10^6 in 32
// bits leaves an angle only 4 digits) and reduced to a quarter turn before they become floats.
// Norms, products and the sums over rows of the weights' gradients are in 32 bits; the outputs are rounded
// once.  Backward: g = the gradient rotated back; dw = sum over rows and heads of g x r;
// dx = r (g w - x r mean(g w x r)).
#include "seqcommon.h"

namespace kl {

enum { POS_PACK = 0, POS_I32 = 1, POS_I64 = 2, POS_F32 = 3 };

struct NormRot {
  Heads q, k;
  int64_t n;
  int hq, hk, dim, half, interleaved, rows;  // half: pairs; rows: rows of a workgroup's table
  float eps;
  const double *freqs;
  int pos_kind;
  const void *pos;                // POS_I32 .. POS_F32
  const int32_t *ids, *starts;    // POS_PACK
  const void *wq, *wk;            // NULL: ones
  int w_f32;                      // the weights are float, whatever x is
};

constexpr int kMaxDim = 256;
constexpr int kTable = 1024;      // pairs in a workgroup's table: 8 KB
constexpr int kNormBlocks = 1024; // workgroups of the backward: partial sums of the weights' gradients

__device__ __forceinline__ double position(const NormRot &a, int64_t row) {
  switch (a.pos_kind) {
    case POS_PACK: {
      const int id = a.ids[row];
      return id < 0 ? 0.0 : (double)(row - a.starts[id]);
    }
    case POS_I32: return (double)((const int32_t *)a.pos)[row];
    case POS_I64: return (double)((const int64_t *)a.pos)[row];
    default: return (double)((const float *)a.pos)[row];
  }
}

// cos and sin: the angle in quarter turns, its nearest whole number of them taken off in 64 bits
__device__ __forceinline__ float2 unit(double angle) {
  const double quarters = angle * 0.63661977236758134308;
  const double whole = rint(quarters);
  float s, c;
  sincospif(0.5f * (float)(quarters - whole), &s, &c);
  const int n = (int)(whole - 4.0 * floor(0.25 * whole)) & 3;
  const float cs = n & 1 ? s : c, sn = n & 1 ? c : s;
  return make_float2(n == 1 || n == 2 ? -cs : cs, n >= 2 ? -sn : sn);
}

template <typename T, int VE>
struct HeadPiece {
  float v[VE];
  __device__ __forceinline__ void load(const T *p) {
    union {
      u32x4 w;
      T t[VE];
    } x;
    x.w = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int e = 0; e < VE; e++) v[e] = (float)x.t[e];
  }
  __device__ __forceinline__ void store(T *p) const {
    union {
      u32x4 w;
      T t[VE];
    } x;
#pragma unroll
    for (int e = 0; e < VE; e++) x.t[e] = (T)v[e];
    *reinterpret_cast<u32x4 *>(p) = x.w;
  }
};

template <typename T, int VE>
__device__ __forceinline__ void load_weight(const NormRot &a, const void *w, int col, float (&out)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; e++) {
    out[e] = 1;
    if (w && col + e < a.dim) out[e] = a.w_f32 ? ((const float *)w)[col + e] : (float)((const T *)w)[col + e];
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Rotates a head held by LANES lanes, VE elements each; dir -1: back.  cs: the row's table.  spare: LDS of
// this head, LANES * VE floats, for the half layout where partners lie at other places of their lanes.
template <int VE, int LANES>
__device__ __forceinline__ void rotate(const NormRot &a, const float2 *cs, float dir, int sub, float *spare,
                                       float (&v)[VE]) {
  const int col = sub * VE;
  if (a.interleaved) {
    if (col < 2 * a.half) {
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        if (col + e < 2 * a.half) {
          const float2 t = cs[(col + e) / 2];
          const float s = dir * t.y, x = v[e], y = v[e + 1];
          v[e] = x * t.x - y * s;
          v[e + 1] = x * s + y * t.x;
        }
      }
    }
    return;
  }
  if (a.half % VE == 0) {  // partners sit at the same place of a lane half / VE away
    const bool first = col < a.half, second = !first && col < 2 * a.half;
    const int other = (int)(threadIdx.x & 63) + (first ? a.half / VE : second ? -(a.half / VE) : 0);
#pragma unroll
    for (int e = 0; e < VE; e++) {
      const float y = __shfl(v[e], other);
      if (first || second) {
        const float2 t = cs[first ? col + e : col + e - a.half];
        v[e] = v[e] * t.x + (first ? -dir : dir) * t.y * y;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < VE; e++) spare[col + e] = v[e];
  __builtin_amdgcn_wave_barrier();  // one wave writes and reads; LDS keeps its order
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int e = 0; e < VE; e++) {
    const int i = col + e;
    if (i < 2 * a.half) {
      const bool first = i < a.half;
      const int j = first ? i : i - a.half;
      const float2 t = cs[j];
      v[e] = v[e] * t.x + (first ? -dir : dir) * t.y * spare[first ? i + a.half : j];
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ void fill_table(const NormRot &a, int64_t row0, int rows, float2 *table) {
  for (int i = threadIdx.x; i < rows * a.half; i += 256) {
    const int r = i / a.half, p = i - r * a.half;
    table[i] = unit(position(a, row0 + r) * a.freqs[p]);
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(256) norm_rotary_kernel(NormRot a, const T *__restrict__ q, const T *__restrict__ k,
                                                        T *__restrict__ yq, T *__restrict__ yk) {
  constexpr int VE = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  __shared__ float2 table[kTable];
  __shared__ float spare[256 * VE];
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.n - row0), heads = a.hq + a.hk;
  const int sub = threadIdx.x % LANES, col = sub * VE;
  const bool in = col < a.dim;
  fill_table(a, row0, rows, table);
  float wq[VE], wk[VE];
  load_weight<T, VE>(a, a.wq, col, wq);
  load_weight<T, VE>(a, a.wk, col, wk);
  __syncthreads();
  // every lane of a wave makes every round: the exchanges take whole waves
  for (int i0 = 0; i0 < rows * heads; i0 += GROUPS) {
    const int i = i0 + threadIdx.x / LANES;
    const bool live = in && i < rows * heads;
    const int r = i < rows * heads ? i / heads : 0, hd = i < rows * heads ? i - r * heads : 0;
    const bool is_q = hd < a.hq;
    const int64_t row = row0 + r;
    HeadPiece<T, VE> x;
#pragma unroll
    for (int e = 0; e < VE; e++) x.v[e] = 0;
    if (live) x.load(is_q ? q + row * a.q.row + hd * a.q.head + col : k + row * a.k.row + (hd - a.hq) * a.k.head + col);
    float ss = 0;
#pragma unroll
    for (int e = 0; e < VE; e++) ss = fmaf(x.v[e], x.v[e], ss);
    const float inv = rsqrtf(lanes_sum<LANES>(ss) / (float)a.dim + a.eps);
#pragma unroll
    for (int e = 0; e < VE; e++) x.v[e] *= inv * (is_q ? wq[e] : wk[e]);
    rotate<VE, LANES>(a, table + r * a.half, 1.f, sub, spare + threadIdx.x / LANES * (LANES * VE), x.v);
    if (live) x.store(is_q ? yq + (row * a.hq + hd) * a.dim + col : yk + (row * a.hk + hd - a.hq) * a.dim + col);
  }
}

// part: (workgroups, 2, dim) partial sums of the weights' gradients (NULL: none wanted)
template <typename T, int LANES>
__global__ void __launch_bounds__(256) norm_rotary_bwd_kernel(NormRot a, const T *__restrict__ gq,
                                                            const T *__restrict__ gk, const T *__restrict__ q,
                                                            const T *__restrict__ k, T *__restrict__ dq,
                                                            T *__restrict__ dk, float *__restrict__ part) {
  constexpr int VE = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  __shared__ float2 table[kTable];
  __shared__ float spare[256 * VE];
  const int heads = a.hq + a.hk, sub = threadIdx.x % LANES, col = sub * VE, group = threadIdx.x / LANES;
  const bool in = col < a.dim;
  float wq[VE], wk[VE], sq[VE], sk[VE];
  load_weight<T, VE>(a, a.wq, col, wq);
  load_weight<T, VE>(a, a.wk, col, wk);
#pragma unroll
  for (int e = 0; e < VE; e++) sq[e] = sk[e] = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.n; row0 += (int64_t)gridDim.x * a.rows) {
    const int rows = (int)min((int64_t)a.rows, a.n - row0);
    __syncthreads();
    fill_table(a, row0, rows, table);
    __syncthreads();
    for (int i0 = 0; i0 < rows * heads; i0 += GROUPS) {
      const int i = i0 + group;
      const bool live = in && i < rows * heads;
      const int r = i < rows * heads ? i / heads : 0, hd = i < rows * heads ? i - r * heads : 0;
      const bool is_q = hd < a.hq;
      const int64_t row = row0 + r;
      HeadPiece<T, VE> x, g;
#pragma unroll
      for (int e = 0; e < VE; e++) x.v[e] = g.v[e] = 0;
      const int64_t at = is_q ? (row * a.hq + hd) * a.dim + col : (row * a.hk + hd - a.hq) * a.dim + col;
      if (live) {
        x.load(is_q ? q + row * a.q.row + hd * a.q.head + col : k + row * a.k.row + (hd - a.hq) * a.k.head + col);
        g.load((is_q ? gq : gk) + at);
      }
      rotate<VE, LANES>(a, table + r * a.half, -1.f, sub, spare + group * (LANES * VE), g.v);
      float ss = 0;
#pragma unroll
      for (int e = 0; e < VE; e++) ss = fmaf(x.v[e], x.v[e], ss);
      const float inv = rsqrtf(lanes_sum<LANES>(ss) / (float)a.dim + a.eps);
      float dot = 0;
#pragma unroll
      for (int e = 0; e < VE; e++) {
        x.v[e] *= inv;
        const float t = g.v[e] * x.v[e];
        sq[e] += is_q && live ? t : 0.f;
        sk[e] += is_q || !live ? 0.f : t;
        g.v[e] *= is_q ? wq[e] : wk[e];
        dot = fmaf(g.v[e], x.v[e], dot);
      }
      const float mean = lanes_sum<LANES>(dot) / (float)a.dim;
#pragma unroll
      for (int e = 0; e < VE; e++) g.v[e] = inv * (g.v[e] - x.v[e] * mean);
      if (live) g.store((is_q ? dq : dk) + at);
    }
  }
  if (!part) return;
  // the groups' sums, added in their order
#pragma unroll
  for (int w = 0; w < 2; w++) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VE; e++) spare[group * (LANES * VE) + col + e] = w ? sk[e] : sq[e];
    __syncthreads();
    for (int d = threadIdx.x; d < a.dim; d += 256) {
      float s = 0;
      for (int j = 0; j < GROUPS; j++) s += spare[j * (LANES * VE) + d];
      part[((int64_t)blockIdx.x * 2 + w) * a.dim + d] = s;
    }
  }
}

// One element of a weight's gradient a wave: the workgroups' partial sums, in an order that their number fixes.
__global__ void __launch_bounds__(256) norm_weight_grad_kernel(int dim, int parts, const float *__restrict__ part,
                                                             kl_dtype type, void *dwq, void *dwk) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 + wave;
  if (i >= 2 * dim) return;
  double s = 0;
  for (int p = lane; p < parts; p += 64) s += part[(int64_t)p * 2 * dim + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  void *out = i < dim ? dwq : dwk;
  const int d = i < dim ? i : i - dim;
  if (lane || !out) return;
  if (type == KL_F32) ((float *)out)[d] = (float)s;
  if (type == KL_F16) ((f16_t *)out)[d] = (f16_t)(float)s;
  if (type == KL_BF16) ((bf16_t *)out)[d] = (bf16_t)(float)s;
}

// Rows of a workgroup: its table holds them, and each group of lanes gets some four heads, unless that leaves
// too few workgroups for the chip.
static int norm_rows(int64_t n, int heads, int half, int groups) {
  int64_t rows = std::max<int64_t>(1, std::min<int64_t>({16, half ? kTable / half : 16, cdiv(4 * groups, heads)}));
  while (rows > 1 && cdiv(n, rows) < 1024) rows /= 2;
  return (int)rows;
}

template <typename F>
static int with_lanes(int lanes, F f) {
  if (lanes <= 8) return f(std::integral_constant<int, 8>());
  if (lanes <= 16) return f(std::integral_constant<int, 16>());
  if (lanes <= 32) return f(std::integral_constant<int, 32>());
  return f(std::integral_constant<int, 64>());
}

static int fill_norm(NormRot &a, int64_t n, int hq, int hk, int dim, int turn, int interleaved,
                     const int64_t *strides, const double *freqs, int pos_kind, const void *pos, const int32_t *ids,
                     const int32_t *starts, const void *wq, const void *wk, int w_f32, float eps) {
  KL_REQUIRE(n >= 0 && n < ((int64_t)1 << 31) - 256 && hq >= 0 && hk >= 0 && hq + hk <= 1 << 16,
             "norm_rotary: sizes out of range");
  KL_REQUIRE(dim > 0 && dim <= kMaxDim && dim % 8 == 0, "norm_rotary: the head size must be a multiple of 8 up to 256");
  KL_REQUIRE(turn >= 0 && turn <= dim && turn % 2 == 0, "norm_rotary: an even part of each head is rotated");
  KL_REQUIRE(eps >= 0 && eps < INFINITY, "norm_rotary: eps must not be negative");
  KL_REQUIRE(pos_kind >= POS_PACK && pos_kind <= POS_F32, "norm_rotary: unknown kind of positions");
  a.q = {strides[0], strides[1]};
  a.k = {strides[2], strides[3]};
  a.n = n;
  a.hq = hq;
  a.hk = hk;
  a.dim = dim;
  a.half = turn / 2;
  a.interleaved = interleaved ? 1 : 0;
  a.eps = eps;
  a.freqs = freqs;
  a.pos_kind = pos_kind;
  a.pos = pos;
  a.ids = ids;
  a.starts = starts;
  a.wq = wq;
  a.wk = wk;
  a.w_f32 = w_f32;
  return KL_OK;
}

static unsigned norm_bwd_blocks(int64_t n, int rows) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv(n, rows), kNormBlocks));
}

}  // namespace kl

using namespace kl;

extern "C" int kl_norm_rotary_forward(kl_dtype dtype, int64_t num_rows, int q_heads, int k_heads, int dim, int turn,
                                      int interleaved, const void *q, const void *k, const int64_t *strides_host,
                                      const void *q_weight, const void *k_weight, int weight_f32, const double *freqs,
                                      int pos_kind, const void *positions, const int32_t *ids, const int32_t *starts,
                                      float eps, void *out_q, void *out_k, kl_stream stream) {
  NormRot a;
  KL_CHECK_RC(fill_norm(a, num_rows, q_heads, k_heads, dim, turn, interleaved, strides_host, freqs, pos_kind, positions,
                        ids, starts, q_weight, k_weight, weight_f32, eps));
  if (num_rows == 0 || q_heads + k_heads == 0) return KL_OK;
  return with_type(dtype, "norm_rotary", [&](auto t) -> int {
    using T = decltype(t);
    return with_lanes(dim * (int)sizeof(T) / 16, [&](auto lanes) -> int {
      constexpr int L = decltype(lanes)::value;
      a.rows = norm_rows(num_rows, q_heads + k_heads, a.half, 256 / L);
      hipLaunchKernelGGL((norm_rotary_kernel<T, L>), dim3((unsigned)cdiv(num_rows, a.rows)), dim3(256), 0, S(stream), a,
                         (const T *)q, (const T *)k, (T *)out_q, (T *)out_k);
      KL_CHECK_LAUNCH();
      return KL_OK;
    });
  });
}

extern "C" size_t kl_norm_rotary_bwd_workspace_bytes(int dim) { return (size_t)kNormBlocks * 2 * std::max(dim, 0) * 4 + 256; }

extern "C" int kl_norm_rotary_backward(kl_dtype dtype, int64_t num_rows, int q_heads, int k_heads, int dim, int turn,
                                       int interleaved, const void *grad_q_out, const void *grad_k_out, const void *q,
                                       const void *k, const int64_t *strides_host, const void *q_weight,
                                       const void *k_weight, int weight_f32, const double *freqs, int pos_kind,
                                       const void *positions, const int32_t *ids, const int32_t *starts, float eps,
                                       void *grad_q, void *grad_k, void *grad_q_weight, void *grad_k_weight, void *ws,
                                       size_t ws_bytes, kl_stream stream) {
  NormRot a;
  KL_CHECK_RC(fill_norm(a, num_rows, q_heads, k_heads, dim, turn, interleaved, strides_host, freqs, pos_kind, positions,
                        ids, starts, q_weight, k_weight, weight_f32, eps));
  const bool weights = grad_q_weight || grad_k_weight;
  KL_REQUIRE(!weights || ws_bytes >= kl_norm_rotary_bwd_workspace_bytes(dim),
             "norm_rotary: the workspace is too small");
  if (q_heads + k_heads == 0 && !weights) return KL_OK;
  return with_type(dtype, "norm_rotary", [&](auto t) -> int {
    using T = decltype(t);
    return with_lanes(dim * (int)sizeof(T) / 16, [&](auto lanes) -> int {
      constexpr int L = decltype(lanes)::value;
      a.rows = norm_rows(num_rows, std::max(1, q_heads + k_heads), a.half, 256 / L);
      const unsigned blocks = norm_bwd_blocks(num_rows, a.rows);
      hipLaunchKernelGGL((norm_rotary_bwd_kernel<T, L>), dim3(blocks), dim3(256), 0, S(stream), a,
                         (const T *)grad_q_out, (const T *)grad_k_out, (const T *)q, (const T *)k, (T *)grad_q,
                         (T *)grad_k, weights ? (float *)ws : nullptr);
      KL_CHECK_LAUNCH();
      if (weights) {
        hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((unsigned)cdiv(2 * dim, 4)), dim3(256), 0, S(stream), dim,
                           (int)blocks, (const float *)ws, weight_f32 ? KL_F32 : dtype, grad_q_weight, grad_k_weight);
        KL_CHECK_LAUNCH();
      }
      return KL_OK;
    });
  });
}
