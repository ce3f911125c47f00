// normrotary.hip -- RMS norm of each head of queries and keys and the rotation of its first elements by the
// row's position, in one pass: y = x * rsqrt(mean(x^2) + eps) * w, then each pair (a, b) of the first
// `turn` elements becomes (a cos - b sin, a sin + b cos), angle = position * freqs[pair].
//
// Bound by memory: every element is read once and written once.  A workgroup first writes the cosines and
// sines of its rows to LDS, one thread a (row, pair), and all heads of both tensors use them; then groups of
// LANES lanes take one head each, 16 bytes a lane, as many heads of a row side by side as there are groups for
// (a lane keeps its row's cosines and sines in registers over them), then rows.  Sums and partners go between
// lanes without LDS where they lie 1, 2, 4 or 8 apart: through LDS, with the table read for each head and the
// weights chosen for each element, the arithmetic was what bound it (16385 rows of 32 + 8 heads of 128, bf16,
// 336 MB: 102 us, now 81, 4.1 TB/s; a copy of as many bytes takes 67).
// Angles are formed in 64 bits (a position of 10^6 in 32 bits leaves an angle only 4 digits) and reduced to a
// quarter turn before they become floats.
// Norms, products and the sums over rows of the weights' gradients are in 32 bits; the outputs are rounded
// once.  Backward: g = the gradient rotated back; dw = sum over rows and heads of g x r;
// dx = r (g w - x r mean(g w x r)).
#include "seqcommon.h"

namespace kl {

enum { POS_PACK = 0, POS_I32 = 1, POS_I64 = 2, POS_F32 = 3 };
// Where an element's partner is: in its own lane (interleaved pairs); at the same place of a lane 8, 4 or any number
// away; anywhere (through LDS)
enum Partner { OWN, AWAY_8, AWAY_4, AWAY, ANYWHERE };

struct NormRot {
  Heads q, k;
  int64_t n;
  int hq, hk, dim, half, rows, partner;  // half: pairs; rows: rows of a workgroup's table; partner: a Partner
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
  __device__ __forceinline__ void set(u32x4 w) {
    union {
      u32x4 w;
      T t[VE];
    } x;
    x.w = w;
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

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Sum over each LANES neighbouring lanes, in every one of them
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<0xb1>(v);   // lanes 1 away
  v += dpp<0x4e>(v);   // 2 away
  if constexpr (LANES >= 8) v += dpp<0x141>(v);   // the other half of 8
  if constexpr (LANES >= 16) v += dpp<0x140>(v);  // of 16
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
  if constexpr (LANES >= 64) v = half_sum(v);
  return v;
}

// 1 / root(mean of squares + eps) of a head.  Where that lies outside 2^-100 .. 2^120, so that squares may have left
// a float's range (float and bf16; heads of 1e25, or of 1e-25 without an eps), the head, the root and eps are taken
// 2^-shift times as large; v is multiplied so.  Other heads: shift 0, for a comparison (forward and backward of 262,147
// rows of 4 + 4 heads of 32, float, 261 us without and 265 with; 16385 rows of 32 + 8 heads of 128, bf16, 215 and 218).
template <typename T, int LANES, int VE>
__device__ __forceinline__ float inverse_root(const NormRot &a, float inv_dim, bool live, float (&v)[VE], int &shift) {
  auto mean = [&](float eps) {
    float ss = 0;
#pragma unroll
    for (int e = 0; e < VE; e++) ss = fmaf(v[e], v[e], ss);
    return fmaf(lanes_sum<LANES>(ss), inv_dim, eps);
  };
  float m = mean(a.eps);
  shift = 0;
  if constexpr (!std::is_same<T, f16_t>::value) {
    const bool far = live && !(m >= 0x1p-100f && m <= 0x1p120f);
    if (__any(far)) {
      float top = sqrtf(a.eps);
#pragma unroll
      for (int e = 0; e < VE; e++) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      if (far && finite(top)) shift = __builtin_amdgcn_frexp_expf(top);
#pragma unroll
      for (int e = 0; e < VE; e++) v[e] = __builtin_amdgcn_ldexpf(v[e], -shift);
      m = mean(__builtin_amdgcn_ldexpf(a.eps, -2 * shift));
    }
  }
  return rsqrtf(m);
}

// What a lane keeps of its row: element e becomes v[e] c[e] + partner[e] s[e]
template <int VE>
struct Turn {
  float c[VE], s[VE];
};

template <int VE>
__device__ __forceinline__ Turn<VE> row_turn(const NormRot &a, const float2 *table, int r, int sub, float dir) {
  Turn<VE> t;
#pragma unroll
  for (int e = 0; e < VE; e++) {
    const int i = sub * VE + e;
    const bool in = i < 2 * a.half, first = a.partner == OWN ? (e & 1) == 0 : i < a.half;
    const int pair = a.partner == OWN ? i / 2 : first ? i : i - a.half;
    const float2 u = in ? table[r * a.half + pair] : make_float2(1, 0);
    t.c[e] = u.x;
    t.s[e] = first ? -dir * u.y : dir * u.y;
  }
  return t;
}

// spare: LDS of this head, LANES * VE floats
template <int VE>
__device__ __forceinline__ void rotate(const NormRot &a, const Turn<VE> &t, int sub, float *spare, float (&v)[VE]) {
  float other[VE];
  switch (a.partner) {
    case OWN:
#pragma unroll
      for (int e = 0; e < VE; e++) other[e] = v[e ^ 1];
      break;
    case AWAY_8:
#pragma unroll
      for (int e = 0; e < VE; e++) other[e] = dpp<0x128>(v[e]);  // rows of 16 lanes, turned by 8
      break;
    case AWAY_4: {
      const bool first = (sub & 7) < 4;
#pragma unroll
      for (int e = 0; e < VE; e++) {
        const float up = dpp<0x104>(v[e]), down = dpp<0x114>(v[e]);  // from 4 lanes on, from 4 lanes back
        other[e] = first ? up : down;
      }
      break;
    }
    case AWAY: {
      const int h = a.half / VE, lane = threadIdx.x & 63, from = sub < h ? lane + h : sub < 2 * h ? lane - h : lane;
#pragma unroll
      for (int e = 0; e < VE; e++) other[e] = __shfl(v[e], from);
      break;
    }
    default: {
      // one wave writes and reads; LDS keeps its order
#pragma unroll
      for (int e = 0; e < VE; e++) spare[sub * VE + e] = v[e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < VE; e++) {
        const int i = sub * VE + e;
        other[e] = i < a.half ? spare[i + a.half] : i < 2 * a.half ? spare[i - a.half] : 0.f;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  if (2 * a.half < a.dim) {  // elements past the rotated ones have no partner, not even an infinite one times 0
#pragma unroll
    for (int e = 0; e < VE; e++) other[e] = sub * VE + e < 2 * a.half ? other[e] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < VE; e++) v[e] = fmaf(other[e], t.s[e], v[e] * t.c[e]);
}

__device__ __forceinline__ void fill_table(const NormRot &a, int64_t row0, int rows, float2 *table) {
  for (int i = threadIdx.x; i < rows * a.half; i += 256) {
    const int r = i / a.half, p = i - r * a.half;
    table[i] = unit(position(a, row0 + r) * a.freqs[p]);
  }
}

// Calls f(row, head, live, turn) for the (row, head)s of one tensor that a group of lanes takes: `side` groups
// side by side along the heads, the others along the rows.  Every lane of a wave makes every call.
template <int GROUPS, int VE, typename F>
__device__ __forceinline__ void each_head(const NormRot &a, int heads, int rows, int group, int sub, float dir,
                                          const float2 *table, F f) {
  int side = 1;
  while (side < GROUPS && side < heads) side *= 2;
  const int h0 = group & (side - 1), r0 = group / side, step = GROUPS / side;
  for (int rb = 0; rb < rows; rb += step) {
    const int r = rb + r0;
    const Turn<VE> t = row_turn<VE>(a, table, min(r, rows - 1), sub, dir);
    for (int hb = 0; hb < heads; hb += side) f(r, hb + h0, r < rows && hb + h0 < heads, t);
  }
}

template <typename T, int LANES>
__global__ void __launch_bounds__(256) norm_rotary_kernel(NormRot a, const T *__restrict__ q, const T *__restrict__ k,
                                                        T *__restrict__ yq, T *__restrict__ yk) {
  constexpr int VE = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  __shared__ float2 table[kTable];
  __shared__ float spare[256 * VE];
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const int rows = (int)min((int64_t)a.rows, a.n - row0);
  const int sub = threadIdx.x % LANES, col = sub * VE, group = threadIdx.x / LANES;
  const bool in = col < a.dim;
  const float inv_dim = 1.f / (float)a.dim;
  fill_table(a, row0, rows, table);
  __syncthreads();
  auto side = [&](const T *x, Heads st, int heads, const void *weight, T *y) {
    float w[VE];
    load_weight<T, VE>(a, weight, col, w);
    each_head<GROUPS, VE>(a, heads, rows, group, sub, 1.f, table, [&](int r, int hd, bool live, const Turn<VE> &t) {
      const int64_t row = row0 + r;
      live = live && in;
      HeadPiece<T, VE> v;
      v.set(live ? *reinterpret_cast<const u32x4 *>(x + row * st.row + hd * st.head + col) : u32x4{0, 0, 0, 0});
      int shift;
      const float inv = inverse_root<T, LANES>(a, inv_dim, live, v.v, shift);
#pragma unroll
      for (int e = 0; e < VE; e++) v.v[e] *= inv * w[e];
      rotate<VE>(a, t, sub, spare + group * (LANES * VE), v.v);
      if (live) v.store(y + (row * heads + hd) * a.dim + col);
    });
  };
  side(q, a.q, a.hq, a.wq, yq);
  side(k, a.k, a.hk, a.wk, yk);
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
  const int sub = threadIdx.x % LANES, col = sub * VE, group = threadIdx.x / LANES;
  const bool in = col < a.dim;
  const float inv_dim = 1.f / (float)a.dim;
  float sq[VE], sk[VE];
#pragma unroll
  for (int e = 0; e < VE; e++) sq[e] = sk[e] = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.n; row0 += (int64_t)gridDim.x * a.rows) {
    const int rows = (int)min((int64_t)a.rows, a.n - row0);
    __syncthreads();
    fill_table(a, row0, rows, table);
    __syncthreads();
    auto side = [&](const T *x, Heads st, const T *gy, int heads, const void *weight, T *dx, float (&sum)[VE]) {
      float w[VE];
      load_weight<T, VE>(a, weight, col, w);
      each_head<GROUPS, VE>(a, heads, rows, group, sub, -1.f, table, [&](int r, int hd, bool live, const Turn<VE> &t) {
        const int64_t row = row0 + r, at = (row * heads + hd) * a.dim + col;
        live = live && in;
        HeadPiece<T, VE> v, g;
        const u32x4 none = {0, 0, 0, 0};
        v.set(live ? *reinterpret_cast<const u32x4 *>(x + row * st.row + hd * st.head + col) : none);
        g.set(live ? *reinterpret_cast<const u32x4 *>(gy + at) : none);
        rotate<VE>(a, t, sub, spare + group * (LANES * VE), g.v);
        int shift;
        const float inv = inverse_root<T, LANES>(a, inv_dim, live, v.v, shift);
        float dot = 0;
#pragma unroll
        for (int e = 0; e < VE; e++) {
          v.v[e] *= inv;
          const float t1 = g.v[e] * v.v[e];
          sum[e] += live ? t1 : 0.f;
          g.v[e] *= w[e];
          dot = fmaf(g.v[e], v.v[e], dot);
        }
        const float mean = lanes_sum<LANES>(dot) * inv_dim;
#pragma unroll
        for (int e = 0; e < VE; e++) g.v[e] = inv * (g.v[e] - v.v[e] * mean);
        if (__any(shift)) {
#pragma unroll
          for (int e = 0; e < VE; e++) g.v[e] = __builtin_amdgcn_ldexpf(g.v[e], -shift);
        }
        if (live) g.store(dx + at);
      });
    };
    side(q, a.q, gq, a.hq, a.wq, dq, sq);
    side(k, a.k, gk, a.hk, a.wk, dk, sk);
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

// Rows of a workgroup: its table holds them, and each group of lanes gets some 32 heads (at the size above 4 take
// 110 us, 8 take 93 and 32 take 81: the table and its barrier come first), unless that leaves too few workgroups; but
// no fewer rows than the lanes take at once (1721 rows of 1 + 1 heads of 128, bf16, forward and backward: 14 + 20 us
// one by one, 7 + 9 by eights).
static int norm_rows(int64_t n, int heads, int half, int groups) {
  int64_t rows = std::max<int64_t>(1, std::min<int64_t>({16, half ? kTable / half : 16, cdiv(32 * groups, heads)}));
  while (rows > 1 && cdiv(n, rows) < 1024 && (rows * heads > groups || rows * half > 256)) rows /= 2;
  return (int)rows;
}

template <typename F>
static int with_lanes(int lanes, F f) {
  if (lanes <= 4) return f(std::integral_constant<int, 4>());
  if (lanes <= 8) return f(std::integral_constant<int, 8>());
  if (lanes <= 16) return f(std::integral_constant<int, 16>());
  if (lanes <= 32) return f(std::integral_constant<int, 32>());
  return f(std::integral_constant<int, 64>());
}

static int fill_norm(NormRot &a, int ve, int64_t n, int hq, int hk, int dim, int turn, int interleaved,
                     const void *q, const void *k, const int64_t *strides, const double *freqs, int pos_kind, const void *pos, const int32_t *ids,
                     const int32_t *starts, const void *wq, const void *wk, int w_f32, float eps) {
  KL_REQUIRE(n >= 0 && n < ((int64_t)1 << 31) - 256 && hq >= 0 && hk >= 0 && hq + hk <= 1 << 16,
             "norm_rotary: sizes out of range");
  KL_REQUIRE(dim > 0 && dim <= kMaxDim && dim % 8 == 0, "norm_rotary: the head size must be a multiple of 8 up to 256");
  KL_REQUIRE(turn >= 0 && turn <= dim && turn % 2 == 0, "norm_rotary: an even part of each head is rotated");
  KL_REQUIRE(eps >= 0 && eps < INFINITY, "norm_rotary: eps must not be negative");
  KL_REQUIRE(pos_kind >= POS_PACK && pos_kind <= POS_F32, "norm_rotary: unknown kind of positions");
  a.q = {strides[0], strides[1]};
  a.k = {strides[2], strides[3]};
  KL_REQUIRE(whole_pieces(q, n, hq, a.q, 16 / ve) && whole_pieces(k, n, hk, a.k, 16 / ve),
             "norm_rotary: rows do not start at multiples of 16 bytes");
  a.n = n;
  a.hq = hq;
  a.hk = hk;
  a.dim = dim;
  a.half = turn / 2;
  const int h = turn / 2 / ve;  // lanes between partners
  a.partner = interleaved ? OWN : turn / 2 % ve ? ANYWHERE : h == 8 ? AWAY_8 : h == 4 ? AWAY_4 : AWAY;
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
  KL_CHECK_RC(fill_norm(a, dtype == KL_F32 ? 4 : 8, num_rows, q_heads, k_heads, dim, turn, interleaved, q, k, strides_host,
                        freqs, pos_kind, positions, ids, starts, q_weight, k_weight, weight_f32, eps));
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
  KL_CHECK_RC(fill_norm(a, dtype == KL_F32 ? 4 : 8, num_rows, q_heads, k_heads, dim, turn, interleaved, q, k, strides_host,
                        freqs, pos_kind, positions, ids, starts, q_weight, k_weight, weight_f32, eps));
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
