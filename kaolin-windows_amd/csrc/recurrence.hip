// recurrence.hip -- gated linear recurrence along packs: h[t] = a[t] h[t-1] + b[t] in every column, from
// `initial` (or 0) at each pack's first row; reverse: from its last row down.
//
// Steps compose: rows t0 .. t1 take a state s to A s + B, so the rows are cut into chunks, and
//   1. every (chunk, columns) thread computes its chunk's (A, B),
//   2. a scan over the chunks gives each chunk the state before it,
//   3. every thread walks its chunk again from that state and writes.
// A pack's first row takes no state: a chunk with one (`reset`) composes to (0, B), and its A is never
// multiplied with the state before it (which may be infinite in another pack).  Order and rounding are
// fixed by the sizes alone.  States, A and B are in 32 bits (64 for double); outputs are rounded once.
//
// Backward: g[t] = dh[t] + a[t+1] g[t+1] is the same recurrence in the other direction with the gate of the
// row walked before; db = g, da[t] = g[t] h[t-1], dinitial = a g at the first row.
#include "seqcommon.h"

namespace kl {

template <typename T>
struct StateOf {
  typedef float S;
};
template <>
struct StateOf<double> {
  typedef double S;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

struct Recur {
  int n, cols, chunk, chunks, packs;  // cols: threads across; chunk: rows of one; packs: rows of initial
  int64_t dim;
  const int32_t *ids, *starts;
};

constexpr int kAhead = 4;  // rows whose loads are in flight together

// One thread's walk over rows first .. last in processing order.  DOWN: rows descend.  GRAD: the backward.
// AGG: only (A, B) are computed, from state 0.
template <typename T, int V, bool DOWN, bool GRAD, bool AGG>
__device__ __forceinline__ void recur_walk(const Recur &r, int64_t first, int64_t last, int64_t col,
                                           const T *__restrict__ a, const T *__restrict__ x, const T *__restrict__ h,
                                           const T *__restrict__ init, T *__restrict__ out, T *__restrict__ da,
                                           T *__restrict__ dinit, typename StateOf<T>::S (&state)[V],
                                           typename StateOf<T>::S (&gain)[V], bool &reset) {
  using S = typename StateOf<T>::S;
  using P = Pack<T, V>;
  const int64_t n = r.n;
  auto row = [&](int64_t i) { return DOWN ? n - 1 - i : i; };
  auto id = [&](int64_t i) { return i >= 0 && i < n ? r.ids[row(i)] : -2; };
  auto at = [&](const T *p, int64_t t) { return *reinterpret_cast<const P *>(p + t * r.dim + col * V); };
  int before = id(first - 1), here = id(first);
  P gate = {};  // GRAD: the gate of the row walked before
  if (GRAD && before == here && here >= 0) gate = at(a, row(first - 1));
  for (int64_t i0 = first; i0 < last; i0 += kAhead) {
    P av[kAhead], xv[kAhead], hv[kAhead];
    int idv[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int64_t i = i0 + u;
      av[u] = P{};
      xv[u] = P{};
      hv[u] = P{};
      idv[u] = -2;
      if (i < last) {
        av[u] = at(a, row(i));
        xv[u] = at(x, row(i));
        idv[u] = id(i + 1);
        if (GRAD && !AGG && idv[u] != -2) hv[u] = at(h, row(i + 1));
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int64_t i = i0 + u;
      if (i >= last) break;
      const int next = idv[u];
      const bool start = here != before, none = here < 0;
      const int64_t t = row(i) * r.dim + col * V;
      reset = reset || start;
      P y, dy;
      if (GRAD) {
        // the forward's state before this row: the next row walked, or the pack's initial state
        const bool end = next != here;
        P hp = hv[u];
        if (!AGG && end) {
          hp = P{};
          if (init && !none && here < r.packs) hp = at(init, here);
        }
#pragma unroll
        for (int c = 0; c < V; c++) {
          const S g = none ? (S)0 : start ? (S)xv[u].v[c] : fma((S)gate.v[c], state[c], (S)xv[u].v[c]);
          if (AGG) gain[c] = start ? (S)0 : gain[c] * (S)gate.v[c];
          state[c] = g;
          y.v[c] = (T)g;
          dy.v[c] = (T)(none ? (S)0 : g * (S)hp.v[c]);
        }
        gate = av[u];
        if (!AGG) {
          *reinterpret_cast<P *>(out + t) = y;
          *reinterpret_cast<P *>(da + t) = dy;
          if (dinit && end && !none && here < r.packs) {
            P d;
#pragma unroll
            for (int c = 0; c < V; c++) d.v[c] = (T)((S)av[u].v[c] * state[c]);
            *reinterpret_cast<P *>(dinit + (int64_t)here * r.dim + col * V) = d;
          }
        }
      } else {
        P h0 = {};
        const bool from = start && init && !none && here < r.packs;
        if (from) h0 = at(init, here);
#pragma unroll
        for (int c = 0; c < V; c++) {
          const S b = (S)xv[u].v[c];
          const S g = none ? (S)0 : start && !from ? b : fma((S)av[u].v[c], from ? (S)h0.v[c] : state[c], b);
          if (AGG) gain[c] = start ? (S)0 : gain[c] * (S)av[u].v[c];
          state[c] = g;
          y.v[c] = (T)g;
        }
        if (!AGG) *reinterpret_cast<P *>(out + t) = y;
      }
      before = here;
      here = next;
    }
  }
}

// Step 1.  The chunk of thread t is t / cols, its columns t % cols.
template <typename T, int V, bool DOWN, bool GRAD>
__global__ void __launch_bounds__(256) recur_chunk_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                        const T *__restrict__ init,
                                                        typename StateOf<T>::S *__restrict__ agg_a,
                                                        typename StateOf<T>::S *__restrict__ agg_b,
                                                        int32_t *__restrict__ resets) {
  using S = typename StateOf<T>::S;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, c = t / r.cols, col = t % r.cols;
  if (c >= r.chunks) return;
  S state[V] = {}, gain[V];
#pragma unroll
  for (int i = 0; i < V; i++) gain[i] = 1;
  bool reset = false;
  const int64_t first = c * r.chunk;
  recur_walk<T, V, DOWN, GRAD, true>(r, first, min((int64_t)r.n, first + r.chunk), col, a, x, nullptr, init, nullptr,
                                     nullptr, nullptr, state, gain, reset);
  using P = Pack<S, V>;
  P pa, pb;
#pragma unroll
  for (int i = 0; i < V; i++) {
    pa.v[i] = gain[i];
    pb.v[i] = state[i];
  }
  *reinterpret_cast<P *>(agg_a + c * r.dim + col * V) = pa;
  *reinterpret_cast<P *>(agg_b + c * r.dim + col * V) = pb;
  if (col == 0) resets[c] = reset;
}

// Step 2: 16 columns and 64 runs of chunks a workgroup; the state before each chunk replaces agg_b.
template <typename S>
__global__ void __launch_bounds__(1024) recur_carry_kernel(Recur r, const S *__restrict__ agg_a, S *__restrict__ agg_b,
                                                         const int32_t *__restrict__ resets) {
  __shared__ S s_a[64][17], s_b[64][17];
  __shared__ int s_reset[64][17];
  const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + lane;
  const int per = (r.chunks + 63) / 64, begin = min(r.chunks, run * per), end = min(r.chunks, begin + per);
  S ga = 1, gb = 0;
  int reset = 0;
  if (col < r.dim) {
#pragma unroll 4
    for (int c = begin; c < end; c++) {
      const S a = agg_a[c * r.dim + col], b = agg_b[c * r.dim + col];
      const int z = resets[c];
      gb = z ? b : fma(a, gb, b);
      ga = z ? (S)0 : ga * a;
      reset |= z;
    }
  }
  s_a[run][lane] = ga;
  s_b[run][lane] = gb;
  s_reset[run][lane] = reset;
  __syncthreads();
  S state = 0;
  for (int i = 0; i < run; i++) state = s_reset[i][lane] ? s_b[i][lane] : fma(s_a[i][lane], state, s_b[i][lane]);
  if (col < r.dim) {
#pragma unroll 4
    for (int c = begin; c < end; c++) {
      const S a = agg_a[c * r.dim + col], b = agg_b[c * r.dim + col];
      agg_b[c * r.dim + col] = state;
      state = resets[c] ? b : fma(a, state, b);
    }
  }
}

// Step 3.  carry: the state before each chunk (NULL with one chunk).  Threads past the chunks write the
// gradients of initial states that no pack has.
template <typename T, int V, bool DOWN, bool GRAD>
__global__ void __launch_bounds__(256) recur_write_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                        const T *__restrict__ h, const T *__restrict__ init,
                                                        const typename StateOf<T>::S *__restrict__ carry,
                                                        T *__restrict__ out, T *__restrict__ da,
                                                        T *__restrict__ dinit) {
  using S = typename StateOf<T>::S;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, c = t / r.cols, col = t % r.cols;
  if (c >= r.chunks) {
    const int64_t p = c - r.chunks;
    if (dinit && p < r.packs && (p >= r.n || r.starts[p] >= r.n))
      *reinterpret_cast<Pack<T, V> *>(dinit + p * r.dim + col * V) = Pack<T, V>{};
    return;
  }
  S state[V] = {}, gain[V];
  bool reset = false;
  if (carry) {
    const Pack<S, V> s = *reinterpret_cast<const Pack<S, V> *>(carry + c * r.dim + col * V);
#pragma unroll
    for (int i = 0; i < V; i++) state[i] = s.v[i];
  }
  const int64_t first = c * r.chunk;
  recur_walk<T, V, DOWN, GRAD, false>(r, first, min((int64_t)r.n, first + r.chunk), col, a, x, h, init, out, da, dinit,
                                      state, gain, reset);
}

// Rows of a chunk: 2^18 threads fill the chip, and longer chunks save carries from there on.
static int recur_chunk_rows(int64_t n, int64_t dim) {
  const int64_t v = dim % 4 == 0 ? 4 : 1;
  return (int)std::min<int64_t>(256, std::max<int64_t>(16, cdiv(n * (dim / v), 1 << 18)));
}

template <typename T, int V, bool DOWN, bool GRAD>
static int recur_run(Recur r, const void *a, const void *x, const void *h, const void *init, void *out, void *da,
                     void *dinit, void *ws, hipStream_t st) {
  using S = typename StateOf<T>::S;
  r.cols = (int)(r.dim / V);
  S *agg_a = (S *)ws, *agg_b = (S *)((char *)ws + al256((size_t)r.chunks * r.dim * sizeof(S)));
  int32_t *resets = (int32_t *)((char *)agg_b + al256((size_t)r.chunks * r.dim * sizeof(S)));
  const unsigned blocks = (unsigned)cdiv((int64_t)r.chunks * r.cols, 256);
  if (r.chunks > 1) {
    hipLaunchKernelGGL((recur_chunk_kernel<T, V, DOWN, GRAD>), dim3(blocks), dim3(256), 0, st, r, (const T *)a,
                       (const T *)x, (const T *)init, agg_a, agg_b, resets);
    KL_CHECK_LAUNCH();
    hipLaunchKernelGGL(recur_carry_kernel<S>, dim3((unsigned)cdiv(r.dim, 16)), dim3(1024), 0, st, r, agg_a, agg_b,
                       resets);
    KL_CHECK_LAUNCH();
  }
  const unsigned all = (unsigned)cdiv((r.chunks + (dinit ? (int64_t)r.packs : 0)) * r.cols, 256);
  hipLaunchKernelGGL((recur_write_kernel<T, V, DOWN, GRAD>), dim3(all), dim3(256), 0, st, r, (const T *)a,
                     (const T *)x, (const T *)h, (const T *)init, r.chunks > 1 ? agg_b : (S *)nullptr, (T *)out,
                     (T *)da, (T *)dinit);
  KL_CHECK_LAUNCH();
  return KL_OK;
}

template <typename T, int V>
static int recur_direction(const Recur &r, bool down, bool grad, const void *a, const void *x, const void *h,
                           const void *init, void *out, void *da, void *dinit, void *ws, hipStream_t st) {
  if (grad) {
    return down ? recur_run<T, V, true, true>(r, a, x, h, init, out, da, dinit, ws, st)
                : recur_run<T, V, false, true>(r, a, x, h, init, out, da, dinit, ws, st);
  }
  return down ? recur_run<T, V, true, false>(r, a, x, h, init, out, da, dinit, ws, st)
              : recur_run<T, V, false, false>(r, a, x, h, init, out, da, dinit, ws, st);
}

// Columns per thread: four (loads of 8 to 32 bytes) where every row is aligned to that, else one
template <typename T>
static int recur_type(const Recur &r, bool down, bool grad, const void *a, const void *x, const void *h,
                      const void *init, void *out, void *da, void *dinit, void *ws, hipStream_t st) {
  const uintptr_t all = (uintptr_t)a | (uintptr_t)x | (uintptr_t)h | (uintptr_t)init | (uintptr_t)out |
                        (uintptr_t)da | (uintptr_t)dinit;
  if (r.dim % 4 == 0 && all % (4 * sizeof(T)) == 0)
    return recur_direction<T, 4>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
  return recur_direction<T, 1>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
}

static int recurrence(kl_dtype dtype, bool down, bool grad, int64_t n, int64_t dim, int64_t packs, const void *a,
                      const void *x, const void *h, const void *init, const int32_t *ids, const int32_t *starts,
                      void *out, void *da, void *dinit, void *ws, size_t ws_bytes, hipStream_t st) {
  KL_REQUIRE(n >= 0 && n < ((int64_t)1 << 31) - 256 && dim >= 0 && dim < (int64_t)1 << 24 && packs >= 0 &&
                 packs < (int64_t)1 << 31,
             "linear_recurrence: sizes out of range");
  KL_REQUIRE(ws_bytes >= kl_linear_recurrence_workspace_bytes(dtype, n, dim),
             "linear_recurrence: the workspace is too small");
  if (dim == 0 || (n == 0 && !(dinit && packs))) return KL_OK;
  Recur r;
  r.n = (int)n;
  r.dim = dim;
  r.chunk = recur_chunk_rows(n, dim);
  r.chunks = (int)cdiv(n, r.chunk);
  r.packs = init ? (int)packs : 0;
  r.ids = ids;
  r.starts = starts;
  KL_REQUIRE(cdiv(((int64_t)r.chunks + packs) * dim, 256) < (int64_t)1 << 31, "linear_recurrence: too many elements");
  switch (dtype) {
    case KL_F32: return recur_type<float>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_F64: return recur_type<double>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_F16: return recur_type<f16_t>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_BF16: return recur_type<bf16_t>(r, down, grad, a, x, h, init, out, da, dinit, ws, st);
    default: set_error("linear_recurrence: expected a Half, BFloat16, Float or Double tensor"); return KL_E_INVALID;
  }
}

}  // namespace kl

using namespace kl;

extern "C" size_t kl_linear_recurrence_workspace_bytes(kl_dtype dtype, int64_t num_rows, int64_t dim) {
  if (num_rows <= 0 || dim <= 0) return 256;
  const size_t chunks = (size_t)cdiv(num_rows, recur_chunk_rows(num_rows, dim));
  if (chunks <= 1) return 256;
  return 2 * al256(chunks * dim * (dtype == KL_F64 ? 8 : 4)) + al256(chunks * 4);
}

extern "C" int kl_linear_recurrence_forward(kl_dtype dtype, int64_t num_rows, int64_t dim, const void *gates,
                                            const void *feats, const void *initial, int64_t num_initial,
                                            const int32_t *ids, const int32_t *starts, int reverse, void *out, void *ws,
                                            size_t ws_bytes, kl_stream stream) {
  return recurrence(dtype, reverse != 0, false, num_rows, dim, num_initial, gates, feats, nullptr, initial, ids, starts,
                    out, nullptr, nullptr, ws, ws_bytes, S(stream));
}

extern "C" int kl_linear_recurrence_backward(kl_dtype dtype, int64_t num_rows, int64_t dim, const void *grad_out,
                                             const void *gates, const void *out, const void *initial,
                                             int64_t num_initial, const int32_t *ids, const int32_t *starts,
                                             int reverse, void *grad_gates, void *grad_feats, void *grad_initial,
                                             void *ws, size_t ws_bytes, kl_stream stream) {
  return recurrence(dtype, reverse == 0, true, num_rows, dim, num_initial, gates, grad_out, out, initial, ids, starts,
                    grad_feats, grad_gates, initial ? grad_initial : nullptr, ws, ws_bytes, S(stream));
}
