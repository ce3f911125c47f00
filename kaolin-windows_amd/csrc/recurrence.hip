// recurrence.hip -- gated linear recurrence along packs: h[t] = a[t] h[t-1] + b[t] in every column, from
// `initial` (or 0) at each pack's first row; reverse: from its last row down.
//
// Steps compose: rows t0 .. t1 take a state s to A s + B.  The rows are cut into chunks, one a thread and piece
// of columns:
//   1. every chunk's (A, B), from the start of its last pack on: what lies before has no effect past the chunk;
//   2. within segments of chunks, the (A, B) of what lies before each chunk, and each segment's own;
//   3. every chunk's state before it from those, back to the nearest segment with a pack's start; then it is
//      walked and written.
// A chunk in which a pack starts (`reset`) has A = 0, and that is never multiplied with the state before it, which
// may be infinite in another pack.  Order and rounding follow from the sizes alone.
//
// Bound by memory: a and b are read 1 + (share of 1) times and h is written once.  Step 3 takes the chunks in the
// other order, so that it finds what 1 read last in the 256 MB cache.  One pass, with workgroups that publish and
// await each other's (A, B), measured no faster: it reads less, but waits.
// 311,000 rows of 64 columns, float, packs of 38 rows: forward 24 + 8 + 40 us (239 MB at least, 47 us at the rate of
// a copy), backward 26 + 8 + 67 us (397 MB, 79 us); 65,537 x 1024, bf16, two packs: 70 + 13 + 72 and
// 60 + 13 + 124 us (403 MB, 80 us, and 671 MB, 133 us).
//
// States, A and B are in 32 bits (64 for double); outputs are rounded once.  A is a product of gates alone, and may pass a
// float's range both ways where the states that it meets do not (they are 0, or small, or other gates undo it): it has
// an exponent of its own (Gain).
// Backward: g[t] = dh[t] + a[t+1] g[t+1] is the same recurrence in the other direction with the gate of the
// row walked before; db = g, da[t] = g[t] h[t-1] with h as it was rounded, dinitial = a g at the first row.
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

// V elements at any address of the type's.  Rows of any length are walked in pieces of 16 bytes, the last of a row
// ending with it: its first columns are the piece's before it as well, computed and written twice alike.
template <int V, typename T>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  Pack<T, V> x;
  __builtin_memcpy(x.v, p, sizeof(T) * V);
  return x;
}
template <int V, typename T>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &x) {
  __builtin_memcpy(p, x.v, sizeof(T) * V);
}

// A = m 2^e with |m| in [0.5, 1), 0 or not finite.  Exponents are whole: a segment's are under 256 chunks * 64 rows * 1074
// (saturated at 2^+-16384, in 16 bits, a double's state came back to life behind 20 gates of 2^-1000 and 16 of 2^1000).
// Against products in a float: 65,537 x 1024 in bf16, training, 360 us for 351; 8192 rows of one pack, which fold up to
// 64 segments with three operations for one, 47 for 39.
__device__ __forceinline__ float mantissa(float x) { return __builtin_amdgcn_frexp_mantf(x); }
__device__ __forceinline__ double mantissa(double x) { return __builtin_amdgcn_frexp_mant(x); }
__device__ __forceinline__ int exponent(float x) { return __builtin_amdgcn_frexp_expf(x); }
__device__ __forceinline__ int exponent(double x) { return __builtin_amdgcn_frexp_exp(x); }
__device__ __forceinline__ float times_two_to(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }
__device__ __forceinline__ double times_two_to(double x, int e) { return __builtin_amdgcn_ldexp(x, e); }
template <typename S>
struct Gain {
  S m;
  int e;
  __device__ __forceinline__ void take(S gate) {  // up to 64 gates, then settle(): m stays over 2^-65
    m *= mantissa(gate);
    e += exponent(gate);
  }
  __device__ __forceinline__ void settle() {
    e += exponent(m);
    m = mantissa(m);
  }
  // the gains of rows before this one's as well
  __device__ __forceinline__ Gain after(const Gain &before) const {
    Gain g = {m * before.m, e + before.e};
    g.settle();
    return g;
  }
  __device__ __forceinline__ S of(S state, S add) const { return times_two_to(m * state, e) + add; }
};

struct Recur {
  int n, chunk, chunks, packs, down;  // chunk: rows of one; packs: rows of initial; down: rows descend
  int64_t dim, cols;                  // cols: pieces across
  int segment, few;                   // log2 of a segment's chunks; few: the number of segments if one wave holds them
  int wide;                           // log2 of a workgroup's pieces across, where steps 1 and 2 are one
  const int32_t *ids, *starts;
  template <int V>
  __device__ __forceinline__ int64_t column(int64_t piece) const { return min(piece * V, dim - V); }
  // rows are numbered in the order they are walked
  __device__ __forceinline__ int64_t row(int64_t i) const { return down ? n - 1 - i : i; }
  __device__ __forceinline__ int id(int64_t i) const { return i >= 0 && i < n ? ids[row(i)] : -2; }
  // row i goes on with the pack of the row before
  __device__ __forceinline__ bool carried(int64_t i) const {
    const int p = id(i);
    return p >= 0 && id(i - 1) == p;
  }
  // the first row walked of pack p
  __device__ __forceinline__ int64_t first(int p) const { return down ? n - starts[p + 1] : starts[p]; }
};

constexpr int kAhead = 8;       // rows whose loads are in flight together in step 1
constexpr int kAheadWrite = 4;  // and in step 3, which keeps more of each
constexpr int kRunChunks = 4;   // chunks of a thread of step 2
constexpr int kSegmentLog = 8, kSegment = 64 * kRunChunks;
static_assert(kSegment == 1 << kSegmentLog, "a segment of step 2");
constexpr int kFewSegments = 64;  // what a wave's lanes can look through at once

// (A, B) of chunks and segments: A = a 2^e and b (count, dim), resets (count)
template <typename S>
struct Composed {
  S *a, *b;
  int32_t *e, *resets;
};
template <typename S>
struct ComposedIn {
  const S *a, *b;
  const int32_t *e, *resets;
};

template <int V, typename S>
__device__ __forceinline__ void store_gains(const Composed<S> &m, int64_t at, const Gain<S> (&g)[V]) {
  Pack<S, V> a;
  Pack<int32_t, V> e;
#pragma unroll
  for (int v = 0; v < V; v++) {
    a.v[v] = g[v].m;
    e.v[v] = g[v].e;
  }
  store_pack<V>(m.a + at, a);
  store_pack<V>(m.e + at, e);
}

// (A, B) of rows [begin, end) of a piece of columns from the start of their last pack on, or of all of them.  True: a
// pack (or rows of none) starts there.
template <typename T, int V, bool GRAD>
__device__ __forceinline__ bool recur_compose(const Recur &r, const T *__restrict__ a, const T *__restrict__ x,
                                              const T *__restrict__ init, int64_t begin, int64_t end, int64_t col,
                                              Gain<typename StateOf<T>::S> (&gain)[V],
                                              typename StateOf<T>::S (&state)[V]) {
  using S = typename StateOf<T>::S;
  using P = Pack<T, V>;
  auto at = [&](const T *p, int64_t i) { return load_pack<V>(p + r.row(i) * r.dim + col); };
  const int last = r.id(end - 1);
  const int64_t start = last < 0 ? end : r.first(last);
  const bool reset = start >= begin;
#pragma unroll
  for (int v = 0; v < V; v++) {
    gain[v] = {(S)(reset ? 0 : 1), 0};
    state[v] = 0;
  }
  int64_t i = max(begin, start);
  if (reset && i < end) {  // the pack's first row
    const P x0 = at(x, i);
#pragma unroll
    for (int v = 0; v < V; v++) state[v] = (S)x0.v[v];
    if (!GRAD && init && last < r.packs) {
      const P a0 = at(a, i), h0 = load_pack<V>(init + (int64_t)last * r.dim + col);
#pragma unroll
      for (int v = 0; v < V; v++) state[v] = fma((S)a0.v[v], (S)h0.v[v], state[v]);
    }
    i++;
  }
  for (; i < end; i += kAhead) {
    P av[kAhead], xv[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) {  // past the last row: that row again
      const int64_t j = min(i + u, end - 1);
      av[u] = at(a, GRAD ? j - 1 : j);
      xv[u] = at(x, j);
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const bool in = i + u < end;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const S g = (S)av[u].v[v], next = fma(g, state[v], (S)xv[u].v[v]);
        state[v] = in ? next : state[v];
        gain[v].take(in ? g : (S)1);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; v++) gain[v].settle();
  return reset;
}

// Step 1.  Thread t: the chunk t / cols, the piece t % cols.
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(256) recur_chunk_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                        const T *__restrict__ init,
                                                        Composed<typename StateOf<T>::S> chunks) {
  using S = typename StateOf<T>::S;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, c = t / r.cols, piece = t - c * r.cols, col = r.column<V>(piece);
  if (c >= r.chunks) return;
  const int64_t begin = c * r.chunk, end = min((int64_t)r.n, begin + r.chunk);
  Gain<S> gain[V];
  Pack<S, V> state;
  const bool reset = recur_compose<T, V, GRAD>(r, a, x, init, begin, end, col, gain, state.v);
  store_gains<V>(chunks, c * r.dim + col, gain);
  store_pack<V>(chunks.b + c * r.dim + col, state);
  if (piece == 0) chunks.resets[c] = reset;
}

// Step 2: 16 columns and a segment a workgroup, 64 runs of kRunChunks chunks.  What lies before a chunk in its
// segment replaces its (A, B); whether a pack starts there goes to `before` (resets is still read by others).
template <typename S>
__global__ void __launch_bounds__(1024) recur_scan_kernel(Recur r, Composed<S> chunks, int32_t *__restrict__ before,
                                                        Composed<S> segments) {
  __shared__ S s_b[1024];
  __shared__ Gain<S> s_a[1024];
  __shared__ int s_reset[1024];
  const int me = threadIdx.x;
  const int64_t col = (int64_t)blockIdx.x * 16 + me % 16, at = min(col, r.dim - 1);
  const int c0 = blockIdx.y * kSegment + me / 16 * kRunChunks;
  const Gain<S> one = {1, 0}, none = {0, 0};
  Gain<S> a[kRunChunks], ga = one;
  S b[kRunChunks], gb = 0;
  int z[kRunChunks], reset = 0;
#pragma unroll
  for (int k = 0; k < kRunChunks; k++) {
    const bool in = c0 + k < r.chunks;
    const int64_t from = (int64_t)(in ? c0 + k : 0) * r.dim + at;
    a[k] = in ? Gain<S>{chunks.a[from], chunks.e[from]} : one;
    b[k] = in ? chunks.b[from] : (S)0;
    z[k] = in ? chunks.resets[c0 + k] : 0;
  }
  auto step = [&](int k) {
    gb = z[k] ? b[k] : a[k].of(gb, b[k]);
    ga = z[k] ? none : a[k].after(ga);
    reset |= z[k];
  };
#pragma unroll
  for (int k = 0; k < kRunChunks; k++) step(k);
  // inclusive over the runs in doubling steps
  for (int off = 16; off < 1024; off *= 2) {
    s_a[me] = ga;
    s_b[me] = gb;
    s_reset[me] = reset;
    __syncthreads();
    if (me >= off && !reset) {
      gb = ga.of(s_b[me - off], gb);
      reset = s_reset[me - off];
      ga = reset ? none : ga.after(s_a[me - off]);
    }
    __syncthreads();
  }
  s_a[me] = ga;
  s_b[me] = gb;
  s_reset[me] = reset;
  __syncthreads();
  if (col < r.dim && me >= 1008) {
    const int64_t to = (int64_t)blockIdx.y * r.dim + col;
    segments.a[to] = ga.m;
    segments.e[to] = ga.e;
    segments.b[to] = gb;
    if (col == 0) segments.resets[blockIdx.y] = reset;
  }
  ga = me >= 16 ? s_a[me - 16] : one;
  gb = me >= 16 ? s_b[me - 16] : (S)0;
  reset = me >= 16 ? s_reset[me - 16] : 0;
  if (col >= r.dim) return;
#pragma unroll
  for (int k = 0; k < kRunChunks; k++) {
    if (c0 + k >= r.chunks) break;
    const int64_t to = (int64_t)(c0 + k) * r.dim + col;
    chunks.a[to] = ga.m;
    chunks.e[to] = ga.e;
    chunks.b[to] = gb;
    if (col == 0) before[c0 + k] = reset;
    step(k);
  }
}

// Steps 1 and 2 in one, where segments of 256 / 2^wide chunks are few: a workgroup takes one, 2^wide pieces across,
// and step 3 folds the segments before a chunk from the last one with a pack's start.  With the pack arrays, every row a
// pack / one pack: 4096 rows of 64 columns, float, 11.5 / 18.9 us, in three launches 15.6 / 17.9; 8192 rows of 1024, bf16,
// 22.5 / 44.8, in three launches 33.5 / 39.9.
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(256) recur_segment_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                          const T *__restrict__ init,
                                                          Composed<typename StateOf<T>::S> chunks,
                                                          int32_t *__restrict__ before,
                                                          Composed<typename StateOf<T>::S> segments) {
  using S = typename StateOf<T>::S;
  __shared__ S s_m[V][256], s_b[V][256];  // a column's, side by side: no bank conflicts
  __shared__ int s_e[V][256], s_reset[256];
  const int me = threadIdx.x, w = 1 << r.wide;
  const int64_t c = (int64_t)blockIdx.y * (256 >> r.wide) + (me >> r.wide);
  const int64_t piece = (int64_t)blockIdx.x * w + (me & (w - 1)), col = r.column<V>(piece);
  const bool live = c < r.chunks && piece < r.cols;
  Gain<S> ga[V];
  Pack<S, V> gb;
#pragma unroll
  for (int v = 0; v < V; v++) {
    ga[v] = {1, 0};
    gb.v[v] = 0;
  }
  int reset = 0;
  if (live) {
    const int64_t begin = c * r.chunk, end = min((int64_t)r.n, begin + r.chunk);
    reset = recur_compose<T, V, GRAD>(r, a, x, init, begin, end, col, ga, gb.v);
  }
  auto publish = [&]() {
#pragma unroll
    for (int v = 0; v < V; v++) {
      s_m[v][me] = ga[v].m;
      s_e[v][me] = ga[v].e;
      s_b[v][me] = gb.v[v];
    }
    s_reset[me] = reset;
    __syncthreads();
  };
  // inclusive over the chunks in doubling steps; nothing to do where every chunk has a reset
  if (__syncthreads_or(live && !reset)) {
    for (int off = w; off < 256; off *= 2) {
      publish();
      if (me >= off && !reset) {
        reset = s_reset[me - off];
#pragma unroll
        for (int v = 0; v < V; v++) {
          gb.v[v] = ga[v].of(s_b[v][me - off], gb.v[v]);
          ga[v] = reset ? Gain<S>{0, 0} : ga[v].after({s_m[v][me - off], s_e[v][me - off]});
        }
      }
      __syncthreads();
    }
  }
  publish();
  if (piece < r.cols && me >= 256 - w) {
    store_gains<V>(segments, (int64_t)blockIdx.y * r.dim + col, ga);
    store_pack<V>(segments.b + (int64_t)blockIdx.y * r.dim + col, gb);
    if (piece == 0) segments.resets[blockIdx.y] = reset;
  }
  if (!live) return;
#pragma unroll
  for (int v = 0; v < V; v++) {
    ga[v] = me >= w ? Gain<S>{s_m[v][me - w], s_e[v][me - w]} : Gain<S>{1, 0};
    gb.v[v] = me >= w ? s_b[v][me - w] : (S)0;
  }
  store_gains<V>(chunks, c * r.dim + col, ga);
  store_pack<V>(chunks.b + c * r.dim + col, gb);
  if (piece == 0) before[c] = me >= w ? s_reset[me - w] : 0;
}

// Rows [begin, end) of a piece of columns walked and written, from the state before them where it is `carried`
template <typename T, int V, bool GRAD>
__device__ __forceinline__ void recur_walk(const Recur &r, const T *__restrict__ a, const T *__restrict__ x,
                                           const T *__restrict__ h, const T *__restrict__ init, int64_t begin,
                                           int64_t end, int64_t col, bool carried,
                                           typename StateOf<T>::S (&state)[V], T *__restrict__ out,
                                           T *__restrict__ da, T *__restrict__ dinit) {
  using S = typename StateOf<T>::S;
  using P = Pack<T, V>;
  const int64_t n = r.n;
  auto at = [&](const T *p, int64_t i) { return load_pack<V>(p + r.row(i) * r.dim + col); };
  int ids[kAheadWrite + 2];  // of the rows before, of and after a batch
#pragma unroll
  for (int u = 0; u < kAheadWrite + 2; u++) ids[u] = r.id(begin - 1 + u);
  P gate = {};  // GRAD: the gate of the row walked before
  if (GRAD && carried) gate = at(a, begin - 1);
  for (int64_t i0 = begin; i0 < end; i0 += kAheadWrite) {
    P av[kAheadWrite], xv[kAheadWrite], hv[kAheadWrite];
    int next_ids[kAheadWrite + 2];
#pragma unroll
    for (int u = 0; u < kAheadWrite; u++) {  // past the last row: that row again
      const int64_t i = min(i0 + u, end - 1);
      av[u] = at(a, i);
      xv[u] = at(x, i);
      // the state on the far side of a pack's border is its initial one; GRAD: elsewhere the forward's before
      // this row, which is that of the next row walked
      const bool none = ids[u + 1] < 0, border = GRAD ? ids[u + 2] != ids[u + 1] : ids[u + 1] != ids[u];
      hv[u] = P{};
      if (border) {
        if (init && !none && ids[u + 1] < r.packs && i0 + u < end)
          hv[u] = load_pack<V>(init + (int64_t)ids[u + 1] * r.dim + col);
      } else if (GRAD) {
        hv[u] = at(h, min(i + 1, n - 1));
      }
    }
#pragma unroll
    for (int u = 0; u < kAheadWrite + 2; u++) next_ids[u] = r.id(i0 + kAheadWrite - 1 + u);
#pragma unroll
    for (int u = 0; u < kAheadWrite; u++) {
      const int64_t i = i0 + u;
      if (i >= end) continue;
      const bool none = ids[u + 1] < 0, start = none || ids[u + 1] != ids[u], last = ids[u + 2] != ids[u + 1];
      const bool from = init && !none && ids[u + 1] < r.packs;
      const int64_t to = r.row(i) * r.dim + col;
      P y;
      if (GRAD) {
        P dy;
#pragma unroll
        for (int v = 0; v < V; v++) {
          const S b = (S)xv[u].v[v], with = fma((S)gate.v[v], state[v], b);
          state[v] = none ? (S)0 : start ? b : with;
          y.v[v] = (T)state[v];
          dy.v[v] = (T)(none ? (S)0 : state[v] * (S)hv[u].v[v]);
        }
        gate = av[u];
        store_pack<V>(da + to, dy);
        if (dinit && last && from) {
          P d;
#pragma unroll
          for (int v = 0; v < V; v++) d.v[v] = (T)((S)av[u].v[v] * state[v]);
          store_pack<V>(dinit + (int64_t)ids[u + 1] * r.dim + col, d);
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; v++) {
          const S b = (S)xv[u].v[v], h0 = (S)hv[u].v[v], prev = start ? h0 : state[v];
          const S with = fma((S)av[u].v[v], prev, b);
          state[v] = none ? (S)0 : start && !from ? b : with;
          y.v[v] = (T)state[v];
        }
      }
      store_pack<V>(out + to, y);
    }
#pragma unroll
    for (int u = 0; u < kAheadWrite + 2; u++) ids[u] = next_ids[u];
  }
}

// Step 3.  Threads past the chunks write the gradients of initial states that no pack has.
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(256) recur_write_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                        const T *__restrict__ h, const T *__restrict__ init,
                                                        ComposedIn<typename StateOf<T>::S> chunks,
                                                        const int32_t *__restrict__ chunk_before,
                                                        ComposedIn<typename StateOf<T>::S> segments,
                                                        T *__restrict__ out, T *__restrict__ da,
                                                        T *__restrict__ dinit) {
  using S = typename StateOf<T>::S;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, place = t / r.cols, col = r.column<V>(t - place * r.cols);
  const int64_t c = r.chunks - 1 - place;
  const int lane = threadIdx.x & 63;
  const uint64_t marks = ballot(lane < r.few && segments.resets[lane] != 0);
  if (c < 0) {
    const int64_t p = -1 - c;
    if (dinit && p < r.packs && (p >= r.n || r.starts[p] >= r.n))
      store_pack<V>(dinit + p * r.dim + col, Pack<T, V>{});
    return;
  }
  const int64_t begin = c * r.chunk, end = min((int64_t)r.n, begin + r.chunk);
  const bool carried = r.carried(begin);
  S state[V];
#pragma unroll
  for (int v = 0; v < V; v++) state[v] = 0;
  if (carried) {
    auto step = [&](const ComposedIn<S> &m, int64_t k, bool reset) {
      const Pack<S, V> ka = load_pack<V>(m.a + k * r.dim + col), kb = load_pack<V>(m.b + k * r.dim + col);
      const Pack<int32_t, V> ke = load_pack<V>(m.e + k * r.dim + col);
#pragma unroll
      for (int v = 0; v < V; v++) {
        const S with = Gain<S>{ka.v[v], ke.v[v]}.of(state[v], kb.v[v]);
        state[v] = reset ? kb.v[v] : with;
      }
    };
    const bool here = chunk_before[c] != 0;
    if (!here) {
      const int64_t mine = c >> r.segment;
      int64_t k = mine - 1;
      if (r.few) {
        const uint64_t left = marks & (((uint64_t)1 << mine) - 1);
        k = left ? 63 - __clzll(left) : 0;
        constexpr int kFold = V >= 4 ? 4 : 8;  // loads in flight together
        for (; k < mine; k += kFold) {
          Pack<S, V> ka[kFold], kb[kFold];
          Pack<int32_t, V> ke[kFold];
#pragma unroll
          for (int u = 0; u < kFold; u++) {
            const int64_t at = min(k + u, mine - 1) * r.dim + col;
            ka[u] = load_pack<V>(segments.a + at);
            ke[u] = load_pack<V>(segments.e + at);
            kb[u] = load_pack<V>(segments.b + at);
          }
#pragma unroll
          for (int u = 0; u < kFold; u++) {
            const bool in = k + u < mine, reset = marks >> ((k + u) & 63) & 1;
#pragma unroll
            for (int v = 0; v < V; v++) {
              const S with = Gain<S>{ka[u].v[v], ke[u].v[v]}.of(state[v], kb[u].v[v]);
              state[v] = !in ? state[v] : reset ? kb[u].v[v] : with;
            }
          }
        }
      } else {
        while (k > 0 && !segments.resets[k]) k--;
        for (; k >= 0 && k < mine; k++) step(segments, k, segments.resets[k] != 0);
      }
    }
    step(chunks, c, here);
  }
  recur_walk<T, V, GRAD>(r, a, x, h, init, begin, end, col, carried, state, out, da, dinit);
}

// All three steps in one launch, for up to kShortRows rows (one step of a batch of sequences): a workgroup takes one
// piece of columns, each thread a row of it.  256 rows of 1024 columns, bf16, with the pack arrays: 7.0 us if every row
// is a pack and 13.8 us if one pack has them all, 11.3 and 17.3 in two launches.  Rows of one piece lie in different
// lines of memory: with four rows a thread 1024 rows took 19 and 32 us, in two launches 12 and 17, and 256 rows of 512
// pieces (2048 columns, float) 12 and 19 us, in two launches 11 and 15 (64 rows of them 6.4 and 9.4 us, 10 and 13).
constexpr int kShortRows = 256, kShortPieces = 1 << 16;  // pieces: of all rows
template <typename T, int V, bool GRAD>
__global__ void __launch_bounds__(kShortRows) recur_short_kernel(Recur r, const T *__restrict__ a, const T *__restrict__ x,
                                                         const T *__restrict__ h, const T *__restrict__ init,
                                                         T *__restrict__ out, T *__restrict__ da,
                                                         T *__restrict__ dinit) {
  using S = typename StateOf<T>::S;
  constexpr int kWaves = kShortRows / 64;
  __shared__ Gain<S> s_a[kWaves][V];
  __shared__ S s_b[kWaves][V];
  __shared__ int s_reset[kWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t col = r.column<V>(blockIdx.x);
  const int64_t begin = threadIdx.x, end = begin + 1;
  const bool live = begin < r.n, carried = live && r.carried(begin);
  Gain<S> ga[V];
  S gb[V];
#pragma unroll
  for (int v = 0; v < V; v++) {
    ga[v] = {1, 0};
    gb[v] = 0;
  }
  auto shifted = [](const Gain<S> &g, int off) { return Gain<S>{__shfl_up(g.m, off), __shfl_up(g.e, off)}; };
  int reset = 0;
  if (live) reset = recur_compose<T, V, GRAD>(r, a, x, init, begin, end, col, ga, gb);
  const bool needed = __any(carried);  // a thread whose state is not carried has a reset
  if (needed) {
    // inclusive over the wave in doubling steps
    for (int off = 1; off < 64; off *= 2) {
      const int before = __shfl_up(reset, off);
      const bool in = lane >= off && !reset;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const Gain<S> pa = shifted(ga[v], off);
        const S pb = __shfl_up(gb[v], off);
        gb[v] = in ? ga[v].of(pb, gb[v]) : gb[v];
        ga[v] = in ? (before ? Gain<S>{0, 0} : ga[v].after(pa)) : ga[v];
      }
      reset = in ? before : reset;
    }
  }
  if (lane == 63) {
#pragma unroll
    for (int v = 0; v < V; v++) {
      s_a[wave][v] = ga[v];
      s_b[wave][v] = gb[v];
    }
    s_reset[wave] = reset;
  }
  __syncthreads();
  S state[V];
#pragma unroll
  for (int v = 0; v < V; v++) state[v] = 0;
  if (needed) {
    for (int w = 0; w < wave; w++) {
#pragma unroll
      for (int v = 0; v < V; v++) state[v] = s_reset[w] ? s_b[w][v] : s_a[w][v].of(state[v], s_b[w][v]);
    }
    const int before = __shfl_up(reset, 1);
#pragma unroll
    for (int v = 0; v < V; v++) {
      const Gain<S> pa = shifted(ga[v], 1);
      const S pb = __shfl_up(gb[v], 1), with = before ? pb : pa.of(state[v], pb);
      state[v] = lane > 0 ? with : state[v];
    }
  }
  if (!carried) {
#pragma unroll
    for (int v = 0; v < V; v++) state[v] = 0;
  }
  if (live) recur_walk<T, V, GRAD>(r, a, x, h, init, begin, end, col, carried, state, out, da, dinit);
  if (dinit) {
    for (int64_t p = threadIdx.x; p < r.packs; p += blockDim.x) {
      if (p >= r.n || r.starts[p] >= r.n) store_pack<V>(dinit + p * r.dim + col, Pack<T, V>{});
    }
  }
}

// Elements of a thread's piece: 16 bytes; one where rows are not whole numbers of such pieces and there are few of
// them, so that more threads share the work (20,070 rows of 676, bf16, training, 164 us by elements and 106 by pieces;
// 6030 of 140 36 and 49).
static int recur_piece(int64_t n, int64_t dim, size_t esize) {
  const int64_t v = 16 / (int64_t)esize;
  return dim % v == 0 || (dim > v && n * cdiv(dim, v) >= 1 << 17) ? (int)v : 1;
}

// Rows of a chunk: 2^17 threads keep the memory busy; longer chunks from there on, for fewer (A, B)
static int recur_chunk_rows(kl_dtype dtype, int64_t n, int64_t dim) {
  const int64_t cols = cdiv(dim, recur_piece(n, dim, dtype == KL_F64 ? 8 : dtype == KL_F32 ? 4 : 2));
  return (int)std::min<int64_t>(64, std::max<int64_t>(8, cdiv(n * cols, 1 << 17)));
}

// The workspace: (A, B) of chunks and of segments
template <typename S>
struct RecurSpace {
  Composed<S> chunks = {}, segments = {};
  int32_t *before = nullptr;
  size_t bytes = 0;
  RecurSpace(char *ws, int64_t num_chunks, int64_t dim) {
    auto take = [&](size_t n) {
      char *p = ws ? ws + bytes : nullptr;
      bytes += al256(n);
      return p;
    };
    const int64_t num = std::max(cdiv(num_chunks, kSegment), std::min<int64_t>(cdiv(num_chunks, 16), kFewSegments));
    chunks.a = (S *)take(num_chunks * dim * sizeof(S));
    chunks.b = (S *)take(num_chunks * dim * sizeof(S));
    segments.a = (S *)take(num * dim * sizeof(S));
    segments.b = (S *)take(num * dim * sizeof(S));
    chunks.e = (int32_t *)take(num_chunks * dim * 4);
    segments.e = (int32_t *)take(num * dim * 4);
    chunks.resets = (int32_t *)take(num_chunks * 4);
    before = (int32_t *)take(num_chunks * 4);
    segments.resets = (int32_t *)take(num * 4);
  }
};

template <typename T, int V, bool GRAD>
static int recur_run(Recur r, const void *a, const void *x, const void *h, const void *init, void *out, void *da,
                     void *dinit, void *ws, hipStream_t st) {
  using S = typename StateOf<T>::S;
  r.cols = cdiv(r.dim, V);
  if (r.n > 1 && r.n <= kShortRows && r.n * r.cols <= kShortPieces) {
    hipLaunchKernelGGL((recur_short_kernel<T, V, GRAD>), dim3((unsigned)r.cols), dim3((unsigned)cdiv(r.n, 64) * 64), 0, st, r, (const T *)a,
                       (const T *)x, (const T *)h, (const T *)init, (T *)out, (T *)da, (T *)dinit);
    KL_CHECK_LAUNCH();
    return KL_OK;
  }
  const RecurSpace<S> m((char *)ws, r.chunks, r.dim);
  r.segment = kSegmentLog;
  while (r.wide < 4 && 1 << r.wide < r.cols) r.wide++;
  const int64_t segments = cdiv(r.chunks, 256 >> r.wide);
  if (r.chunks > 1 && segments <= kFewSegments) {
    r.segment = 8 - r.wide;
    r.few = (int)segments;
    hipLaunchKernelGGL((recur_segment_kernel<T, V, GRAD>),
                       dim3((unsigned)cdiv(r.cols, 1 << r.wide), (unsigned)segments), dim3(256), 0, st, r, (const T *)a,
                       (const T *)x, (const T *)init, m.chunks, m.before, m.segments);
    KL_CHECK_LAUNCH();
  } else if (r.chunks > 1) {
    const int64_t all = cdiv(r.chunks, kSegment);
    r.few = all <= kFewSegments ? (int)all : 0;
    hipLaunchKernelGGL((recur_chunk_kernel<T, V, GRAD>), dim3((unsigned)cdiv(r.chunks * r.cols, 256)), dim3(256), 0, st,
                       r, (const T *)a, (const T *)x, (const T *)init, m.chunks);
    KL_CHECK_LAUNCH();
    hipLaunchKernelGGL(recur_scan_kernel<S>, dim3((unsigned)cdiv(r.dim, 16), (unsigned)cdiv(r.chunks, kSegment)),
                       dim3(1024), 0, st, r, m.chunks, m.before, m.segments);
    KL_CHECK_LAUNCH();
  }
  const dim3 grid((unsigned)cdiv((r.chunks + (dinit ? (int64_t)r.packs : 0)) * r.cols, 256));
  hipLaunchKernelGGL((recur_write_kernel<T, V, GRAD>), grid, dim3(256), 0, st, r, (const T *)a, (const T *)x,
                     (const T *)h, (const T *)init, ComposedIn<S>{m.chunks.a, m.chunks.b, m.chunks.e, m.chunks.resets},
                     m.before, ComposedIn<S>{m.segments.a, m.segments.b, m.segments.e, m.segments.resets}, (T *)out,
                     (T *)da, (T *)dinit);
  KL_CHECK_LAUNCH();
  return KL_OK;
}

template <typename T>
static int recur_type(const Recur &r, bool grad, const void *a, const void *x, const void *h, const void *init,
                      void *out, void *da, void *dinit, void *ws, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool pieces = recur_piece(r.n, r.dim, sizeof(T)) == V;
  if (grad) {
    return pieces ? recur_run<T, V, true>(r, a, x, h, init, out, da, dinit, ws, st)
                  : recur_run<T, 1, true>(r, a, x, h, init, out, da, dinit, ws, st);
  }
  return pieces ? recur_run<T, V, false>(r, a, x, h, init, out, da, dinit, ws, st)
                : recur_run<T, 1, false>(r, a, x, h, init, out, da, dinit, ws, st);
}

static int recurrence(kl_dtype dtype, bool down, bool grad, int64_t n, int64_t dim, int64_t packs, const void *a,
                      const void *x, const void *h, const void *init, const int32_t *ids, const int32_t *starts,
                      void *out, void *da, void *dinit, void *ws, size_t ws_bytes, hipStream_t st) {
  KL_REQUIRE(n >= 0 && n < ((int64_t)1 << 31) - 256 && dim >= 0 && dim < (int64_t)1 << 24 && packs >= 0 &&
                 packs < (int64_t)1 << 31,
             "linear_recurrence: sizes out of range");
  KL_REQUIRE(cdiv((cdiv(n, 8) + packs) * dim, 256) < (int64_t)1 << 31 &&
                 cdiv(n, recur_chunk_rows(dtype, n, dim)) <= (int64_t)kSegment * 65535,
             "linear_recurrence: too many elements");
  KL_REQUIRE(ws_bytes >= kl_linear_recurrence_workspace_bytes(dtype, n, dim),
             "linear_recurrence: the workspace is too small");
  if (dim == 0 || (n == 0 && !(dinit && packs))) return KL_OK;
  Recur r = {};
  r.n = (int)n;
  r.dim = dim;
  r.chunk = recur_chunk_rows(dtype, n, dim);
  r.chunks = (int)cdiv(n, r.chunk);
  r.down = down ? 1 : 0;
  r.packs = init ? (int)packs : 0;
  r.ids = ids;
  r.starts = starts;
  switch (dtype) {
    case KL_F32: return recur_type<float>(r, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_F64: return recur_type<double>(r, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_F16: return recur_type<f16_t>(r, grad, a, x, h, init, out, da, dinit, ws, st);
    case KL_BF16: return recur_type<bf16_t>(r, grad, a, x, h, init, out, da, dinit, ws, st);
    default: set_error("linear_recurrence: expected a Half, BFloat16, Float or Double tensor"); return KL_E_INVALID;
  }
}

}  // namespace kl

using namespace kl;

extern "C" size_t kl_linear_recurrence_workspace_bytes(kl_dtype dtype, int64_t num_rows, int64_t dim) {
  if (num_rows <= 0 || dim <= 0) return 256;
  const size_t chunks = (size_t)cdiv(num_rows, recur_chunk_rows(dtype, num_rows, dim));
  return dtype == KL_F64 ? RecurSpace<double>(nullptr, chunks, dim).bytes : RecurSpace<float>(nullptr, chunks, dim).bytes;
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
