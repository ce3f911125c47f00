// packs.hip -- the pack arrays of a boundary mask (seqcommon.h): each row's pack and each pack's first
// row, with nothing read back, so the operators that use them can be captured into a graph.
//
// A workgroup counts the marks of the rows before its own and of all rows, then writes its part.  Up to
// kOneLaunchRows rows every workgroup counts the whole mask itself (one byte a row, from L2), in one
// launch; past that a first launch leaves one count per workgroup.  Two masks share their launches: each takes
// some 4 us, whatever a small mask's few workgroups have to do (16,385 rows 5.6 us, 311,094 rows 5 + 6).
#include "seqcommon.h"

namespace kl {

constexpr int kLayoutRows = 1024;        // rows per workgroup: 256 threads of four
constexpr int64_t kOneLaunchRows = 65536;  // 64 KB per workgroup and 64 workgroups

__device__ __forceinline__ int block_sum(int v, int *s_wave) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  const int t = s_wave[0] + s_wave[1] + s_wave[2] + s_wave[3];
  __syncthreads();
  return t;
}

// marks among rows [begin, end): 16 rows a thread where the address allows
__device__ __forceinline__ int count_marks(const uint8_t *__restrict__ b, int64_t begin, int64_t end) {
  int n = 0;
  const int64_t head = min(end, begin + (int64_t)((16 - ((uintptr_t)(b + begin) & 15)) & 15));
  if (begin + threadIdx.x < head) n += b[begin + threadIdx.x] != 0;
  const int64_t vecs = (end - head) / 16;
  const uint4 *v = reinterpret_cast<const uint4 *>(b + head);
  for (int64_t i = threadIdx.x; i < vecs; i += 256) {
    const uint4 w = v[i];
    // a byte of a mask is 0 or 1; any non-zero byte counts once all the same
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; k++) n += __popc(((((x[k] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x[k]) & 0x80808080u));
  }
  const int64_t tail = head + vecs * 16;
  if (tail + threadIdx.x < end) n += b[tail + threadIdx.x] != 0;
  return n;
}

struct Mask {
  const uint8_t *b;
  int64_t n;
  int blocks;               // 0: no mask
  int32_t *counts;          // NULL: every workgroup counts
  int32_t *ids, *starts;
};

__global__ void __launch_bounds__(256) pack_count_kernel(Mask one, Mask two) {
  __shared__ int s_wave[4];
  const bool is_two = (int)blockIdx.x >= one.blocks;
  const Mask m = is_two ? two : one;
  const int block = (int)blockIdx.x - (is_two ? one.blocks : 0);
  if (!m.counts) return;
  const int64_t begin = (int64_t)block * kLayoutRows;
  const int c = block_sum(count_marks(m.b, begin, min(m.n, begin + kLayoutRows)), s_wave);
  if (threadIdx.x == 0) m.counts[block] = c;
}

__global__ void __launch_bounds__(256) pack_layout_kernel(Mask one, Mask two) {
  __shared__ int s_wave[4];
  const bool is_two = (int)blockIdx.x >= one.blocks;
  const Mask m = is_two ? two : one;
  const int block = (int)blockIdx.x - (is_two ? one.blocks : 0);
  const uint8_t *b = m.b;
  int32_t *ids = m.ids, *starts = m.starts;
  const int64_t n = m.n, first = (int64_t)block * kLayoutRows;
  int before = 0, all = 0;
  if (m.counts) {
    for (int i = threadIdx.x; i < m.blocks; i += 256) {
      const int c = m.counts[i];
      all += c;
      before += i < block ? c : 0;
    }
  } else {
    before = count_marks(b, 0, first);
    all = before + count_marks(b, first, n);
  }
  before = block_sum(before, s_wave);
  all = block_sum(all, s_wave);
  const int64_t row = first + 4 * (int64_t)threadIdx.x;
  int mark[4], mine = 0;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    mark[k] = row + k < n && b[row + k] != 0;
    mine += mark[k];
  }
  int total;
  int id = before + block_exclusive_scan(mine, s_wave, &total) - 1;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if (row + k >= n) break;
    id += mark[k];
    ids[row + k] = id;
    if (mark[k]) starts[id] = (int32_t)(row + k);
    if (row + k >= all) starts[row + k] = (int32_t)n;  // past the last pack
  }
  if (block == 0 && threadIdx.x == 0) starts[n] = (int32_t)n;
}

static int take_mask(Mask &m, const char *func, int64_t n, const uint8_t *b, int32_t *ids, int32_t *starts, char *ws) {
  KL_REQUIRE(n >= 0 && n < (int64_t)1 << 31, std::string(func) + ": the number of rows is out of range");
  m = {b, n, (int)std::max<int64_t>(1, cdiv(n, kLayoutRows)), n > kOneLaunchRows ? (int32_t *)ws : nullptr, ids, starts};
  return KL_OK;
}

static int write_layouts(const Mask &one, const Mask &two, hipStream_t st) {
  const dim3 blocks((unsigned)(one.blocks + two.blocks));
  if (one.counts || two.counts) {
    hipLaunchKernelGGL(pack_count_kernel, blocks, dim3(256), 0, st, one, two);
    KL_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL(pack_layout_kernel, blocks, dim3(256), 0, st, one, two);
  KL_CHECK_LAUNCH();
  return KL_OK;
}

}  // namespace kl

using namespace kl;

extern "C" size_t kl_pack_layout_workspace_bytes(int64_t num_rows) {
  return num_rows > kOneLaunchRows ? al256((size_t)cdiv(num_rows, kLayoutRows) * 4) : 256;
}

extern "C" int kl_pack_layout(int64_t num_rows, const uint8_t *boundaries, int32_t *ids, int32_t *starts, void *ws,
                              size_t ws_bytes, kl_stream stream) {
  Mask one, none = {};
  KL_CHECK_RC(take_mask(one, "pack_layout", num_rows, boundaries, ids, starts, (char *)ws));
  KL_REQUIRE(ws_bytes >= kl_pack_layout_workspace_bytes(num_rows), "pack_layout: the workspace is too small");
  return write_layouts(one, none, S(stream));
}

extern "C" int kl_pack_layout_pair(int64_t num_rows, const uint8_t *boundaries, int32_t *ids, int32_t *starts,
                                   int64_t num_rows2, const uint8_t *boundaries2, int32_t *ids2, int32_t *starts2,
                                   void *ws, size_t ws_bytes, kl_stream stream) {
  Mask one, two;
  const size_t bytes = num_rows < 0 ? 0 : kl_pack_layout_workspace_bytes(num_rows);
  KL_CHECK_RC(take_mask(one, "pack_layout_pair", num_rows, boundaries, ids, starts, (char *)ws));
  KL_CHECK_RC(take_mask(two, "pack_layout_pair", num_rows2, boundaries2, ids2, starts2, (char *)ws + bytes));
  KL_REQUIRE(ws_bytes >= bytes + kl_pack_layout_workspace_bytes(num_rows2),
             "pack_layout_pair: the workspace is too small");
  return write_layouts(one, two, S(stream));
}
