// Blocks of the KV pool copied to other blocks, and moved (copied, with the
// block tables redirected).
//
//   pool[plane][dst[i]] = pool[plane][src[i]]   for every plane and pair i
//   tables[t] = dst[i]  where tables[t] == src[i]                (move only)
//
// A plane is what one stride of num_blocks * block_bytes covers: K or V of a
// layer in the bf16 pool, a whole layer in the FP8 pool; both keep a block's
// bytes of one plane contiguous.  Pure memory traffic, 2 * planes * pairs *
// block_bytes: 16-byte loads, kUnroll of them in flight per thread before the
// first store, a grid of a few waves striding over (plane, pair) units.
#include "pkv_device.cuh"
#include "pkv_kernels.h"

namespace pkv {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kUnroll = 2;      // 16-byte loads in flight per thread and unit
constexpr int kCtasPerSm = 8;   // 2048 threads

struct PageParams {
  uint8_t* pool;
  int64_t plane_stride;  // bytes
  int64_t block_bytes;
  const int32_t* src;
  const int32_t* dst;
  int32_t* tables;  // nullptr: copy only
  int64_t pitch;
  int64_t units;  // planes * n
  int32_t n, num_blocks, table_rows, table_cols, copy_ctas;
  int32_t* err;
};

// The table entries that name a moved block.  src ascends, so an entry is
// looked up by bisection, and one outside [src[0], src[n - 1]] (every block
// that stays, after a compaction) is left after the first comparison.
__device__ void redirect_tables(const PageParams& p) {
  const int lo_id = p.src[0], hi_id = p.src[p.n - 1];
  const int64_t total = static_cast<int64_t>(p.table_rows) * p.table_cols;
  const int64_t step = static_cast<int64_t>(gridDim.x - p.copy_ctas) * kCopyThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x - p.copy_ctas) * kCopyThreads + threadIdx.x;
       i < total; i += step) {
    const int64_t row = i / p.table_cols;
    int32_t* cell = p.tables + row * p.pitch + (i - row * p.table_cols);
    const int id = *cell;
    if (id < lo_id || id > hi_id) continue;
    int a = 0, z = p.n;  // first index whose src is >= id
    while (a < z) {
      const int mid = (a + z) >> 1;
      if (__ldg(p.src + mid) < id)
        a = mid + 1;
      else
        z = mid;
    }
    if (a < p.n && __ldg(p.src + a) == id) {
      const int to = __ldg(p.dst + a);
      if (to >= 0 && to < p.num_blocks && id >= 0 && id < p.num_blocks) *cell = to;
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const PageParams p) {
  pdl_trigger();
  pdl_wait();
  if (static_cast<int>(blockIdx.x) >= p.copy_ctas) {
    redirect_tables(p);
    return;
  }
  const DevErr err{p.err};
  for (int64_t u = blockIdx.x; u < p.units; u += p.copy_ctas) {
    const int64_t plane = u / p.n;
    const int pair = static_cast<int>(u - plane * p.n);
    const int s = __ldg(p.src + pair), d = __ldg(p.dst + pair);
    if ((s < 0 && d < 0) || s == d) continue;  // a padding pair, or nothing to do
    if (s < 0 || d < 0 || s >= p.num_blocks || d >= p.num_blocks) {
      if (threadIdx.x == 0) err.raise(PKV_DEVERR_BLOCK_ID);
      continue;
    }
    uint8_t* base = p.pool + plane * p.plane_stride;
    const uint8_t* from = base + s * p.block_bytes;
    uint8_t* to = base + d * p.block_bytes;
    for (int64_t o = threadIdx.x * 16; o < p.block_bytes; o += kUnroll * kCopyThreads * 16) {
      uint4 v[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int64_t at = o + k * kCopyThreads * 16;
        if (at < p.block_bytes) v[k] = __ldcs(reinterpret_cast<const uint4*>(from + at));
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int64_t at = o + k * kCopyThreads * 16;
        if (at < p.block_bytes) __stcs(reinterpret_cast<uint4*>(to + at), v[k]);
      }
    }
  }
}

}  // namespace

cudaError_t launch_copy_blocks(const PageLaunch& a, cudaStream_t stream) {
  PageParams p{};
  p.pool = static_cast<uint8_t*>(a.pool);
  p.plane_stride = a.plane_stride;
  p.block_bytes = a.block_bytes;
  p.src = a.src;
  p.dst = a.dst;
  p.tables = a.tables;
  p.pitch = a.table_pitch;
  p.n = a.n;
  p.num_blocks = a.num_blocks;
  p.table_rows = a.table_rows;
  p.table_cols = a.table_cols;
  p.units = static_cast<int64_t>(a.num_planes) * a.n;
  p.err = a.err;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t most = static_cast<int64_t>(sms) * kCtasPerSm;
  p.copy_ctas = static_cast<int32_t>(p.units < most ? p.units : most);
  int64_t table_ctas = 0;
  if (a.tables) {
    const int64_t cells = static_cast<int64_t>(a.table_rows) * a.table_cols;
    table_ctas = (cells + 4 * kCopyThreads - 1) / (4 * kCopyThreads);
    if (table_ctas > sms) table_ctas = sms;
  }
  return launch_k(copy_blocks_kernel, dim3(static_cast<unsigned>(p.copy_ctas + table_ctas)),
                  dim3(kCopyThreads), 0, stream, p);
}

}  // namespace pkv
