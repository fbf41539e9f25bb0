// What the two packed-chunk kernels (chunk.cu, chunk_short.cu) share.
#pragma once

#include "pkv_device.cuh"
#include "pkv_kernels.h"

namespace pkv {

constexpr int kShortRows = 32;    // query rows of a chunk of the short kernel
constexpr float kLazyLog2 = 8.f;  // a running maximum moves by more than this

struct ShortParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const uint8_t* kv8;
  const int32_t* tables;
  int64_t pitch;
  const int32_t* rows;
  const int32_t* q_starts;
  const int32_t* kv_lens;
  int32_t tokens, hkv, group, num_blocks, causal;
  int32_t most_rows;   // sequences of more rows per KV head are not its
  int32_t chunks;      // of kShortRows rows, for each sequence
  int32_t min_blocks;  // a partition holds at least this many
  int32_t beside;      // launched right behind chunk.cu's kernel, to run beside it
  float scale_log2;
  int32_t* err;
};

// parts: partitions of a sequence's blocks at most, a power of two up to 16
cudaError_t launch_chunk_short(const ShortParams& p, const CUtensorMap& kmap,
                               const CUtensorMap& vmap, int32_t batch, int32_t parts,
                               cudaStream_t stream);

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3, int c4,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "l"(policy)
      : "memory");
}

}  // namespace pkv
