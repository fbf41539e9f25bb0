// What the two packed-chunk kernels (chunk.cu, chunk_short.cu) share.
#pragma once

#include "pkv_device.cuh"
#include "pkv_kernels.h"

namespace pkv {

// Sequences with at most this many query rows per KV head (new tokens times
// heads of a group) are the short kernel's, the others the tensor-memory one's.
constexpr int kShortRows = 32;
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
  int32_t max_parts;   // grid.x
  int32_t min_blocks;  // a partition holds at least this many
  int32_t part_rows;
  float scale_log2;
  float* part_lse;  // [sequences * hkv * max_parts][part_rows]
  float* part_o;    // ... [128]
  int32_t* err;
};

// A sequence's share of the short kernel: T = 0 if it has none.
struct ShortRow {
  int first, T, kv, nblk, per_part, nparts;
  bool cut;  // kv_len past the table
};
__device__ __forceinline__ ShortRow short_row(const ShortParams& p, int b) {
  ShortRow r;
  const int s0 = min(max(__ldg(p.q_starts + b), 0), p.tokens);
  const int s1 = min(max(__ldg(p.q_starts + b + 1), s0), p.tokens);
  const int kv = max(__ldg(p.kv_lens + b), 0);
  r.first = s0;
  r.T = s1 - s0 <= kShortRows / p.group ? s1 - s0 : 0;
  r.kv = static_cast<int>(min(static_cast<int64_t>(kv),
                              min(p.pitch, int64_t(1) << 26) * kBlockTokens));
  r.cut = kv > r.kv;
  r.nblk = (r.kv + kBlockTokens - 1) / kBlockTokens;
  // equal partitions of whole rounds of the four warps; no position: one
  // empty partition, which writes the NaN rows
  const int np = min(p.max_parts, max(1, r.nblk / p.min_blocks));
  r.per_part = max(4, ((r.nblk + np - 1) / np + 3) / 4 * 4);
  r.nparts = max(1, (r.nblk + r.per_part - 1) / r.per_part);
  return r;
}

cudaError_t launch_chunk_short(const ShortParams& p, const CUtensorMap& kmap,
                               const CUtensorMap& vmap, int32_t batch, cudaStream_t stream);

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
