// Attention of the newest tokens of each sequence over its paged cache
// (tokens of all sequences packed, any number per sequence).
#include <math.h>

#include "pkv_device.cuh"
#include "pkv_kernels.h"

namespace pkv {
namespace {

struct ChunkParams {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const uint8_t* k;  // bf16 K plane, or the FP8 chunks of the layer
  const uint8_t* v;
  const int32_t* tables;
  int64_t pitch;
  const int32_t* rows;
  const int32_t* q_starts;
  const int32_t* kv_lens;
  int32_t batch, tokens, hkv, group, num_blocks, causal;
  float scale_log2;
  int32_t* err;
};

// One warp per (token, query head): lane l holds dims 4l .. 4l+3 of q and of
// the running output; keys one by one, the score summed across the warp.
template <bool kFp8>
__global__ void __launch_bounds__(128) chunk_simple_kernel(const ChunkParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int hq = p.hkv * p.group;
  const int64_t n = w / hq;
  const int head = static_cast<int>(w - n * hq);
  if (n >= p.tokens) return;
  const int h = head / p.group;
  const DevErr err{p.err};
  // the row that holds token n: the last one that starts at or before it
  int a = 0, z = p.batch;
  while (a < z) {
    const int mid = (a + z) >> 1;
    if (p.q_starts[mid + 1] <= n)
      a = mid + 1;
    else
      z = mid;
  }
  if (a >= p.batch || n < p.q_starts[a]) return;
  const int first = max(p.q_starts[a], 0), last = min(p.q_starts[a + 1], p.tokens);
  int kv = max(p.kv_lens[a], 0);
  if (kv > p.pitch * kBlockTokens) {
    if (lane == 0) err.raise(PKV_DEVERR_POSITION);
    kv = static_cast<int>(p.pitch) * kBlockTokens;
  }
  const int lim = p.causal ? min(kv, kv - (last - first) + static_cast<int>(n - first) + 1) : kv;
  const int32_t* trow = p.tables + static_cast<int64_t>(p.rows ? p.rows[a] : a) * p.pitch;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int e = 0; e < 4; ++e)
    q[e] = __bfloat162float(p.q[n * p.q_st + head * p.q_sh + lane * 4 + e]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j < lim; ++j) {
    int blk = trow[j / kBlockTokens];
    if (blk < 0 || blk >= p.num_blocks) {
      if (lane == 0) err.raise(PKV_DEVERR_BLOCK_ID);
      blk = 0;
    }
    const int t = j % kBlockTokens;
    float k[4], v[4];
    if constexpr (kFp8) {
      const uint8_t* c = p.k + (static_cast<int64_t>(blk) * p.hkv + h) * kFp8HeadBlockBytes;
      const float ks = reinterpret_cast<const float*>(c + kFp8KScaleOff)[t];
      const float vs = reinterpret_cast<const float*>(c + kFp8VScaleOff)[t];
      for (int e = 0; e < 4; ++e) {
        const int d = lane * 4 + e, x = d & 15;
        const int place = x < 8 ? 4 * (x >> 1) + (x & 1) : 4 * ((x - 8) >> 1) + 2 + (x & 1);
        const int tp = t < 8 ? 4 * (t >> 1) + (t & 1) : 4 * ((t - 8) >> 1) + 2 + (t & 1);
        uint32_t lo, hi;
        e4m3x4_to_f16x2x2(c[t * 128 + (((d >> 4) ^ (t & 7)) << 4) + place] |
                              (c[kFp8VOff + d * 16 + tp] << 8), lo, hi);
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&lo));
        k[e] = f.x * ks;
        v[e] = f.y * vs;
      }
    } else {
      const int64_t at = ((static_cast<int64_t>(blk) * kBlockTokens + t) * p.hkv + h) * kHeadDim;
      for (int e = 0; e < 4; ++e) {
        k[e] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.k)[at + lane * 4 + e]);
        v[e] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.v)[at + lane * 4 + e]);
      }
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float al = ex2(m - base), pr = ex2(s - base);
    m = mn;
    l = l * al + pr;
    for (int e = 0; e < 4; ++e) o[e] = o[e] * al + pr * v[e];
  }
  const float inv = 1.f / l;  // 0/0 -> NaN for a query that sees no key
  for (int e = 0; e < 4; ++e)
    p.out[n * p.o_st + head * p.o_sh + lane * 4 + e] = __float2bfloat16(o[e] * inv);
}

}  // namespace

size_t chunk_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

cudaError_t launch_chunk(const ChunkLaunch& a, cudaStream_t stream) {
  ChunkParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.o_st = a.o_st;
  p.o_sh = a.o_sh;
  p.k = static_cast<const uint8_t*>(a.kv8 ? a.kv8 : a.k_pool);
  p.v = static_cast<const uint8_t*>(a.v_pool);
  p.tables = a.tables;
  p.pitch = a.pitch;
  p.rows = a.rows;
  p.q_starts = a.q_starts;
  p.kv_lens = a.kv_lens;
  p.batch = a.batch;
  p.tokens = a.num_tokens;
  p.hkv = a.num_kv_heads;
  p.group = a.num_q_heads / a.num_kv_heads;
  p.num_blocks = a.num_blocks;
  p.causal = a.causal;
  p.scale_log2 = a.sm_scale * 1.4426950408889634f;
  p.err = a.err;
  const int64_t warps = static_cast<int64_t>(a.num_tokens) * a.num_q_heads;
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4));
  return a.kv8 ? launch_k(chunk_simple_kernel<true>, grid, dim3(128), 0, stream, p)
               : launch_k(chunk_simple_kernel<false>, grid, dim3(128), 0, stream, p);
}

}  // namespace pkv
