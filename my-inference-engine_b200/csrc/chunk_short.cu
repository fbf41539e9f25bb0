// Packed-chunk attention, sequences of few new tokens (at most 32 query rows,
// tokens times heads of a group, per KV head), and small calls altogether, in
// chunks of 32 rows.  HBM-bound: every K/V block is read once for the chunk.
//
//   grid    = (partitions, KV heads, sequences x chunks)
//   cluster = the partitions of one unit (up to 16): they join through
//             distributed shared memory, so a call is one launch and needs no
//             workspace
//   block   = 4 warps; warp w takes blocks w, w + 4, ... of its partition and
//             streams them through its own ring of copies (bf16: TMA boxes of
//             K and V; FP8: one bulk copy of the block's chunk)
//
// One warp, one 16-token block, keys in M and query rows in N (mma.sync
// m16n8k16; NT tiles of 8 rows: token n / group, head n % group):
//   S^T[16 x 8 NT]  = K[16 x 128] . Q^T       Q fragments from shared memory
//   online softmax per row over the lanes that hold its 16 keys, its base
//   moved (and O rescaled) only when a score passes it by more than 2^8
//   O^T[128 x 8 NT] += V^T[128 x 16] . P^T    P^T by movmatrix, V^T by
//                                             ldmatrix.trans
// FP8: fragments are e4m3 pairs widened to f16 in registers (exact), q / 16 as
// f16, the key's scale applied to its scores and the value's to its
// probabilities after the row's sum, relative to 4 times the largest scale that
// the warp has met (its `cap`): the product is a f16 of up to 2^15, off by at
// most 2^-11 of itself, or 2^-30 of the row's largest probability times the
// largest value where it falls below f16's normal range, so that thousands of
// small terms of a long cache keep their weight.  (Values that a row does not
// see, or that have no weight, raise the cap too.)  bf16: probabilities are
// rounded to bf16, by at most 2^-8 of themselves, since both operands of a
// product have the pool's type.
// The warps join in shared memory, then the partitions.  Every row's partitions
// follow from its own length, so a captured call replays for other lengths.
//
// mma.sync runs at about a tenth of the tensor cores' rate: 32 rows of bf16
// are bound by it (64 sequences of up to 5 tokens at 6 heads, 347 MB: 83 us
// here, 73 us in chunk.cu), 16 are not.
#include <math.h>

#include <atomic>

#include "chunk.cuh"

namespace pkv {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxNT = kShortRows / 8;

template <bool kFp8>
struct Short {
  static constexpr int kStageBytes = kFp8 ? kFp8HeadBlockBytes : 2 * kHeadBlockBytes;
  static constexpr int kStages = kFp8 ? 5 : 3;
  static constexpr int kOffQ = kWarps * kStages * kStageBytes;    // [32][128] 16-bit, swizzled
  static constexpr int kOffBar = kOffQ + kShortRows * 256;
  static constexpr int kSmem = kOffBar + kWarps * kStages * 8 + 1024;
  // where the CTA leaves its joined rows for the cluster: [32][128], [32][2]
  static constexpr int kOffJoin = kWarps * kShortRows * (kHeadDim + 2) * 4;
  static_assert(kOffQ >= kOffJoin + kShortRows * (kHeadDim + 2) * 4,
                "the join of the warps reuses the ring");
  static_assert(kSmem <= 113 * 1024, "two CTAs per SM");
};

// Four bf16 or f16 8x8 fragments.
template <bool kFp8>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (kFp8)
    mma_f16(d, a0, a1, a2, a3, b0, b1);
  else
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
}

// A cluster's barrier, and 16 bytes of another of its CTAs' shared memory.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 cluster_ld4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 cluster_ld2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

struct ShortItem {
  int first, T, kv;      // packed token, tokens, positions
  int row0, rows;        // the chunk's rows of the sequence
  int blk0, blk1;        // blocks of this partition
  int part, nparts;
  const int32_t* trow;
};

// One partition of one (sequence, KV head) with at most 8 NT rows.
template <bool kFp8, int NT>
__device__ __forceinline__ void short_part(const ShortParams& p, const CUtensorMap* kmap,
                                           const CUtensorMap* vmap, uint8_t* smem, uint64_t* bars,
                                           const ShortItem& it, int kvh) {
  using C = Short<kFp8>;
  constexpr int NST = C::kStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const DevErr err{p.err};
  const int rows = it.rows;
  const int span = it.blk1 - it.blk0;
  const int my_n = span > warp ? (span - warp + kWarps - 1) / kWarps : 0;

  uint8_t* wstage = smem + warp * NST * C::kStageBytes;
  uint64_t* wbar = bars + warp * NST;
  const uint64_t policy = policy_evict_first();
  // Block ids of this warp's iterations, 32 at a time, the next 32 ahead.
  auto load_ids = [&](int c) -> int {
    const int i = c * 32 + lane;
    if (i >= my_n) return 0;
    int id = __ldg(it.trow + it.blk0 + warp + kWarps * i);
    if (id < 0 || id >= p.num_blocks) {
      err.raise(PKV_DEVERR_BLOCK_ID);
      id = 0;
    }
    return id;
  };
  int ids_cur = load_ids(0);
  int ids_next = my_n > 32 ? load_ids(1) : 0;
  auto issue = [&](int i, int blk) {  // one lane
    const int st = i % NST;
    uint8_t* dst = wstage + st * C::kStageBytes;
    mbar_arrive_expect_tx(&wbar[st], C::kStageBytes);
    if constexpr (kFp8) {
      bulk_load(dst, p.kv8 + (static_cast<int64_t>(blk) * p.hkv + kvh) * kFp8HeadBlockBytes,
                kFp8HeadBlockBytes, &wbar[st], policy);
    } else {
      tma_load_5d(dst, kmap, &wbar[st], 0, 0, 0, blk * 2, kvh, policy);
      tma_load_5d(dst + kHeadBlockBytes, vmap, &wbar[st], 0, 0, 0, blk * 2, kvh, policy);
    }
  };
  for (int i = 0; i < min(NST, my_n); ++i) {
    const int blk = __shfl_sync(0xffffffffu, ids_cur, i);
    if (lane == 0) issue(i, blk);
  }

  // Q rows to shared memory, chunk c of row n at chunk c ^ (n & 7) of its
  // 128-byte halves; rows past the sequence's are zero
  uint8_t* sq = smem + C::kOffQ;
  for (int i = tid; i < 8 * NT * 16; i += kWarps * 32) {
    const int n = i >> 4, c = i & 15;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n < rows) {
      const int tok = (it.row0 + n) / p.group, head = kvh * p.group + it.row0 + n - tok * p.group;
      v = *reinterpret_cast<const uint4*>(p.q + (it.first + tok) * p.q_st + head * p.q_sh + c * 8);
      if constexpr (kFp8) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[e]));
          w[e] = pack_f16(f.x * 0.0625f, f.y * 0.0625f);
        }
      }
    }
    *reinterpret_cast<uint4*>(sq + n * 256 + (c >> 3) * 128 + (((c & 7) ^ (n & 7)) << 4)) = v;
  }
  __syncthreads();

  // keys below lim are visible to rows 2t and 2t + 1 of each tile
  int lim[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int n = nt * 8 + 2 * t + u;
      lim[nt][u] = n >= rows ? 0 : (p.causal ? min(it.kv, it.kv - it.T + (it.row0 + n) / p.group + 1) : it.kv);
    }
  // keys below are visible to all rows
  const int clear = p.causal ? it.kv - it.T + it.row0 / p.group + 1 : it.kv;

  float m[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
  }
  float cap = 0.f, unit = 0.f;  // FP8: O is kept in units of cap / 128; unit = 128 / cap
  const uint32_t sqa = smem_u32(sq);
  // ldmatrix lane roles
  const int a_row = (lane & 7) + ((lane >> 3) & 1) * 8, a_chk = lane >> 4;  // K rows
  const int v_tok = (lane & 7) + ((lane >> 4) & 1) * 8, v_chk = (lane >> 3) & 1;
  const int q_row = lane & 7, q_chk = lane >> 3;

  int i = 0;
  bool ok = true;
  for (; i < my_n; ++i) {
    const int st = i % NST;
    ok = __all_sync(0xffffffffu, mbar_wait(&wbar[st], (i / NST) & 1, err));
    if (!ok) break;
    uint8_t* stage = wstage + st * C::kStageBytes;
    const uint32_t ks = smem_u32(stage);
    const int key0 = (it.blk0 + warp + kWarps * i) * kBlockTokens;
    if (key0 + kBlockTokens > it.kv) {
      // the last block's end holds no position: zero V there, so that P's
      // zeros do not meet whatever is stored
      const int from = it.kv - key0;
      if constexpr (kFp8) {
        for (int c = lane; c < kHeadDim; c += 32) {
          uint8_t* row = stage + kFp8VOff + c * 16;
          for (int tok = from; tok < kBlockTokens; ++tok)
            row[tok < 8 ? 4 * (tok >> 1) + (tok & 1) : 4 * ((tok - 8) >> 1) + 2 + (tok & 1)] = 0;
        }
        if (lane < kBlockTokens && lane >= from)
          reinterpret_cast<float*>(stage + kFp8VScaleOff)[lane] = 0.f;
      } else {
        for (int c = from * 16 + lane; c < kBlockTokens * 16; c += 32) {
          const int tok = c >> 4;
          *reinterpret_cast<uint4*>(stage + kHeadBlockBytes + (tok >> 3) * 2048 +
                                    ((c >> 3) & 1) * 1024 + (tok & 7) * 128 + (c & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        }
      }
      __syncwarp();
    }
    // ---- S^T
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {  // 32 dims a step
      uint32_t a[8];
      if constexpr (kFp8) {
        uint32_t r0, r1, r2, r3;
        ldsm_x4(ks + a_row * 128 + (((2 * kk + a_chk) ^ (a_row & 7)) << 4), r0, r1, r2, r3);
        e4m3x4_to_f16x2x2(r0, a[0], a[2]);
        e4m3x4_to_f16x2x2(r1, a[1], a[3]);
        e4m3x4_to_f16x2x2(r2, a[4], a[6]);
        e4m3x4_to_f16x2x2(r3, a[5], a[7]);
      } else {
        // token row r of a block: group r >> 3 at 2 KiB, halves of 64 dims at 1 KiB
        const uint32_t row = ks + (a_row >> 3) * 2048 + (kk >> 1) * 1024 + (a_row & 7) * 128;
        const int c0 = (kk & 1) * 4;
        ldsm_x4(row + (((c0 + a_chk) ^ (a_row & 7)) << 4), a[0], a[1], a[2], a[3]);
        ldsm_x4(row + (((c0 + 2 + a_chk) ^ (a_row & 7)) << 4), a[4], a[5], a[6], a[7]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NT > 1 && nt * 8 >= rows) break;
        uint32_t b0, b1, b2, b3;  // dims 32kk .. +7, +8 .., +16 .., +24 ..
        ldsm_x4(sqa + (nt * 8 + q_row) * 256 + (kk >> 1) * 128 +
                    ((((kk & 1) * 4 + q_chk) ^ q_row) << 4),
                b0, b1, b2, b3);
        mma16<kFp8>(s[nt], a[0], a[1], a[2], a[3], b0, b1);
        mma16<kFp8>(s[nt], a[4], a[5], a[6], a[7], b2, b3);
      }
    }
    // ---- softmax over this block's keys g and g + 8
    float k0 = p.scale_log2, k1 = p.scale_log2, v0 = 1.f, v1 = 1.f;
    if constexpr (kFp8) {
      const float* sc = reinterpret_cast<const float*>(stage + kFp8KScaleOff);
      k0 = sc[g] * (16.f * p.scale_log2);
      k1 = sc[g + 8] * (16.f * p.scale_log2);
      v0 = sc[16 + g];
      v1 = sc[24 + g];
    }
    bool over = kFp8 && fmaxf(v0, v1) > cap;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s[nt][0] *= k0;
      s[nt][1] *= k0;
      s[nt][2] *= k1;
      s[nt][3] *= k1;
      if (key0 + kBlockTokens > clear) {
        if (key0 + g >= lim[nt][0]) s[nt][0] = -INFINITY;
        if (key0 + g >= lim[nt][1]) s[nt][1] = -INFINITY;
        if (key0 + g + 8 >= lim[nt][0]) s[nt][2] = -INFINITY;
        if (key0 + g + 8 >= lim[nt][1]) s[nt][3] = -INFINITY;
      }
      over |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + kLazyLog2 ||
              fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + kLazyLog2;
    }
    if (__any_sync(0xffffffffu, over)) {
      float to_unit = 1.f;  // from the old unit of O to the new one
      if constexpr (kFp8) {
        float top = fmaxf(v0, v1);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (top > cap) {
          const float next = 4.f * top;  // (some room, so that scales a little larger pass)
          to_unit = cap / next;
          cap = next;
          unit = 128.f / next;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float mx = fmaxf(s[nt][u], s[nt][2 + u]);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
          const float mn = fmaxf(m[nt][u], mx);
          const float al = ex2(m[nt][u] - (mn == -INFINITY ? 0.f : mn));
          l[nt][u] *= al;
          m[nt][u] = mn;
          const float ao = kFp8 ? al * to_unit : al;
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[nt][mt][u] *= ao;
            o[nt][mt][2 + u] *= ao;
          }
        }
      }
    }
    if constexpr (kFp8) {
      v0 *= unit;
      v1 *= unit;
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float b0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0];
      const float b1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
      const float p0 = ex2(s[nt][0] - b0), p1 = ex2(s[nt][1] - b1);
      const float p2 = ex2(s[nt][2] - b0), p3 = ex2(s[nt][3] - b1);
      l[nt][0] += p0 + p2;
      l[nt][1] += p1 + p3;
      if constexpr (kFp8) {
        pb[nt][0] = movm_t(pack_f16(p0 * v0, p1 * v0));
        pb[nt][1] = movm_t(pack_f16(p2 * v1, p3 * v1));
      } else {
        pb[nt][0] = movm_t(pack_bf16(p0, p1));
        pb[nt][1] = movm_t(pack_bf16(p2, p3));
      }
    }
    // ---- O^T
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // 32 dims
      uint32_t a[8];
      if constexpr (kFp8) {
        uint32_t r0, r1, r2, r3;
        ldsm_x4(ks + kFp8VOff +
                    (32 * c + (lane & 7) + ((lane >> 3) & 1) * 8 + (lane >> 4) * 16) * 16,
                r0, r1, r2, r3);
        e4m3x4_to_f16x2x2(r0, a[0], a[2]);
        e4m3x4_to_f16x2x2(r1, a[1], a[3]);
        e4m3x4_to_f16x2x2(r2, a[4], a[6]);
        e4m3x4_to_f16x2x2(r3, a[5], a[7]);
      } else {
        const uint32_t row = ks + kHeadBlockBytes + (v_tok >> 3) * 2048 + (c >> 1) * 1024 +
                             (v_tok & 7) * 128;
        const int c0 = (c & 1) * 4;
        ldsm_x4_t(row + (((c0 + v_chk) ^ (v_tok & 7)) << 4), a[0], a[1], a[2], a[3]);
        ldsm_x4_t(row + (((c0 + 2 + v_chk) ^ (v_tok & 7)) << 4), a[4], a[5], a[6], a[7]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NT > 1 && nt * 8 >= rows) break;
        mma16<kFp8>(o[nt][2 * c], a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
        mma16<kFp8>(o[nt][2 * c + 1], a[4], a[5], a[6], a[7], pb[nt][0], pb[nt][1]);
      }
    }
    __syncwarp();
    const int nx = i + NST;
    if (nx < my_n) {
      if ((nx & 31) == 0) {
        ids_cur = ids_next;
        ids_next = load_ids((nx >> 5) + 1);
      }
      const int blk = __shfl_sync(0xffffffffu, ids_cur, nx & 31);
      if (lane == 0) issue(nx, blk);
    }
  }
  if (!ok) {
    // copies in flight get a bounded time to land before the memory is
    // reused; this warp contributes nothing
    for (int k = i; k < min(my_n, i + NST); ++k) mbar_wait(&wbar[k % NST], (k / NST) & 1, err);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
        o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int off = 4; off < 32; off <<= 1)
        l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], off);

  if constexpr (kFp8) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int u = 0; u < 4; ++u) o[nt][mt][u] *= cap * (1.f / 128.f);
  }

  // ---- join the four warps (in the ring's memory)
  __syncthreads();
  float* co = reinterpret_cast<float*>(smem);                    // [4][8 NT][128]
  float* cm = co + kWarps * 8 * NT * kHeadDim;                   // [4][8 NT]
  float* cl = cm + kWarps * 8 * NT;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (g == 0) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        cm[warp * 8 * NT + nt * 8 + 2 * t + u] = m[nt][u];
        cl[warp * 8 * NT + nt * 8 + 2 * t + u] = l[nt][u];
      }
    }
    float* cw = co + (warp * 8 * NT + nt * 8) * kHeadDim;
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) {
      const int d = mt * 16 + g;
      cw[(2 * t) * kHeadDim + d] = o[nt][mt][0];
      cw[(2 * t + 1) * kHeadDim + d] = o[nt][mt][1];
      cw[(2 * t) * kHeadDim + d + 8] = o[nt][mt][2];
      cw[(2 * t + 1) * kHeadDim + d + 8] = o[nt][mt][3];
    }
  }
  __syncthreads();
  float* po = reinterpret_cast<float*>(smem + C::kOffJoin);   // [32][128]
  float* pm = po + kShortRows * kHeadDim;                      // [32] (base, sum)
  auto store = [&](int n, float4 acc, float sum) {
    const float inv = 1.f / sum;  // 0/0 -> NaN for a token that sees no key
    const int tok = (it.row0 + n) / p.group, head = kvh * p.group + it.row0 + n - tok * p.group;
    uint2 pk;
    pk.x = pack_bf16(acc.x * inv, acc.y * inv);
    pk.y = pack_bf16(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(p.out + (it.first + tok) * p.o_st + head * p.o_sh + lane * 4) = pk;
  };
  for (int n = warp; n < rows; n += kWarps) {  // a warp per row, lane: dims 4l .. 4l + 3
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, cm[w * 8 * NT + n]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(cm[w * 8 * NT + n] - base);
      L += f * cl[w * 8 * NT + n];
      const float4 v =
          *reinterpret_cast<const float4*>(co + (w * 8 * NT + n) * kHeadDim + lane * 4);
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    if (it.nparts == 1) {
      store(n, acc, L);
    } else {
      *reinterpret_cast<float4*>(po + n * kHeadDim + lane * 4) = acc;
      if (lane == 0) *reinterpret_cast<float2*>(pm + 2 * n) = make_float2(M, L);
    }
  }
  if (it.nparts == 1) return;
  // ---- join the partitions, in key order; each CTA of the cluster finishes
  // every nparts-th row.  CTAs past the last partition have left, or, beside
  // chunk.cu's kernel, wait for its end: a unit with fewer partitions than the
  // cluster is then joined behind it (the barrier asks for every thread that
  // has not left; that kernel waits for nothing here).
  cluster_sync();
  for (int n = it.part + it.nparts * warp; n < rows; n += it.nparts * kWarps) {
    float M = -INFINITY;
    for (int c = 0; c < it.nparts; ++c) M = fmaxf(M, cluster_ld2(cluster_addr(pm + 2 * n, c)).x);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < it.nparts; ++c) {
      const float2 ml = cluster_ld2(cluster_addr(pm + 2 * n, c));
      const float4 v = cluster_ld4(cluster_addr(po + n * kHeadDim + lane * 4, c));
      const float f = ex2(ml.x - base);
      L += f * ml.y;
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    store(n, acc, L);
  }
  cluster_sync();  // no CTA leaves while another reads its rows
}

// The CTA's partition of (sequence b, its chunk of rows, KV head), if it has one.
template <bool kFp8>
__device__ __forceinline__ void short_unit(const ShortParams& p, const CUtensorMap* kmap,
                                           const CUtensorMap* vmap, uint8_t* smem, uint64_t* bars,
                                           int b, int chunk, int kvh) {
  // (a whole cluster takes the same way here: all of it is one unit)
  const int s0 = min(max(__ldg(p.q_starts + b), 0), p.tokens);
  const int s1 = min(max(__ldg(p.q_starts + b + 1), s0), p.tokens);
  const int len = max(__ldg(p.kv_lens + b), 0);
  ShortItem it;
  it.first = s0;
  it.T = s1 - s0;
  it.row0 = chunk * kShortRows;
  it.rows = min(it.T * p.group - it.row0, kShortRows);
  if (it.rows <= 0 || it.T * p.group > p.most_rows) return;
  it.kv = static_cast<int>(min(static_cast<int64_t>(len),
                               min(p.pitch, int64_t(1) << 26) * kBlockTokens));
  if (len > it.kv && blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
    DevErr{p.err}.raise(PKV_DEVERR_POSITION);
  // equal partitions of whole rounds of the four warps; no position: one
  // empty partition, which writes the NaN rows
  const int nblk = (it.kv + kBlockTokens - 1) / kBlockTokens;
  const int np = min(static_cast<int>(gridDim.x), max(1, nblk / p.min_blocks));
  const int per = max(kWarps, ((nblk + np - 1) / np + kWarps - 1) / kWarps * kWarps);
  it.nparts = max(1, (nblk + per - 1) / per);
  it.part = blockIdx.x;
  if (it.part >= it.nparts) return;
  it.blk0 = it.part * per;
  it.blk1 = min(nblk, it.blk0 + per);
  it.trow = p.tables + static_cast<int64_t>(p.rows ? p.rows[b] : b) * p.pitch;
  if (it.rows <= 8)
    short_part<kFp8, 1>(p, kmap, vmap, smem, bars, it, kvh);
  else if (it.rows <= 16)
    short_part<kFp8, 2>(p, kmap, vmap, smem, bars, it, kvh);
  else
    short_part<kFp8, kMaxNT>(p, kmap, vmap, smem, bars, it, kvh);
}

template <bool kFp8>
__global__ void __launch_bounds__(kWarps * 32, 2)
    chunk_short_kernel(const ShortParams p, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
  using C = Short<kFp8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z / p.chunks, chunk = blockIdx.z - b * p.chunks, kvh = blockIdx.y;
  pdl_trigger();
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(&bars[warp * C::kStages + s], 1);
    fence_mbar_init();
    if (warp == 0 && !kFp8) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
  }
  __syncwarp();
  // Beside chunk.cu's kernel (launched just before): that one has waited for
  // the stream's earlier work before it let this one start, so the two run at
  // the same time; waiting for it at the end keeps the stream's order for
  // what comes after.
  if (!p.beside) pdl_wait();
  short_unit<kFp8>(p, &kmap, &vmap, smem, bars, b, chunk, kvh);
  if (p.beside) pdl_wait();
}

template <bool kFp8>
cudaError_t launch_short_t(const ShortParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                           dim3 grid, cudaStream_t stream) {
  using C = Short<kFp8>;
  auto kern = chunk_short_kernel<kFp8>;
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = grid.x;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p, kmap, vmap);
}

}  // namespace

cudaError_t launch_chunk_short(const ShortParams& p, const CUtensorMap& kmap,
                               const CUtensorMap& vmap, int32_t batch, int32_t parts,
                               cudaStream_t stream) {
  const dim3 grid(parts, p.hkv, batch * p.chunks);
  return p.kv8 ? launch_short_t<true>(p, kmap, vmap, grid, stream)
               : launch_short_t<false>(p, kmap, vmap, grid, stream);
}

}  // namespace pkv
