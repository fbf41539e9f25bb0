// Attention of the newest tokens of each sequence over its paged cache, the
// tokens of all sequences packed (sm_100a: tcgen05 + TMEM).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j      j < kv_len, and, causal,
//                                                   j <= kv_len - T + i
//
// Rows of a tile.  The query heads that share a KV head are packed with the
// tokens: tile row r is token r / group, head r % group, so 128 rows are
// 128 / group tokens (21 of 6 heads) and every K/V tile is read once for all
// heads of the group.  A check of a few drafted tokens then costs one pass
// over the cache.
//
// Work split.  An item is (row, KV head, block of tokens); its cost is its
// visible keys (per tile) plus a constant.  The items' costs are laid end to
// end and cut into one equal range per CTA, so the SMs finish together
// whatever mix of prompt chunks and single tokens a call holds.  A CTA walks
// its range; an item that a boundary cuts leaves fp32 partials (o / l and
// log2-sum-exp) that merge_kernel joins in key order.  Every CTA works the
// same ranges out for itself from q_starts and kv_lens (a block-wide sum), so
// nothing but the sizes of the launch comes from the host and a captured call
// replays for other lengths.
//
// CTA (one per SM), warps:
//   0      K/V copies: one 5-D TMA box of 4 KiB per block for K and for V
//          (FP8: one bulk copy of a block's chunk), through the block table
//   1      owns TMEM, issues tcgen05.mma
//   2, 3   write the next item's Q tile(s) to shared memory (FP8: as f16 of
//          q / 16); warp 3 also walks the range and hands the items out
//   4-7    softmax of slot A, 8-11 of slot B: a thread owns a tile row
//   12-15  (FP8) widen e4m3 to f16 tiles (exact)
// Two slots, each one S / P and one O tile in tensor memory, keep the tensor
// cores busy while the other slot's softmax runs.  An item of more than 128
// rows gives each slot one of its two tiles (the K/V tiles are shared); a
// smaller one gives the slots alternate key tiles and joins them at its end.
// Order of the tensor instructions: P.V(j) of a slot, then Q.K(j + 1) of it;
// one commit after Q.K therefore says that P.V(j) is done too, and O may be
// rescaled without another wait.
//
// P takes S's columns as 16-bit pairs and is the A operand from tensor
// memory.  bf16 pool: P in bf16.  FP8 pool: scores are scaled per key, and
// the value scale goes into the exponent, p' = 2^(s + log2 vs - base), so
// that P'V needs no scale; l sums p' / vs.  P' in f16 against base = max - 7
// (at most 2^15 with the lazy maximum): 11 bits, and 2^-29 of the largest
// term before a term falls below f16's normal range.
#include <math.h>

#include "pkv_device.cuh"
#include "pkv_kernels.h"
#include "tc_device.cuh"

namespace pkv {
namespace {

constexpr int kRows = 128;                         // rows of a tile (MMA M)
constexpr int kKeys = 128;                         // keys of a tile
constexpr int kTileBlocks = kKeys / kBlockTokens;  // 8
constexpr int kRegion = kRows * 128;               // 128 rows x 64 elements
constexpr int kOperand = 2 * kRegion;              // 32 KiB
constexpr float kLazyLog2 = 8.f;  // the running maximum moves by more than this
constexpr float kP8Shift = 7.f;   // FP8: P' up to 2^(8 + 7)
// cost model, in keys of one tile: what an item costs besides its keys, and
// the least a CTA is given
constexpr int kItemCost = 384;
constexpr int kMinStep = kItemCost + 4 * kKeys;
constexpr int kItemRing = 3;

template <bool kFp8>
struct Cfg {
  static constexpr int kThreads = kFp8 ? 512 : 384;
  static constexpr int kTiles = kFp8 ? 1 : 2;   // tiles of a full item
  static constexpr int kStages = kFp8 ? 4 : 5;  // 32 KiB K or V tiles
  static constexpr int kRaw = kFp8 ? 13 : 0;    // chunks in flight
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = kOffQ + kTiles * kOperand;
  static constexpr int kOffRaw = kOffKV + kStages * kOperand;
  static constexpr int kOffScale = kOffRaw + kRaw * kFp8HeadBlockBytes;  // [4][3][128]
  static constexpr int kOffMl = kOffScale + (kFp8 ? 4 * 3 * kKeys * 4 : 0);  // [2][128] float2
  static constexpr int kOffItem = kOffMl + 2 * kRows * 8;
  static constexpr int kOffBar = kOffItem + kItemRing * 64;
  static constexpr int kBars = 2 * kItemRing + 2 + 2 * kStages + 6 + 3 + 2 * kRaw + 4;
  static constexpr int kOffScan = kOffBar + kBars * 8 + 16;  // 16 warp sums, base, row
  static constexpr int kSmem = kOffScan + 18 * 8;
  // setmaxnreg: launch registers x threads covers the warpgroups' shares
  static constexpr int kRegsLaunch = kFp8 ? 128 : 168;
  static constexpr int kRegsLow = kFp8 ? 72 : 80;    // warps 0-3
  static constexpr int kRegsConv = 72;               // warps 12-15
  static constexpr int kRegsSoftmax = kFp8 ? 184 : 208;
  static_assert(128 * kRegsLow + 256 * kRegsSoftmax + (kFp8 ? 128 * kRegsConv : 0) <=
                    kRegsLaunch * kThreads,
                "register split exceeds the launch allocation");
  static_assert(kSmem <= 227 * 1024, "shared memory exceeds the per-CTA limit");
};

struct ChunkParams {
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
  int32_t batch, tokens, hkv, group, num_blocks, causal;
  float scale_log2;
  int32_t part_rows;  // rows of a partial slot
  int4* desc;         // [grid]: parts, first token, tokens, KV head
  float* part_lse;    // [grid][2][part_rows]
  float* part_o;      // [grid][2][part_rows][128]
  int32_t* err;
};

// ---------------------------------------------------------------- work split
struct RowWork {
  int first, T, kv;  // first packed token, tokens, visible positions
  int n;             // items per KV head
  int a;             // causal: keys that token -1 would see; else kv
  int i0;            // causal: items that see no key
  int64_t head;      // cost of one KV head's items
};

struct Work {
  const ChunkParams& p;
  int tpt, block, wfull;  // tokens per tile and per full item, tiles of a full item

  __device__ Work(const ChunkParams& prm, int tiles)
      : p(prm), tpt(kRows / prm.group), block(tpt * tiles), wfull(tiles) {}

  // Keys that item i's last token sees (0: none of its tokens sees any).
  __device__ int key_end(const RowWork& r, int i) const {
    if (!p.causal) return r.kv;
    return max(0, r.kv - r.T + min(r.T, (i + 1) * block));
  }
  __device__ int weight(const RowWork& r, int i) const {
    return min(r.T - i * block, block) > tpt ? wfull : 1;
  }
  // Cost of a KV head's items before item i <= n - 1 (all of them full).
  __device__ int64_t before(const RowWork& r, int i) const {
    int64_t keys;
    if (!p.causal) {
      keys = static_cast<int64_t>(i) * r.kv;
    } else {
      const int64_t m = max(0, i - r.i0), z = r.i0;
      keys = m * r.a + static_cast<int64_t>(block) * (m * (m + 1) / 2 + m * z);
    }
    return static_cast<int64_t>(i) * kItemCost + keys * wfull;
  }
  __device__ int64_t cost(const RowWork& r, int i) const {
    return kItemCost + static_cast<int64_t>(weight(r, i)) * key_end(r, i);
  }
  __device__ RowWork row(int b) const {
    RowWork r;
    const int s0 = min(max(__ldg(p.q_starts + b), 0), p.tokens);
    const int s1 = min(max(__ldg(p.q_starts + b + 1), s0), p.tokens);
    r.first = s0;
    r.T = s1 - s0;
    r.kv = static_cast<int>(min(static_cast<int64_t>(max(__ldg(p.kv_lens + b), 0)),
                                min(p.pitch, int64_t(1) << 26) * kBlockTokens));
    r.n = (r.T + block - 1) / block;
    r.a = r.kv - r.T;
    r.i0 = p.causal && r.a < 0 ? -r.a / block : 0;
    r.head = r.n ? before(r, r.n - 1) + cost(r, r.n - 1) : 0;
    return r;
  }
};

// What the roles need of an item; 64 bytes in the ring.
struct __align__(16) Item {
  int table_row, first, ntok, kvh;  // first: packed token of tile row 0
  int kv, key_end, t0, t1;          // key tiles [t0, t1) of the cache; t1 < 0: no more items
  int lim0;                         // keys that token 0 of the item sees, causal
  int two;                          // two tiles
  int slot;                         // partial slot, < 0: whole item, written to out
  int pad;
};
static_assert(sizeof(Item) <= 64, "item ring");

__device__ __forceinline__ uint64_t kmajor(uint32_t base, int kk) {
  return sdesc(base + (kk >> 2) * kRegion + (kk & 3) * 32, 16, 1024);
}
// bf16 tiles as the 5-D boxes land: block b's 8-token groups of 64 dims at
// b * 4096 + group * 2048 + half * 1024 (128-byte rows, 128B swizzle).
__device__ __forceinline__ uint64_t box_k(uint32_t base, int kk) {
  return sdesc(base + (kk >> 2) * 1024 + (kk & 3) * 32, 16, 2048);
}
__device__ __forceinline__ uint64_t box_v(uint32_t base, int kb) {
  return sdesc(base + kb * 4096, 1024, 2048);
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3, int c4,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "l"(policy)
      : "memory");
}

constexpr uint64_t kWaitNs = 4000000000ull;
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

template <bool kFp8>
struct Ctx {
  using C = Cfg<kFp8>;
  uint8_t* smem;
  uint64_t *item_full, *item_empty, *q_full, *q_free, *kv_full, *kv_empty, *s_full, *p_full,
      *o_full, *ml_bar, *ep_bar, *mma_done, *raw_full, *raw_empty, *sc_full;
  DevErr err;

  __device__ Ctx(uint8_t* s, int32_t* e) : smem(s), err{e} {
    uint64_t* b = reinterpret_cast<uint64_t*>(s + C::kOffBar);
    auto take = [&](int n) {
      uint64_t* r = b;
      b += n;
      return r;
    };
    item_full = take(kItemRing);
    item_empty = take(kItemRing);
    q_full = take(1);
    q_free = take(1);
    kv_full = take(C::kStages);
    kv_empty = take(C::kStages);
    s_full = take(2);
    p_full = take(2);
    o_full = take(2);
    ml_bar = take(1);
    ep_bar = take(1);
    mma_done = take(1);
    raw_full = take(C::kRaw);
    raw_empty = take(C::kRaw);
    sc_full = take(4);
  }
  __device__ uint32_t* tmem_slot() const {
    return reinterpret_cast<uint32_t*>(smem + C::kOffBar + C::kBars * 8);
  }
  __device__ Item* item(int n) const {
    return reinterpret_cast<Item*>(smem + C::kOffItem + (n % kItemRing) * 64);
  }
  // Bounded by time: a role may wait for a whole item, nothing waits seconds.
  __device__ bool wait(uint64_t* bar, uint32_t phase) const {
    if (mbar_test(bar, phase & 1)) return true;
    const uint64_t t0 = now_ns();
    do {
      for (int i = 0; i < 64; ++i)
        if (mbar_test(bar, phase & 1)) return true;
    } while (now_ns() - t0 < kWaitNs);
    err.raise(PKV_DEVERR_TIMEOUT);
    return false;
  }
  __device__ bool wait_warp(uint64_t* bar, uint32_t phase) const {
    return __all_sync(0xffffffffu, wait(bar, phase));
  }
  // Item n, read by a whole warp; false after a wait that ran out.
  __device__ bool next(int n, Item& it) const {
    if (!wait_warp(&item_full[n % kItemRing], n / kItemRing)) return false;
    it = *item(n);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&item_empty[n % kItemRing]);
    return true;
  }
};

// ---------------------------------------------------------------- Q tiles
// Warps 2 and 3: rows of the item, 16-byte chunk c of row r at chunk
// c ^ (r & 7) of its 128-byte line (K-major, 128B swizzle).  Rows past the
// item's are not written: they only reach their own rows of S and O.
template <bool kFp8>
__device__ void load_q(const ChunkParams& p, uint8_t* smem, const Item& it, int tpt, int thread) {
  const int rows = it.ntok * p.group;
  constexpr int kBatch = 8;
  for (int base = 0; base < rows * 16; base += 64 * kBatch) {
    uint4 v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = base + k * 64 + thread;
      if (i < rows * 16) {
        const int r = i >> 4, tok = r / p.group, head = it.kvh * p.group + r - tok * p.group;
        v[k] = *reinterpret_cast<const uint4*>(p.q + (it.first + tok) * p.q_st + head * p.q_sh +
                                               (i & 15) * 8);
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = base + k * 64 + thread;
      if (i < rows * 16) {
        int r = i >> 4;
        const int c = i & 15;
        uint8_t* dst = smem + Cfg<kFp8>::kOffQ;
        if (Cfg<kFp8>::kTiles == 2 && r >= tpt * p.group) {
          r -= tpt * p.group;
          dst += kOperand;
        }
        if constexpr (kFp8) {
          uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[e]));
            w[e] = pack_f16(f.x * 0.0625f, f.y * 0.0625f);
          }
        }
        *reinterpret_cast<uint4*>(dst + (c >> 3) * kRegion + swz128(r, c & 7)) = v[k];
      }
    }
  }
}

// ---------------------------------------------------------------- epilogue
// Columns [c0, c0 + 32 * N) of a row of O (already divided by its sum): bf16 to out or fp32
// to the row's partial.
__device__ __forceinline__ void store_cols(const float (&v)[32], __nv_bfloat16* out, float* part) {
  if (out) {
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      uint4 pk;
      pk.x = pack_bf16(v[e + 0], v[e + 1]);
      pk.y = pack_bf16(v[e + 2], v[e + 3]);
      pk.z = pack_bf16(v[e + 4], v[e + 5]);
      pk.w = pack_bf16(v[e + 6], v[e + 7]);
      *reinterpret_cast<uint4*>(out + e) = pk;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; e += 4)
      *reinterpret_cast<float4*>(part + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
}

// ---------------------------------------------------------------- softmax
template <bool kFp8>
__device__ void softmax_role(const ChunkParams& p, const Ctx<kFp8>& x, uint32_t tmem, int slot,
                             int tpt) {
  using C = Cfg<kFp8>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3;
  const int r = quarter * 32 + lane;
  const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t col_s = lane_addr + slot * 128, col_o = lane_addr + 256 + slot * 128;
  const int rtok = r / p.group, rhead = r - rtok * p.group;
  float2* ml = reinterpret_cast<float2*>(x.smem + C::kOffMl);
  uint32_t n_tile = 0, n_done = 0, n_ml = 0;  // phases waited for on this slot's barriers
  uint32_t n_key = 0;                         // key tiles of all items so far (FP8 scale ring)
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    const bool whole = it.two;  // this slot has a tile of its own
    const int tok = rtok + (whole ? slot * tpt : 0);
    const bool live = rtok < tpt && tok < it.ntok;
    const int head = it.kvh * p.group + rhead;
    if (it.t1 == 0) {  // no key for any token of the item
      if (live && (whole || slot == 0)) {
        __nv_bfloat16* o = p.out + (it.first + tok) * p.o_st + head * p.o_sh;
        const uint4 nv = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
#pragma unroll
        for (int e = 0; e < 128; e += 8) *reinterpret_cast<uint4*>(o + e) = nv;
      }
      continue;
    }
    const int lim = !live ? 0 : (p.causal ? min(it.kv, it.lim0 + tok) : it.kv);
    const bool busy = __any_sync(0xffffffffu, live);
    float m = -INFINITY, l = 0.f;
    bool first = true;
    for (int j = it.t0 + (whole ? 0 : slot); j < it.t1; j += whole ? 1 : 2) {
      if (!x.wait_warp(&x.s_full[slot], n_tile)) return;
      ++n_tile;
      if (busy) {
        tc_fence_after();
        float s[128];
        tmem_ld32x4_sync(col_s, s);
        const int left = lim - j * kKeys;  // visible keys of this tile
        const float* sc = nullptr;
        if constexpr (kFp8) {
          const uint32_t kt = n_key + (j - it.t0);
          if (!x.wait_warp(&x.sc_full[kt & 3], kt >> 2)) return;
          sc = reinterpret_cast<const float*>(x.smem + C::kOffScale) + (kt & 3) * 3 * kKeys;
#pragma unroll
          for (int i = 0; i < 128; i += 4) {
            const float4 a = *reinterpret_cast<const float4*>(sc + i);
            const float4 b = *reinterpret_cast<const float4*>(sc + kKeys + i);
            s[i + 0] = fmaf(s[i + 0], a.x, b.x);
            s[i + 1] = fmaf(s[i + 1], a.y, b.y);
            s[i + 2] = fmaf(s[i + 2], a.z, b.z);
            s[i + 3] = fmaf(s[i + 3], a.w, b.w);
          }
        }
        if (left < kKeys) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= left) s[i] = -INFINITY;
        }
        float pm[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) pm[u] = fmaxf(s[u], s[u + 8]);
#pragma unroll
        for (int i = 16; i < 128; ++i) pm[i & 7] = fmaxf(pm[i & 7], s[i]);
        float mx = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])),
                         fmaxf(fmaxf(pm[4], pm[5]), fmaxf(pm[6], pm[7])));
        if constexpr (!kFp8) mx *= p.scale_log2;
        // the running maximum moves only by more than 2^8
        const float mn = (mx > m + kLazyLog2 || m == -INFINITY) ? mx : m;
        const float alpha = mn == m ? 1.f : ex2(m - mn);  // 0 from m = -inf
        const float base = mn == -INFINITY ? 0.f : (kFp8 ? mn - kP8Shift : mn);
        m = mn;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
        // P(j) as 16-bit pairs over columns [0, 64) of S, already read
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              e[u] = ex2(kFp8 ? s[c * 32 + i + u] - base
                              : fmaf(s[c * 32 + i + u], p.scale_log2, -base));
            if constexpr (kFp8) {
              const float4 iv = *reinterpret_cast<const float4*>(sc + 2 * kKeys + c * 32 + i);
              ps[0] = fmaf(e[0], iv.x, ps[0]);
              ps[1] = fmaf(e[1], iv.y, ps[1]);
              ps[2] = fmaf(e[2], iv.z, ps[2]);
              ps[3] = fmaf(e[3], iv.w, ps[3]);
              pk[i / 2] = pack_f16(e[0], e[1]);
              pk[i / 2 + 1] = pack_f16(e[2], e[3]);
            } else {
#pragma unroll
              for (int u = 0; u < 4; ++u) ps[u] += e[u];
              pk[i / 2] = pack_bf16(e[0], e[1]);
              pk[i / 2 + 1] = pack_bf16(e[2], e[3]);
            }
          }
          tmem_st16u(col_s + c * 16, pk);
        }
        l = l * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
        if (!first && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32_sync(col_o + c * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= alpha;
            tmem_st32(col_o + c * 32, v);
          }
        }
        first = false;
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&x.p_full[slot]);
    }
    n_key += it.t1 - it.t0;
    // ---- end of the item
    if (whole || slot == 0 || it.t1 - it.t0 > 1) {
      if (!x.wait_warp(&x.o_full[slot], n_done)) return;
      ++n_done;
    }
    tc_fence_after();
    const float base = m == -INFINITY ? 0.f : (kFp8 ? m - kP8Shift : m);
    const bool direct = it.slot < 0;
    const int prow = r + (whole ? slot * kRows : 0);
    const int64_t pslot = static_cast<int64_t>(blockIdx.x) * 2 + max(it.slot, 0);
    __nv_bfloat16* out = direct ? p.out + (it.first + (live ? tok : 0)) * p.o_st + head * p.o_sh
                                : nullptr;
    float* part = direct ? nullptr : p.part_o + (pslot * p.part_rows + prow) * kHeadDim;
    if (whole) {
      if (busy) {
        // a token without a visible key: NaN, but 0 in a partial (its weight is 0)
        const float inv = (direct || l > 0.f) ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld32_sync(col_o + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = (direct || l > 0.f) ? v[i] * inv : 0.f;
          if (live) store_cols(v, out ? out + c * 32 : nullptr, part + c * 32);
        }
        if (live && !direct)
          p.part_lse[pslot * p.part_rows + prow] = l > 0.f ? base + log2f(l) : -INFINITY;
      }
    } else {
      // the slots' halves of the keys: exchange (base, l), then slot s
      // finishes columns [64 s, 64 s + 64) of both O tiles
      ml[slot * kRows + r] = make_float2(m == -INFINITY ? -INFINITY : base, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x.ml_bar);
      if (!x.wait_warp(x.ml_bar, n_ml)) return;
      tc_fence_after();
      if (busy) {
        const float2 A = ml[r], B = ml[kRows + r];
        const float top = fmaxf(A.x, B.x);
        const float fa = A.y > 0.f ? ex2(A.x - top) : 0.f;
        const float fb = B.y > 0.f ? ex2(B.x - top) : 0.f;
        const float sum = A.y * fa + B.y * fb;
        const float inv = (direct || sum > 0.f) ? 1.f / sum : 0.f;
        // a slot without a tile never wrote its O (t1 - t0 = 1)
        const bool has_b = it.t1 - it.t0 > 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v[32], w[32];
          const uint32_t at = lane_addr + 256 + slot * 64 + c * 32;
          tmem_ld32_sync(at, v);
          if (has_b) {
            tmem_ld32_sync(at + 128, w);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = (v[i] * fa + w[i] * fb) * inv;
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= fa * inv;
          }
          if (!direct && !(sum > 0.f)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
          }
          if (live)
            store_cols(v, out ? out + slot * 64 + c * 32 : nullptr, part + slot * 64 + c * 32);
        }
        if (live && !direct && slot == 0)
          p.part_lse[pslot * p.part_rows + prow] = sum > 0.f ? top + log2f(sum) : -INFINITY;
      }
      // both O tiles are read: the next item may overwrite them
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x.ep_bar);
      if (!x.wait_warp(x.ep_bar, n_ml)) return;
      ++n_ml;
    }
    tc_fence_before();
  }
}

// ---------------------------------------------------------------- tensor core
template <bool kFp8>
__device__ void mma_role(const ChunkParams& p, const Ctx<kFp8>& x, uint32_t tmem) {
  using C = Cfg<kFp8>;
  constexpr uint32_t kFmt = kFp8 ? 0u : ((1u << 7) | (1u << 10));  // f16 / bf16 operands
  constexpr uint32_t kIdesc = (1u << 4) | kFmt | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
  constexpr uint32_t kIdescPV = kFp8 ? kIdesc : kIdesc | (1u << 16);  // bf16 V: MN-major
  const int lane = threadIdx.x & 31;
  const uint32_t sq = smem_u32(x.smem + C::kOffQ), skv = smem_u32(x.smem + C::kOffKV);
  uint32_t seq = 0;               // K/V tiles taken so far: K(j) at seq + 2j, V(j) after it
  uint32_t n_q = 0, n_p0 = 0, n_p1 = 0;  // phases of q_full and of p_full[0], [1]
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    const int nt = it.t1 - it.t0;
    if (nt == 0) continue;
    if (!x.wait_warp(x.q_full, n_q)) return;
    ++n_q;
    // S of `slot` = Q (tile of the slot) . K(j)
    auto qk = [&](int j, int slot, bool last_use) -> bool {
      const uint32_t i = seq + 2 * j, st = i % C::kStages;
      if (!x.wait_warp(&x.kv_full[st], i / C::kStages)) return false;
      if (lane == 0) {
        tc_fence_after();
        const uint32_t a = sq + (it.two ? slot * kOperand : 0), b = skv + st * kOperand;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma(tmem + slot * 128, kmajor(a, kk), kFp8 ? kmajor(b, kk) : box_k(b, kk), kIdesc,
               kk > 0 ? 1u : 0u);
        umma_commit(&x.s_full[slot]);
        if (last_use) umma_commit(&x.kv_empty[st]);
      }
      __syncwarp();
      return true;
    };
    // O of `slot` (+)= P . V(j)
    auto pv = [&](int j, int slot, bool fresh, bool first_use, bool last_use) -> bool {
      const uint32_t i = seq + 2 * j + 1, st = i % C::kStages;
      if (!x.wait_warp(&x.kv_full[st], i / C::kStages)) return false;
      const int key0 = (it.t0 + j) * kKeys;
      const int nb = min(kTileBlocks, (it.key_end - key0 + kBlockTokens - 1) / kBlockTokens);
      if (!kFp8 && first_use) {
        // the rest of the cache's last block holds no position: zero rows, so
        // that P's zeros do not meet whatever is stored there
        const int end = it.kv - key0, t = end & (kBlockTokens - 1);
        if (t && end < nb * kBlockTokens) {
          uint8_t* blk = x.smem + C::kOffKV + st * kOperand + (end / kBlockTokens) * 4096;
          for (int c = t * 16 + lane; c < kBlockTokens * 16; c += 32) {
            const int tok = c >> 4, half = (c >> 3) & 1;
            *reinterpret_cast<uint4*>(blk + (tok >> 3) * 2048 + half * 1024 + (tok & 7) * 128 +
                                      (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
        }
      }
      uint32_t& np = slot ? n_p1 : n_p0;
      if (!x.wait_warp(&x.p_full[slot], np)) return false;
      ++np;
      if (lane == 0) {
        tc_fence_after();
        const uint32_t b = skv + st * kOperand;
        for (int kb = 0; kb < nb; ++kb)
          umma_ts(tmem + 256 + slot * 128, tmem + slot * 128 + kb * 8,
                  kFp8 ? kmajor(b, kb) : box_v(b, kb), kIdescPV, (!fresh || kb > 0) ? 1u : 0u);
        if (last_use) umma_commit(&x.kv_empty[st]);
      }
      __syncwarp();
      return true;
    };
    auto commit = [&](uint64_t* bar) {
      if (lane == 0) umma_commit(bar);
      __syncwarp();
    };
    if (it.two) {
      if (!qk(0, 0, false) || !qk(0, 1, true)) return;
      if (nt == 1) commit(x.q_free);
      for (int j = 0; j < nt; ++j) {
        if (!pv(j, 0, j == 0, true, false)) return;
        if (j + 1 < nt) {
          if (!qk(j + 1, 0, false)) return;
        } else {
          commit(&x.o_full[0]);
        }
        if (!pv(j, 1, j == 0, false, true)) return;
        if (j + 1 < nt) {
          if (!qk(j + 1, 1, true)) return;
          if (j + 2 == nt) commit(x.q_free);
        } else {
          commit(&x.o_full[1]);
        }
      }
    } else {
      if (!qk(0, 0, true) || (nt > 1 && !qk(1, 1, true))) return;
      if (nt <= 2) commit(x.q_free);
      for (int j = 0; j < nt; ++j) {
        if (!pv(j, j & 1, j < 2, true, true)) return;
        if (j + 2 < nt) {
          if (!qk(j + 2, j & 1, true)) return;
          if (j + 3 == nt) commit(x.q_free);
        }
      }
      commit(&x.o_full[0]);
      // a slot without a tile waits for nothing of this item, so its barrier
      // must not move on: two phases unseen look like none
      if (nt > 1) commit(&x.o_full[1]);
    }
    seq += 2 * nt;
  }
}

// ---------------------------------------------------------------- copies
// The block ids of an item, 32 at a time: lane k holds block 32c + k of the
// range, the next 32 loaded ahead.  Bad ids read block 0 and set the flag.
struct BlockIds {
  const int32_t* trow;
  int first, count, num_blocks;
  int cur, nxt;
  __device__ int load(int c, const DevErr& err) const {
    const int i = c * 32 + (threadIdx.x & 31);
    if (i >= count) return 0;
    int id = __ldg(trow + first + i);
    if (id < 0 || id >= num_blocks) {
      err.raise(PKV_DEVERR_BLOCK_ID);
      id = 0;
    }
    return id;
  }
  __device__ void start(const DevErr& err) {
    cur = load(0, err);
    nxt = load(1, err);
  }
  // The id of block i (whole warp; i ascends by at most one chunk at a time).
  __device__ int at(int i) const { return __shfl_sync(0xffffffffu, cur, i & 31); }
  __device__ void advance(int i, const DevErr& err) {  // called with i = 32, 64, ...
    cur = nxt;
    nxt = load(i / 32 + 1, err);
  }
};

template <bool kFp8>
__device__ void copy_role(const ChunkParams& p, const Ctx<kFp8>& x, const CUtensorMap* kmap,
                          const CUtensorMap* vmap) {
  using C = Cfg<kFp8>;
  const int lane = threadIdx.x & 31;
  const uint64_t keep = policy_evict_last();
  uint32_t seq = 0;  // K/V tiles (FP8: chunks) issued so far
  bool ok = true;
  for (int n = 0; ok; ++n) {
    Item it;
    ok = x.next(n, it);
    if (!ok || it.t1 < 0) break;
    const int nt = it.t1 - it.t0;
    if (nt == 0) continue;
    BlockIds ids;
    ids.trow = p.tables + static_cast<int64_t>(it.table_row) * p.pitch;
    ids.first = it.t0 * kTileBlocks;
    ids.count = min(it.t1 * kTileBlocks, (it.key_end + kBlockTokens - 1) / kBlockTokens) - ids.first;
    ids.num_blocks = p.num_blocks;
    ids.start(x.err);
    for (int j = 0; j < nt && ok; ++j) {
      const int b0 = j * kTileBlocks;
      if (j && (b0 & 31) == 0) ids.advance(b0, x.err);
      const int nb = min(kTileBlocks, ids.count - b0);
      if constexpr (kFp8) {
        for (int b = 0; b < nb && ok; ++b, ++seq) {
          const uint32_t st = seq % C::kRaw, ph = seq / C::kRaw;
          const int id = ids.at(b0 + b);
          if (ph) ok = x.wait_warp(&x.raw_empty[st], ph - 1);
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&x.raw_full[st], kFp8HeadBlockBytes);
            bulk_load(x.smem + C::kOffRaw + st * kFp8HeadBlockBytes,
                      p.kv8 + (static_cast<int64_t>(id) * p.hkv + it.kvh) * kFp8HeadBlockBytes,
                      kFp8HeadBlockBytes, &x.raw_full[st], keep);
          }
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int which = 0; which < 2; ++which, ++seq) {
          const uint32_t st = seq % C::kStages, ph = seq / C::kStages;
          if (ph && !x.wait_warp(&x.kv_empty[st], ph - 1)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(&x.kv_full[st], nb * 4096);
          for (int b = 0; b < nb; ++b) {
            const int id = ids.at(b0 + b);
            if (lane == 0)
              tma_load_5d(x.smem + C::kOffKV + st * kOperand + b * 4096, which ? vmap : kmap,
                          &x.kv_full[st], 0, 0, 0, id * 2, it.kvh, keep);
          }
          __syncwarp();
        }
      }
    }
  }
  if (!ok) {
    // copies still in flight get a bounded time to land before the CTA ends
    const uint32_t ring = kFp8 ? C::kRaw : C::kStages;
    for (uint32_t s = seq > ring ? seq - ring : 0; s < seq; ++s)
      x.wait(kFp8 ? &x.raw_full[s % ring] : &x.kv_full[s % ring], s / ring);
  }
}

// ---------------------------------------------------------------- FP8 widening
// Warps 12-15: thread c of 128.  K: one 16-byte group (token t, dims 16g ..)
// per block; the lanes of a quarter-warp take tokens t and t ^ 5 with four
// groups each, which keeps both the load (group ^ t) and the two stores
// (chunk 2g + h ^ t) free of bank conflicts.  V is stored by dim, so its tile
// is K-major with the keys contiguous; thread = dim.
__device__ __forceinline__ void widen16(const uint4 raw, uint4& lo, uint4& hi) {
  e4m3x4_to_f16x2x2(raw.x, lo.x, hi.x);
  e4m3x4_to_f16x2x2(raw.y, lo.y, hi.y);
  e4m3x4_to_f16x2x2(raw.z, lo.z, hi.z);
  e4m3x4_to_f16x2x2(raw.w, lo.w, hi.w);
}

// The 16-bit halves of a pair (tokens t, t + 1) that lie before `valid`.
__device__ __forceinline__ uint32_t keep_pair(uint32_t w, int t, int valid) {
  return t + 1 < valid ? w : (t < valid ? w & 0xffffu : 0u);
}

__device__ void widen_role(const ChunkParams& p, const Ctx<true>& x) {
  using C = Cfg<true>;
  const int c = threadIdx.x - 384, lane = c & 31;
  const int pair = ((lane >> 4) & 1) + 2 * (c >> 5);
  const int tok = ((pair & 3) + (pair >> 2) * 8) ^ ((lane >> 2) & 1 ? 5 : 0);
  const int grp = (lane & 3) + ((lane >> 3) & 1) * 4;
  const uint32_t k_src = tok * 128 + ((grp ^ (tok & 7)) << 4);
  const uint32_t k_dst = (grp >> 2) * kRegion + tok * 128;
  const uint32_t k_lo = ((((grp & 3) * 2) ^ (tok & 7)) << 4);
  const uint32_t k_hi = ((((grp & 3) * 2 + 1) ^ (tok & 7)) << 4);
  uint32_t seq = 0, raw = 0, key = 0;
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    const int nt = it.t1 - it.t0;
    const int nblk = (it.key_end + kBlockTokens - 1) / kBlockTokens;
    for (int j = 0; j < nt; ++j) {
      const int b0 = (it.t0 + j) * kTileBlocks, nb = min(kTileBlocks, nblk - b0);
      // ---- K tile and the keys' scales
      uint32_t st = seq % C::kStages, ph = seq / C::kStages;
      if (ph && !x.wait_warp(&x.kv_empty[st], ph - 1)) return;
      uint8_t* dst = x.smem + C::kOffKV + st * kOperand;
      for (int b = 0; b < nb; ++b) {
        const uint32_t rs = (raw + b) % C::kRaw;
        if (!x.wait_warp(&x.raw_full[rs], (raw + b) / C::kRaw)) return;
        const uint8_t* src = x.smem + C::kOffRaw + rs * kFp8HeadBlockBytes;
        uint4 lo, hi;
        widen16(*reinterpret_cast<const uint4*>(src + k_src), lo, hi);
        *reinterpret_cast<uint4*>(dst + k_dst + b * 2048 + k_lo) = lo;
        *reinterpret_cast<uint4*>(dst + k_dst + b * 2048 + k_hi) = hi;
      }
      {
        float ks = 0.f, lv = 0.f, iv = 0.f;
        const int pos = b0 * kBlockTokens + c;
        if (c < nb * kBlockTokens && pos < it.kv) {
          const uint32_t rs = (raw + c / kBlockTokens) % C::kRaw;
          const float* sc = reinterpret_cast<const float*>(
              x.smem + C::kOffRaw + rs * kFp8HeadBlockBytes + kFp8KScaleOff);
          ks = sc[c % kBlockTokens] * (16.f * p.scale_log2);
          // a value row below 2^-91 in size counts as if at that scale
          const float vs = fmaxf(sc[16 + c % kBlockTokens], 0x1p-100f);
          lv = log2f(vs);
          iv = 1.f / vs;
        }
        float* sc = reinterpret_cast<float*>(x.smem + C::kOffScale) + (key & 3) * 3 * kKeys;
        sc[c] = ks;
        sc[kKeys + c] = lv;
        sc[2 * kKeys + c] = iv;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&x.sc_full[key & 3]);
        mbar_arrive(&x.kv_full[st]);
      }
      ++key;
      ++seq;
      // ---- V tile
      st = seq % C::kStages;
      ph = seq / C::kStages;
      if (ph && !x.wait_warp(&x.kv_empty[st], ph - 1)) return;
      dst = x.smem + C::kOffKV + st * kOperand;
      for (int b = 0; b < nb; ++b) {
        const uint32_t rs = (raw + b) % C::kRaw;
        const uint8_t* src = x.smem + C::kOffRaw + rs * kFp8HeadBlockBytes + kFp8VOff;
        uint4 lo, hi;
        widen16(*reinterpret_cast<const uint4*>(src + c * 16), lo, hi);
        __syncwarp();
        if (lane == 0) mbar_arrive(&x.raw_empty[rs]);
        const int valid = it.kv - (b0 + b) * kBlockTokens;
        if (valid < kBlockTokens) {  // no position there: zeros for P's zeros
          lo.x = keep_pair(lo.x, 0, valid);
          lo.y = keep_pair(lo.y, 2, valid);
          lo.z = keep_pair(lo.z, 4, valid);
          lo.w = keep_pair(lo.w, 6, valid);
          hi.x = keep_pair(hi.x, 8, valid);
          hi.y = keep_pair(hi.y, 10, valid);
          hi.z = keep_pair(hi.z, 12, valid);
          hi.w = keep_pair(hi.w, 14, valid);
        }
        uint8_t* row = dst + (b >> 2) * kRegion + c * 128;
        *reinterpret_cast<uint4*>(row + ((((b & 3) * 2) ^ (c & 7)) << 4)) = lo;
        *reinterpret_cast<uint4*>(row + ((((b & 3) * 2 + 1) ^ (c & 7)) << 4)) = hi;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&x.kv_full[st]);
      ++seq;
      raw += nb;
    }
  }
}

// ---------------------------------------------------------------- items
// Warp 3: the items of this CTA's range [lo, hi) of the summed costs, from row
// b whose first item starts at `base`; then its half of each Q tile.
template <bool kFp8>
__device__ void item_role(const ChunkParams& p, const Ctx<kFp8>& x, const Work& w, int b,
                          int64_t base, int64_t lo, int64_t hi, int64_t step) {
  const int lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  int n = 0;
  uint32_t n_load = 0;
  int4 desc = make_int4(0, 0, 0, 0);
  bool ok = true;
  auto push = [&](const Item& it) -> bool {
    const int st = n % kItemRing;
    if (n >= kItemRing && !x.wait_warp(&x.item_empty[st], n / kItemRing - 1)) return false;
    if (lane == 0) {
      *x.item(n) = it;
      mbar_arrive(&x.item_full[st]);
    }
    __syncwarp();
    ++n;
    return true;
  };
  for (; ok && b < p.batch && base < hi; ++b) {
    const RowWork r = w.row(b);
    if (!r.T) continue;
    const int64_t row_end = base + r.head * p.hkv;
    if (row_end <= lo) {
      base = row_end;
      continue;
    }
    const int trow = p.rows ? __ldg(p.rows + b) : b;
    int h = lo > base ? static_cast<int>((lo - base) / r.head) : 0;
    for (; ok && h < p.hkv && base + h * r.head < hi; ++h) {
      const int64_t h0 = base + h * r.head;
      int i = 0;
      if (lo > h0) {  // the last item that starts at or before lo
        int z = r.n - 1;
        while (i < z) {
          const int mid = (i + z + 1) >> 1;
          if (h0 + w.before(r, mid) <= lo)
            i = mid;
          else
            z = mid - 1;
        }
      }
      for (; ok && i < r.n; ++i) {
        const int64_t s = h0 + w.before(r, i);
        if (s >= hi) break;
        const int wt = w.weight(r, i), ke = w.key_end(r, i);
        const int64_t end = s + kItemCost + static_cast<int64_t>(wt) * ke;
        const int kt = (ke + kKeys - 1) / kKeys;
        // tiles before a boundary inside the item
        auto cut = [&](int64_t at) -> int {
          const int64_t d = at - s - kItemCost;
          return d <= 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(kt), d / (wt * kKeys)));
        };
        Item it;
        it.t0 = lo <= s ? 0 : cut(lo);
        it.t1 = hi >= end ? kt : cut(hi);
        if (kt == 0 ? lo > s : it.t0 >= it.t1) continue;
        it.table_row = trow;
        it.first = r.first + i * w.block;
        it.ntok = min(w.block, r.T - i * w.block);
        it.kvh = h;
        it.kv = r.kv;
        it.key_end = ke;
        it.lim0 = r.kv - r.T + i * w.block + 1;
        it.two = wt == 2;
        it.slot = (it.t0 == 0 && it.t1 == kt) ? -1 : (it.t0 == 0 ? 1 : 0);
        it.pad = 0;
        if (it.slot == 1)  // this CTA holds the item's first keys: it names the parts
          desc = make_int4(static_cast<int>((end - 1) / step) - cta + 1, it.first, it.ntok, h);
        ok = push(it);
        if (ok && it.t1 > 0) {
          if (n_load) ok = x.wait_warp(x.q_free, n_load - 1);
          if (ok) {
            load_q<kFp8>(p, x.smem, it, w.tpt, 32 + lane);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(x.q_full);
            ++n_load;
          }
        }
      }
    }
    base = row_end;
  }
  if (p.desc && lane == 0) p.desc[cta] = desc;
  if (ok) {
    Item stop;
    stop.t0 = 0;
    stop.t1 = -1;
    push(stop);
  }
}

template <bool kFp8>
__device__ void q_role(const ChunkParams& p, const Ctx<kFp8>& x, int tpt) {
  const int lane = threadIdx.x & 31;
  uint32_t n_load = 0;
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    if (it.t1 == 0) continue;
    if (n_load && !x.wait_warp(x.q_free, n_load - 1)) return;
    load_q<kFp8>(p, x.smem, it, tpt, lane);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(x.q_full);
    ++n_load;
  }
}

template <bool kFp8>
__global__ void __launch_bounds__(Cfg<kFp8>::kThreads, 1)
    chunk_kernel(const ChunkParams p, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<kFp8>;
  // No static shared memory and 1024-byte alignment asked for: the tiles'
  // swizzle needs it, and 1 KiB of slack for aligning by hand does not fit.
  extern __shared__ __align__(1024) uint8_t smem[];
  const Ctx<kFp8> x(smem, p.err);
  if (smem_u32(smem) & 1023u) {  // a loader that ignores the alignment: nothing can run
    if (threadIdx.x == 0) x.err.raise(PKV_DEVERR_TIMEOUT);
    return;
  }
  int64_t* s_warp = reinterpret_cast<int64_t*>(smem + C::kOffScan);
  int64_t& s_base = s_warp[16];
  int64_t& s_row = s_warp[17];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Work w(p, C::kTiles);

  if (tid == 0) {
    if constexpr (!kFp8) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
    for (int i = 0; i < kItemRing; ++i) {
      mbar_init(&x.item_full[i], 1);
      mbar_init(&x.item_empty[i], kFp8 ? 15 : 11);  // every warp but warp 3
    }
    mbar_init(x.q_full, 2);
    mbar_init(x.q_free, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&x.kv_full[i], kFp8 ? 4 : 1);
      mbar_init(&x.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&x.s_full[i], 1);
      mbar_init(&x.p_full[i], 4);
      mbar_init(&x.o_full[i], 1);
    }
    mbar_init(x.ml_bar, 8);
    mbar_init(x.ep_bar, 8);
    mbar_init(x.mma_done, 1);
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(&x.raw_full[i], 1);
      mbar_init(&x.raw_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&x.sc_full[i], 4);
    fence_mbar_init();
    s_row = p.batch;
    s_base = 0;
  }
  if (warp == 1) tmem_alloc(x.tmem_slot(), 512);
  pdl_wait();

  // The summed cost, and the row in which this CTA's range starts: thread t
  // sums rows [t * per, (t + 1) * per).
  const int per = (p.batch + C::kThreads - 1) / C::kThreads;
  const int rb = min(p.batch, tid * per), re = min(p.batch, rb + per);
  int64_t mine = 0;
  for (int b = rb; b < re; ++b) {
    const RowWork r = w.row(b);
    mine += r.head * p.hkv;
    if (r.T && __ldg(p.kv_lens + b) > r.kv) x.err.raise(PKV_DEVERR_POSITION);
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // dependents launch once this CTA holds its TMEM
  int64_t total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < C::kThreads / 32; ++i) {
    if (i < warp) before += s_warp[i];
    total += s_warp[i];
  }
  const int64_t step = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kMinStep));
  const int64_t lo = step * blockIdx.x, hi = min(total, lo + step);
  const int64_t excl = before + incl - mine;
  if (mine && lo >= excl && lo < excl + mine) {
    int64_t at = excl;
    int b = rb;
    for (; b < re; ++b) {
      const int64_t c = w.row(b).head * p.hkv;
      if (lo < at + c) break;
      at += c;
    }
    s_row = b;
    s_base = at;
  }
  __syncthreads();
  const uint32_t tmem = *x.tmem_slot();

  // Each role's code sits inside the branch that set its register limit.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsLow));
    if (warp == 0) {
      copy_role<kFp8>(p, x, &kmap, &vmap);
    } else if (warp == 1) {
      mma_role<kFp8>(p, x, tmem);
      // every tensor instruction has retired before TMEM is freed (after a
      // wait that ran out, some may be in flight here)
      if (lane == 0) umma_commit(x.mma_done);
      __syncwarp();
      x.wait_warp(x.mma_done, 0);
    } else if (warp == 2) {
      q_role<kFp8>(p, x, w.tpt);
    } else {
      item_role<kFp8>(p, x, w, static_cast<int>(s_row), s_base, lo, hi, step);
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
    softmax_role<kFp8>(p, x, tmem, (warp - 4) >> 2, w.tpt);
  } else if constexpr (kFp8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsConv));
    widen_role(p, x);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp per packed row of a cut item: o = sum 2^(lse_c - L) o_c over its
// parts in key order, lane l holding dims 4l .. 4l+3.
__global__ void __launch_bounds__(256) merge_kernel(const ChunkParams p) {
  pdl_trigger();
  pdl_wait();
  const int4 d = __ldcg(p.desc + blockIdx.x);
  if (d.x < 2) return;
  const int lane = threadIdx.x & 31;
  const int tpt = kRows / p.group, rows = d.z * p.group;
  for (int i = blockIdx.y * 8 + (threadIdx.x >> 5); i < rows; i += gridDim.y * 8) {
    const int tok = i / p.group, head = d.w * p.group + i - tok * p.group;
    const int prow = (d.z > tpt && tok >= tpt) ? kRows + i - tpt * p.group : i;
    auto slot = [&](int c) -> int64_t {
      return ((static_cast<int64_t>(blockIdx.x) + c) * 2 + (c == 0 ? 1 : 0)) * p.part_rows + prow;
    };
    float top = -INFINITY;
    for (int c = lane; c < d.x; c += 32) top = fmaxf(top, __ldcg(p.part_lse + slot(c)));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < d.x; ++c) {
      const float f = ex2(__ldcg(p.part_lse + slot(c)) - base);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot(c) * kHeadDim) + lane);
      sum += f;
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    const float inv = 1.f / sum;  // 0/0 -> NaN for a token that sees no key
    uint2 pk;
    pk.x = pack_bf16(acc.x * inv, acc.y * inv);
    pk.y = pack_bf16(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(d.y + tok) * p.o_st + head * p.o_sh +
                              lane * 4) = pk;
  }
}

// ---------------------------------------------------------------- host
struct ChunkPlan {
  int grid, part_rows;
};

// One CTA per SM, fewer where the launch's sizes cannot give each kMinStep.
ChunkPlan plan_chunk(int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t max_kv_len,
                     bool fp8) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaGetLastError();
  const int group = hq / hkv, tpt = kRows / group, tiles = fp8 ? 1 : 2;
  const int64_t items = (static_cast<int64_t>(tokens) / (tpt * tiles) + batch) * hkv;
  const int64_t item = kItemCost + static_cast<int64_t>(tiles) * max_kv_len;
  const int64_t want = items > (int64_t(1) << 40) / item ? sms : (items * item + kMinStep - 1) / kMinStep;
  ChunkPlan pl;
  pl.grid = static_cast<int>(want < 1 ? 1 : (want < sms ? want : sms));
  // rows of a partial: those of one item (tile B starts at row 128)
  const int64_t most = static_cast<int64_t>(tokens) * group;
  pl.part_rows = tokens > tpt ? tiles * kRows : static_cast<int>((most + 7) / 8 * 8);
  return pl;
}

size_t plan_bytes(const ChunkPlan& pl) {
  if (pl.grid < 2) return 0;
  return static_cast<size_t>(pl.grid) * (16 + 2 * static_cast<size_t>(pl.part_rows) * (kHeadDim + 1) * 4);
}

template <bool kFp8>
cudaError_t launch_chunk_t(const ChunkParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                           int grid, cudaStream_t stream) {
  using C = Cfg<kFp8>;
  auto kern = chunk_kernel<kFp8>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  return launch_k(kern, dim3(grid), dim3(C::kThreads), static_cast<size_t>(C::kSmem), stream, p,
                  kmap, vmap);
}

// setmaxnreg.inc draws on what the block was launched with: a build in which
// the compiler chose another register count must not run.
template <bool kFp8>
bool registers_as_planned() {
  cudaFuncAttributes a{};
  return cudaFuncGetAttributes(&a, chunk_kernel<kFp8>) == cudaSuccess &&
         a.numRegs == Cfg<kFp8>::kRegsLaunch;
}

}  // namespace

size_t chunk_workspace_bytes(int32_t batch, int32_t tokens, int32_t hq, int32_t hkv,
                             int32_t max_kv_len) {
  const size_t a = plan_bytes(plan_chunk(batch, tokens, hq, hkv, max_kv_len, false));
  const size_t b = plan_bytes(plan_chunk(batch, tokens, hq, hkv, max_kv_len, true));
  return a > b ? a : b;
}

cudaError_t launch_chunk(const ChunkLaunch& a, cudaStream_t stream) {
  const bool fp8 = a.kv8 != nullptr;
  static const bool usable[2] = {registers_as_planned<false>(), registers_as_planned<true>()};
  if (!usable[fp8]) return cudaErrorInvalidKernelImage;
  const ChunkPlan pl =
      plan_chunk(a.batch, a.num_tokens, a.num_q_heads, a.num_kv_heads, a.max_kv_len, fp8);
  ChunkParams p{};
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.q_st = a.q_st;
  p.q_sh = a.q_sh;
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.o_st = a.o_st;
  p.o_sh = a.o_sh;
  p.kv8 = static_cast<const uint8_t*>(a.kv8);
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
  p.part_rows = pl.part_rows;
  if (pl.grid > 1) {
    p.desc = static_cast<int4*>(a.workspace);
    p.part_lse = reinterpret_cast<float*>(p.desc + pl.grid);
    p.part_o = p.part_lse + static_cast<int64_t>(pl.grid) * 2 * pl.part_rows;
  }
  const cudaError_t e = fp8 ? launch_chunk_t<true>(p, a.kmap, a.vmap, pl.grid, stream)
                            : launch_chunk_t<false>(p, a.kmap, a.vmap, pl.grid, stream);
  if (e != cudaSuccess || pl.grid < 2) return e;
  const int item_rows = pl.part_rows;
  return launch_k(merge_kernel, dim3(pl.grid, (item_rows + 15) / 16), dim3(256), 0, stream, p);
}

}  // namespace pkv
