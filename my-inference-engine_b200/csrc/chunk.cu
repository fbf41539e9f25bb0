// Attention of the newest tokens of each sequence over its paged cache, the
// tokens of all sequences packed (sm_100a: tcgen05 + TMEM).  Sequences of few
// new tokens, and small calls, are chunk_short.cu's.
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
//   0, 15  copies of K and of V, a 5-D TMA box of 4 KiB per block, through the
//          block table (FP8: warp 0, one bulk copy of a block's chunk)
//   1      owns TMEM, issues the Q.K's
//   2      issues the P.V's
//   3      walks the range and hands the items out
//   4-7    softmax of slot A, 8-11 of slot B: a thread owns a tile row
//   12-14  write the items' Q tiles to shared memory
//   12-15  (FP8) do so as f16 of q / 16, and widen K and V to f16 tiles
// The loops of these roles together are near what the instruction cache holds,
// so code is kept small where it costs nothing: loops rolled, one copy of a
// loop that two warps run (2048 tokens on a 30k cache 377 -> 340 us).
// Two slots, each with a P and an O tile in tensor memory, share one S tile:
// softmax warps take S into registers and free it at once, so the next Q.K
// (the other slot's) runs under their exponentials.  An item of more than 128
// rows gives each slot one of its two tiles (the K/V tiles are shared); a
// smaller one gives the slots alternate key tiles and joins them at its end.
//
// P, as 16-bit pairs, is the A operand from tensor memory: bf16, and f16 over
// the FP8 pool, whose e4m3 keys and values are widened to f16 with their scale
// applied, relative to a power of two for the tile (a score or probability then
// needs no scale of its own; as columns of S the scales cost every softmax
// thread 96 loads a tile).  f16's range is
// used up to 2^(8 + 7): base = maximum - 7, so a term keeps 11 bits down to
// 2^-21 of the largest and is off by at most 2^-32 of it below.  (Both operands
// of a product have one type: with bf16 values a probability is off by up to
// 2^-8 of itself, as in the other bf16 kernels; in f16 by up to 2^-11.)
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "chunk.cuh"
#include "tc_device.cuh"

namespace pkv {
namespace {

constexpr int kRows = 128;                         // rows of a tile (MMA M)
constexpr int kKeys = 128;                         // keys of a tile
constexpr int kTileBlocks = kKeys / kBlockTokens;  // 8
constexpr int kRegion = kRows * 128;               // 128 rows x 64 elements
constexpr int kOperand = 2 * kRegion;              // 32 KiB
constexpr float kP8Shift = 7.f;   // FP8: P' up to 2^(8 + 7)
// cost model, in keys of one tile: what an item costs besides its keys, and
// the least a CTA is given (384 and 896: 512 tokens without a cache 25.3 us
// instead of 22.4, 24 ragged suffixes 150 us either way)
constexpr int kItemCost = 512;
constexpr int kMinStep = kItemCost + 2 * kKeys;
constexpr int kItemRing = 3;
constexpr int kGroup = 2;  // FP8: blocks to a copy barrier
constexpr int kUnitRing = 4;  // FP8: tiles whose units are published (3 would do, see widen_role)
// tensor memory columns: S, then each slot's P, then each slot's O
constexpr uint32_t kColP = 128, kColO = 256;

template <bool kFp8>
struct Cfg {
  static constexpr int kThreads = 512;
  static constexpr int kTiles = 2;              // tiles of a full item
  // 32 KiB tiles; a ring each, so that no barrier is polled by two copiers of
  // whom each sees every second phase only
  static constexpr int kKStages = kFp8 ? 2 : 3, kVStages = 2;
  static constexpr int kRaw = kFp8 ? 3 : 0;  // groups of kGroup chunks in flight
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + kTiles * kOperand;
  static constexpr int kOffV = kOffK + kKStages * kOperand;
  static constexpr int kOffRaw = kOffV + kVStages * kOperand;
  static constexpr int kOffMl = kOffRaw + kRaw * kGroup * kFp8HeadBlockBytes;  // [2][128] float2
  static constexpr int kOffItem = kOffMl + 2 * kRows * 8;
  // FP8: the tiles' units, float2 (key, value), and each slot's at an item's end
  static constexpr int kOffUnit = kOffItem + kItemRing * 64;
  static constexpr int kOffBar = kOffUnit + (kFp8 ? kUnitRing * 8 + 2 * 4 : 0);
  static constexpr int kBars = 2 * kItemRing + 2 + 2 * (kKStages + kVStages) + 7 + 3 + 2 * kRaw;
  static constexpr int kOffScan = kOffBar + kBars * 8 + 16;  // 16 warp sums, base, row
  static constexpr int kSmem = kOffScan + 18 * 8;
  // setmaxnreg: the warpgroups' shares of the launch's 128 per thread
  static constexpr int kRegsLaunch = 128;
  // (bf16 72 / 200 / 40 spilled and was no faster: 2048 tokens on 30k 312 us, ragged 150 against 149)
  static constexpr int kRegsLow = kFp8 ? 72 : 64;    // warps 0-3
  static constexpr int kRegsSoftmax = kFp8 ? 184 : 192;
  static constexpr int kRegsAux = kFp8 ? 72 : 64;    // warps 12-15
  static_assert(kRegsLow + 2 * kRegsSoftmax + kRegsAux <= 4 * kRegsLaunch,
                "register split exceeds the launch allocation");
  static_assert(kRegsLow == kRegsAux, "warps 0 and 15 run one copy of the copy loop");
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
  int32_t short_rows;  // sequences of more rows per KV head are this kernel's
  int32_t part_rows;   // rows of a partial slot
  int4* desc;         // [grid]: parts, first token, tokens, KV head
  float* part_lse;    // [grid][2][part_rows]
  float* part_o;      // [grid][2][dims / 4][part_rows][4]
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
    r.T = (s1 - s0) * p.group > p.short_rows ? s1 - s0 : 0;  // else the short kernel's
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

// Shared-memory descriptors as (low word, high word): the high word is a
// constant of the layout, the low word the start address and the leading
// byte offset, both in 16-byte units, so a step along K is one addition.
// K-major tiles (Q, FP8's K and V): 64-element regions of 128 rows, 8-row
// groups 1 KiB apart; a step of 16 elements is 32 bytes, four per region.
// bf16 tiles as the 5-D boxes land: block b's 8-token groups of 64 dims at
// b * 4096 + group * 2048 + half * 1024 (128-byte rows, 128B swizzle).
constexpr uint32_t kDescHi = (1u << 14) | (2u << 29);  // version, 128B swizzle
constexpr uint32_t kHiKMajor = kDescHi | (1024 >> 4);
constexpr uint32_t kHiBoxK = kDescHi | (2048 >> 4);
constexpr uint32_t kHiBoxV = kDescHi | (2048 >> 4);
constexpr uint32_t kLoKMajor = 1u << 16;              // leading offset unused (16 bytes)
constexpr uint32_t kLoBoxV = (1024u >> 4) << 16;      // 64-dim groups 1 KiB apart

// Eight tensor instructions (K = 8 x 16) by a converged warp: elect.sync
// inside the statement picks one lane, so control and operands stay uniform
// for the compiler; a warp that shares its scheduler with two softmax warps
// gets few issue slots, and every instruction between two tensor
// instructions costs tens of cycles.  STEP4: from step 3 to step 4 of an
// operand, in 16-byte units (steps within a half: STEP).
#define PKV_MMA_STEP(a, da, b, db) "add.u32 " a ", " a ", " da ";\n\tadd.u32 " b ", " b ", " db ";\n\t"
template <uint32_t kHiA, uint32_t kHiB, uint32_t kJumpA, uint32_t kJumpB, uint32_t kStepB>
__device__ __forceinline__ void mma_ss8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#define PKV_SS(acc) \
  "mov.b64 da, {la, %4};\n\tmov.b64 db, {lb, %5};\n\t" \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, " acc ";\n\t"
  asm volatile(
      "{\n\t.reg .pred t, f, e;\n\t.reg .b32 la, lb;\n\t.reg .b64 da, db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\tsetp.eq.u32 t, 0, 0;\n\tsetp.ne.u32 f, 0, 0;\n\t"
      "mov.b32 la, %1;\n\tmov.b32 lb, %2;\n\t" PKV_SS("f") PKV_MMA_STEP("la", "2", "lb", "%8")
          PKV_SS("t") PKV_MMA_STEP("la", "2", "lb", "%8") PKV_SS("t") PKV_MMA_STEP("la", "2", "lb", "%8")
              PKV_SS("t") PKV_MMA_STEP("la", "%6", "lb", "%7") PKV_SS("t")
                  PKV_MMA_STEP("la", "2", "lb", "%8") PKV_SS("t") PKV_MMA_STEP("la", "2", "lb", "%8")
                      PKV_SS("t") PKV_MMA_STEP("la", "2", "lb", "%8") PKV_SS("t") "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(kHiA), "n"(kHiB), "n"(kJumpA), "n"(kJumpB), "n"(kStepB)
      : "memory");
#undef PKV_SS
}
// A from tensor memory, 8 columns per step.
template <uint32_t kHiB, uint32_t kJumpB, uint32_t kStepB>
__device__ __forceinline__ void mma_ts8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                        uint32_t accumulate) {
#define PKV_TS(acc) \
  "mov.b64 db, {lb, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [la], db, %3, " acc ";\n\t"
  asm volatile(
      "{\n\t.reg .pred t, f, e;\n\t.reg .b32 la, lb;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\tsetp.eq.u32 t, 0, 0;\n\tsetp.ne.u32 f, %4, 0;\n\t"
      "mov.b32 la, %1;\n\tmov.b32 lb, %2;\n\t" PKV_TS("f") PKV_MMA_STEP("la", "8", "lb", "%7")
          PKV_TS("t") PKV_MMA_STEP("la", "8", "lb", "%7") PKV_TS("t") PKV_MMA_STEP("la", "8", "lb", "%7")
              PKV_TS("t") PKV_MMA_STEP("la", "8", "lb", "%6") PKV_TS("t")
                  PKV_MMA_STEP("la", "8", "lb", "%7") PKV_TS("t") PKV_MMA_STEP("la", "8", "lb", "%7")
                      PKV_TS("t") PKV_MMA_STEP("la", "8", "lb", "%7") PKV_TS("t") "}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kHiB), "n"(kJumpB), "n"(kStepB)
      : "memory");
#undef PKV_TS
}
#undef PKV_MMA_STEP
__device__ __forceinline__ void mma_ts1(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\telect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar))
      : "memory");
}

// try_wait with a time hint: the warp sleeps until the phase completes or 1 ms
// has passed.  Without one it comes back at once, and a dozen roles that poll
// take the issue slots of the ones that work (a call then takes up to twice
// as long).
__device__ __forceinline__ bool suspend_on(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

constexpr uint64_t kWaitNs = 4000000000ull;
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// A place in a ring of N, and the phase of its barriers' use.
template <int N>
struct RingPos {
  uint32_t st = 0, ph = 0;
  __device__ void next(uint32_t n = N) {
    if (++st == n) {
      st = 0;
      ph ^= 1;
    }
  }
};

template <bool kFp8>
struct Ctx {
  using C = Cfg<kFp8>;
  uint8_t* smem;
  uint64_t *item_full, *item_empty, *q_full, *q_free, *k_full, *k_empty, *v_full, *v_empty, *s_full, *s_free, *p_full,
      *pv_done, *ml_bar, *ep_bar, *mma_done, *raw_full, *raw_empty;
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
    k_full = take(C::kKStages);
    k_empty = take(C::kKStages);
    v_full = take(C::kVStages);
    v_empty = take(C::kVStages);
    s_full = take(2);
    s_free = take(1);
    p_full = take(2);
    pv_done = take(2);
    ml_bar = take(1);
    ep_bar = take(1);
    mma_done = take(1);
    raw_full = take(C::kRaw);
    raw_empty = take(C::kRaw);
  }
  __device__ uint32_t* tmem_slot() const {
    return reinterpret_cast<uint32_t*>(smem + C::kOffBar + C::kBars * 8);
  }
  __device__ Item* item(int n) const {
    return reinterpret_cast<Item*>(smem + C::kOffItem + (n % kItemRing) * 64);
  }
  __device__ float2* unit(uint32_t key_tile) const {
    return reinterpret_cast<float2*>(smem + C::kOffUnit) + key_tile % kUnitRing;
  }
  __device__ float* slot_unit(int slot) const {
    return reinterpret_cast<float*>(smem + C::kOffUnit + kUnitRing * 8) + slot;
  }
  // A whole warp waits for a phase: false after kWaitNs (a role may wait for
  // a whole item, nothing waits seconds).
  __device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t phase) const {
    uint64_t since = 0;
    while (!__all_sync(0xffffffffu, suspend_on(bar, phase & 1))) {
      const uint64_t t = now_ns();
      if (since == 0) since = t;
      if (t - since > kWaitNs) {
        err.raise(PKV_DEVERR_TIMEOUT);
        return false;
      }
    }
    return true;
  }
  // Item n, read by a whole warp; false after a wait that ran out.
  __device__ bool next(int n, Item& it) const {
    if (!wait_warp(&item_full[n % kItemRing], n / kItemRing)) return false;
    it = *item(n);
    // An arrive does not wait for loads in flight, so what they bring has to
    // be used before it: here one word of each 16 bytes.
    it.kvh = __shfl_sync(0xffffffffu, it.kvh, 0);
    it.t1 = __shfl_sync(0xffffffffu, it.t1, 0);
    it.slot = __shfl_sync(0xffffffffu, it.slot, 0);
    if ((threadIdx.x & 31) == 0) mbar_arrive(&item_empty[n % kItemRing]);
    return true;
  }
};

// ---------------------------------------------------------------- Q tiles
// The item's rows, 16-byte chunk c of row r at chunk c ^ (r & 7) of its
// 128-byte line (K-major, 128B swizzle).  Rows past the item's are not
// written: they only reach their own rows of S and O.
// A thread takes one 16-byte chunk of every kThreads / 16th row; heads and
// tokens advance without a division (one per 16 bytes made the Q tiles of an
// item take 9k cycles, which nothing hides in its first tiles).
template <int kThreads>
struct QWalk {
  const __nv_bfloat16* src;
  int64_t step, wrap;  // elements to the next row, and from past a token's last head
  int r, rows, head, dhead, group, per_tile, c;
  __device__ QWalk(const ChunkParams& p, const Item& it, int tpt, int thread)
      : r(thread >> 4), rows(it.ntok * p.group), group(p.group), per_tile(tpt * p.group), c(thread & 15) {
    constexpr int kRowStep = kThreads / 16;
    const int dtok = kRowStep / group, tok = r / group;
    dhead = kRowStep - dtok * group;
    head = r - tok * group;
    step = dtok * p.q_st + dhead * p.q_sh;
    wrap = p.q_st - group * p.q_sh;
    src = p.q + static_cast<int64_t>(it.first + tok) * p.q_st + (it.kvh * group + head) * p.q_sh + c * 8;
  }
  __device__ bool more() const { return r < rows; }
  __device__ uint32_t dst() const {
    const bool b = r >= per_tile;
    return (b ? kOperand : 0) + (c >> 3) * kRegion + swz128(b ? r - per_tile : r, c & 7);
  }
  __device__ void next() {
    r += kThreads / 16;
    src += step;
    head += dhead;
    if (head >= group) {
      head -= group;
      src += wrap;
    }
  }
};

// bf16 pool: three warps, asynchronous copies, all in flight at once.
__device__ void load_q(const ChunkParams& p, uint8_t* tiles, const Item& it, int tpt, int thread) {
  const uint32_t base = smem_u32(tiles);
  for (QWalk<96> q(p, it, tpt, thread); q.more(); q.next())
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + q.dst()), "l"(q.src)
                 : "memory");
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// FP8 pool: q / 16 as f16, 128 threads.  (1/16 keeps any |q| below 2^20 in
// f16's range; it is exact from 2^-10 up, below that off by at most 2^-21.)
__device__ void load_q_f16(const ChunkParams& p, uint8_t* tiles, const Item& it, int tpt,
                           int thread) {
  constexpr int kBatch = 4;
  QWalk<128> q(p, it, tpt, thread);
  while (q.more()) {
    uint4 v[kBatch];
    uint32_t at[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      at[k] = q.more() ? q.dst() : ~0u;
      if (q.more()) v[k] = *reinterpret_cast<const uint4*>(q.src);
      q.next();
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (at[k] != ~0u) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[e]));
          w[e] = pack_f16(f.x * 0.0625f, f.y * 0.0625f);
        }
        *reinterpret_cast<uint4*>(tiles + at[k]) = v[k];
      }
    }
  }
}

// ---------------------------------------------------------------- epilogue
// A thread holds a row, and a store whose lanes lie in 32 rows takes 32 cycles
// whatever its width, so four lanes exchange their 16-byte vectors and each
// store then covers 64 bytes of eight rows (the epilogue of an item took 4k
// cycles a tile, 8k of fp32, with a store per thread).
struct OutRows {
  __nv_bfloat16* row[4];  // the rows of this lane's group of four
  bool live[4];
  __device__ OutRows(__nv_bfloat16* mine, bool is_live) {
    const int lane = threadIdx.x & 31;
    const unsigned mask = __ballot_sync(0xffffffffu, is_live);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int from = (lane & ~3) + j;
      row[j] = reinterpret_cast<__nv_bfloat16*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), from));
      live[j] = (mask >> from) & 1;
    }
  }
  // Columns [col, col + 32) as bf16, by a whole warp.
  __device__ __forceinline__ void store(const float (&v)[32], int col) const {
    const int q = threadIdx.x & 3;
    uint32_t w[4][4];  // this row's four 16-byte vectors
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 2][i & 3] = pack_bf16(v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // 4 x 4 transpose of the vectors among four lanes
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (q & 1) ? w[i][e] : w[i + 1][e], 1);
        if (q & 1)
          w[i][e] = got;
        else
          w[i + 1][e] = got;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (q & 2) ? w[i][e] : w[i + 2][e], 2);
        if (q & 2)
          w[i][e] = got;
        else
          w[i + 2][e] = got;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (live[j])
        *reinterpret_cast<uint4*>(row[j] + col + q * 8) = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
  }
};

// The same columns as fp32 to a partial, whose rows are its fast axis.
__device__ __forceinline__ void store_part(const float (&v)[32], float* part, int part_rows, int col) {
#pragma unroll
  for (int e = 0; e < 32; e += 4)
    *reinterpret_cast<float4*>(part + static_cast<int64_t>(col + e) * part_rows) =
        make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
}

// ---------------------------------------------------------------- softmax
// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ void fma2(float& x0, float& x1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 x, a, b;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\tfma.rn.f32x2 x, x, a, b;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float a0, float a1) {
  asm("{\n\t.reg .b64 x, a;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, a;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(a0), "f"(a1));
}
__device__ __forceinline__ void mul2(float& x0, float& x1, float a) {
  asm("{\n\t.reg .b64 x, a;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 a, {%2, %2};\n\t"
      "mul.rn.f32x2 x, x, a;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(a));
}

// a / b of two powers of two.
__device__ __forceinline__ float exp2i_ratio(float a, float b) {
  return __int_as_float(max(__float_as_int(a) - __float_as_int(b) + (127 << 23), 0));
}

template <bool kFp8>
__device__ void softmax_role(const ChunkParams& p, const Ctx<kFp8>& x, uint32_t tmem, int slot,
                             int tpt) {
  using C = Cfg<kFp8>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3;
  const int r = quarter * 32 + lane;
  const uint32_t lane_addr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t col_p = lane_addr + kColP + slot * 64, col_o = lane_addr + kColO + slot * 128;
  const int rtok = r / p.group, rhead = r - rtok * p.group;
  float2* ml = reinterpret_cast<float2*>(x.smem + C::kOffMl);
  uint32_t n_tile = 0, n_ml = 0;  // tiles of this slot, joins of the two slots so far
  uint32_t n_key = 0;             // key tiles of the items so far
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
    // A row of no token is never masked and its maximum stays 0: whatever it
    // holds reaches only its own P and O, and it must not send its warp
    // through the mask or the rescale (two such rows of 128, with groups of 6,
    // made every tile's mask run: 340 us instead of 310 for 2048 tokens on a
    // 30k cache).
    const int lim = !live ? INT_MAX : (p.causal ? min(it.kv, it.lim0 + tok) : it.kv);
    const bool busy = __any_sync(0xffffffffu, live);
    float m = -INFINITY, l = 0.f;
    float unit = 1.f;  // O is kept in this unit (FP8: the last tile's value unit)
    bool first = true;
    for (int j = it.t0 + (whole ? 0 : slot); j < it.t1; j += whole ? 1 : 2) {
      if (!x.wait_warp(&x.s_full[slot], n_tile)) return;
      ++n_tile;
      if (busy) {
        tc_fence_after();
        float s[128];
        tmem_ld32x4_sync(lane_addr, s);
        // FP8: S and this tile's part of O are in the tile's units
        float scale = p.scale_log2, to_unit = 1.f;
        if constexpr (kFp8) {
          float2 u = *x.unit(n_key + (j - it.t0));
          u.x = __shfl_sync(0xffffffffu, u.x, 0);  // (loaded before the arrival below)
          scale = fmaxf(scale * u.x, FLT_MIN);     // (0 * -inf is no mask)
          // powers of two, never falling within an item
          if (!first && u.y != unit) to_unit = exp2i_ratio(unit, u.y);
          unit = u.y;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(x.s_free);
        const int left = lim - j * kKeys;  // visible keys of this tile
        if (left < kKeys) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int n = left - c * 32;
            const uint32_t seen = n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(seen >> i & 1)) s[c * 32 + i] = -INFINITY;
          }
        }
        float pm[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) pm[u] = fmaxf(s[u], s[u + 4]);
#pragma unroll
        for (int i = 8; i < 128; i += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u) pm[u] = fmaxf(fmaxf(pm[u], s[i + u]), s[i + u + 4]);
        float mx = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
        mx = live ? mx * scale : 0.f;
        // the running maximum moves only by more than 2^8
        const float mn = (mx > m + kLazyLog2 || m == -INFINITY) ? mx : m;
        const float alpha = mn == m ? 1.f : ex2(m - mn);  // 0 from m = -inf
        const float alpha_o = kFp8 ? alpha * to_unit : alpha;
        const float base = mn == -INFINITY ? 0.f : (kFp8 ? mn - kP8Shift : mn);
        m = mn;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
        // P(j) as 16-bit pairs
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float* e = s + c * 32 + i;
            fma2(e[0], e[1], scale, scale, -base, -base);
            fma2(e[2], e[3], scale, scale, -base, -base);
#pragma unroll
            for (int u = 0; u < 4; ++u) e[u] = ex2(e[u]);
            add2(ps[0], ps[1], e[0], e[1]);
            add2(ps[2], ps[3], e[2], e[3]);
            pk[i / 2] = kFp8 ? pack_f16(e[0], e[1]) : pack_bf16(e[0], e[1]);
            pk[i / 2 + 1] = kFp8 ? pack_f16(e[2], e[3]) : pack_bf16(e[2], e[3]);
          }
          if (c == 0) {  // P and O are the slot's again once its last P.V is done
            if (!first && !x.wait_warp(&x.pv_done[slot], n_tile - 2)) return;
            tc_fence_after();
          }
          tmem_st16u(col_p + c * 16, pk);
        }
        l = l * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
        if (!first && __any_sync(0xffffffffu, alpha_o != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float v[32];
            tmem_ld32_sync(col_o + c * 32, v);
#pragma unroll
            for (int i = 0; i < 32; i += 2) mul2(v[i], v[i + 1], alpha_o);
            tmem_st32(col_o + c * 32, v);
          }
        }
        tmem_wait_st();
        tc_fence_before();
      } else {
        if (lane == 0) mbar_arrive(x.s_free);
        // without rows too: an arrival a tile ahead would end the wrong phase
        if (!first && !x.wait_warp(&x.pv_done[slot], n_tile - 2)) return;
      }
      first = false;
      __syncwarp();
      if (lane == 0) mbar_arrive(&x.p_full[slot]);
    }
    // ---- end of the item
    if (!first && !x.wait_warp(&x.pv_done[slot], n_tile - 1)) return;
    tc_fence_after();
    const float base = m == -INFINITY ? 0.f : (kFp8 ? m - kP8Shift : m);
    const bool direct = it.slot < 0;
    const int prow = r + (whole ? slot * kRows : 0);
    const int64_t pslot = static_cast<int64_t>(blockIdx.x) * 2 + max(it.slot, 0);
    const OutRows out(p.out + (it.first + (live ? tok : 0)) * p.o_st + head * p.o_sh, live);
    float* part = p.part_o + pslot * p.part_rows * kHeadDim + prow * 4;
    if (whole) {
      if (busy) {
        // a token without a visible key: NaN, but 0 in a partial (its weight is 0)
        const float inv = (direct || l > 0.f) ? unit / l : 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld32_sync(col_o + c * 32, v);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = (direct || l > 0.f) ? v[i] * inv : 0.f;
          if (direct)
            out.store(v, c * 32);
          else if (live)
            store_part(v, part, p.part_rows, c * 32);
        }
        if (live && !direct)
          p.part_lse[pslot * p.part_rows + prow] = l > 0.f ? base + log2f(l) : -INFINITY;
      }
    } else {
      // the slots' halves of the keys: exchange (base, l), then slot s
      // finishes columns [64 s, 64 s + 64) of both O tiles
      ml[slot * kRows + r] = make_float2(m == -INFINITY ? -INFINITY : base, l);
      if (kFp8 && busy && lane == 0) *x.slot_unit(slot) = unit;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(x.ml_bar);
      if (!x.wait_warp(x.ml_bar, n_ml)) return;
      tc_fence_after();
      if (busy) {
        const float2 A = ml[r], B = ml[kRows + r];
        const float top = fmaxf(A.x, B.x);
        float fa = A.y > 0.f ? ex2(A.x - top) : 0.f;
        float fb = B.y > 0.f ? ex2(B.x - top) : 0.f;
        const float sum = A.y * fa + B.y * fb;
        const float inv = (direct || sum > 0.f) ? 1.f / sum : 0.f;
        if constexpr (kFp8) {
          fa *= *x.slot_unit(0);
          fb *= *x.slot_unit(1);
        }
        // a slot without a tile never wrote its O (t1 - t0 = 1)
        const bool has_b = it.t1 - it.t0 > 1;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          float v[32], w[32];
          const uint32_t at = lane_addr + kColO + slot * 64 + c * 32;
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
          if (direct)
            out.store(v, slot * 64 + c * 32);
          else if (live)
            store_part(v, part, p.part_rows, slot * 64 + c * 32);
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
    n_key += it.t1 - it.t0;
    tc_fence_before();
  }
}

// ---------------------------------------------------------------- tensor core
// Two warps issue, one the Q.K's and one the P.V's: the tensor cores' queue
// holds a few instructions only, and a single warp that waits for P leaves
// them idle although the next Q.K could start (and the other way round).
template <bool kFp8>
struct Tensor {
  using C = Cfg<kFp8>;
  static constexpr uint32_t kFmt = kFp8 ? 0u : ((1u << 7) | (1u << 10));  // f16 / bf16 operands
  static constexpr uint32_t kIdesc =
      (1u << 4) | kFmt | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
  static constexpr uint32_t kIdescPV = kFp8 ? kIdesc : kIdesc | (1u << 16);  // bf16 V: MN-major
};

// S = Q (tile of the slot) . K, tile by tile, each when the slot before has
// taken S.
template <bool kFp8>
__device__ void qk_role(const ChunkParams& p, const Ctx<kFp8>& x, uint32_t tmem) {
  using C = Cfg<kFp8>;
  const uint32_t sq = kLoKMajor | (smem_u32(x.smem + C::kOffQ) >> 4);
  const uint32_t sk = kLoKMajor | (smem_u32(x.smem + C::kOffK) >> 4);
  RingPos<C::kKStages> k;
  uint32_t n_q = 0, n_s = 0;  // Q tiles, Q.K's so far
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    const int nt = it.t1 - it.t0;
    if (nt == 0) continue;
    if (!x.wait_warp(x.q_full, n_q)) return;
    ++n_q;
    for (int j = 0; j < nt; ++j) {
      if (!x.wait_warp(&x.k_full[k.st], k.ph)) return;
      const uint32_t b = sk + k.st * (kOperand >> 4);
#pragma unroll 1
      for (int t = 0; t <= (it.two ? 1 : 0); ++t) {
        if (n_s && !x.wait_warp(x.s_free, n_s - 1)) return;
        ++n_s;
        tc_fence_after();
        if constexpr (kFp8)
          mma_ss8<kHiKMajor, kHiKMajor, (kRegion >> 4) - 6, (kRegion >> 4) - 6, 2>(
              tmem, sq + t * (kOperand >> 4), b, Tensor<kFp8>::kIdesc);
        else
          mma_ss8<kHiKMajor, kHiBoxK, (kRegion >> 4) - 6, (1024 >> 4) - 6, 2>(
              tmem, sq + t * (kOperand >> 4), b, Tensor<kFp8>::kIdesc);
        mma_commit(&x.s_full[it.two ? t : j & 1]);
      }
      mma_commit(&x.k_empty[k.st]);
      k.next();
    }
    mma_commit(x.q_free);
  }
}

// O of the slot (+)= P . V
template <bool kFp8>
__device__ void pv_role(const ChunkParams& p, const Ctx<kFp8>& x, uint32_t tmem) {
  using C = Cfg<kFp8>;
  constexpr uint32_t kIdesc = Tensor<kFp8>::kIdescPV;
  const int lane = threadIdx.x & 31;
  const uint32_t sv = (kFp8 ? kLoKMajor : kLoBoxV) | (smem_u32(x.smem + C::kOffV) >> 4);
  RingPos<C::kVStages> v;
  uint32_t n_p0 = 0, n_p1 = 0;  // P.V's of each slot so far
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    const int nt = it.t1 - it.t0;
    for (int j = 0; j < nt; ++j) {
      if (!x.wait_warp(&x.v_full[v.st], v.ph)) return;
      const int left = it.key_end - (it.t0 + j) * kKeys;  // keys of this tile, and beyond
      if (!kFp8 && left < kKeys) {
        // the rest of the cache's last block holds no position: zero rows, so
        // that P's zeros do not meet whatever is stored there
        const int nb = (left + kBlockTokens - 1) / kBlockTokens;
        const int end = it.kv - (it.t0 + j) * kKeys, t = end & (kBlockTokens - 1);
        if (t && end < nb * kBlockTokens) {
          uint8_t* blk = x.smem + C::kOffV + v.st * kOperand + (end / kBlockTokens) * 4096;
          for (int c = t * 16 + lane; c < kBlockTokens * 16; c += 32) {
            const int tok = c >> 4, half = (c >> 3) & 1;
            *reinterpret_cast<uint4*>(blk + (tok >> 3) * 2048 + half * 1024 + (tok & 7) * 128 +
                                      (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
          __syncwarp();
        }
      }
      const uint32_t b = sv + v.st * (kOperand >> 4);
#pragma unroll 1
      for (int t = 0; t <= (it.two ? 1 : 0); ++t) {
        const int slot = it.two ? t : j & 1;
        uint32_t& np = slot ? n_p1 : n_p0;
        if (!x.wait_warp(&x.p_full[slot], np)) return;
        ++np;
        tc_fence_after();
        const uint32_t d = tmem + kColO + slot * 128, a = tmem + kColP + slot * 64;
        const bool more = it.two ? j > 0 : j > 1;  // onto what the item has so far
        if (left > kKeys - kBlockTokens) {
          if constexpr (kFp8)
            mma_ts8<kHiKMajor, (kRegion >> 4) - 6, 2>(d, a, b, kIdesc, more);
          else
            mma_ts8<kHiBoxV, 256, 256>(d, a, b, kIdesc, more);
        } else {
          const int nb = (left + kBlockTokens - 1) / kBlockTokens;
#pragma unroll 1
          for (int kb = 0; kb < nb; ++kb)
            mma_ts1(d, a + kb * 8,
                    b + (kFp8 ? (kb >> 2) * (kRegion >> 4) + (kb & 3) * 2 : kb * 256),
                    kFp8 ? kHiKMajor : kHiBoxV, kIdesc, (more || kb > 0) ? 1u : 0u);
        }
        mma_commit(&x.pv_done[slot]);
      }
      mma_commit(&x.v_empty[v.st]);
      v.next();
    }
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
  __device__ BlockIds(const ChunkParams& p, const Item& it, const DevErr& err)
      : trow(p.tables + static_cast<int64_t>(it.table_row) * p.pitch),
        first(it.t0 * kTileBlocks),
        count(min(it.t1 * kTileBlocks, (it.key_end + kBlockTokens - 1) / kBlockTokens) - first),
        num_blocks(p.num_blocks) {
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

// Copies issued by a converged warp (elect.sync in the statement): no branch
// around each, which with the softmax on the same scheduler is what a copy
// costs.
__device__ __forceinline__ void box_load(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                         int slot8, int head, uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%6, %6, %6, %3, %4}], [%2], %5;\n\t}" ::"r"(dst),
      "l"(map), "r"(bar), "r"(slot8), "r"(head), "l"(policy), "r"(0)
      : "memory");
}
__device__ __forceinline__ void chunk_load(uint32_t dst, const void* src, uint32_t bar,
                                           uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1], %2, [%3], %4;\n\t}" ::"r"(dst),
      "l"(src), "r"(kFp8HeadBlockBytes), "r"(bar), "l"(policy)
      : "memory");
}

// bf16 pool: one warp copies the K tiles, another the V tiles: a
// thread takes over 100 cycles per box, 16 of them a tile of both.
__device__ void copy_role(const ChunkParams& p, const Ctx<false>& x, const CUtensorMap* map,
                          uint64_t* full, uint64_t* empty, uint8_t* ring, uint32_t stages) {
  const int lane = threadIdx.x & 31;
  const uint64_t keep = policy_evict_last();
  RingPos<0> r;
  uint32_t n_tile = 0;
  bool ok = true;
  for (int n = 0; ok; ++n) {
    Item it;
    ok = x.next(n, it);
    if (!ok || it.t1 < 0) break;
    const int nt = it.t1 - it.t0;
    if (nt == 0) continue;
    BlockIds ids(p, it, x.err);
    for (int j = 0; j < nt; ++j) {
      const int b0 = j * kTileBlocks;
      if (j && (b0 & 31) == 0) ids.advance(b0, x.err);
      const int nb = min(kTileBlocks, ids.count - b0);
      if (n_tile >= stages && !x.wait_warp(&empty[r.st], r.ph ^ 1)) {
        ok = false;
        break;
      }
      const uint32_t dst = smem_u32(ring) + r.st * kOperand, bar = smem_u32(&full[r.st]);
      if (lane == 0) mbar_arrive_expect_tx(&full[r.st], nb * 4096);
      __syncwarp();
#pragma unroll 1  // (the warp has time: unrolled by 8 it costs others their instruction cache)
      for (int b = 0; b < nb; ++b)
        box_load(dst + b * 4096, map, bar, ids.at(b0 + b) * 2, it.kvh, keep);
      r.next(stages);
      ++n_tile;
    }
  }
  if (!ok) {  // copies still in flight get a bounded time to land before the CTA ends
    for (uint32_t t = n_tile > stages ? n_tile - stages : 0; t < n_tile; ++t)
      x.wait_warp(&full[t % stages], t / stages);
  }
}

// FP8 pool: one bulk copy per block, kGroup blocks to a barrier.
__device__ void copy_role(const ChunkParams& p, const Ctx<true>& x) {
  using C = Cfg<true>;
  const int lane = threadIdx.x & 31;
  const uint64_t keep = policy_evict_last();
  const uint64_t stride = static_cast<uint64_t>(p.hkv) * kFp8HeadBlockBytes;
  RingPos<C::kRaw> r;
  uint32_t n_group = 0;
  bool ok = true;
  for (int n = 0; ok; ++n) {
    Item it;
    ok = x.next(n, it);
    if (!ok || it.t1 < 0) break;
    if (it.t1 == it.t0) continue;
    BlockIds ids(p, it, x.err);
    const uint8_t* from = p.kv8 + static_cast<int64_t>(it.kvh) * kFp8HeadBlockBytes;
    for (int b0 = 0; b0 < ids.count; b0 += kGroup) {
      if (b0 && (b0 & 31) == 0) ids.advance(b0, x.err);
      if (n_group >= C::kRaw && !x.wait_warp(&x.raw_empty[r.st], r.ph ^ 1)) {
        ok = false;
        break;
      }
      const int nb = min(kGroup, ids.count - b0);
      const uint32_t dst = smem_u32(x.smem + C::kOffRaw) + r.st * kGroup * kFp8HeadBlockBytes;
      const uint32_t bar = smem_u32(&x.raw_full[r.st]);
      if (lane == 0) mbar_arrive_expect_tx(&x.raw_full[r.st], nb * kFp8HeadBlockBytes);
      __syncwarp();
      if (nb == kGroup) {
#pragma unroll
        for (int b = 0; b < kGroup; ++b)
          chunk_load(dst + b * kFp8HeadBlockBytes,
                     from + static_cast<uint32_t>(ids.at(b0 + b)) * stride, bar, keep);
      } else {
        for (int b = 0; b < nb; ++b)
          chunk_load(dst + b * kFp8HeadBlockBytes,
                     from + static_cast<uint32_t>(ids.at(b0 + b)) * stride, bar, keep);
      }
      ++n_group;
      r.next();
    }
  }
  if (!ok)
    for (uint32_t g = n_group > C::kRaw ? n_group - C::kRaw : 0; g < n_group; ++g)
      x.wait_warp(&x.raw_full[g % C::kRaw], g / C::kRaw);
}

// ---------------------------------------------------------------- FP8 widening
// Warps 12-15: e4m3 * scale as f16 (the chunks hold 4 bits, f16 holds 11).
// f16 spans 30 powers of two and fp32 scales many more, so a tile holds its
// keys, and its values, in a unit, a power of two: unit = cap / 128, where the
// cap lies above every scale of the item so far (128 * 448 is within f16) and
// is raised when a group brings one that is not below it; what the tile holds
// by then is brought down to the new unit.  (2 x 1024 tokens on a 15k cache 367 us;
// with a fixed unit, which loses values past 1023 and keys past 65504, 335 us.)  The softmax folds the key unit into its scale, keeps O in the value
// unit of its last tile (units never fall within an item) and multiplies by it
// at the end.  What is much smaller than the largest scale so far is off by
// f16's least steps, at most 2^-30 of the largest key or value.  A tile's units
// go through a ring: entry n is written again for tile n + kUnitRing, after
// Q.K(n + kUnitRing - 2) has freed its K buffer, which was issued after all of
// S(n + kUnitRing - 3) had been taken, and the units are read before that.
// A key's scale is two f16 terms: rounded to one it would move all of the
// key's products, and so its score, by up to 2^-11 together, where their own
// roundings average out.  For a value it is one more rounding among many.
// One thread's chain of load, convert, scale and store is what bounds a group,
// so its two blocks go through without a branch or a barrier between them and
// every thread rounds the scales it needs (344 -> 322 us; with a copy of the
// scales in shared memory 324 us).
// K: one 16-byte group (token t, dims 16g ..) per block and thread; the lanes
// of a quarter-warp take tokens t and t ^ 5 with four groups each, which keeps
// the two stores (chunk 2g + h ^ t) free of bank conflicts.  V is stored by
// dim, so its tile is K-major with the keys contiguous; thread = dim.
__device__ __forceinline__ __half2 as_half2(uint32_t x) {
  return *reinterpret_cast<const __half2*>(&x);
}
__device__ __forceinline__ uint32_t as_u32(__half2 x) {
  return *reinterpret_cast<const uint32_t*>(&x);
}
// Four e4m3 bytes -> elements (2i, 2i + 1) and (2i + 8, 2i + 9).
__device__ __forceinline__ void widen_k(uint32_t four, uint32_t s, uint32_t rest, uint32_t& lo,
                                        uint32_t& hi) {
  uint32_t a, b;
  e4m3x4_to_f16x2x2(four, a, b);
  lo = as_u32(__hfma2(as_half2(a), as_half2(s), __hmul2(as_half2(a), as_half2(rest))));
  hi = as_u32(__hfma2(as_half2(b), as_half2(s), __hmul2(as_half2(b), as_half2(rest))));
}
__device__ __forceinline__ void widen_v(uint32_t four, uint32_t s_lo, uint32_t s_hi, uint32_t& lo,
                                        uint32_t& hi) {
  uint32_t a, b;
  e4m3x4_to_f16x2x2(four, a, b);
  lo = as_u32(__hmul2(as_half2(a), as_half2(s_lo)));
  hi = as_u32(__hmul2(as_half2(b), as_half2(s_hi)));
}

// The unit of one tile ring's keys or values: the cap's biased exponent.
struct Unit {
  static constexpr int kLeast = 27;  // 2^-100: scales far below it count as 0
  int exp;
  float up;  // 128 / cap
  __device__ Unit() {
    exp = kLeast;
    up = __int_as_float((261 - kLeast) << 23);
  }
  // The cap above `scale` (a positive float's bits); its former unit over the new one.
  __device__ __forceinline__ __half2 raise(uint32_t scale) {
    const int to = min(max(static_cast<int>(scale >> 23) + 1, exp), 250);
    const int by = to - exp;
    exp = to;
    up = __int_as_float((261 - to) << 23);
    return __float2half2_rn(by < 100 ? __int_as_float((127 - by) << 23) : 0.f);
  }
  __device__ __forceinline__ bool holds(uint32_t scale) const { return scale < static_cast<uint32_t>(exp) << 23; }
  __device__ __forceinline__ float value() const { return __int_as_float((exp - 7) << 23); }
};
__device__ __forceinline__ void scale8(uint8_t* at, __half2 by) {
  uint4 w = *reinterpret_cast<uint4*>(at);
  w.x = as_u32(__hmul2(as_half2(w.x), by));
  w.y = as_u32(__hmul2(as_half2(w.y), by));
  w.z = as_u32(__hmul2(as_half2(w.z), by));
  w.w = as_u32(__hmul2(as_half2(w.w), by));
  *reinterpret_cast<uint4*>(at) = w;
}

// The 16-bit halves of a pair (tokens t, t + 1) that lie before `valid`.
__device__ __forceinline__ uint32_t keep_pair(uint32_t w, int t, int valid) {
  return t + 1 < valid ? w : (t < valid ? w & 0xffffu : 0u);
}

__device__ void widen_role(const ChunkParams& p, const Ctx<true>& x, int tpt) {
  using C = Cfg<true>;
  const int c = threadIdx.x - 384, lane = c & 31;
  const int pair = ((lane >> 4) & 1) + 2 * (c >> 5);
  const int tok = ((pair & 3) + (pair >> 2) * 8) ^ ((lane >> 2) & 1 ? 5 : 0);
  const int grp = (lane & 3) + ((lane >> 3) & 1) * 4;
  const uint32_t k_src = tok * 128 + ((grp ^ (tok & 7)) << 4);
  const uint32_t k_dst = (grp >> 2) * kRegion + tok * 128;
  const uint32_t k_lo = ((((grp & 3) * 2) ^ (tok & 7)) << 4);
  const uint32_t k_hi = ((((grp & 3) * 2 + 1) ^ (tok & 7)) << 4);
  uint32_t key = 0, n_load = 0;  // key tiles, Q tiles so far
  RingPos<C::kRaw> g;            // the next copy group
  RingPos<C::kKStages> k;
  RingPos<C::kVStages> v;
  Item it;
  for (int n = 0;; ++n) {
    if (!x.next(n, it) || it.t1 < 0) return;
    const int nt = it.t1 - it.t0;
    if (nt) {
      if (n_load && !x.wait_warp(x.q_free, n_load - 1)) return;
      ++n_load;
      load_q_f16(p, x.smem + C::kOffQ, it, tpt, c);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(x.q_full);
    }
    const int nblk = (it.key_end + kBlockTokens - 1) / kBlockTokens;
    const int positions = min(it.kv, nblk * kBlockTokens);
    Unit ku, vu;  // the same in every thread
    for (int j = 0; j < nt; ++j) {
      const int b0 = (it.t0 + j) * kTileBlocks, nb = min(kTileBlocks, nblk - b0);
      if (key >= C::kKStages && !x.wait_warp(&x.k_empty[k.st], k.ph ^ 1)) return;
      if (key >= C::kVStages && !x.wait_warp(&x.v_empty[v.st], v.ph ^ 1)) return;
      uint8_t* k_tile = x.smem + C::kOffK + k.st * kOperand + k_dst;
      uint8_t* v_tile = x.smem + C::kOffV + v.st * kOperand + c * 128;
      for (int first = 0; first < nb; first += kGroup) {
        if (!x.wait_warp(&x.raw_full[g.st], g.ph)) return;
        const uint8_t* raw = x.smem + C::kOffRaw + g.st * kGroup * kFp8HeadBlockBytes;
        // the group's scales, lane: one of its 32 positions
        const float* mine = reinterpret_cast<const float*>(
            raw + (lane >> 4) * kFp8HeadBlockBytes + kFp8KScaleOff + (lane & 15) * 4);
        const bool held = (b0 + first) * kBlockTokens + lane < positions;
        const uint32_t k_top = __reduce_max_sync(0xffffffffu, held ? __float_as_uint(mine[0]) : 0u);
        const uint32_t v_top = __reduce_max_sync(
            0xffffffffu, held ? __float_as_uint(mine[(kFp8VScaleOff - kFp8KScaleOff) / 4]) : 0u);
        if (!ku.holds(k_top) || !vu.holds(v_top)) {
          const __half2 k_by = ku.raise(k_top), v_by = vu.raise(v_top);
#pragma unroll 1
          for (int b = 0; b < first; ++b) {  // (what this thread wrote itself)
            scale8(k_tile + b * 2048 + k_lo, k_by);
            scale8(k_tile + b * 2048 + k_hi, k_by);
            uint8_t* row = v_tile + (b >> 2) * kRegion;
            scale8(row + ((((b & 3) * 2) ^ (c & 7)) << 4), v_by);
            scale8(row + ((((b & 3) * 2 + 1) ^ (c & 7)) << 4), v_by);
          }
        }
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int b = first + i;  // (past the item's last block: rows that nothing uses)
          const uint4 kr = *reinterpret_cast<const uint4*>(raw + i * kFp8HeadBlockBytes + k_src);
          const uint4 vr =
              *reinterpret_cast<const uint4*>(raw + i * kFp8HeadBlockBytes + kFp8VOff + c * 16);
          const float* fs = reinterpret_cast<const float*>(raw + i * kFp8HeadBlockBytes + kFp8KScaleOff);
          const float ks = fs[tok] * ku.up;
          const __half2 top = __float2half2_rn(ks);
          const uint2 sc = make_uint2(as_u32(top), as_u32(__float2half2_rn(ks - __low2float(top))));
          const float4* fv = reinterpret_cast<const float4*>(raw + i * kFp8HeadBlockBytes + kFp8VScaleOff);
          const float4 f0 = fv[0], f1 = fv[1], f2 = fv[2], f3 = fv[3];
          auto pair = [&](float x, float y) { return pack_f16(x * vu.up, y * vu.up); };
          const uint4 sl = make_uint4(pair(f0.x, f0.y), pair(f0.z, f0.w), pair(f1.x, f1.y), pair(f1.z, f1.w));
          const uint4 sh = make_uint4(pair(f2.x, f2.y), pair(f2.z, f2.w), pair(f3.x, f3.y), pair(f3.z, f3.w));
          uint4 lo, hi;
          widen_k(kr.x, sc.x, sc.y, lo.x, hi.x);
          widen_k(kr.y, sc.x, sc.y, lo.y, hi.y);
          widen_k(kr.z, sc.x, sc.y, lo.z, hi.z);
          widen_k(kr.w, sc.x, sc.y, lo.w, hi.w);
          *reinterpret_cast<uint4*>(k_tile + b * 2048 + k_lo) = lo;
          *reinterpret_cast<uint4*>(k_tile + b * 2048 + k_hi) = hi;
          widen_v(vr.x, sl.x, sh.x, lo.x, hi.x);
          widen_v(vr.y, sl.y, sh.y, lo.y, hi.y);
          widen_v(vr.z, sl.z, sh.z, lo.z, hi.z);
          widen_v(vr.w, sl.w, sh.w, lo.w, hi.w);
          uint8_t* row = v_tile + (b >> 2) * kRegion;
          *reinterpret_cast<uint4*>(row + ((((b & 3) * 2) ^ (c & 7)) << 4)) = lo;
          *reinterpret_cast<uint4*>(row + ((((b & 3) * 2 + 1) ^ (c & 7)) << 4)) = hi;
        }
        // behind the stores: every load of the chunks has returned by then,
        // which an arrive right behind the loads would not wait for
        __syncwarp();
        if (lane == 0) mbar_arrive(&x.raw_empty[g.st]);
        g.next();
      }
      const int valid = it.kv - b0 * kBlockTokens;  // positions from the tile's first on
      if (valid < nb * kBlockTokens) {
        // no positions at the end of the last block: zeros for P's zeros
        const int b = nb - 1, t = valid - b * kBlockTokens;
        uint8_t* row = v_tile + (b >> 2) * kRegion;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint4* at = reinterpret_cast<uint4*>(row + ((((b & 3) * 2 + half) ^ (c & 7)) << 4));
          uint4 w = *at;
          w.x = keep_pair(w.x, half * 8, t);
          w.y = keep_pair(w.y, half * 8 + 2, t);
          w.z = keep_pair(w.z, half * 8 + 4, t);
          w.w = keep_pair(w.w, half * 8 + 6, t);
          *at = w;
        }
      }
      if (c == 0) *x.unit(key) = make_float2(ku.value(), vu.value());
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&x.k_full[k.st]);
        mbar_arrive(&x.v_full[v.st]);
      }
      k.next();
      v.next();
      ++key;
    }
  }
}

// ---------------------------------------------------------------- items
// Warp 3: the items of this CTA's range [lo, hi) of the summed costs, from row
// b whose first item starts at `base`.
template <bool kFp8>
__device__ void item_role(const ChunkParams& p, const Ctx<kFp8>& x, const Work& w, int b,
                          int64_t base, int64_t lo, int64_t hi, int64_t step) {
  const int lane = threadIdx.x & 31;
  const int cta = blockIdx.x;
  int n = 0;
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
        // tiles before a boundary inside the item (128 or 256 of cost each)
        auto cut = [&](int64_t at) -> int {
          const int64_t d = at - s - kItemCost;
          return d <= 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(kt), d >> (6 + wt)));
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

__device__ void q_role(const ChunkParams& p, const Ctx<false>& x, int tpt) {
  uint32_t n_load = 0;
  for (int n = 0;; ++n) {
    Item it;
    if (!x.next(n, it) || it.t1 < 0) return;
    if (it.t1 == 0) continue;
    if (n_load && !x.wait_warp(x.q_free, n_load - 1)) return;
    load_q(p, x.smem + Cfg<false>::kOffQ, it, tpt, threadIdx.x - 384);
    fence_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(x.q_full);
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
      mbar_init(&x.item_empty[i], 15);  // every warp but warp 3
    }
    mbar_init(x.q_full, kFp8 ? 4 : 3);
    mbar_init(x.q_free, 1);
    for (int i = 0; i < C::kKStages; ++i) {
      mbar_init(&x.k_full[i], kFp8 ? 4 : 1);
      mbar_init(&x.k_empty[i], 1);
    }
    for (int i = 0; i < C::kVStages; ++i) {
      mbar_init(&x.v_full[i], kFp8 ? 4 : 1);
      mbar_init(&x.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&x.s_full[i], 1);
      mbar_init(&x.p_full[i], 4);
      mbar_init(&x.pv_done[i], 1);
    }
    mbar_init(x.s_free, 4);
    mbar_init(x.ml_bar, 8);
    mbar_init(x.ep_bar, 8);
    mbar_init(x.mma_done, 2);
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(&x.raw_full[i], 1);
      mbar_init(&x.raw_empty[i], 4);
    }
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

  // Each role's code sits inside the branch that set its register limit, but
  // for the copy loop that warps 0 and 15, of one limit, share (bf16).
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsLow));
    if (warp == 0) {
      if constexpr (kFp8) copy_role(p, x);
    } else if (warp == 1) {
      qk_role<kFp8>(p, x, tmem);
      // every tensor instruction has retired before TMEM is freed (after a
      // wait that ran out, some may be in flight here)
      mma_commit(x.mma_done);
      x.wait_warp(x.mma_done, 0);
    } else if (warp == 2) {
      pv_role<kFp8>(p, x, tmem);
      mma_commit(x.mma_done);
      x.wait_warp(x.mma_done, 0);
    } else {
      item_role<kFp8>(p, x, w, static_cast<int>(s_row), s_base, lo, hi, step);
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
    softmax_role<kFp8>(p, x, tmem, (warp - 4) >> 2, w.tpt);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsAux));
    if constexpr (kFp8) {
      widen_role(p, x, w.tpt);
    } else if (warp < 15) {
      q_role(p, x, w.tpt);
    }
  }
  if constexpr (!kFp8) {  // (not on one scheduler)
    if (warp == 0 || warp == 15) {
      const bool k = warp == 0;
      copy_role(p, x, k ? &kmap : &vmap, k ? x.k_full : x.v_full, k ? x.k_empty : x.v_empty,
                smem + (k ? C::kOffK : C::kOffV), k ? C::kKStages : C::kVStages);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// What was cut, joined in key order: o = sum 2^(lse_c - L) o_c.  Block (CTA,
// y): the item that chunk_kernel's CTA cut, where it has its first keys; eight
// rows at a time, warp w their dims [16 w, 16 w + 16), lane (row, four dims).
__global__ void __launch_bounds__(256) merge_kernel(const ChunkParams p) {
  pdl_trigger();
  pdl_wait();
  const int cta = blockIdx.x;
  const int4 d = __ldcg(p.desc + cta);
  if (d.x < 2) return;
  const int lane = threadIdx.x & 31, dims = ((threadIdx.x >> 5) * 4 + (lane >> 3)) * 4;
  const int tpt = kRows / p.group, rows = d.z * p.group;
  for (int i0 = blockIdx.y * 8; i0 < rows; i0 += gridDim.y * 8) {
    const int i = min(i0 + (lane & 7), rows - 1);
    const int tok = i / p.group, head = d.w * p.group + i - tok * p.group;
    const int prow = (d.z > tpt && tok >= tpt) ? kRows + i - tpt * p.group : i;
    auto slot = [&](int c) -> int64_t {  // part c's, in rows
      return ((static_cast<int64_t>(cta) + c) * 2 + (c == 0 ? 1 : 0)) * p.part_rows;
    };
    float top = -INFINITY;
#pragma unroll 4
    for (int c = lane >> 3; c < d.x; c += 4) top = fmaxf(top, __ldcg(p.part_lse + slot(c) + prow));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float base = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < d.x; ++c) {
      const float f = ex2(__ldcg(p.part_lse + slot(c) + prow) - base);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(
          p.part_o + slot(c) * kHeadDim + static_cast<int64_t>(dims) * p.part_rows + prow * 4));
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
    if (i0 + (lane & 7) < rows)
      *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(d.y + tok) * p.o_st + head * p.o_sh + dims) = pk;
  }
}

// ---------------------------------------------------------------- host
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  std::atomic<int>& k = known[dev & 63];
  int sms = k.load();
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    k.store(sms);
  }
  return sms;
}

struct ChunkPlan {
  int grid, part_rows;             // chunk_kernel; grid 0: not needed
  int short_rows, chunks, parts;   // short kernel; short_rows 0: not needed
};

// Which sequences are the short kernel's: those of at most 16 query rows per
// KV head (up to 32 rows of bf16 the tensor cores win: 64 sequences of up to 30
// rows 73 us there, 83 us here); 32 over FP8, where widening K and V costs
// chunk_kernel as much for few rows as for many (96 sequences of 24 rows on 6k
// caches: 91 us here, 127 us there), unless the call's sequences have more on
// average, so that it runs anyway and takes the others along (24 sequences
// of up to 60 rows on 3k caches: 32 us, with the short kernel beside it 47 us);
// and all sequences of a call of at most kSmallRows rows, which is one launch.
constexpr int kSmallRows = 128;
constexpr int kShortCtas = 148 * 2;  // CTAs that long enough caches are split into: two per SM of a B200
constexpr int kShortMinBlocks = 8;       // per partition: two per warp
// chunk_kernel: one CTA per SM, fewer where the launch's sizes cannot give
// each kMinStep.
ChunkPlan plan_chunk(int32_t batch, int32_t tokens, int32_t hq, int32_t hkv, int32_t max_kv_len,
                     bool fp8) {
  const int group = hq / hkv, tpt = kRows / group, tiles = 2;
  const int64_t most = static_cast<int64_t>(tokens) * group;  // rows of one sequence
  ChunkPlan pl{};
  const bool few = static_cast<int64_t>(tokens) * group <= int64_t(32) * batch;
  pl.short_rows = most <= kSmallRows ? kSmallRows : (fp8 && few ? 32 : 16);
  pl.chunks = most <= kSmallRows ? static_cast<int>((most + kShortRows - 1) / kShortRows) : 1;
  if (pl.short_rows < group) pl.short_rows = pl.chunks = 0;  // not one token
  if (pl.short_rows) {
    const int64_t units = static_cast<int64_t>(batch) * hkv * pl.chunks;
    const int nblk = max_kv_len / kBlockTokens + 1;
    const int64_t want = std::min<int64_t>((kShortCtas + units - 1) / units,
                                           std::max(1, nblk / kShortMinBlocks));
    pl.parts = 1;
    while (pl.parts * 2 <= want && pl.parts < 16) pl.parts *= 2;
  }
  if (most > pl.short_rows) {
    const int64_t longest = std::min<int64_t>(batch, tokens / (pl.short_rows / group + 1));
    const int64_t items = (static_cast<int64_t>(tokens) / (tpt * tiles) + longest) * hkv;
    const int64_t item = kItemCost + static_cast<int64_t>(tiles) * max_kv_len;
    const int sms = sm_count();
    const int64_t want =
        items > (int64_t(1) << 40) / item ? sms : (items * item + kMinStep - 1) / kMinStep;
    pl.grid = static_cast<int>(want < 1 ? 1 : (want < sms ? want : sms));
    // rows of a partial: those of one item (tile B starts at row 128)
    pl.part_rows = tokens > tpt ? tiles * kRows : static_cast<int>((most + 7) / 8 * 8);
  }
  return pl;
}

// Descriptors, sums and partials of chunk_kernel.
size_t plan_bytes(const ChunkPlan& pl) {
  if (pl.grid < 2) return 0;
  return static_cast<size_t>(pl.grid) * (16 + 2 * static_cast<size_t>(pl.part_rows) * (kHeadDim + 1) * 4);
}

template <bool kFp8>
cudaError_t launch_chunk_t(const ChunkParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                           int grid, cudaStream_t stream) {
  using C = Cfg<kFp8>;
  auto kern = chunk_kernel<kFp8>;
  static std::atomic<uint64_t> ready{0};  // a bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(ready.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(bit);
  }
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
  return std::max(plan_bytes(plan_chunk(batch, tokens, hq, hkv, max_kv_len, false)),
                  plan_bytes(plan_chunk(batch, tokens, hq, hkv, max_kv_len, true)));
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
  p.scale_log2 = a.sm_scale * 1.4426950408889634f * (fp8 ? 16.f : 1.f);  // FP8: q / 16
  p.err = a.err;
  p.part_rows = pl.part_rows;
  if (pl.grid > 1) {
    p.desc = static_cast<int4*>(a.workspace);
    p.part_lse = reinterpret_cast<float*>(p.desc + pl.grid);
    p.part_o = p.part_lse + static_cast<int64_t>(pl.grid) * 2 * pl.part_rows;
  }
  p.short_rows = pl.short_rows;
  cudaError_t e = cudaSuccess;
  if (pl.grid > 0)
    e = fp8 ? launch_chunk_t<true>(p, a.kmap, a.vmap, pl.grid, stream)
            : launch_chunk_t<false>(p, a.kmap, a.vmap, pl.grid, stream);
  if (e != cudaSuccess) return e;
  if (pl.short_rows > 0) {
    ShortParams q{};
    q.q = p.q;
    q.q_st = p.q_st;
    q.q_sh = p.q_sh;
    q.out = p.out;
    q.o_st = p.o_st;
    q.o_sh = p.o_sh;
    q.kv8 = p.kv8;
    q.tables = p.tables;
    q.pitch = p.pitch;
    q.rows = p.rows;
    q.q_starts = p.q_starts;
    q.kv_lens = p.kv_lens;
    q.tokens = p.tokens;
    q.hkv = p.hkv;
    q.group = p.group;
    q.num_blocks = p.num_blocks;
    q.causal = p.causal;
    q.most_rows = pl.short_rows;
    q.chunks = pl.chunks;
    q.min_blocks = kShortMinBlocks;
    q.beside = pl.grid > 0;
    q.scale_log2 = a.sm_scale * 1.4426950408889634f;
    q.err = a.err;
    e = launch_chunk_short(q, a.kmap, a.vmap, a.batch, pl.parts, stream);
    if (e != cudaSuccess) return e;
  }
  if (pl.grid < 2) return cudaSuccess;
  return launch_k(merge_kernel, dim3(pl.grid, (pl.part_rows + 15) / 16), dim3(256), 0, stream, p);
}

}  // namespace pkv
