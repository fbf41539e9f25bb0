"""Cases, plain forms and exact values of the paged-cache operators.

Two pairs of operators, each over a bf16 pool and over the FP8 (e4m3) pool:

  chunk   attention of each sequence's newest tokens over its paged cache: the
          tokens of all sequences are packed into one [tokens, heads, 128]
          tensor, sequence b owning rows q_starts[b] .. q_starts[b + 1] and
          kv_lens[b] cached positions (its new tokens the last of them)
  copy    blocks of the cache copied to other blocks, in every layer (a forked
          sequence's partly filled last block)
  move    blocks of the cache moved into free blocks, in every layer, and the
          block tables redirected to them (compaction)

`run` computes them from elementary torch operations, or, with `own` set, with
the library's entry points.  Lengths come from the case alone; values, block
numbers and table orders come from the seed.
"""
import math
import random
import sys

import numpy as np
import torch

own = False

HEAD_DIM = 128
BLOCK = 16
CHUNK_BYTES = 4224  # one (16-token block, KV head) of the FP8 pool
SCALE = 1.0 / math.sqrt(HEAD_DIM)


def listed():
    return [
        # bf16 pool, the engine's own head layout (12 query heads, 2 KV heads)
        # four chats check four drafted tokens each: a few microseconds of work
        chunk("draft_check_4_rows", "bf16", rows=4, new=4, cached=900),
        # a full batch checks five drafted tokens per chat, histories of 2k to 8k
        chunk("draft_check_64_rows", "bf16", rows=64, new=5, cached=8000, spread=True),
        # one tick of a serving loop: a 512-token prompt beside 32 decoding chats
        chunk("mixed_step", "bf16", rows=33, singles=32, new=512, cached=2000, spread=True),
        # messages of up to 200 tokens after a cached history, wider head layout
        chunk("ragged_suffixes", "bf16", rows=24, new=200, cached=3000, spread=True, hq=32, hkv=8),
        # the last chunk of a long document
        chunk("document_chunk", "bf16", rows=1, new=2048, cached=30000),
        # FP8 pool
        # one chat, one token, a 4k history: latency
        chunk("fp8_one_token", "fp8", rows=1, new=1, cached=4001),
        # a large batch checks drafted tokens
        chunk("fp8_draft_check_96_rows", "fp8", rows=96, new=4, cached=6000, spread=True),
        # two prompts continue after a cached document
        chunk("fp8_document_chunks", "fp8", rows=2, new=1024, cached=15001),
        # forks of four chats: one partly filled block each
        pages("copy_four_forks", "copy", "bf16", blocks=1024, pairs=4),
        # every beam of a wide search copies its last blocks
        pages("copy_beams_fp8", "copy", "fp8", blocks=2048, pairs=333),
        # compaction of a pool after its chats ended in another order
        pages("compact", "move", "bf16", blocks=4096, pairs=1100, table_rows=256, pitch=128),
        pages("compact_fp8", "move", "fp8", blocks=3001, pairs=517, table_rows=61, pitch=301),
    ]


def chunk(name, pool, rows, new, cached, singles=0, spread=False, hq=12, hkv=2, lens=1):
    """`rows` sequences; `singles` of them with one new token, the others with
    `new` (1 .. new if `spread`) after `cached` (0 .. cached) earlier ones."""
    case = {"op": "chunk", "pool": pool, "rows": rows, "singles": singles, "new": new,
            "cached": cached, "spread": spread, "hq": hq, "hkv": hkv, "lens": lens}
    return dict(case, name=name) if name else case


def pages(name, op, pool, blocks, pairs, layers=28, hkv=2, table_rows=0, pitch=0):
    case = {"op": op, "pool": pool, "layers": layers, "blocks": blocks, "pairs": pairs, "hkv": hkv,
            "table_rows": table_rows, "pitch": pitch}
    return dict(case, name=name) if name else case


def spread_int(rng, low, high):
    """An integer of [low, high], even over its logarithm."""
    x = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
    return max(low, min(high, int(x)))


def draw(rng):
    pool = rng.choice(["bf16", "fp8"])
    if rng.random() < 0.65:
        while True:
            hq, hkv = rng.choice([(12, 2), (12, 2), (2, 2), (8, 1), (16, 4), (28, 4), (32, 8), (6, 6)])
            rows = spread_int(rng, 1, 96)
            case = chunk(None, pool, rows, new=spread_int(rng, 1, 2048), cached=spread_int(rng, 1, 32000),
                         singles=rng.choice([0, 0, rng.randrange(rows)]), spread=rng.random() < 0.6,
                         hq=hq, hkv=hkv, lens=rng.randrange(1 << 30))
            new, kv = lengths(case)
            padded = rows * max(new) * max(kv) * hq
            if (padded <= 800_000_000 and rows * max(kv) * hkv <= 1_500_000
                    and work(case)["flops"] <= 380e9):
                return case
    while True:
        op = rng.choice(["copy", "move"])
        blocks = spread_int(rng, 40, 4096)
        case = pages(None, op, pool, blocks, pairs=spread_int(rng, 1, max(1, blocks // 4)),
                     layers=rng.randint(1, 28), hkv=rng.choice([1, 2, 2, 4, 8]),
                     table_rows=spread_int(rng, 1, 256) if op == "move" else 0,
                     pitch=spread_int(rng, 1, 500) if op == "move" else 0)
        if work(case)["bytes"] <= 1_000_000_000 and pool_bytes(case) <= 4_000_000_000:
            return case


def lengths(case):
    """New tokens and cached positions (the new ones included) of each row."""
    rng = random.Random(case["lens"])
    new, kv = [], []
    for b in range(case["rows"]):
        t = case["new"] if b >= case["singles"] else 1
        old = case["cached"]
        if case["spread"]:
            t = rng.randint((t + 1) // 2, t)
            old = rng.randint(old // 4, old)
        new.append(t)
        kv.append(t + old)
    order = list(range(case["rows"]))
    rng.shuffle(order)
    return [new[i] for i in order], [kv[i] for i in order]


def block_bytes(case):
    """Bytes of one block in one plane (bf16: K or V of a layer; FP8: a layer)."""
    return case["hkv"] * (BLOCK * HEAD_DIM * 2 if case["pool"] == "bf16" else CHUNK_BYTES)


def pool_bytes(case):
    planes = case["layers"] * (2 if case["pool"] == "bf16" else 1)
    return planes * case["blocks"] * block_bytes(case)


def work(case):
    if case["op"] == "chunk":
        new, kv = lengths(case)
        tokens, hq, hkv = sum(new), case["hq"], case["hkv"]
        per_key = 2 * HEAD_DIM * 2 if case["pool"] == "bf16" else 2 * (HEAD_DIM + 4)
        pairs = sum(t * s - t * (t - 1) // 2 for t, s in zip(new, kv))  # query i sees s - t + i + 1 keys
        return {"bytes": (2 * tokens * hq * HEAD_DIM * 2 + sum(kv) * hkv * per_key
                          + sum(4 * -(-s // BLOCK) for s in kv) + 4 * (2 * len(kv) + 1)),
                "flops": 4 * HEAD_DIM * hq * pairs}
    planes = case["layers"] * (2 if case["pool"] == "bf16" else 1)
    table = case["table_rows"] * case["pitch"]
    return {"bytes": 2 * planes * case["pairs"] * block_bytes(case) + 8 * case["pairs"] + 8 * table,
            "flops": 0}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    if case["op"] != "chunk":
        return dict(case, err=err, **page_inputs(case, gen, dev))
    new, kv = lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    need = [-(-s // BLOCK) for s in kv]
    num_blocks = sum(need) + 3
    order = torch.randperm(num_blocks, generator=gen, device=dev).to(torch.int32)
    tables = torch.zeros(len(kv), max(need) + 2, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    # keys with a few strong channels and queries of unit size: scores of a
    # few units, as rotated projections give; values of differing size per token
    slots = num_blocks * BLOCK
    k = torch.randn(slots, hkv, HEAD_DIM, generator=gen, device=dev)
    k *= torch.exp(0.5 * torch.randn(hkv, HEAD_DIM, generator=gen, device=dev))
    v = torch.randn(slots, hkv, HEAD_DIM, generator=gen, device=dev)
    v *= torch.exp(0.5 * torch.randn(slots, hkv, 1, generator=gen, device=dev))
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    tokens = sum(new)
    state = dict(case, err=err, tables=tables, max_kv=max(kv), max_new=max(new), tokens=tokens,
                 q=torch.randn(tokens, hq, HEAD_DIM, generator=gen, device=dev).to(torch.bfloat16),
                 q_starts=torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=dev),
                 kv_lens=torch.tensor(kv, dtype=torch.int32, device=dev))
    if case["pool"] == "bf16":
        state.update(k=k, v=v)
    else:
        state.update(pool8=quantise(k.view(num_blocks, BLOCK, hkv, HEAD_DIM),
                                    v.view(num_blocks, BLOCK, hkv, HEAD_DIM)))
    return state


def quantise(k, v):
    """[blocks, 16, hkv, 128] keys and values -> the FP8 pool's bytes of one
    layer [blocks, hkv, 4224]: e4m3 rows with one fp32 scale per token."""
    def rows(x):
        x = x.float()
        amax = x.abs().amax(-1, keepdim=True)
        y = x * torch.where(amax > 0, 448.0 / amax, torch.zeros_like(amax))
        scale = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax)).squeeze(-1)
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale

    dev, n, hkv = k.device, k.shape[0], k.shape[2]
    (kb, ks), (vb, vs) = rows(k), rows(v)
    out = torch.empty(n, hkv, CHUNK_BYTES, dtype=torch.uint8, device=dev)
    out[..., k_bytes(dev).view(-1)] = kb.permute(0, 2, 1, 3).reshape(n, hkv, -1)
    out[..., v_bytes(dev).view(-1)] = vb.permute(0, 2, 1, 3).reshape(n, hkv, -1)
    out[..., 4096:4160] = ks.permute(0, 2, 1).contiguous().view(torch.uint8)
    out[..., 4160:4224] = vs.permute(0, 2, 1).contiguous().view(torch.uint8)
    return out


def place(e):
    """Byte of element e (0 .. 15) in a 16-byte group."""
    return torch.where(e < 8, 4 * (e // 2) + e % 2, 4 * ((e - 8) // 2) + 2 + e % 2)


def k_bytes(dev):
    """Byte of token t's key dim d in a chunk, [16, 128]."""
    t = torch.arange(BLOCK, device=dev)[:, None]
    d = torch.arange(HEAD_DIM, device=dev)[None, :]
    return t * 128 + ((d // 16) ^ (t % 8)) * 16 + place(d % 16)


def v_bytes(dev):
    t = torch.arange(BLOCK, device=dev)[:, None]
    d = torch.arange(HEAD_DIM, device=dev)[None, :]
    return 2048 + d * 16 + place(t)


def page_inputs(case, gen, dev):
    blocks, n, layers, hkv = case["blocks"], case["pairs"], case["layers"], case["hkv"]
    if case["pool"] == "bf16":
        pool = torch.empty(layers, 2, blocks * BLOCK, hkv, HEAD_DIM, dtype=torch.bfloat16, device=dev)
        for plane in pool.view(-1, blocks * BLOCK * hkv * HEAD_DIM):
            plane.normal_(generator=gen)
    else:
        pool = torch.empty(layers, blocks, hkv, CHUNK_BYTES, dtype=torch.uint8, device=dev)
        for plane in pool:
            plane.random_(0, 256, generator=gen)
    order = torch.randperm(blocks, generator=gen, device=dev)
    if case["op"] == "copy":  # a source may be copied several times, a target is written once
        src = order[n:][torch.randint(max(1, (blocks - n) // 2), (n,), generator=gen, device=dev)]
        return {"block_pool": pool, "src": src.to(torch.int32), "dst": order[:n].to(torch.int32)}
    # live blocks end up as 0 .. live - 1: the n live ones above move into the n holes below
    live = blocks - n - (blocks - 2 * n) // 3
    low = torch.randperm(live, generator=gen, device=dev)
    high = live + torch.randperm(blocks - live, generator=gen, device=dev)
    src, dst = high[:n].sort().values, low[:n]
    used = torch.cat([low[n:], src])
    pick = torch.randint(used.numel(), (case["table_rows"], case["pitch"]), generator=gen, device=dev)
    return {"block_pool": pool, "src": src.to(torch.int32), "dst": dst.to(torch.int32),
            "tables": used[pick].to(torch.int32)}


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return run_own(state)
    if state["op"] == "chunk":
        return plain_chunk(state)
    pool, src, dst = state["block_pool"], state["src"].long(), state["dst"].long()
    if state["pool"] == "bf16":
        pages = pool.view(*pool.shape[:2], -1, BLOCK, *pool.shape[3:])
        pages[:, :, dst] = pages[:, :, src]
    else:
        pool[:, dst] = pool[:, src]
    if state["op"] == "copy":
        return pool
    to = torch.arange(state["blocks"], dtype=torch.int32, device=pool.device)
    to[src] = state["dst"]
    state["tables"].copy_(to[state["tables"].long()])
    return pool, state["tables"]


def run_own(s):
    if "my-inference-engine_b200" not in sys.path:
        sys.path.insert(0, "my-inference-engine_b200")
    import pagedkv

    if s["op"] == "copy":
        pagedkv.copy_blocks(s["block_pool"], s["src"], s["dst"], s["err"])
        return s["block_pool"]
    if s["op"] == "move":
        pagedkv.move_blocks(s["block_pool"], s["src"], s["dst"], s["tables"], s["err"])
        return s["block_pool"], s["tables"]
    out = torch.empty_like(s["q"])
    if s["pool"] == "bf16":
        pagedkv.paged_chunk(s["q"], s["k"], s["v"], s["tables"], None, s["q_starts"], s["kv_lens"],
                            s["max_kv"], out, True, SCALE, s["hkv"], s["err"])
    else:
        pagedkv.paged_chunk_fp8(s["q"], s["pool8"], s["tables"], None, s["q_starts"], s["kv_lens"],
                                s["max_kv"], out, True, SCALE, s["err"])
    return out


def plain_chunk(s):
    """softmax(scale q k^T) v with the rows padded to the longest, in 32 bits."""
    rows, hq, hkv = s["rows"], s["hq"], s["hkv"]
    group, most, keys = hq // hkv, s["max_new"], s["max_kv"]
    dev = s["q"].device
    first, kv = s["q_starts"].long(), s["kv_lens"].long()
    new = first[1:] - first[:-1]
    # packed tokens <-> [rows, most]
    row = torch.repeat_interleave(torch.arange(rows, device=dev), new, output_size=s["tokens"])
    col = torch.arange(s["tokens"], device=dev) - first[row]
    q = torch.zeros(rows, most, hq, HEAD_DIM, device=dev)
    q[row, col] = s["q"].float()
    q = q.view(rows, most, hkv, group, HEAD_DIM)
    # the rows' keys and values through their tables, [rows, keys, hkv, 128]
    pos = torch.arange(keys, device=dev)
    blocks = s["tables"].long()[:, pos // BLOCK]
    if s["pool"] == "bf16":
        slot = blocks * BLOCK + pos % BLOCK
        k, v = s["k"][slot].float(), s["v"][slot].float()
    else:
        k, v = plain_dequantise(s["pool8"], s["tables"].long(), keys)
    score = torch.einsum("bthgd,bshd->bhgts", q, k) * SCALE
    see = pos[None, None, :] <= (kv - new)[:, None, None] + torch.arange(most, device=dev)[None, :, None]
    see &= pos[None, None, :] < kv[:, None, None]
    score.masked_fill_(~see[:, None, None], -math.inf)
    # rows past a sequence's last token see its whole cache and are not taken
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.einsum("bhgts,bshd->bthgd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    return out.reshape(rows, most, hq, HEAD_DIM)[row, col].to(torch.bfloat16)


def plain_dequantise(pool8, tables, keys):
    dev = pool8.device
    chunks = pool8[tables[:, :-(-keys // BLOCK)]]  # [rows, blocks, hkv, 4224]
    rows, n, hkv = chunks.shape[:3]

    def values(place, at):
        e = chunks[..., place.view(-1)].view(torch.float8_e4m3fn).float().view(rows, n, hkv, BLOCK, HEAD_DIM)
        scale = chunks[..., at:at + 64].contiguous().view(torch.float32)
        x = (e * scale[..., None]).permute(0, 1, 3, 2, 4).reshape(rows, n * BLOCK, hkv, HEAD_DIM)
        return x[:, :keys]

    return values(k_bytes(dev), 4096), values(v_bytes(dev), 4160)


# ---------------------------------------------------------------- 64 bits
E4M3 = [(-1.0 if b & 128 else 1.0) * (2.0 ** -9 * (b & 7) if not b & 0x78
                                     else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3 & 15) - 7))
        for b in range(256)]


def exact(case, seed):
    if case["op"] != "chunk":
        return None  # blocks and tables are copied, not computed
    s = prepare(case, seed)
    new, kv = lengths(case)
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    out = torch.empty(sum(new), case["hq"], HEAD_DIM, dtype=torch.float64, device="cuda")
    table = torch.tensor(E4M3, dtype=torch.float64, device="cuda")
    at = 0
    for b, (t, n) in enumerate(zip(new, kv)):
        ids = s["tables"][b, :-(-n // BLOCK)].long()
        for h in range(hkv):
            k, v = cached(s, ids, h, table)
            for g in range(group):
                head = h * group + g
                for a in range(0, t, 512):  # pieces of the queries, to bound memory
                    z = min(t, a + 512)
                    sc = s["q"][at + a:at + z, head].double() @ k[:n].T / math.sqrt(HEAD_DIM)
                    limit = n - t + torch.arange(a, z, device="cuda")
                    hidden = torch.arange(n, device="cuda")[None, :] > limit[:, None]
                    out[at + a:at + z, head] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v[:n]
        at += t
    return out


def cached(s, ids, h, table):
    """Keys and values of KV head h in the blocks `ids`, in 64 bits."""
    if s["pool"] == "bf16":
        slots = (ids[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).view(-1)
        return s["k"][slots, h].double(), s["v"][slots, h].double()
    c = s["pool8"][ids, h]  # [blocks, 4224]
    i = torch.arange(16, device="cuda")
    # byte 4i + u of a group holds element 2i + u (u = 0, 1) or 2i + 6 + u (u = 2, 3)
    element = 2 * (i // 4) + i % 4 + 6 * (i % 4 >= 2)
    group = torch.empty(len(ids), BLOCK, 8, 16, dtype=torch.float64, device="cuda")
    group[..., element] = table[c[:, :2048].view(-1, BLOCK, 8, 16).long()]
    stored = torch.arange(8, device="cuda")[None, :] ^ (i % 8)[:, None]  # [token, group] -> stored group
    k = group[:, i[:, None], stored].reshape(-1, BLOCK, HEAD_DIM)
    v = torch.empty(len(ids), HEAD_DIM, BLOCK, dtype=torch.float64, device="cuda")
    v[..., element] = table[c[:, 2048:4096].view(-1, HEAD_DIM, 16).long()]
    scales = c[:, 4096:].contiguous().view(torch.float32).double().view(-1, 2, BLOCK, 1)
    return (k * scales[:, 0]).view(-1, HEAD_DIM), (v.transpose(1, 2) * scales[:, 1]).reshape(-1, HEAD_DIM)
