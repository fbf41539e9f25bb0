"""Packed steps on a cache whose sequences share, copy, roll back and move
blocks: prepare_packed -> append -> packed_attention between fork, truncate and
compact, on both pools; then the whole model (forward_packed) checking drafted
tokens, and chats that fork.

The tolerance of the attention is test_chunk_gpu's; the K/V of every sequence
must be, byte for byte, what the one-sequence-at-a-time path stores."""
import copy

import pytest
import torch

from test_chunk_gpu import plain, read_fp8
from test_model_gpu import (MARGIN_BF16, MARGIN_FP32, _agreement, _teacher_forced,
                            models)  # noqa: F401 (fixture)

pytestmark = pytest.mark.gpu

FMT = pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3"])
HQ, HKV = 12, 2
LAYERS = 3


def _cache(blocks, cuda, fmt):
    from kv_cache import KVCache

    c = KVCache(blocks, 16, cuda, torch.bfloat16, num_layers=LAYERS, kv_format=fmt)
    if c.fp8:  # positions that were never written are no number
        c.pool8.fill_(0xFF)
    else:
        c.buf.fill_(float("nan"))
    return c


class Runner:
    """A cache driven by packed steps, and what each of its sequences holds."""

    def __init__(self, blocks, cuda, fmt, seed=0):
        self.c, self.cuda, self.fmt = _cache(blocks, cuda, fmt), cuda, fmt
        self.g = torch.Generator(device=cuda).manual_seed(seed)
        self.kv = {}  # seq -> [tokens, layers, 2, HKV, 128]
        # cos 1, sin 0: the roped k is k
        self.cos = torch.ones(4096, 128, device=cuda, dtype=torch.bfloat16)
        self.sin = torch.zeros_like(self.cos)

    def alloc(self):
        s = self.c.alloc()
        self.kv[s] = torch.zeros(0, LAYERS, 2, HKV, 128, device=self.cuda, dtype=torch.bfloat16)
        return s

    def fork(self, seqs, lengths=None):
        new = self.c.fork_many(seqs, lengths)
        for f, s, n in zip(new, seqs, lengths or [None] * len(seqs)):
            self.kv[f] = self.kv[s][:n]
        return new

    def truncate(self, s, n):
        self.c.truncate(s, n)
        self.kv[s] = self.kv[s][:n]

    def free(self, s):
        self.c.free(s)
        del self.kv[s]

    def slots(self, s):
        table = torch.tensor(self.c.host_table(s) or [0], device=self.cuda)
        pos = torch.arange(self.c.length(s), device=self.cuda)
        return table[pos // 16] * 16 + pos % 16

    def read(self, s, layer):
        slots = self.slots(s)
        if self.c.fp8:
            return read_fp8(self.c.pool8[layer], slots)
        return tuple(self.c.buf[layer, i][slots].double() for i in range(2))

    def expected(self, s, layer):
        """The same through a cache of its own and the unpacked append."""
        if not self.c.fp8:
            return tuple(self.kv[s][:, layer, i].double() for i in range(2))
        own = _cache(max(1, -(-len(self.kv[s]) // 16)), self.cuda, self.fmt)
        r = Runner.__new__(Runner)
        r.c, r.cuda = own, self.cuda
        q = own.alloc()
        if len(self.kv[s]):
            _, step, _ = own.prepare([q], len(self.kv[s]))
            k, v = (self.kv[s][:, layer, i].transpose(0, 1)[None] for i in range(2))
            own.write(layer, step, k, v)
            own.advance([q], len(self.kv[s]))
        return r.read(q, layer)

    def step(self, seqs, new_lens, causal=True):
        """A packed step with random q, k, v; attention checked in every layer."""
        from kernels.fa2 import packed_attention

        c, N = self.c, sum(new_lens)
        qkv = torch.randn(N, LAYERS, HQ + 2 * HKV, 128, generator=self.g, device=self.cuda)
        qkv[:, :, HQ:] *= torch.exp(torch.randn(N, LAYERS, 1, 1, generator=self.g, device=self.cuda))
        qkv = qkv.to(torch.bfloat16)
        starts, step = c.prepare_packed(seqs, new_lens)
        assert starts == [c.length(s) for s in seqs]
        outs = []
        for layer in range(LAYERS):
            part = qkv[:, layer][:, :, None]  # [N, heads, 1, 128]
            q_rot = torch.empty(N, HQ, 128, device=self.cuda, dtype=torch.bfloat16)
            c.append(layer, step.tokens, part[:, :HQ], part[:, HQ:HQ + HKV], part[:, HQ + HKV:],
                     self.cos, self.sin, q_rot[:, :, None])
            assert torch.equal(q_rot, qkv[:, layer, :HQ])
            k, v = c.read(layer, step)
            outs.append(packed_attention(q_rot, k, v, causal))
        c.advance_packed(seqs, new_lens)
        c.check_errors()
        at = 0
        for s, n in zip(seqs, new_lens):
            new = qkv[at:at + n, :, HQ:].view(n, LAYERS, 2, HKV, 128)
            self.kv[s] = torch.cat([self.kv[s], new])
            at += n
        for layer in range(LAYERS):
            case = dict(q=qkv[:, layer, :HQ], hq=HQ, hkv=HKV, new=new_lens,
                        kv=[c.length(s) for s in seqs], read=[self.read(s, layer) for s in seqs],
                        fmt="fp8" if c.fp8 else "bf16")
            want, tol = plain(case, causal)
            over = (outs[layer].double() - want).abs() - tol
            assert N == 0 or over.max().item() <= 0, f"layer {layer}: {over.max().item()} over"
        self.check()

    def check(self):
        for s in self.kv:
            assert self.c.length(s) == len(self.kv[s])
            for layer in range(LAYERS):
                for a, b in zip(self.read(s, layer), self.expected(s, layer)):
                    assert torch.equal(a, b), f"seq {s}, layer {layer}"


@FMT
def test_a_run_of_sharing_attending_rolling_back_and_moving(cuda, fmt):
    r = Runner(80, cuda, fmt)
    a, b = r.alloc(), r.alloc()
    r.step([a, b], [200, 37])               # two prompts
    f, g, h = r.fork([a, a, b], [200, 128, 37])
    r.step([f, a, g, h, b], [3, 1, 20, 0, 1])  # checks, a decode token, a suffix, an idle row
    r.step([f, a], [0, 0])                  # nothing to do in a whole step
    r.truncate(f, 201)
    r.truncate(a, 64)                       # whole shared blocks dropped
    r.truncate(g, 100)                      # into a block that a held too: copied
    r.check()
    r.step([a, f, g], [5, 1, 1])
    beams = r.fork([f, f, g, b])            # one beam twice
    for s in (f, g):
        r.free(s)
    r.step(beams, [1, 1, 1, 1])
    r.free(b)
    used = r.c.compact()
    assert used == r.c.num_blocks - r.c.free_block_count() < 80
    r.check()
    c = r.alloc()                           # new blocks come right above
    r.step([*beams, a, c], [1, 1, 2, 1, 9, 150])
    r.step([c], [1], causal=False)
    for s in list(r.kv):
        r.free(s)
    assert r.c.free_block_count() == 80 and not r.c._shared


@FMT
def test_random_runs(cuda, fmt):
    import random

    rng = random.Random(5)
    r = Runner(120, cuda, fmt, seed=1)
    for _ in range(40):
        live = list(r.kv)
        op = rng.choice(["step", "step", "fork", "truncate", "free", "compact"])
        if len(live) < 2:
            r.alloc()
        elif op == "step":
            seqs = rng.sample(live, rng.randint(1, len(live)))
            lens = [rng.choice([0, 1, 1, 4, 17, 90]) for _ in seqs]
            try:
                r.step(seqs, lens)
            except RuntimeError as e:
                assert "exhausted" in str(e)
                r.free(rng.choice(live))
        elif op == "fork" and len(live) < 12 and r.c.free_block_count() > 3:
            seqs = [rng.choice(live) for _ in range(rng.randint(1, 3))]
            r.fork(seqs, rng.choice([None, [rng.randint(0, r.c.length(s)) for s in seqs]]))
        elif op == "truncate" and r.c.free_block_count():
            s = rng.choice(live)
            r.truncate(s, rng.randint(0, r.c.length(s)))
        elif op == "free":
            r.free(rng.choice(live))
        elif op == "compact":
            r.c.compact()
    r.check()


def test_refusals(cuda):
    from kernels.fa2 import flash_attention, packed_attention

    r = Runner(8, cuda, "bf16")
    a, b = r.alloc(), r.alloc()
    _, step = r.c.prepare_packed([a, b], [3, 2])
    k, v = r.c.read(0, step)
    q = torch.zeros(5, HQ, 128, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="packed_attention"):
        flash_attention(q[:2, :, None], k, v)
    with pytest.raises(AssertionError, match="new tokens"):
        packed_attention(q[:4], k, v)
    with pytest.raises(AssertionError, match="GQA"):
        packed_attention(q[:, :5], k, v)
    with pytest.raises(AssertionError, match="bf16"):
        packed_attention(q.float(), k, v)
    _, plain_step, _ = r.c.prepare([a], 1)
    k1, v1 = r.c.read(0, plain_step)
    with pytest.raises(AssertionError, match="prepare_packed"):
        packed_attention(q[:1], k1, v1)
    with pytest.raises(AssertionError, match="one read"):
        packed_attention(q, k, r.c.read(0, step)[1].__class__(r.c, 0, 1, plain_step))
    with pytest.raises(ValueError, match="twice"):
        r.c.prepare_packed([a, a], [1, 1])
    with pytest.raises(RuntimeError, match="exhausted"):
        r.c.prepare_packed([a, b], [100, 100])
    _, empty = r.c.prepare_packed([], [])
    assert packed_attention(q[:0], *r.c.read(0, empty)).shape == (0, HQ, 128)
    _, idle = r.c.prepare_packed([a, b], [0, 0])
    assert packed_attention(q[:0], *r.c.read(0, idle)).shape == (0, HQ, 128)


@pytest.mark.parametrize("fmt,gemm", [("bf16", "cublas"), ("bf16", "skinny"), ("fp8_e4m3", "skinny")])
def test_checking_drafts_gives_the_greedy_ids(cuda, models, fmt, gemm):  # noqa: F811
    """Both prompts in one packed forward, row 0 forked; then steps that check
    three drafted tokens per row (some right, some wrong, by a fixed pattern),
    keep those that the model would have chosen and truncate the rest.  The
    ids must be the oracle's greedy ids wherever its margin is decisive, as in
    the one-token-at-a-time paths, and the K/V that stays is untouched by the
    rejected tokens."""
    from kv_cache import KVCache

    ours, ref32, ref16, fx = models
    m = copy.deepcopy(ours).fuse_weights_()
    m.skinny_linears = gemm == "skinny"
    m.persistent_decode = True  # one packed token per row is still no decode step
    fp8 = fmt != "bf16"
    prompts, steps = fx["prompts"], fx["steps"]
    c = KVCache(64, 16, cuda, torch.bfloat16, kv_format=fmt)
    seqs = [c.alloc(), c.alloc()]
    ids, logits = [[], [], []], [[], [], []]

    def take(r, lg):
        logits[r].append(lg)
        ids[r].append(int(lg.argmax()))

    with torch.no_grad():
        lg = m.forward_packed(torch.tensor(prompts[0] + prompts[1]), c, seqs,
                              [len(p) for p in prompts]).float()
        seqs.append(c.fork(seqs[0]))
        for r in range(3):
            take(r, lg[r % 2])
        turn = 0
        while min(len(x) for x in ids) <= steps:
            rows = [r for r in range(3) if len(ids[r]) <= steps]
            if turn % 2 == 0:  # drafts of the reference's ids, spoiled at a moving place
                drafts = []
                for r in rows:
                    ref = fx["ids"][r % 2] + [1, 2, 3]
                    d = [int(x) for x in ref[len(ids[r]):len(ids[r]) + 3]]
                    d = (d + [4, 5, 6])[:3]
                    d[(turn + r) % 3] ^= 1 if turn % 4 else 0
                    drafts.append(d)
            else:  # a plain decode step of every row, through the packed forward
                drafts = [[] for _ in rows]
            new = [[ids[r][-1]] + d for r, d in zip(rows, drafts)]
            live = [seqs[r] for r in rows]
            at = 0
            lg = m.forward_packed(torch.tensor(sum(new, [])), c, live, [len(x) for x in new],
                                  all_logits=True).float()
            for r, d in zip(rows, drafts):
                start = c.length(seqs[r]) - len(d) - 1
                take(r, lg[at])
                kept = 0
                while kept < len(d) and d[kept] == ids[r][-1]:
                    kept += 1
                    take(r, lg[at + kept])
                table = c.host_table(seqs[r])
                pool = c.pool8 if fp8 else c.buf.view(28, 2, 64, 16, -1)
                first = table[:(start + 1 + kept) // 16]
                before = pool[:, first].clone() if fp8 else pool[:, :, first].clone()
                c.truncate(seqs[r], start + 1 + kept)
                after = pool[:, first] if fp8 else pool[:, :, first]
                assert torch.equal(before, after)
                at += len(d) + 1
            turn += 1
            if turn == 3:
                extra = c.fork(seqs[1])
                c.free(extra)
                c.compact()
    torch.cuda.synchronize()
    c.check_errors()
    for r in range(3):  # every id but the last is in the cache
        assert c.length(seqs[r]) == len(prompts[r % 2]) + len(ids[r]) - 1
    torch.backends.cuda.matmul.allow_tf32 = False
    every = [prompts[0], prompts[1], prompts[0]]
    flat = [t for row in ids for t in row]
    flat_logits = [x for row in logits for x in row]
    for ref, dtype, margin in ((ref16, torch.bfloat16, MARGIN_BF16), (ref32, torch.float32, MARGIN_FP32)):
        want = [x for row in _teacher_forced(ref, dtype, every, ids, cuda, fp8) for x in row]
        decisive, agree, bad = _agreement(want, flat, margin)
        off = max(float((x - y).abs().max()) for x, y in zip(flat_logits, want))
        print(fmt, gemm, dtype, decisive, agree, bad, off)
        assert decisive >= 3 and agree == decisive, (decisive, agree, bad, off)


def test_packed_forward_refusals(cuda, models):  # noqa: F811
    from kv_cache import KVCache

    m = copy.deepcopy(models[0]).fuse_weights_()
    c = KVCache(4, 16, cuda, torch.bfloat16)
    s = c.alloc()
    for ids, seqs, lens in ((torch.tensor([1, 2]), [s], [3]), (torch.tensor([[1, 2]]), [s], [2]),
                            (torch.tensor([1]), [s, c.alloc()], [1, 0]),
                            (torch.zeros(0, dtype=torch.long), [], [])):
        with pytest.raises(ValueError):
            m.forward_packed(ids, c, seqs, lens)
    with pytest.raises(RuntimeError, match="exhausted"):
        m.forward_packed(torch.zeros(80, dtype=torch.long), c, [s], [80])
    assert c.length(s) == 0 and c.free_block_count() == 4


def test_a_forked_chat_reads_its_parents_blocks(cuda, models, monkeypatch):  # noqa: F811
    """The scheduler on the real model: a fork prefills only its own message on
    top of shared blocks, and both chats' K/V of the history stay equal."""
    import queue

    import chat
    from kv_cache import KVCache
    from oracle.scheduler_trace import FakeTokenizer

    m = copy.deepcopy(models[0]).fuse_weights_()
    monkeypatch.setattr(chat, "_job_queue", queue.Queue())
    monkeypatch.setattr(chat, "MAX_REPLY_TOKENS", 8)
    for state in (chat.active, chat._deferred, chat._resident, chat._mixed):
        state.clear()
    cache = KVCache(64, 16, cuda, torch.bfloat16)
    chat.init(kv_cache=cache, start_worker=False)
    try:
        a = chat.Chat(FakeTokenizer())
        a.submit(m, "x" * 60)
        chat.run_until_idle()
        n = cache.length(a.seq)
        b = a.fork()
        b.submit(m, "one way")
        a.submit(m, "or another")
        chat.run_until_idle()
        cache.check_errors()
        ta, tb = cache.host_table(a.seq), cache.host_table(b.seq)
        assert n % 16 and ta[:n // 16] == tb[:n // 16] and not set(ta[n // 16:]) & set(tb)
        last = cache.buf.view(28, 2, 64, 16, -1)[:, :, :, :n % 16]
        assert torch.equal(last[:, :, ta[n // 16]], last[:, :, tb[n // 16]])
        assert not cache.buf.isnan().any()
        a.release()
        b.release()
        assert cache.free_block_count() == 64
    finally:
        chat._kv_cache = None
        chat._resident.clear()
