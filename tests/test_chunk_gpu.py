"""Packed-chunk attention over the paged cache (pkv_paged_chunk, bf16 and FP8
pools) against a plain implementation in 64 bits.

Tolerance, elementwise.  With o = sum p_j v_j and A = sum p_j |v_j| (p the
exact softmax): the result's rounding is off by at most half a bf16 step,
2^-8 |o|; the products take p_j rounded to bf16 (f16 for the FP8 pool, a finer
step), 2^-8 A; scores are fp32 sums of 128 products, off by at most
130 * 2^-24 * S with S = scale * sum |q_d k_d|, which moves p by twice that
relatively, and ex2, the sums over keys and the running rescale add a few
2^-22 each: 2^-16 A covers them up to 64 rescales.

The FP8 kernel takes e4m3 * scale as f16.  A key element is off by at most
2^-12 of itself (one rounding to 11 bits; the scale is held in two terms), so a
score by 2^-12 S and p by twice that relatively; a value element by 2^-12 for
its scale and 2^-12 for the product, 2^-11 A in all.  The kernel holds values
times 2^6, so one of less than 2^-20 lies below f16's normal range there and is
off by at most half its least step, 2^-25 / 2^6 = 2^-31 (weights sum to 1, so
the result by no more).  Its products take p_j as f16 too: one that has fallen
below f16's normal range is off by half its least step, 2^-25, of a number that
holds the largest p as 2^7, so by 2^-32 of the largest; the short kernel rounds
p_j times its row's scale, relative to four times the largest scale, 2^-30 of
the largest value.  Over n keys that is at most n 2^-30 max |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 1.0 / math.sqrt(128)


def make(device, new, kv, hq, hkv, fmt="bf16", seed=0, poison=True, spare_rows=0, amp=1.0, edit=None):
    """Pool, tables, packed q of rows with `new` tokens and `kv` positions.
    Everything that belongs to no position (other blocks, the tail of the last
    block) holds NaN when `poison`.  edit(keys, values) changes a sequence's
    before they are stored."""
    import pagedkv

    g = torch.Generator(device=device).manual_seed(seed)
    need = [-(-n // 16) for n in kv]
    nb = sum(need) + 3
    order = torch.randperm(nb, generator=g, device=device).to(torch.int32)
    pitch = max(need) + 1
    tables = torch.full((len(kv) + 2, pitch), 0, dtype=torch.int32, device=device)
    rows = torch.randperm(len(kv) + 2, generator=g, device=device)[:len(kv)].to(torch.int32)
    k = torch.full((nb * 16, hkv, 128), float("nan"), device=device)
    v = k.clone()
    if not poison:
        k.zero_(), v.zero_()
    at = 0
    dense = []
    for b, n in enumerate(kv):
        ids = order[at:at + need[b]]
        at += need[b]
        tables[rows[b].item(), :need[b]] = ids
        pos = torch.arange(n, device=device)
        slot = ids.long()[pos // 16] * 16 + pos % 16
        kk = torch.randn(n, hkv, 128, generator=g, device=device) * amp
        vv = torch.randn(n, hkv, 128, generator=g, device=device)
        vv *= torch.exp(torch.randn(n, hkv, 1, generator=g, device=device))
        if edit is not None:
            edit(kk, vv)
        k[slot], v[slot] = kk, vv
        dense.append(slot)
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    N = sum(new) + spare_rows
    q = torch.randn(N, hq, 128, generator=g, device=device).to(torch.bfloat16)
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)
    kv_lens = torch.tensor(kv, dtype=torch.int32, device=device)
    c = dict(q=q, k=k, v=v, tables=tables, rows=rows, starts=starts, kv_lens=kv_lens, new=new, kv=kv,
             hq=hq, hkv=hkv, slots=dense, fmt=fmt)
    if fmt == "fp8":
        # write the positions through the library's own quantising append
        pool8 = torch.zeros(nb, hkv, pagedkv.fp8_block_bytes(), dtype=torch.uint8, device=device)
        if poison:  # NaN bytes and NaN scales everywhere but the written slots
            pool8[..., :4096] = 0x7F
            pool8[..., 4096:] = 0xFF
        for b, n in enumerate(kv):
            if n:
                kk = k[dense[b]].view(1, n, hkv, 128).transpose(1, 2)
                vv = v[dense[b]].view(1, n, hkv, 128).transpose(1, 2)
                pagedkv.append_rope_fp8(None, kk, vv, None, None, None, pool8, tables, rows[b:b + 1],
                                        torch.zeros(1, dtype=torch.int32, device=device))
        c["pool8"] = pool8
        c["k"], c["v"] = None, None
        c["read"] = []
        for b, n in enumerate(kv):
            c["read"].append(read_fp8(pool8, dense[b]))
    else:
        c["read"] = [(k[s].double(), v[s].double()) for s in dense]
    return c


def read_fp8(pool8, slots):
    """[n, hkv, 128] keys and values (64 bits) of the given slots."""
    from oracle import fp8_ref

    lut = torch.from_numpy(fp8_ref.e4m3_decode(torch.arange(256).numpy())).double().to(pool8.device)
    c = pool8[slots // 16]  # [n, hkv, chunk]
    t = (slots % 16).cpu()
    d = torch.arange(128)
    pl = torch.from_numpy(fp8_ref.fp8_pos(torch.arange(16).numpy()))
    ko = (t[:, None] * 128 + (((d >> 4)[None] ^ (t[:, None] & 7)) << 4) + pl[d & 15][None]).to(pool8.device)
    vo = (2048 + d[None] * 16 + pl[t][:, None]).to(pool8.device)
    hkv = pool8.shape[1]
    kb = torch.gather(c, 2, ko[:, None].expand(-1, hkv, -1))
    vb = torch.gather(c, 2, vo[:, None].expand(-1, hkv, -1))
    sc = c[..., 4096:].contiguous().view(torch.float32).double()  # [n, hkv, 32]
    ti = t.to(pool8.device)[:, None, None].expand(-1, hkv, 1)
    return lut[kb.long()] * sc.gather(2, ti), lut[vb.long()] * sc.gather(2, ti + 16)


def plain(c, causal=True):
    """(o, tolerance) in 64 bits, rows of no sequence NaN in both."""
    q = c["q"].double()
    o = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = o.clone()
    group = c["hq"] // c["hkv"]
    at = 0
    for b, (t, n) in enumerate(zip(c["new"], c["kv"])):
        k, v = (x.repeat_interleave(group, 1) for x in c["read"][b])  # [n, hq, 128]
        for a in range(0, t, 256):
            z = min(t, a + 256)
            qq = q[at + a:at + z]
            s = torch.einsum("thd,shd->hts", qq, k) * SCALE
            big = torch.einsum("thd,shd->hts", qq.abs(), k.abs()) * SCALE
            if causal:
                i = torch.arange(a, z, device=q.device)[:, None]
                hide = torch.arange(n, device=q.device)[None] > n - t + i
                s = s.masked_fill(hide, -math.inf)
                big = big.masked_fill(hide, 0.0)
            p = torch.softmax(s, -1) if n else s  # no visible key: NaN
            if n == 0:
                continue
            oo = torch.einsum("hts,shd->thd", p, v)
            A = torch.einsum("hts,shd->thd", p, v.abs())
            S = big.amax(-1).transpose(0, 1)[..., None] if n else 0.0
            o[at + a:at + z] = oo
            rel = 2.0 ** -8 + 2.0 ** -16 + 2 * 130 * 2.0 ** -24 * S
            if c["fmt"] == "fp8":
                rel = rel + 2 * 2.0 ** -12 * S + 2.0 ** -11
            least = 0.0
            if c["fmt"] == "fp8":
                least = 2.0 ** -31 + n * 2.0 ** -30 * v.abs().amax((0, 2))[None, :, None]
            tol[at + a:at + z] = 2.0 ** -8 * oo.abs() + rel * A + least
        at += t
    return o, tol


def call(c, causal=True, out=None, max_kv=None, err=None):
    import pagedkv

    out = torch.full_like(c["q"], 7.0) if out is None else out
    err = torch.zeros(1, dtype=torch.int32, device=out.device) if err is None else err
    mk = max(c["kv"] + [0]) if max_kv is None else max_kv
    if c["fmt"] == "fp8":
        pagedkv.paged_chunk_fp8(c["q"], c["pool8"], c["tables"], c["rows"], c["starts"], c["kv_lens"],
                                mk, out, causal, SCALE, err)
    else:
        pagedkv.paged_chunk(c["q"], c["k"], c["v"], c["tables"], c["rows"], c["starts"], c["kv_lens"],
                            mk, out, causal, SCALE, c["hkv"], err)
    torch.cuda.synchronize()
    return out, int(err.item())


def check(c, causal=True, **kw):
    out, err = call(c, causal, **kw)
    assert err == 0, f"device error bits {err:#x}"
    want, tol = plain(c, causal)
    n = sum(c["new"])
    got = out[:n].double()
    want, tol = want[:n], tol[:n]
    assert torch.equal(got.isnan(), want.isnan()), "NaN in other places than the formula's"
    ok = ~want.isnan()
    over = (got - want).abs()[ok] - tol[ok]
    assert over.numel() == 0 or over.max().item() <= 0, \
        f"off by {(got - want).abs()[ok].max().item()}, {over.max().item()} over the tolerance"
    assert bool((out[n:] == 7.0).all()), "rows of no sequence were written"
    return out


FMT = pytest.mark.parametrize("fmt", ["bf16", "fp8"])


@FMT
@pytest.mark.parametrize("new,kv", [
    ([1], [1]), ([1], [16]), ([1], [17]), ([1], [129]), ([3], [3]), ([5], [128]), ([21], [127]),
    ([22], [300]), ([42], [42]), ([43], [555]), ([64], [1000]), ([130], [257]), ([300], [300]),
    ([1, 1, 1], [5, 1030, 64]), ([2, 0, 7, 1], [40, 33, 7, 2000]), ([4] * 9, [100 * i + 4 for i in range(9)]),
    ([200, 1, 1, 33, 1], [700, 15, 1600, 33, 257]),
])
def test_lengths(cuda, fmt, new, kv):
    check(make(cuda, new, kv, 12, 2, fmt, spare_rows=3))


@FMT
@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (8, 1), (16, 4), (28, 4), (32, 8), (6, 6), (15, 3),
                                    (13, 1), (64, 1), (48, 2), (33, 1)])
def test_head_layouts(cuda, fmt, hq, hkv):
    check(make(cuda, [1, 37, 5], [300, 130, 517], hq, hkv, fmt, seed=hq))


@FMT
@pytest.mark.parametrize("new,kv", [([1], [9000]), ([4], [20001]), ([60], [8195]), ([1, 1], [40000, 3]),
                                    ([7] * 5, [6000, 129, 4097, 7, 2050]), ([700], [5000]),
                                    ([2] * 40, [900 + 31 * i for i in range(40)])])
def test_long_caches_split_over_keys(cuda, fmt, new, kv):
    check(make(cuda, new, kv, 12, 2, fmt, seed=len(kv)))


@FMT
def test_all_positions_visible(cuda, fmt):
    """causal = 0: every token of a row sees all its positions."""
    check(make(cuda, [1, 50, 3, 129], [700, 90, 1, 131], 12, 2, fmt), causal=False)


@FMT
@pytest.mark.parametrize("causal", [True, False])
def test_rows_without_a_visible_key_are_nan(cuda, fmt, causal):
    """More tokens than positions (the first ones see nothing), and no position at all."""
    check(make(cuda, [5, 3, 1, 60, 300], [2, 0, 0, 13, 150], 12, 2, fmt), causal=causal)


@FMT
def test_no_token_at_all(cuda, fmt):
    c = make(cuda, [0, 0], [40, 0], 12, 2, fmt, spare_rows=4)
    out, err = call(c)
    assert err == 0 and bool((out == 7.0).all())


@FMT
def test_large_scores(cuda, fmt):
    """Scores of several hundred: one key takes a row, then another moves the maximum."""
    check(make(cuda, [30, 2], [900, 3000], 12, 2, fmt, seed=5, amp=60.0))


@FMT
@pytest.mark.parametrize("new", [[1], [5], [40], [2, 40]])
@pytest.mark.parametrize("value", [1e-4, 1.0, 90.0])
def test_small_terms_of_a_long_cache_keep_their_weight(cuda, fmt, new, value):
    """One key far above the others (e^12.5) and 30000 that together weigh a
    tenth of it: neither the small terms nor values as small as f16's least
    normal numbers may be lost to a narrow format."""
    def edit(kk, vv):
        kk *= 0.02
        kk[5] = 12.5 / SCALE / 128
        vv.fill_(value)
        vv[5] = -value

    c = make(cuda, new, [30000] * len(new), 12, 2, fmt, seed=6, edit=edit)
    c["q"].fill_(1.0)
    out = check(c)
    assert float(out.max()) > -0.95 * value  # the tail counts


@FMT
def test_strided_q_and_out(cuda, fmt):
    """q as a slice of a merged q/k/v buffer, out with another token pitch and head order."""
    c = make(cuda, [9, 1, 40], [300, 70, 40], 12, 2, fmt)
    n = c["q"].shape[0]
    wide = torch.zeros(n, 16, 128, dtype=torch.bfloat16, device=cuda)
    wide[:, 2:14] = c["q"]
    want = check(c)
    c["q"] = wide[:, 2:14]
    buf = torch.full((13, n + 2, 136), 7.0, dtype=torch.bfloat16, device=cuda)
    out = buf[:12, :n, :128].transpose(0, 1)
    got, err = call(c, out=out)
    assert err == 0 and torch.equal(got, want)
    assert bool((buf[12:] == 7.0).all() and (buf[:, n:] == 7.0).all() and (buf[..., 128:] == 7.0).all())


@FMT
def test_same_bits_on_every_call_and_capacity(cuda, fmt):
    """The result does not depend on the order in which parts finish, nor the call on an earlier one."""
    c = make(cuda, [1, 4, 90, 1], [5000, 2000, 700, 12000], 12, 2, fmt)
    a, _ = call(c)
    for _ in range(3):
        b, _ = call(c)
        assert torch.equal(a, b)
    check(c, max_kv=c["tables"].shape[1] * 16)


@FMT
@pytest.mark.parametrize("new,kv", [([21] * 40, [2048] * 40), ([10] * 40, [2000 + i for i in range(40)]),
                                    ([700], [5000]), ([1500, 3], [9000, 20000])])
def test_repeated_calls_give_the_same_bits(cuda, fmt, new, kv):
    """Items back to back in every CTA, the rings full: a copy or a tile
    released before it was read shows as other bits on some call."""
    c = make(cuda, new, kv, 12, 2, fmt)
    first = check(c)
    for _ in range(40):
        out, err = call(c)
        assert err == 0 and torch.equal(out, first)


@FMT
def test_captured_graph_replays_on_other_lengths(cuda, fmt):
    """A call captured for a capacity of tokens and positions replays for any
    lengths within it: rows are padded with T = 0."""
    import pagedkv

    base = make(cuda, [40, 1, 1, 6], [900, 400, 30, 2500], 12, 2, fmt)
    q, starts, kv_lens = torch.zeros(64, 12, 128, dtype=torch.bfloat16, device=cuda), \
        torch.zeros(5, dtype=torch.int32, device=cuda), torch.zeros(4, dtype=torch.int32, device=cuda)
    out, err = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device=cuda)
    cap = base["tables"].shape[1] * 16

    def go():
        if fmt == "fp8":
            pagedkv.paged_chunk_fp8(q, base["pool8"], base["tables"], base["rows"], starts, kv_lens, cap,
                                    out, True, SCALE, err)
        else:
            pagedkv.paged_chunk(q, base["k"], base["v"], base["tables"], base["rows"], starts, kv_lens,
                                cap, out, True, SCALE, 2, err)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for new in ([40, 1, 1, 6], [0, 1, 0, 0], [1, 1, 1, 1], [64, 0, 0, 0], [3, 20, 2, 30]):
        kv = [n if t else 0 for t, n in zip(new, base["kv"])]
        c = dict(base, new=new, kv=kv, q=q)
        c["read"] = [(k[:n], v[:n]) for (k, v), n in zip(base["read"], kv)]
        q.copy_(torch.randn(q.shape, device=cuda))
        starts.copy_(torch.tensor([sum(new[:i]) for i in range(5)], dtype=torch.int32))
        kv_lens.copy_(torch.tensor(kv, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        want, tol = plain(c)
        n = sum(new)
        assert torch.equal(out[:n].isnan(), want[:n].isnan())
        ok = ~want[:n].isnan()
        assert bool(((out[:n].double() - want[:n]).abs()[ok] <= tol[:n][ok]).all())
        assert bool((out[n:] == 7.0).all())


@FMT
def test_two_streams_at_once(cuda, fmt):
    cs = [make(cuda, [4, 1], [9000 + i, 700], 12, 2, fmt, seed=i) for i in range(4)]
    want = [call(c)[0] for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [torch.full_like(c["q"], 7.0) for c in cs]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    import pagedkv

    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, o in zip(cs, streams, outs):
            with torch.cuda.stream(s):
                if fmt == "fp8":
                    pagedkv.paged_chunk_fp8(c["q"], c["pool8"], c["tables"], c["rows"], c["starts"],
                                            c["kv_lens"], max(c["kv"]), o, True, SCALE, err)
                else:
                    pagedkv.paged_chunk(c["q"], c["k"], c["v"], c["tables"], c["rows"], c["starts"],
                                        c["kv_lens"], max(c["kv"]), o, True, SCALE, 2, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


@FMT
def test_bad_block_ids_are_flagged(cuda, fmt):
    """A table entry outside the pool reads block 0 and sets the flag; the other rows are right."""
    c = make(cuda, [4, 3], [200, 300], 12, 2, fmt, poison=False)
    c["tables"][c["rows"][0].item(), 3] = 1 << 28
    c["tables"][c["rows"][0].item(), 4] = -5
    out, err = call(c)
    assert err == 1
    want, tol = plain(c)
    assert bool(((out[4:].double() - want[4:]).abs() <= tol[4:]).all())


@FMT
def test_positions_past_the_table_are_flagged(cuda, fmt):
    c = make(cuda, [2], [100], 12, 2, fmt, poison=False)
    c["kv_lens"].fill_(100000)
    _, err = call(c, max_kv=100000)
    assert err & 2


@FMT
def test_blocks_past_4_gib(cuda, fmt):
    """The rows' blocks lie past the first 4 GiB of a plane."""
    c = make(cuda, [5, 1], [500, 77], 12, 2, fmt)
    if fmt == "fp8":
        unit = c["pool8"][0].numel()
        nb = c["pool8"].shape[0]
        far = (5 << 30) // unit
        big = torch.empty(far + nb, *c["pool8"].shape[1:], dtype=torch.uint8, device=cuda)
        big[far:] = c["pool8"]
        c["pool8"] = big
    else:
        nb = c["k"].shape[0] // 16
        far = (5 << 30) // (16 * 2 * 256)
        for name in "kv":
            big = torch.empty((far + nb) * 16, 2, 128, dtype=torch.bfloat16, device=cuda)
            big[far * 16:] = c[name]
            c[name] = big
    c["tables"] += far
    check(c)


def test_decode_rows_agree_with_the_decode_kernel(cuda):
    """T = 1 rows: the same attention as pkv_paged_decode, each within its
    rounding.  (The pool is finite throughout: the decode kernel multiplies
    the tail of a row's last block by zero probabilities.)"""
    import pagedkv

    c = make(cuda, [1] * 6, [1, 16, 700, 33, 5000, 128], 12, 2, poison=False)
    out, _ = call(c)
    other = torch.empty_like(out)
    pagedkv.paged_decode(c["q"], c["k"], c["v"], c["tables"], c["rows"], c["kv_lens"], 5000, other,
                         SCALE, 2)
    want, tol = plain(c)
    assert bool(((out.double() - want).abs() <= tol).all())
    assert bool(((out.double() - other.double()).abs() <= 2 * tol).all())


def test_refused_arguments(cuda):
    import pagedkv

    c = make(cuda, [4, 1], [40, 20], 12, 2, poison=False)
    ok = dict(q=c["q"], k=c["k"], v=c["v"], tables=c["tables"], rows=c["rows"], starts=c["starts"],
              kv_lens=c["kv_lens"], out=torch.empty_like(c["q"]), hkv=2, scale=SCALE)

    def go(**kw):
        a = dict(ok, **kw)
        pagedkv.paged_chunk(a["q"], a["k"], a["v"], a["tables"], a["rows"], a["starts"], a["kv_lens"], 40,
                            a["out"], True, a["scale"], a["hkv"])

    go()
    for kw in (dict(q=c["q"].float()), dict(q=c["q"].cpu()), dict(out=c["q"][:3]),
               dict(starts=c["starts"][:2]), dict(starts=c["starts"].long()), dict(kv_lens=c["kv_lens"].long()),
               dict(rows=c["rows"][:1]), dict(tables=c["tables"].long()), dict(k=c["k"].float()),
               dict(k=c["k"][:, :1]), dict(v=c["v"][:16]), dict(tables=c["tables"][:1], rows=None),
               dict(tables=c["tables"].cpu())):
        with pytest.raises(ValueError):
            go(**kw)
    with pytest.raises(pagedkv.PagedKVError):
        go(hkv=2, scale=0.0)
    with pytest.raises(pagedkv.PagedKVError):  # token rows not 16-byte aligned
        w = torch.empty(5, 12, 129, dtype=torch.bfloat16, device=cuda)
        go(q=w[..., :128])
    q = torch.empty(5, 130, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(pagedkv.PagedKVError):  # 65 query heads per KV head
        go(q=q, out=torch.empty_like(q))
