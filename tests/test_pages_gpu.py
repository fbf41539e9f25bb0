"""Blocks copied and moved in every plane of a pool (pkv_copy_blocks,
pkv_move_blocks): bytes equal to indexed copies, tables to a lookup."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def pool_of(device, fmt, layers, blocks, hkv, seed=0):
    import pagedkv

    g = torch.Generator(device=device).manual_seed(seed)
    if fmt == "bf16":
        raw = torch.randint(0, 1 << 16, (layers, 2, blocks * 16, hkv, 128), generator=g, device=device,
                            dtype=torch.int32).to(torch.int16)
        return raw.view(torch.bfloat16)
    return torch.randint(0, 256, (layers, blocks, hkv, pagedkv.fp8_block_bytes()), generator=g,
                         device=device, dtype=torch.int32).to(torch.uint8)


def blocks_of(pool):
    """[planes, blocks, bytes] view."""
    p = pool.view(torch.uint8)
    if pool.dtype == torch.bfloat16:
        return p.view(-1, pool.shape[-3] // 16, 16 * pool.shape[-2] * 256)
    return p.view(-1, pool.shape[-3], pool.shape[-2] * pool.shape[-1])


def pairs(device, blocks, n, seed):
    """n distinct targets, sources among the other blocks (with repeats)."""
    g = torch.Generator(device=device).manual_seed(seed)
    order = torch.randperm(blocks, generator=g, device=device)
    src = order[n:][torch.randint(blocks - n, (n,), generator=g, device=device)]
    return src.to(torch.int32), order[:n].to(torch.int32)


FMT = pytest.mark.parametrize("fmt", ["bf16", "fp8"])


@FMT
@pytest.mark.parametrize("layers,blocks,hkv,n", [(1, 2, 1, 1), (28, 40, 2, 1), (3, 100, 8, 37),
                                                 (28, 600, 2, 290), (2, 3000, 1, 1400), (1, 9, 5, 0)])
def test_copy(cuda, fmt, layers, blocks, hkv, n):
    import pagedkv

    pool = pool_of(cuda, fmt, layers, blocks, hkv, seed=n)
    want = blocks_of(pool).clone()
    src, dst = pairs(cuda, blocks, n, n) if n else (torch.empty(0, dtype=torch.int32, device=cuda),) * 2
    want[:, dst.long()] = want[:, src.long()]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    pagedkv.copy_blocks(pool, src, dst, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(blocks_of(pool), want)


@FMT
def test_one_layer_view(cuda, fmt):
    import pagedkv

    pool = pool_of(cuda, fmt, 4, 30, 2)
    want = blocks_of(pool).clone().view(4, -1, *blocks_of(pool).shape[1:])
    want[2][:, 5] = want[2][:, 9]
    ids = torch.tensor([9, 5], dtype=torch.int32, device=cuda)
    pagedkv.copy_blocks(pool[2], ids[:1], ids[1:])
    torch.cuda.synchronize()
    assert torch.equal(blocks_of(pool), want.view_as(blocks_of(pool)))


@FMT
def test_padding_pairs_and_bad_ids(cuda, fmt):
    """Both ids negative: skipped in silence; another id outside the pool: skipped and flagged."""
    import pagedkv

    pool = pool_of(cuda, fmt, 2, 20, 2)
    want = blocks_of(pool).clone()
    want[:, 3] = want[:, 7]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)

    def go(src, dst):
        err.zero_()
        pagedkv.copy_blocks(pool, torch.tensor(src, dtype=torch.int32, device=cuda),
                            torch.tensor(dst, dtype=torch.int32, device=cuda), err)
        torch.cuda.synchronize()
        assert torch.equal(blocks_of(pool), want)
        return int(err.item())

    assert go([-1, 7, -1, 4], [-1, 3, -1, 4]) == 0
    assert go([7, 20], [3, 2]) == 1
    assert go([7, 5], [3, 1 << 30]) == 1
    assert go([7, -1], [3, 5]) == 1
    assert go([7, 5], [3, -1]) == 1


@FMT
@pytest.mark.parametrize("layers,blocks,n,rows,cols", [(1, 8, 2, 1, 1), (28, 400, 90, 33, 50),
                                                       (2, 2000, 700, 256, 301), (3, 50, 1, 7, 4000)])
def test_move(cuda, fmt, layers, blocks, n, rows, cols):
    import pagedkv

    g = torch.Generator(device=cuda).manual_seed(blocks)
    pool = pool_of(cuda, fmt, layers, blocks, 2)
    want = blocks_of(pool).clone()
    order = torch.randperm(blocks, generator=g, device=cuda)
    src, dst = order[:n].sort().values, order[n:2 * n]
    # a wider table whose extra columns must stay; entries of every kind, junk among them
    table = torch.randint(-3, blocks + 3, (rows, cols + 5), generator=g, device=cuda, dtype=torch.int32)
    before = table.clone()
    to = torch.arange(blocks, dtype=torch.int32, device=cuda)
    to[src] = dst.to(torch.int32)
    part = before[:, :cols].long()
    moved = torch.where((part >= 0) & (part < blocks), to[part.clamp(0, blocks - 1)], before[:, :cols])
    want[:, dst] = want[:, src]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    pagedkv.move_blocks(pool, src.to(torch.int32), dst.to(torch.int32), table[:, :cols], err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(blocks_of(pool), want)
    assert torch.equal(table[:, :cols], moved) and torch.equal(table[:, cols:], before[:, cols:])


def test_captured_copy_replays_with_other_pairs(cuda):
    import pagedkv

    pool = pool_of(cuda, "bf16", 2, 64, 2)
    src, dst = (torch.full((8,), -1, dtype=torch.int32, device=cuda) for _ in range(2))
    pagedkv.copy_blocks(pool, src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pagedkv.copy_blocks(pool, src, dst)
    for seed in range(3):
        want = blocks_of(pool).clone()
        s, d = pairs(cuda, 64, 5, seed)
        src.fill_(-1), dst.fill_(-1)
        src[:5], dst[:5] = s, d
        want[:, d.long()] = want[:, s.long()]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(blocks_of(pool), want)


def test_planes_past_4_gib(cuda):
    """Block offsets past 32 bits within one plane."""
    import pagedkv

    blocks = (5 << 30) // (16 * 2 * 256)
    pool = torch.zeros(2, blocks * 16, 2, 128, dtype=torch.bfloat16, device=cuda)
    b = blocks_of(pool)
    b[0, blocks - 1] = 3
    b[1, blocks - 1] = 5
    b[1, 0] = 9
    src = torch.tensor([0, blocks - 1], dtype=torch.int32, device=cuda)
    dst = torch.tensor([blocks - 3, 7], dtype=torch.int32, device=cuda)
    pagedkv.copy_blocks(pool, src, dst)
    torch.cuda.synchronize()
    assert bool((b[0, 7] == 3).all() and (b[1, 7] == 5).all() and (b[1, blocks - 3] == 9).all())
    assert bool((b[0, blocks - 3] == 0).all() and (b[0, 8] == 0).all())


def test_refused_arguments(cuda):
    import pagedkv

    pool = pool_of(cuda, "bf16", 2, 20, 2)
    ids = torch.zeros(3, dtype=torch.int32, device=cuda)
    tables = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    for bad in (lambda: pagedkv.copy_blocks(pool.float(), ids, ids),
                lambda: pagedkv.copy_blocks(pool[:, :, :, :, :64], ids, ids),
                lambda: pagedkv.copy_blocks(pool[:, :, :24], ids, ids),
                lambda: pagedkv.copy_blocks(pool.cpu(), ids.cpu(), ids.cpu()),
                lambda: pagedkv.copy_blocks(pool, ids.long(), ids),
                lambda: pagedkv.copy_blocks(pool, ids, ids[:2]),
                lambda: pagedkv.copy_blocks(pool, ids.cpu(), ids),
                lambda: pagedkv.move_blocks(pool, ids, ids, tables.long()),
                lambda: pagedkv.move_blocks(pool, ids, ids, tables[0]),
                lambda: pagedkv.move_blocks(pool, ids, ids, tables.T)):
        with pytest.raises(ValueError):
            bad()
