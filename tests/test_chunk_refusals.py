"""What the packed-chunk and block entry points refuse, before any CUDA call
(so no GPU is needed): the C entries by status and message, the Python
wrappers by ValueError."""
import math

import pytest
import torch

INVALID, UNSUPPORTED, ALIGN, WORKSPACE = 1, 2, 3, 6

CHUNK = dict(q=16, q_st=1536, q_sh=128, k=16, v=16, slots=64, tables=16, pitch=4, rows=None,
             q_starts=16, kv_lens=16, max_kv=64, batch=1, tokens=4, hq=12, hkv=2, d=128, causal=1,
             scale=0.1, out=16, o_st=1536, o_sh=128, ws=None, ws_bytes=0, err=None, stream=None)
CHUNK8 = {("pool" if k == "k" else "blocks" if k == "slots" else k): (4 if k == "slots" else v)
          for k, v in CHUNK.items() if k != "v"}
COPY = dict(pool=16, planes=2, stride=8192 * 8, block=8192, blocks=8, src=16, dst=16, n=2,
            err=None, stream=None)
MOVE = dict(list(COPY.items())[:8] + [("tables", 16), ("rows", 2), ("cols", 4), ("pitch", 4)]
            + list(COPY.items())[8:])


def _refused(name, args, change, status):
    import pagedkv

    L = pagedkv.lib()
    unknown = set(change) - set(args)
    assert not unknown, unknown
    assert getattr(L, name)(*{**args, **change}.values()) == status, L.pkv_last_error()


COMMON = [
    (dict(hq=5), INVALID), (dict(hkv=0), INVALID), (dict(hq=0), INVALID), (dict(hkv=-2), INVALID),
    (dict(hq=130, hkv=2), UNSUPPORTED), (dict(d=64), UNSUPPORTED),
    (dict(batch=-1), INVALID), (dict(tokens=-1), INVALID), (dict(max_kv=-1), INVALID),
    (dict(batch=16384), UNSUPPORTED), (dict(tokens=1 << 27), UNSUPPORTED),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(q_starts=None), INVALID),
    (dict(kv_lens=None), INVALID), (dict(tables=None), INVALID), (dict(pitch=0), INVALID),
    (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(q=24), ALIGN), (dict(out=20), ALIGN),
    (dict(q_st=1540), ALIGN), (dict(q_sh=132), ALIGN), (dict(o_st=1540), ALIGN), (dict(o_sh=129), ALIGN),
    (dict(tokens=4096, batch=2), WORKSPACE), (dict(tokens=4096, ws=24, ws_bytes=1 << 40), ALIGN),
]


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=24), ALIGN), (dict(v=40), ALIGN),
    (dict(slots=17), INVALID), (dict(slots=0), INVALID)], ids=str)
def test_chunk(change, status):
    _refused("pkv_paged_chunk", CHUNK, change, status)


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(pool=None), INVALID), (dict(pool=24), ALIGN), (dict(blocks=0), INVALID)], ids=str)
def test_chunk_fp8(change, status):
    _refused("pkv_paged_chunk_fp8", CHUNK8, change, status)


def test_an_empty_call_is_no_error():
    import pagedkv

    L = pagedkv.lib()
    assert L.pkv_paged_chunk(*{**CHUNK, "batch": 0}.values()) == 0
    assert L.pkv_paged_chunk(*{**CHUNK, "tokens": 0}.values()) == 0
    assert L.pkv_copy_blocks(*{**COPY, "n": 0, "src": None, "dst": None}.values()) == 0
    assert L.pkv_move_blocks(*{**MOVE, "n": 0}.values()) == 0


PAGES = [(dict(n=-1), INVALID), (dict(planes=-1), INVALID), (dict(pool=None), INVALID),
         (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(blocks=0), INVALID),
         (dict(block=0), INVALID), (dict(block=8), ALIGN), (dict(stride=8192 * 8 + 8), ALIGN),
         (dict(pool=24), ALIGN), (dict(stride=8192 * 7), INVALID)]


@pytest.mark.parametrize("change,status", PAGES, ids=str)
def test_copy_blocks(change, status):
    _refused("pkv_copy_blocks", COPY, change, status)


@pytest.mark.parametrize("change,status", PAGES + [
    (dict(tables=None), INVALID), (dict(rows=-1), INVALID), (dict(pitch=3), INVALID)], ids=str)
def test_move_blocks(change, status):
    _refused("pkv_move_blocks", MOVE, change, status)


def test_workspace_size_needs_no_gpu():
    import pagedkv

    size = pagedkv.lib().pkv_chunk_workspace_size
    assert size(1, 4, 12, 2, 64) == 0  # one launch that joins its parts itself
    assert size(0, 0, 12, 2, 64) == 0
    assert 0 < size(4, 4096, 12, 2, 4096) < 1 << 30
    for bad in ((-1, 4, 12, 2, 64), (1, -4, 12, 2, 64), (1, 4, 5, 2, 64), (1, 4, 12, 0, 64)):
        assert size(*bad) == 0


def test_python_wrappers_refuse_host_tensors():
    import pagedkv

    q = torch.zeros(4, 12, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(64, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        pagedkv.paged_chunk(q, kv, kv, i.view(1, 2), None, i, i[:1], 4, q, True, 0.1, 2)
    with pytest.raises(ValueError, match="CUDA"):
        pagedkv.copy_blocks(kv, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        pagedkv.move_blocks(kv, i, i, i.view(1, 2))
