"""A packed step's `tokens` (one row per token) where any step goes: written,
read and attended over."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FMT = pytest.mark.parametrize("fmt", ["bf16", "fp8_e4m3"])


def _cache(cuda, fmt):
    from kv_cache import KVCache

    return KVCache(40, 16, cuda, torch.bfloat16, num_layers=1, kv_format=fmt)


def _kv(cuda, n, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(2, n, 2, 1, 128, generator=g, device=cuda).to(torch.bfloat16)


@FMT
def test_a_step_of_idle_rows_is_written_and_attended(cuda, fmt):
    from kernels.fa2 import packed_attention

    c = _cache(cuda, fmt)
    seqs = [c.alloc(), c.alloc()]
    before = (c.pool8 if c.fp8 else c.buf).clone()
    _, step = c.prepare_packed(seqs, [0, 0])
    k, v = _kv(cuda, 0, 0)
    c.write(0, step.tokens, k, v)
    q = torch.empty(0, 12, 128, dtype=torch.bfloat16, device=cuda)
    c.append(0, step.tokens, q[:, :, None], k, v, before.new_zeros(1, 128).to(torch.bfloat16),
             before.new_zeros(1, 128).to(torch.bfloat16), q[:, :, None])
    assert packed_attention(q, *c.read(0, step)).shape == (0, 12, 128)
    assert torch.equal(c.pool8 if c.fp8 else c.buf, before)


@FMT
def test_tokens_are_rows_of_one_token(cuda, fmt):
    """`tokens` reads as N rows, and decode attention over them (row i up to
    token i's position) is the packed attention: both are within half a bf16
    step and 2^-8 of the weighted values (the tolerance of test_chunk_gpu) of
    the same formula; over the FP8 pool the packed one takes keys to 2^-11 and
    values to 2^-10: with scale sum |q_d k_d| below 12, 2 * 12 * 2^-11 + 3 * 2^-11
    < 2^-6 of the weighted values more."""
    from kernels.fa2 import flash_attention, packed_attention

    c = _cache(cuda, fmt)
    seqs = [c.alloc(), c.alloc()]
    _, step = c.prepare_packed(seqs, [37, 5])
    k, v = _kv(cuda, 42, 1)
    c.write(0, step.tokens, k, v)
    assert step.tokens.batch == 42 and c.read(0, step.tokens)[0].shape == (42, 2, 37, 128)
    q = torch.randn(42, 12, 128, device=cuda).to(torch.bfloat16)
    got = packed_attention(q, *c.read(0, step)).float()
    rows = flash_attention(q[:, :, None], *c.read(0, step.tokens))[:, :, 0].float()
    largest = v.float().abs().max()
    assert (got - rows).abs().max() <= (2 * 2.0 ** -7 + (2.0 ** -6 if c.fp8 else 0)) * largest
    dense = c.read(0, step.tokens)[1].materialize()
    assert dense.shape == (42, 2, 37, 128)
    if not c.fp8:
        assert torch.equal(dense[41, :, :5], v[37:, :, 0].transpose(0, 1))
    c.check_errors()
