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
