"""Packed-chunk attention over the FP8 pool for keys and values of any size,
against 64 bits of what the pool holds (e4m3 * scale).

Tolerance, elementwise, with u = 2^-11, half an f16 step:
  * a key is f16(e4m3 * scale), its scale held in two f16 terms: off by at most
    u of itself, plus, where f16's least steps count, 2^-30 of the largest key:
    keys and values are held in a unit that follows the largest scale, which
    comes to 64 at least and the largest key to 448 times that; half the least
    step of a scale, times 448, and of a product, twice, are 450 * 2^-25;
  * q is f16(q / 16): exact from 2^-13 up, below that off by at most 2^-21;
  * so a score is off by at most D = u S + 2^-30 max|k| scale sum|q| + 2^-21
    scale sum|k_d| (the d with |q_d| < 2^-13) + 130 * 2^-24 S (fp32 sums), with
    S = scale sum |q_d k_d|, and a probability by a factor of exp(2 D) at most;
  * a value is off by u for its scale and u for the product, 2 u in all, plus
    2^-30 of the largest value, and a probability by u for its f16; the short
    kernel rounds the probability times the value's scale, the same u;
  * a probability below f16's normal range is off by at most 2^-32 of the
    largest (long sequences); the short kernel's product by 2^-30 of the largest
    probability times the largest value: n 2^-30 max|v| over n keys;
  * 2^-16 for ex2, fp32 sums and rescales, as in test_chunk_gpu;
  * the result's own rounding, 2^-8 of itself.
max|k| and max|v| are taken over all positions of the sequence: hidden ones and
those of no weight set the unit too."""
import math

import pytest
import torch

from test_chunk_gpu import SCALE, call, make

pytestmark = pytest.mark.gpu


def plain8(c, causal=True):
    q = c["q"].double()
    o = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    tol = o.clone()
    group = c["hq"] // c["hkv"]
    u = 2.0 ** -11
    at = 0
    for b, (t, n) in enumerate(zip(c["new"], c["kv"])):
        k, v = (x.repeat_interleave(group, 1) for x in c["read"][b])  # [n, hq, 128]
        for a in range(0, t if n else 0, 256):
            z = min(t, a + 256)
            qq = q[at + a:at + z]
            s = torch.einsum("thd,shd->hts", qq, k) * SCALE
            S = torch.einsum("thd,shd->hts", qq.abs(), k.abs()) * SCALE
            small = torch.einsum("thd,shd->hts", (qq.abs() < 2.0 ** -13).double(), k.abs()) * SCALE
            D = (u + 130 * 2.0 ** -24) * S + 2.0 ** -21 * small + \
                2.0 ** -30 * SCALE * (k.abs().amax((0, 2))[None] * qq.abs().sum(-1)).T[..., None]
            if causal:
                hide = torch.arange(n, device=q.device)[None] > n - t + torch.arange(a, z, device=q.device)[:, None]
                s, D = s.masked_fill(hide, -math.inf), D.masked_fill(hide, 0.0)
            p = torch.softmax(s, -1)
            oo = torch.einsum("hts,shd->thd", p, v)
            A = torch.einsum("hts,shd->thd", p, v.abs())
            D = D.amax(-1).T[..., None]
            vmax = v.abs().amax((0, 2))[None, :, None]
            off = (torch.expm1(2 * D) + 3 * u + 2.0 ** -16) * A + (2.0 ** -30 + n * 2.0 ** -30) * vmax
            o[at + a:at + z] = oo
            tol[at + a:at + z] = 2.0 ** -8 * oo.abs() + (1 + 2.0 ** -8) * off
        at += t
    return o, tol


def check8(c, causal=True):
    out, err = call(c, causal)
    assert err == 0, f"device error bits {err:#x}"
    want, tol = plain8(c, causal)
    n = sum(c["new"])
    assert torch.equal(out[:n].isnan(), want[:n].isnan()), "NaN in other places than the formula's"
    ok = ~want[:n].isnan()
    diff = (out[:n].double() - want[:n]).abs()[ok]
    over = (diff - tol[:n][ok]).max().item()
    assert over <= 0, f"off by {diff.max().item()}, {over} over the tolerance"
    return out


# tokens that take the tensor cores' kernel, the short one, and both
NEW = pytest.mark.parametrize("new", [[40], [300], [5], [1], [2, 40], [4] * 6 + [90]], ids=str)


@NEW
@pytest.mark.parametrize("causal", [True, False])
def test_ordinary_values(cuda, new, causal):
    check8(make(cuda, new, [700 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=1), causal)


@NEW
@pytest.mark.parametrize("size", [2.0 ** -20, 3e3, 3e5, 1e20, 1e34])
def test_values_of_any_size(cuda, new, size):
    def edit(kk, vv):
        vv *= size

    check8(make(cuda, new, [700 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=2, edit=edit))


@NEW
def test_large_values_that_the_first_tokens_do_not_see(cuda, new):
    """The newest position holds a value far above the others, which only the
    newest token sees."""
    def edit(kk, vv):
        vv[-1] *= 3e4

    check8(make(cuda, new, [300 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=3, edit=edit))


@NEW
@pytest.mark.parametrize("at", [0, 150, -1])
def test_a_large_value_of_no_weight(cuda, new, at):
    def edit(kk, vv):
        kk[...] = kk * 0.2 + 1.0
        kk[at] = -30.0
        vv[at] *= 1e4

    c = make(cuda, new, [300 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=4, edit=edit)
    c["q"].copy_(c["q"] * 0.2 + 0.5)
    check8(c)


@NEW
def test_a_channel_of_large_keys(cuda, new):
    """Keys past f16's largest number in a dimension that q leaves out."""
    def edit(kk, vv):
        kk *= 1000.0
        kk[..., 7] = 1e5

    c = make(cuda, new, [700 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=5, edit=edit)
    c["q"] *= 2.0 ** -10
    c["q"][..., 7] = 0
    check8(c)


@NEW
def test_small_keys_and_large_queries(cuda, new):
    def edit(kk, vv):
        kk *= 2.0 ** -13

    c = make(cuda, new, [700 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=6, edit=edit)
    c["q"] *= 2.0 ** 13
    check8(c)


@NEW
@pytest.mark.parametrize("step", [1.5, 1 / 1.5])
def test_scales_that_grow_or_fall_along_the_cache(cuda, new, step):
    """Keys and values of every size from 2^-17 to 2^17, in either order: the
    unit moves inside tiles and between them."""
    def edit(kk, vv):
        n = kk.shape[0]
        f = torch.exp2(torch.linspace(-17, 17, n, device=kk.device) * (1 if step > 1 else -1))[:, None, None]
        vv *= f
        kk /= torch.clamp(f, 2.0 ** -4, 2.0 ** 4)

    check8(make(cuda, new, [900 + 13 * i for i in range(len(new))], 12, 2, "fp8", seed=7, edit=edit))


def test_a_head_layout_of_one_tile_and_of_many_items(cuda):
    """Slots that share an item's keys join what they hold in different units."""
    def edit(kk, vv):
        n = kk.shape[0]
        vv *= torch.exp2(torch.linspace(0, 30, n, device=kk.device))[:, None, None]

    for new, hq, hkv in (([20], 12, 2), ([3], 64, 1), ([21, 400], 8, 8), ([130, 33], 32, 8)):
        check8(make(cuda, new, [1500] * len(new), hq, hkv, "fp8", seed=8, edit=edit))
