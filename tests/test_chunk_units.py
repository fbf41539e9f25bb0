"""The units that csrc/chunk.cu holds FP8 keys and values in, modelled on the CPU.

Hand-over: the widening warps publish a tile's units in a ring whose entries no
barrier of their own protects; run under random timing with the barriers that
do (the K buffers' and S's), every softmax warp must read the units of its tile.
The waits for values and probabilities, which only hold the roles back further,
are left out.

Arithmetic: widening in f16 with a unit that follows the largest scale, against
e4m3 * scale in 64 bits."""
import random

import numpy as np
import pytest

from test_prefill_protocol import Barrier, Race


def run_units(items, seed, ring, k_stages=2):
    """items: [(two, key tiles)].  Raises Race when a warp reads another tile's units."""
    rng = random.Random(seed)
    k_full, k_empty = [Barrier(4) for _ in range(k_stages)], [Barrier(1) for _ in range(k_stages)]
    s_full, s_free = [Barrier(1), Barrier(1)], Barrier(4)
    units, pipe = [None] * ring, []
    tiles = [(two, j, n) for n, (two, nt) in enumerate(items) for j in range(nt)]

    def wait(bar, phase):
        return lambda: bar.test(phase & 1)

    def widen(w):
        for t in range(len(tiles)):
            if t >= k_stages:
                yield wait(k_empty[t % k_stages], t // k_stages - 1)
            yield None
            if w == 0:
                units[t % ring] = t
                yield None
            k_full[t % k_stages].arrive()

    def qk():
        n_s = 0
        for t, (two, j, _) in enumerate(tiles):
            yield wait(k_full[t % k_stages], t // k_stages)
            for slot in (0, 1) if two else (j & 1,):
                if n_s:
                    yield wait(s_free, n_s - 1)
                n_s += 1
                pipe.append(s_full[slot])
                yield None
            pipe.append(k_empty[t % k_stages])

    def softmax(slot):
        n_tile = 0
        for t, (two, j, _) in enumerate(tiles):
            if not two and (j & 1) != slot:
                continue
            yield wait(s_full[slot], n_tile)
            n_tile += 1
            yield None
            if units[t % ring] != t:
                raise Race(f"units of tile {units[t % ring]} read for {t}")
            s_free.arrive()

    actors = [widen(w) for w in range(4)] + [qk()] + [softmax(s) for s in range(2) for _ in range(4)]
    live = {i: (a, None) for i, a in enumerate(actors)}
    weight = [rng.choice([1, 1, 3, 10]) for _ in range(len(actors) + 1)]
    while live or pipe:
        ops = [(i, weight[i]) for i, (_, p) in live.items() if p is None or p()]
        if pipe:
            ops.append((-1, weight[-1]))
        if not ops:
            raise Race("hang")
        pick = rng.choices([o for o, _ in ops], [w for _, w in ops])[0]
        if pick < 0:
            pipe.pop(0).arrive()
            continue
        try:
            live[pick] = (live[pick][0], next(live[pick][0]))
        except StopIteration:
            del live[pick]


def some_items(seed):
    rng = random.Random(seed)
    return [(rng.random() < 0.5, rng.choice([0, 1, 1, 2, 3, 4, 5, 9])) for _ in range(rng.randint(1, 6))]


@pytest.mark.parametrize("ring", [3, 4])
def test_every_warp_reads_the_units_of_its_tile(ring):
    for seed in range(300):
        run_units(some_items(seed), seed, ring)


def test_the_model_sees_a_ring_that_is_too_short():
    with pytest.raises(Race):
        for seed in range(300):
            run_units([(True, 9)] * 2, seed, 2)


class Unit:
    """struct Unit of csrc/chunk.cu."""

    LEAST = 27

    def __init__(self):
        self.exp = self.LEAST

    @staticmethod
    def power(biased):
        return 2.0 ** (biased - 127)

    @property
    def up(self):
        return np.float32(self.power(261 - self.exp))

    @property
    def value(self):
        return self.power(self.exp - 7)

    def holds(self, top):
        return int(np.float32(top).view(np.uint32)) < self.exp << 23

    def fit(self, top):
        """What the tile holds so far is multiplied by this."""
        if self.holds(top):
            return np.float16(1)
        to = min(max((int(np.float32(top).view(np.uint32)) >> 23) + 1, self.exp), 250)
        by, self.exp = to - self.exp, to
        return np.float16(self.power(127 - by) if by < 100 else 0.0)


def fma16(a, b, c):
    """f16 a * b + c with one rounding (exact in 64 bits)."""
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(np.float16)


def widen(e, scale, keys):
    """[n, d] e4m3 values and [n] scales, 32 rows (a group) at a time -> 64-bit values held."""
    unit, out = Unit(), np.zeros(e.shape, np.float16)
    for g in range(0, len(e), 32):
        s = scale[g:g + 32].astype(np.float32)
        out[:g] *= unit.fit(s.max())
        x = e[g:g + 32].astype(np.float16)
        s = s * unit.up
        top = s.astype(np.float16)[:, None]
        if keys:
            rest = (s - s.astype(np.float16).astype(np.float32)).astype(np.float16)[:, None]
            out[g:g + 32] = fma16(x, top, x * rest)
        else:
            out[g:g + 32] = x * top
    assert np.isfinite(out).all()
    return out.astype(np.float64) * unit.value


@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("lo,hi", [(-3, 3), (-9, 17), (40, 110), (-90, -60), (-30, 30)])
@pytest.mark.parametrize("order", ["random", "rising", "falling"])
def test_what_a_tile_holds_is_within_the_stated_bounds(keys, lo, hi, order):
    rng = np.random.default_rng(abs(lo) + 7 * abs(hi))
    codes = np.array([m / 8 * 2.0 ** -6 for m in range(8)] +
                     [(1 + m / 8) * 2.0 ** (x - 7) for x in range(1, 16) for m in range(8)][:-1])
    e = rng.choice(codes, (128, 64)) * rng.choice([-1, 1], (128, 64))
    e[:, 0] = 448
    scale = (2.0 ** rng.uniform(lo, hi, 128)).astype(np.float32)
    if order != "random":
        scale = np.sort(scale)[::1 if order == "rising" else -1]
    want = e * scale.astype(np.float64)[:, None]
    off = np.abs(widen(e, scale, keys) - want)
    rel = (2.0 ** -11 if keys else 2.0 ** -10) * (1 + 2.0 ** -9)
    assert (off <= rel * np.abs(want) + 2.0 ** -30 * 448 * scale.max()).all()


def test_one_rounding_to_f16_is_off_by_up_to_half_its_step():
    """2^-11 for a key and close to 2^-10 for a value, whose scale is rounded too."""
    rng = np.random.default_rng(0)
    e = rng.choice([(1 + m / 8) * 2.0 ** x for x in range(-6, 9) for m in range(7)], (4096, 64))
    scale = (2.0 ** rng.uniform(-1, 0, 4096)).astype(np.float32)
    want = e * scale.astype(np.float64)[:, None]
    worst = [np.abs(widen(e, scale, keys) / want - 1).max() for keys in (True, False)]
    assert 2.0 ** -11.2 < worst[0] <= 2.0 ** -11 * (1 + 2.0 ** -9)
    assert 2.0 ** -10.3 < worst[1] <= 2.0 ** -10
