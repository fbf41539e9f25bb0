"""The packed-chunk kernel's synchronisation protocol and work split
(csrc/chunk.cu), modelled on the CPU.

Protocol: the roles (copies, the warp that hands out the items, three that
write Q tiles, one issuing Q.K's and one P.V's, two slots of four softmax
warps, FP8: four widening warps that also write Q) run as generators under random scheduling; copies
land in any order, the tensor instructions and commits of one issuer run in
order but those of the two in any, mbarriers have the hardware's phase parity.  Every read is checked for the tile it was meant for.

Work split: the cut of the summed item costs into one range per CTA, restated
in Python: every key tile of every item is worked exactly once, the parts of a
cut item are the consecutive CTAs that the first one names, and no partial
slot is used twice."""
import random

import pytest

from test_prefill_protocol import Barrier, Race

RING = 3


def run_kernel(items, seed, fp8, shared_ring=False, merge_wait=True, idle_wait=True):
    """items: [(two, nt)].  Raises Race on a wrong read, a lost update or a hang."""
    rng = random.Random(seed)
    k_stages, v_stages = (2, 2) if fp8 else (3, 2)
    raws = 3  # groups of two chunks
    B = {"q_full": Barrier(4 if fp8 else 3), "q_free": Barrier(1), "ml": Barrier(8), "ep": Barrier(8)}
    for i in range(RING):
        B[f"item_full{i}"], B[f"item_empty{i}"] = Barrier(1), Barrier(15)
    for i in range(k_stages + v_stages):
        B[f"kv_full{i}"], B[f"kv_empty{i}"] = Barrier(4 if fp8 else 1), Barrier(1)

    def ring(which, t):
        """(stage, use) of K (0) or V (1) tile t: a ring each; shared_ring: one ring that alternates."""
        if shared_ring:
            return (2 * t + which) % (k_stages + v_stages), (2 * t + which) // (k_stages + v_stages)
        return (k_stages + t % v_stages, t // v_stages) if which else (t % k_stages, t // k_stages)

    B["s_free"] = Barrier(4)
    for s in range(2):
        B[f"s_full{s}"], B[f"p_full{s}"], B[f"pv_done{s}"] = Barrier(1), Barrier(4), Barrier(1)
    for i in range(raws):
        B[f"raw_full{i}"], B[f"raw_empty{i}"] = Barrier(1), Barrier(4)
    item_ring = [None] * RING
    Q = [None] * (4 if fp8 else 3)
    kv = [[None] * 4 for _ in range(k_stages + v_stages)]  # per widening warp; the copy engine writes all four
    raw = [None] * raws
    S = [None] * 4
    P = [[None] * 4 for _ in range(2)]
    O = [set(), set()]
    ml = [[None] * 4 for _ in range(2)]
    tma, qk_pipe, pv_pipe, finished = [], [], [], []
    STOP = (None, -1)

    def wait(name, phase):
        return lambda: B[name].test(phase & 1)

    def need(ok, what):
        if not ok:
            raise Race(what)

    def nxt(n):
        yield wait(f"item_full{n % RING}", n // RING)
        it = item_ring[n % RING]
        need(it[0] == n, "item overwritten")
        B[f"item_empty{n % RING}"].arrive()
        return it[1]

    def q_write(n, which, n_load):
        if n_load:
            yield wait("q_free", n_load - 1)
        for w in which:
            Q[w] = n
        yield None
        B["q_full"].arrive()

    def items_role():
        for n, it in enumerate(list(items) + [STOP]):
            if n >= RING:
                yield wait(f"item_empty{n % RING}", n // RING - 1)
            item_ring[n % RING] = (n, it)
            B[f"item_full{n % RING}"].arrive()
            yield None

    def q_role(w):
        n = n_load = 0
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            if it[1]:
                yield from q_write(n, [w], n_load)
                n_load += 1
            n += 1

    def copy_role(which):
        n = t = 0
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            for j in range(it[1]):
                if fp8:
                    for g in range(4):
                        st = t % raws
                        if t >= raws:
                            yield wait(f"raw_empty{st}", t // raws - 1)
                        B[f"raw_full{st}"].expect_tx(1)
                        tma.append((raw, st, (n, j, g), f"raw_full{st}"))
                        t += 1
                        yield None
                else:
                    st, use = ring(which, t)
                    if use:
                        yield wait(f"kv_empty{st}", use - 1)
                    B[f"kv_full{st}"].expect_tx(1)
                    tma.append((kv, st, [("KV"[which], n, j)] * 4, f"kv_full{st}"))
                    t += 1
                    yield None
            n += 1

    def widen_role(w):
        n = r = n_load = 0
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            if it[1]:
                yield from q_write(n, [w], n_load)
                n_load += 1
            for j in range(it[1]):
                places = [ring(i, r // 4) for i in range(2)]
                for st, use in places:
                    if use:
                        yield wait(f"kv_empty{st}", use - 1)
                for g in range(4):
                    rs = r % raws
                    yield wait(f"raw_full{rs}", r // raws)
                    need(raw[rs] == (n, j, g), "raw chunks")
                    if rng.random() < 0.2:
                        yield None
                    need(raw[rs] == (n, j, g), "raw chunks while read")
                    for what, (st, _) in zip("KV", places):  # a tile is whole with its last group
                        kv[st][w] = (what, n, j) if g == 3 else (what, n, j, g)
                    B[f"raw_empty{rs}"].arrive()
                    r += 1
                yield None
                for st, _ in places:
                    B[f"kv_full{st}"].arrive()
            n += 1

    def qk_role():
        n = k = n_q = n_s = 0
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            two, nt = it
            if nt:
                yield wait("q_full", n_q)
                n_q += 1
            for j in range(nt):
                st, use = ring(0, k)
                k += 1
                yield wait(f"kv_full{st}", use)
                for slot in (0, 1) if two else (j & 1,):
                    if n_s:
                        yield wait("s_free", n_s - 1)
                    n_s += 1
                    qk_pipe.append(("QK", n, j, slot, st))
                    qk_pipe.append(("commit", f"s_full{slot}"))
                qk_pipe.append(("commit", f"kv_empty{st}"))
            if nt:
                qk_pipe.append(("commit", "q_free"))
            n += 1

    def pv_role():
        n = v = 0
        n_p = [0, 0]
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            two, nt = it
            for j in range(nt):
                st, use = ring(1, v)
                v += 1
                yield wait(f"kv_full{st}", use)
                for slot in (0, 1) if two else (j & 1,):
                    yield wait(f"p_full{slot}", n_p[slot])
                    n_p[slot] += 1
                    pv_pipe.append(("PV", n, j, slot, st, j < (1 if two else 2)))
                    pv_pipe.append(("commit", f"pv_done{slot}"))
                pv_pipe.append(("commit", f"kv_empty{st}"))
            n += 1

    def softmax(slot, q):
        n = n_tile = n_ml = 0
        while True:
            it = yield from nxt(n)
            if it[1] < 0:
                return
            two, nt = it
            if not nt:
                n += 1
                continue
            busy = rng.random() < 0.7  # a warp whose rows are past the item's does no work
            mine = list(range(nt)) if two else list(range(slot, nt, 2))
            for a, j in enumerate(mine):
                yield wait(f"s_full{slot}", n_tile)
                n_tile += 1
                need(S[q] == (n, j, slot), f"S {S[q]} for {(n, j, slot)}")
                yield None
                need(S[q] == (n, j, slot), "S while it is taken")
                B["s_free"].arrive()
                if rng.random() < 0.5:
                    yield None
                if a and (busy or idle_wait):
                    yield wait(f"pv_done{slot}", n_tile - 2)
                if busy:
                    if a:
                        need(O[slot] == {(n, i) for i in mine[:a]}, "O during a rescale")
                P[slot][q] = (n, j)
                B[f"p_full{slot}"].arrive()
            if mine:
                yield wait(f"pv_done{slot}", n_tile - 1)
            if two:
                need(O[slot] == {(n, j) for j in mine}, "O at the end")
            else:
                ml[slot][q] = n
                yield None
                B["ml"].arrive()
                yield wait("ml", n_ml)
                need(ml[0][q] == n and ml[1][q] == n, "exchanged sums")
                yield None
                for s in range(2):
                    if len(range(s, nt, 2)):
                        need(O[s] == {(n, j) for j in range(s, nt, 2)}, "O of both slots at the end")
                need(ml[0][q] == n and ml[1][q] == n, "exchanged sums, second read")
                B["ep"].arrive()
                if merge_wait:
                    yield wait("ep", n_ml)
                n_ml += 1
            finished.append((n, slot, q))
            n += 1

    def pipe_step(pipe):
        op = pipe.pop(0)
        if op[0] == "commit":
            B[op[1]].arrive()
        elif op[0] == "QK":
            _, n, j, slot, st = op
            need(set(Q) == {n}, "Q tile")
            need(all(v == ("K", n, j) for v in kv[st]), "K tile")
            S[:] = [(n, j, slot)] * 4
        else:
            _, n, j, slot, st, fresh = op
            need(P[slot] == [(n, j)] * 4, f"P {P[slot]}")
            need(all(v == ("V", n, j) for v in kv[st]), "V tile")
            if fresh:
                O[slot].clear()
            O[slot].add((n, j))

    actors = [items_role(), qk_role(), pv_role()]
    actors += [copy_role(None)] if fp8 else [copy_role(0), copy_role(1)] + [q_role(w) for w in range(3)]
    actors += [softmax(s, q) for s in range(2) for q in range(4)]
    if fp8:
        actors += [widen_role(w) for w in range(4)]
    live = {i: (a, None) for i, a in enumerate(actors)}
    weight = [rng.choice([1, 1, 3, 10]) for _ in range(len(actors) + 3)]
    while live or tma or qk_pipe or pv_pipe:
        ready = [i for i, (_, p) in live.items() if p is None or p()]
        ops = [(i, weight[i]) for i in ready]
        if tma:
            ops.append(("tma", weight[-1]))
        if qk_pipe:
            ops.append(("qk", weight[-2]))
        if pv_pipe:
            ops.append(("pv", weight[-3]))
        if not ops:
            raise Race("hang")
        pick = rng.choices([o for o, _ in ops], [w for _, w in ops])[0]
        if pick == "tma":
            mem, at, val, bar = tma.pop(rng.randrange(len(tma)))
            mem[at] = val
            B[bar].complete_tx(1)
        elif pick in ("qk", "pv"):
            pipe_step(qk_pipe if pick == "qk" else pv_pipe)
        else:
            a = live[pick][0]
            try:
                live[pick] = (a, next(a))
            except StopIteration:
                del live[pick]
    assert len(finished) == 8 * sum(nt > 0 for _, nt in items)


def some_items(rng, fp8):
    return [(rng.random() < 0.5, rng.choice([0, 1, 1, 2, 3, 4, 5, 9])) for _ in range(rng.randint(1, 6))]


@pytest.mark.parametrize("fp8", [False, True])
def test_protocol_under_random_timing(fp8):
    for seed in range(250 if fp8 else 500):
        run_kernel(some_items(random.Random(seed), fp8), seed, fp8)


def test_the_model_sees_a_missing_wait():
    """Without the wait after the slots' join, a slot's next P.V overwrites an O tile still being read."""
    with pytest.raises(Race):
        for seed in range(400):
            run_kernel([(False, 2)] * 4, seed, False, merge_wait=False)


def test_the_model_sees_an_arrival_too_early():
    """A warp without rows that does not wait for its slot's P.V can end the phase of the tile before."""
    with pytest.raises(Race):
        for seed in range(400):
            run_kernel([(True, 6)] * 2, seed, False, idle_wait=False)


def test_the_model_sees_a_ring_with_two_copiers():
    """One ring for K and V of an odd number of stages: each copier sees every second phase of a barrier only."""
    with pytest.raises(Race):
        for seed in range(300):
            run_kernel([(True, 9)] * 2, seed, False, shared_ring=True)


# ---------------------------------------------------------------- work split
ITEM, STEP, KEYS = 512, 512 + 2 * 128, 128


class Split:
    """struct Work and item_role of csrc/chunk.cu."""

    def __init__(self, new, kv, group, hkv, fp8, causal):
        # sequences of few rows per KV head are the short kernel's
        short = 32 if fp8 and sum(new) * group <= 32 * len(new) else 16
        self.new = [t if t * group > short else 0 for t in new]
        self.kv, self.hkv, self.causal = kv, hkv, causal
        self.tpt = 128 // group
        self.wfull = 2
        self.block = self.tpt * self.wfull

    def n(self, b):
        return -(-self.new[b] // self.block)

    def key_end(self, b, i):
        if not self.causal:
            return self.kv[b]
        return max(0, self.kv[b] - self.new[b] + min(self.new[b], (i + 1) * self.block))

    def weight(self, b, i):
        return self.wfull if min(self.new[b] - i * self.block, self.block) > self.tpt else 1

    def before(self, b, i):
        if not self.causal:
            keys = i * self.kv[b]
        else:
            a = self.kv[b] - self.new[b]
            z = -a // self.block if a < 0 else 0
            m = max(0, i - z)
            keys = m * a + self.block * (m * (m + 1) // 2 + m * z)
        return i * ITEM + keys * self.wfull

    def cost(self, b, i):
        return ITEM + self.weight(b, i) * self.key_end(b, i)

    def head(self, b):
        return self.before(b, self.n(b) - 1) + self.cost(b, self.n(b) - 1) if self.n(b) else 0

    def ranges(self, ctas):
        total = sum(self.head(b) * self.hkv for b in range(len(self.new)))
        step = max(-(-total // ctas), STEP)
        return step, [(c * step, min(total, (c + 1) * step)) for c in range(ctas)]

    def cta(self, c, step, lo, hi):
        base, out, desc = 0, [], None
        for b in range(len(self.new)):
            if base >= hi:
                break
            row_end = base + self.head(b) * self.hkv
            for h in range(self.hkv):
                for i in range(self.n(b)):
                    s = base + h * self.head(b) + self.before(b, i)
                    w, ke = self.weight(b, i), self.key_end(b, i)
                    end, kt = s + ITEM + w * ke, -(-ke // KEYS)
                    if s >= hi or end <= lo:
                        continue

                    def cut(at):
                        d = at - s - ITEM
                        return 0 if d <= 0 else min(kt, d // (w * KEYS))

                    t0 = 0 if lo <= s else cut(lo)
                    t1 = kt if hi >= end else cut(hi)
                    if (lo > s) if kt == 0 else t0 >= t1:
                        continue
                    slot = -1 if t0 == 0 and t1 == kt else (1 if t0 == 0 else 0)
                    if slot == 1:
                        assert desc is None
                        desc = ((b, h, i), (end - 1) // step - c + 1)
                    out.append(((b, h, i), t0, t1, kt, slot))
            base = row_end
        return out, desc


@pytest.mark.parametrize("seed", range(60))
def test_every_key_tile_is_worked_once(seed):
    rng = random.Random(seed)
    group, fp8, causal = rng.choice([1, 4, 6, 7, 8, 64]), rng.random() < 0.5, rng.random() < 0.7
    rows = rng.choice([1, 2, 5, 17])
    new = [rng.choice([0, 1, 3, 21, 22, 43, 200, rng.randint(1, 600)]) for _ in range(rows)]
    kv = [rng.choice([0, t, t + rng.randint(0, 3000), rng.randint(0, 400), t + 20000]) for t in new]
    sp = Split(new, kv, group, rng.choice([1, 2, 8]), fp8, causal)
    # the closed form of the summed costs is the sum
    for b in range(rows):
        at = 0
        for i in range(sp.n(b)):
            assert sp.before(b, i) == at
            at += sp.cost(b, i)
        assert sp.head(b) == at
    ctas = rng.choice([2, 11, 148])
    if not any(sp.new):
        return
    step, ranges = sp.ranges(ctas)
    work, slots, descs = {}, {}, {}
    for c, (lo, hi) in enumerate(ranges):
        items, desc = sp.cta(c, step, lo, hi)
        for key, t0, t1, kt, slot in items:
            work.setdefault(key, []).append((t0, t1, kt, c, slot))
            if slot >= 0:
                assert (c, slot) not in slots
                slots[c, slot] = key
        if desc:
            descs[desc[0]] = (c, desc[1])
    for b in range(rows):
        for h in range(sp.hkv):
            for i in range(sp.n(b)):
                parts = sorted(work[b, h, i])
                assert parts[0][0] == 0 and parts[-1][1] == parts[0][2]
                assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
                if len(parts) == 1:
                    assert parts[0][4] == -1 and (b, h, i) not in descs
                else:
                    first, count = descs[b, h, i]
                    assert [p[3] for p in parts] == list(range(first, first + count))
                    assert [p[4] for p in parts] == [1] + [0] * (count - 1)
