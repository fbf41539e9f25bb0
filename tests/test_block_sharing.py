"""Host half of block sharing, roll-back and compaction (kv_cache.BlockTables):
random operations against a pool simulated on the host, in which every sequence
must read back exactly the tokens it was given; refusals that change nothing;
chats that fork (chat.Chat.fork) through the scheduler."""
import queue
import random

import pytest
import torch

from kv_cache import BlockTables
from oracle.scheduler_trace import FakeModel, FakeTokenizer


class Simulated(BlockTables):
    """BlockTables over a host pool and host copies of the device tables."""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.pool = [[None] * self.block_size for _ in range(self.num_blocks)]
        self.device = {}
        self.launches = 0

    def flush(self):
        for r, c, b in self.take_pending():
            self.device[(r, c)] = b

    def _copy(self, src, dst):
        self.launches += 1
        assert len(set(dst)) == len(dst) and not set(dst) & set(src)
        for s, d in zip(src, dst):
            self.pool[d] = list(self.pool[s])

    def _move(self, src, dst):
        self.flush()
        assert src == sorted(set(src))
        self._copy(src, dst)
        to = dict(zip(src, dst))
        self.device = {cell: to.get(b, b) for cell, b in self.device.items()}
        for b in src:
            self.pool[b] = [None] * self.block_size

    def write(self, seq, tokens):
        """Append tokens as a step does: reserve, flush, store, advance."""
        start = self.length(seq)
        self.packed_rows([seq], [len(tokens)])
        self.flush()
        row = self.table_row(seq)
        for i, t in enumerate(tokens, start):
            b = self.device[(row, i // self.block_size)]
            assert b not in self._shared, "a shared block was written"
            self.pool[b][i % self.block_size] = t
        self.advance_packed([seq], [len(tokens)])

    def read(self, seq):
        self.flush()
        row, bs = self.table_row(seq), self.block_size
        return [self.pool[self.device[(row, i // bs)]][i % bs] for i in range(self.length(seq))]

    def check(self):
        held = {}
        for t in self._block_tables.values():
            assert len(set(t)) == len(t)
            for b in t:
                held[b] = held.get(b, 0) + 1
        assert {b: n for b, n in held.items() if n > 1} == self._shared
        assert sorted(list(held) + self._free_blocks) == list(range(self.num_blocks))
        for s, t in self._block_tables.items():
            assert not any(b in self._shared for b in t[self.length(s) // self.block_size:])


def _state(bt):
    return ({s: list(t) for s, t in bt._block_tables.items()}, dict(bt._lengths), dict(bt._shared),
            list(bt._free_blocks), list(bt._free_rows), dict(bt._pending))


@pytest.mark.parametrize("seed", range(12))
def test_sequences_keep_their_tokens_through_random_operations(seed):
    rng = random.Random(seed)
    bt = Simulated(rng.randint(6, 60), 16, max_seqs=rng.choice([4, 40]))
    want = {}
    fresh = iter(range(10 ** 9))
    refused = 0
    for _ in range(400):
        op = rng.choice(["alloc", "write", "write", "fork", "fork", "truncate", "trim", "free",
                         "reserve", "compact"])
        live = list(want)
        before = None
        try:
            if op == "alloc" or not live:
                before = _state(bt)
                want[bt.alloc()] = []
            elif op == "write":
                s = rng.choice(live)
                new = [next(fresh) for _ in range(rng.choice([1, 1, 5, 16, 33]))]
                before = _state(bt)
                bt.write(s, new)
                want[s] = want[s] + new
            elif op == "fork":
                seqs = [rng.choice(live) for _ in range(rng.randint(1, 3))]
                lens = rng.choice([None, [rng.randint(0, len(want[s])) for s in seqs]])
                before = _state(bt)
                launches = bt.launches
                new = bt.fork_many(seqs, lens)
                assert bt.launches <= launches + 1
                for f, s, n in zip(new, seqs, lens or [len(want[s]) for s in seqs]):
                    want[f] = want[s][:n]
            elif op == "truncate":
                s = rng.choice(live)
                n = rng.randint(0, len(want[s]))
                before = _state(bt)
                bt.truncate(s, n)
                want[s] = want[s][:n]
            elif op == "trim":
                bt.trim(rng.choice(live))
            elif op == "free":
                s = rng.choice(live)
                bt.free(s)
                del want[s]
            elif op == "reserve":
                s = rng.choice(live)
                before = _state(bt)
                bt.ensure_capacity(s, bt.length(s) + rng.randint(0, 40))
            else:
                n = bt.compact()
                assert n == bt.num_blocks - bt.free_block_count()
                assert {b for t in bt._block_tables.values() for b in t} == set(range(n))
        except RuntimeError as e:
            assert "exhausted" in str(e)
            assert _state(bt) == before, f"{op} changed something before it was refused"
            refused += 1
        bt.check()
        for s in want:
            assert bt.read(s) == want[s], (op, s)
    assert refused  # the pool was small enough to run dry
    for s in list(want):
        bt.free(s)
    assert sorted(bt._free_blocks) == list(range(bt.num_blocks)) and not bt._shared


def test_fork_shares_full_blocks_and_copies_the_last():
    bt = Simulated(16, 16)
    a = bt.alloc()
    bt.write(a, list(range(40)))
    bt.ensure_capacity(a, 100)  # reserved blocks are not handed on
    b = bt.fork(a)
    ta, tb = bt.host_table(a), bt.host_table(b)
    assert tb[:2] == ta[:2] and len(tb) == 3 and tb[2] not in ta and bt.launches == 1
    c = bt.fork(a, 32)  # ends with a block: nothing to copy
    assert bt.host_table(c) == ta[:2] and bt.launches == 1
    d = bt.fork(a, 0)
    assert bt.host_table(d) == [] and bt.length(d) == 0
    assert bt._shared == {ta[0]: 3, ta[1]: 3}
    free = bt.free_block_count()
    bt.free(a)  # its own third block and the four reserved ones
    assert bt.free_block_count() == free + 5 and bt._shared == {ta[0]: 2, ta[1]: 2}
    assert bt.read(b) == list(range(40)) and bt.read(c) == list(range(32))


def test_truncate_copies_a_block_it_would_write_into():
    bt = Simulated(5, 16)
    a = bt.alloc()
    bt.write(a, list(range(48)))
    b = bt.fork(a)
    bt.truncate(b, 20)
    assert bt.host_table(b)[0] == bt.host_table(a)[0]
    assert bt.host_table(b)[1] not in bt.host_table(a)
    bt.write(b, [99])
    assert bt.read(b) == list(range(20)) + [99] and bt.read(a) == list(range(48))
    bt.truncate(b, 16)  # its copy goes back
    assert bt.free_block_count() == 2
    c = bt.fork(a, 33)
    d = bt.fork(a, 32)
    assert bt.free_block_count() == 1
    bt.write(d, [7])  # takes the last block
    e = bt.fork(a)  # whole blocks only, none needed
    state = _state(bt)
    with pytest.raises(RuntimeError, match="exhausted"):
        bt.truncate(e, 40)
    assert _state(bt) == state
    bt.truncate(d, 24)  # its own released block serves as the copy
    assert bt.read(d) == list(range(24)) and bt.read(c) == list(range(33))


def test_refusals_change_nothing():
    bt = Simulated(4, 16, max_seqs=3)
    a = bt.alloc()
    bt.write(a, list(range(20)))
    state = _state(bt)
    for call in (lambda: bt.fork(a, 21), lambda: bt.fork(a, -1), lambda: bt.truncate(a, 21),
                 lambda: bt.truncate(a, -1), lambda: bt.fork_many([a, a], [1]),
                 lambda: bt.packed_rows([a, a], [1, 1]), lambda: bt.packed_rows([a], [1, 2]),
                 lambda: bt.packed_rows([a], [-1])):
        with pytest.raises(ValueError):
            call()
        assert _state(bt) == state
    for call in (lambda: bt.fork_many([a, a, a]),           # blocks
                 lambda: bt.fork_many([a, a, a], [16] * 3),  # rows
                 lambda: bt.packed_rows([a], [45])):
        with pytest.raises(RuntimeError, match="exhausted"):
            call()
        assert _state(bt) == state
    with pytest.raises(KeyError):
        bt.fork(77)
    assert _state(bt) == state


def test_a_packed_step_is_refused_as_a_whole():
    """Two rows that fit alone but not together: neither is given blocks."""
    bt = BlockTables(4, 16)
    a, b = bt.alloc(), bt.alloc()
    state = _state(bt)
    with pytest.raises(RuntimeError, match="exhausted"):
        bt.packed_rows([a, b], [40, 20])
    assert _state(bt) == state
    wide = BlockTables(8, 16, max_blocks_per_seq=2)  # the second row outgrows its table row
    c, d = wide.alloc(), wide.alloc()
    before = _state(wide)
    with pytest.raises(RuntimeError, match="device table"):
        wide.packed_rows([c, d], [16, 33])
    assert _state(wide) == before
    assert bt.packed_rows([a, b], [40, 16]) == ([0, 0], [bt.table_row(a), bt.table_row(b)])


def test_compact_hands_out_the_lowest_blocks_next():
    bt = Simulated(12, 16)
    seqs = [bt.alloc() for _ in range(4)]
    for i, s in enumerate(seqs):
        bt.write(s, [100 * i + j for j in range(40)])
    bt.free(seqs[1])
    bt.free(seqs[3])
    assert bt.compact() == 6
    assert bt.read(seqs[0]) == [j for j in range(40)]
    assert bt.read(seqs[2]) == [200 + j for j in range(40)]
    bt.write(seqs[0], list(range(9)))
    assert max(bt.host_table(seqs[0])) == 6
    launches = bt.launches
    assert bt.compact() == 7 and bt.launches == launches  # in place already


# ---------------------------------------------------------------- chats
@pytest.fixture
def engine(monkeypatch):
    import chat

    for name, value in (("DEVICE", torch.device("cpu")), ("MAX_REPLY_TOKENS", 12),
                        ("_job_queue", queue.Queue())):
        monkeypatch.setattr(chat, name, value)
    for state in (chat.active, chat._deferred, chat._resident, chat._mixed):
        state.clear()

    def install(blocks):
        chat.init(kv_cache=BlockTables(blocks, 16), start_worker=False)
        return chat._kv()

    yield chat, install
    chat._kv_cache = None
    chat._resident.clear()


def _talk(chat_mod, c, model, text):
    c.submit(model, text)
    chat_mod.run_until_idle()


def test_a_forked_chat_prefills_only_its_own_message(engine):
    chat_mod, install = engine
    cache = install(64)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    _talk(chat_mod, a, model, "x" * 50)
    resident = cache.length(a.seq)
    b = a.fork()
    assert b.seq is None and b.ids == a.ids and b.messages == a.messages
    c = b.fork()  # of a fork that has not spoken yet
    history = list(a.ids)
    model.log.clear()
    _talk(chat_mod, b, model, "another way")
    first = model.log[0]
    assert first["ids"][0] == b.ids[resident:resident + first["T"]] and b.seq != a.seq
    assert cache.length(b.seq) > resident and cache.length(a.seq) == resident
    assert cache.host_table(b.seq)[:resident // 16] == cache.host_table(a.seq)[:resident // 16]
    assert a.ids == history and b.ids[:len(history)] == history and b.parent is None
    _talk(chat_mod, a, model, "on we go")  # the two go on separately
    _talk(chat_mod, c, model, "a third way")
    assert a.ids[:len(history)] == b.ids[:len(history)] == c.ids[:len(history)]
    assert len({tuple(x.ids) for x in (a, b, c)}) == 3
    for x in (a, b, c):
        x.release()
    assert cache.free_block_count() == 64 and not cache._shared


def test_a_fork_of_an_evicted_chat_prefills_the_history(engine):
    chat_mod, install = engine
    cache = install(64)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    _talk(chat_mod, a, model, "hello there")
    b = a.fork()
    a.release()
    model.log.clear()
    _talk(chat_mod, b, model, "again")
    message = b.tokenizer.encode("User: again\nAssistant:")
    assert model.log[0]["ids"][0] == a.ids + message
    assert cache.length(b.seq) >= len(a.ids) and not cache._shared


def test_forked_chats_in_a_full_pool(engine):
    """Forks that compete for a small pool are deferred and evicted like any
    chat; blocks are conserved and every chat ends with its own history."""
    chat_mod, install = engine
    cache = install(12)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    _talk(chat_mod, a, model, "h" * 40)
    forks = [a.fork() for _ in range(4)]
    for i, f in enumerate(forks):
        f.submit(model, f"variant {i} " + "y" * 30)
    for _ in range(400):
        if not chat_mod._tick(block=False) and not chat_mod.active and not chat_mod._deferred:
            break
        held = {b for t in cache._block_tables.values() for b in t}
        assert len(held) + cache.free_block_count() == 12
    for i, f in enumerate(forks):
        assert f.messages[-2] == ("user", f"variant {i} " + "y" * 30)
        assert f.ids[:len(a.ids)] == a.ids
    for x in [a, *forks]:
        x.release()
    assert cache.free_block_count() == 12 and not cache._shared


def test_a_chat_with_a_message_in_flight_does_not_fork(engine):
    chat_mod, install = engine
    install(64)
    a = chat_mod.Chat(FakeTokenizer())
    a.submit(FakeModel([]), "hello")
    with pytest.raises(RuntimeError, match="in flight"):
        a.fork()
    chat_mod._tick(block=False)
    with pytest.raises(RuntimeError, match="in flight"):
        a.fork()
    chat_mod.run_until_idle()
    a.fork()


def test_a_message_is_taken_over_in_one_piece(engine):
    """A fork on another thread waits while the worker turns a queued message
    into history, or sees it still queued; it never copies half of it."""
    chat_mod, install = engine
    install(64)
    a = chat_mod.Chat(FakeTokenizer())
    seen = []

    class Ids(list):
        def extend(self, new):
            seen.append(chat_mod._cache_lock.locked())
            super().extend(new)

    a.ids = Ids()
    a.submit(FakeModel([]), "hello")
    chat_mod._tick(block=False)
    assert seen[0]
    chat_mod.run_until_idle()
    a.fork()
