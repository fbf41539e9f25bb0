"""Chats on a cache with fewer table rows than chats: rows, like blocks, are
made by evicting idle chats, and a message waits when there are none, so that
admission cannot raise on the scheduler's thread (nothing would answer after
that)."""
import queue

import pytest
import torch

from kv_cache import BlockTables
from oracle.scheduler_trace import FakeModel, FakeTokenizer


@pytest.fixture
def engine(monkeypatch):
    import chat

    for name, value in (("DEVICE", torch.device("cpu")), ("MAX_REPLY_TOKENS", 12),
                        ("_job_queue", queue.Queue())):
        monkeypatch.setattr(chat, name, value)
    for state in (chat.active, chat._deferred, chat._resident, chat._mixed):
        state.clear()

    def install(*a, **kw):
        chat.init(kv_cache=BlockTables(*a, **kw), start_worker=False)
        return chat._kv()

    yield chat, install
    chat._kv_cache = None
    for state in (chat.active, chat._deferred, chat._resident, chat._mixed):
        state.clear()


def _drain(chat_mod, ticks=600):
    for _ in range(ticks):
        if not chat_mod._tick(block=False) and not chat_mod.active and not chat_mod._deferred:
            return
    raise AssertionError("messages left over")


def _talk(chat_mod, c, model, text):
    c.submit(model, text)
    _drain(chat_mod)


def _conserved(cache):
    held = {b for t in cache._block_tables.values() for b in t}
    assert len(held) + cache.free_block_count() == cache.num_blocks
    assert len(cache._block_tables) + cache.free_row_count() == cache.max_seqs


@pytest.mark.parametrize("rows", [1, 2, 3, 5])
def test_more_queued_forks_than_rows(engine, rows):
    chat_mod, install = engine
    cache = install(64, 16, max_seqs=rows)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    _talk(chat_mod, a, model, "h" * 40)
    forks = [a.fork() for _ in range(6)]
    for i, f in enumerate(forks):
        f.submit(model, f"variant {i}")
    for _ in range(600):
        more = chat_mod._tick(block=False)
        _conserved(cache)
        if not more and not chat_mod.active and not chat_mod._deferred:
            break
    for i, f in enumerate(forks):
        assert f.messages[-2] == ("user", f"variant {i}") and f.parent is None
        assert f.ids[:len(a.ids)] == a.ids
    _talk(chat_mod, a, model, "still there")
    for x in [a, *forks]:
        x.release()
    assert cache.free_block_count() == 64 and cache.free_row_count() == rows and not cache._shared


def test_deferred_forks_use_up_the_rows_but_not_the_blocks(engine):
    """Forks of a history of whole blocks hold a row and no block of their own
    while they wait for room."""
    chat_mod, install = engine
    cache = install(12, 16, max_seqs=4)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    _talk(chat_mod, a, model, "h" * 40)
    forks = [a.fork() for _ in range(8)]
    for f in forks:
        f.submit(model, "y" * 60)
    _drain(chat_mod)
    for f in forks:
        assert f.messages[-2] == ("user", "y" * 60) and f.messages[-1][0] == "assistant"
    _conserved(cache)


def test_a_fork_still_shares_when_an_idle_chat_gives_its_row(engine):
    chat_mod, install = engine
    cache = install(64, 16, max_seqs=2)
    model = FakeModel([])
    a, other = (chat_mod.Chat(FakeTokenizer()) for _ in range(2))
    _talk(chat_mod, other, model, "someone else")
    _talk(chat_mod, a, model, "h" * 50)
    resident = cache.length(a.seq)
    b = a.fork()
    model.log.clear()
    _talk(chat_mod, b, model, "another way")
    assert other.seq is None and a.seq is not None  # the longest idle one gave way
    assert model.log[0]["ids"][0] == b.ids[resident:resident + model.log[0]["T"]]


def test_ordinary_chats_take_turns_on_few_rows(engine):
    chat_mod, install = engine
    cache = install(64, 16, max_seqs=2)
    model = FakeModel([])
    chats = [chat_mod.Chat(FakeTokenizer()) for _ in range(5)]
    for turn in range(2):
        for i, c in enumerate(chats):
            c.submit(model, f"message {turn} of chat {i}")
        _drain(chat_mod)
    for c in chats:
        assert [r for r, _ in c.messages] == ["user", "assistant"] * 2
    _conserved(cache)
