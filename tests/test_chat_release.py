"""A chat that is released (on a request thread) between the making of room for
its message and the message's admission: a fork's shared blocks do not come
back to the pool then, so the room has to be looked at again."""
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

    def install(blocks):
        chat.init(kv_cache=BlockTables(blocks, 16), start_worker=False)
        return chat._kv()

    yield chat, install
    chat._kv_cache = None
    for state in (chat.active, chat._deferred, chat._resident, chat._mixed):
        state.clear()


def _drain(chat_mod):
    for _ in range(600):
        if not chat_mod._tick(block=False) and not chat_mod.active and not chat_mod._deferred:
            return
    raise AssertionError("messages left over")


@pytest.mark.parametrize("deferred_first", [False, True])
def test_a_fork_released_while_it_is_admitted(engine, monkeypatch, deferred_first):
    chat_mod, install = engine
    cache = install(14)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    a.submit(model, "h" * 80)
    _drain(chat_mod)
    b = a.fork()
    make_room, released = chat_mod._make_room, []

    def raced(job):
        if deferred_first and not released:
            released.append(None)
            return False
        ok = make_room(job)
        if job.chat is b and ok and b not in released:
            assert cache._shared
            b.release()
            released.append(b)
        return ok

    monkeypatch.setattr(chat_mod, "_make_room", raced)
    b.submit(model, "another way")
    _drain(chat_mod)
    assert b in released and b.messages[-2] == ("user", "another way")
    assert b.messages[-1][0] == "assistant" and b.ids[:len(a.ids)] == a.ids
    held = {x for t in cache._block_tables.values() for x in t}
    assert len(held) + cache.free_block_count() == 14


def test_a_message_that_no_longer_fits_waits(engine, monkeypatch):
    """The same while other chats are active: no room is left, the message is deferred."""
    chat_mod, install = engine
    cache = install(16)
    model = FakeModel([])
    a = chat_mod.Chat(FakeTokenizer())
    a.submit(model, "h" * 80)
    _drain(chat_mod)
    b = a.fork()
    a.submit(model, "on we go")  # a's blocks cannot be evicted while it talks
    chat_mod._tick(block=False)
    make_room, released = chat_mod._make_room, []

    def raced(job):
        ok = make_room(job)
        if job.chat is b and ok and not released:
            b.release()
            released.append(b)
        return ok

    monkeypatch.setattr(chat_mod, "_make_room", raced)
    b.submit(model, "another way")
    chat_mod._tick(block=False)
    assert released and len(chat_mod._deferred) == 1 and b.pending == ["another way"]
    _drain(chat_mod)
    assert b.messages[-2] == ("user", "another way") and a.messages[-1][0] == "assistant"
    assert not chat_mod._deferred
