"""The staging buffer of small uploads is guarded on the stream that copies from
it, whichever device is current (checked with a CUDA that is not there)."""
import numpy as np
import torch

import kv_cache


class Host(torch.Tensor):
    """A host tensor that says it was copied to another device."""

    @staticmethod
    def of(t):
        return t.as_subclass(Host)

    def to(self, device, non_blocking=False):
        assert non_blocking and device == torch.device("cuda", 1)
        out = self.clone()
        out.where = device
        return out

    @property
    def device(self):
        return getattr(self, "where", torch.device("cpu"))


def test_the_event_is_recorded_on_the_copys_stream(monkeypatch):
    seen = []

    class Event:
        def record(self, stream=None):
            seen.append(stream)

        def synchronize(self):
            seen.append("waited")

    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda n, dtype, pin_memory: Host.of(empty(n, dtype=dtype)))
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: ("stream of", device))
    up = kv_cache._PinnedUpload(torch.int32)
    dev = torch.device("cuda", 1)
    for _ in range(2):
        assert up.send(np.arange(5, dtype=np.int32), dev).tolist() == [0, 1, 2, 3, 4]
    assert seen == [("stream of", dev), "waited", ("stream of", dev)]
