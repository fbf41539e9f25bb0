"""Packed-chunk attention of many sequences in one call: more than the kernel
has threads (so that a thread sums the work of several rows and a CTA's range
starts inside them), the most that a call takes, and short sequences of one to
four partitions beside a long one."""
import random

import pytest
import torch

from test_chunk_fp8_gpu import check8
from test_chunk_gpu import FMT, check, make

pytestmark = pytest.mark.gpu


def both(c, causal=True):
    return check8(c, causal) if c["fmt"] == "fp8" else check(c, causal)


@FMT
@pytest.mark.parametrize("count", [512, 513, 1025, 1700])
def test_more_sequences_than_threads(cuda, fmt, count):
    rng = random.Random(count)
    new = [rng.choice([0, 0, 0, 1, 1, 3, 9, 22, 45]) for _ in range(count)]
    kv = [t + rng.choice([0, 0, 1, 15, 60, 200]) if t else rng.choice([0, 7]) for t in new]
    new[-1], kv[-1] = 70, 333
    both(make(cuda, new, kv, 12, 2, fmt, seed=count, spare_rows=2))


@FMT
def test_long_runs_of_idle_rows_between_long_sequences(cuda, fmt):
    """CTAs' ranges start in the first, a middle and the last of a thread's rows."""
    for at in (0, 2, 3):
        new, kv = [0] * 2000, [3] * 2000
        for i in range(at, 2000, 200):
            new[i], kv[i] = 150 + i % 7, 1500 + i
        both(make(cuda, new, kv, 8, 1, fmt, seed=at))


@FMT
@pytest.mark.parametrize("long", [0, 60])
def test_the_most_sequences_of_a_call(cuda, fmt, long):
    """16383 rows, all but a few idle; with `long` the tensor cores' kernel runs too."""
    count = 16383
    new, kv = [0] * count, [0] * count
    for i, (t, n) in {0: (1, 20), 1: (0, 9), 4095: (16, 100), 9001: (2, 31), count - 1: (1, 65)}.items():
        new[i], kv[i] = t, n
    if long:
        new[7000], kv[7000] = long, 300
    both(make(cuda, new, kv, 12, 2, fmt, seed=9))


@FMT
@pytest.mark.parametrize("kv_long", [300, 20000])
def test_short_sequences_of_every_partition_count_beside_a_long_one(cuda, fmt, kv_long):
    """Clusters in which some partitions are empty join beside the long sequence's work."""
    new = [1, 2, 1, 1, 2, 1, 1, 600]
    kv = [5, 130, 256, 300, 400, 520, 700, kv_long + 600]
    c = make(cuda, new, kv, 12, 2, fmt, seed=11)
    first = both(c)
    for _ in range(5):
        assert torch.equal(both(c), first)
