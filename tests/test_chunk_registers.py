"""Register limits of the packed-chunk kernel's warpgroups (csrc/chunk.cu).

A warp that has given registers back with setmaxnreg must not run code compiled
for more: code that warps of two warpgroups share needs one limit in both, and
the limits together must not exceed what the block was launched with."""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "my-inference-engine_b200" / "csrc" / "chunk.cu").read_text()


def _constant(name, fp8):
    value = re.search(rf"constexpr int {name} = ([^;]+);", SOURCE).group(1)
    both = re.fullmatch(r"kFp8 \? (\d+) : (\d+)", value)
    return int(both.group(1 if fp8 else 2)) if both else int(value)


@pytest.mark.parametrize("fp8", [False, True])
def test_the_shares_fit_the_launch(fp8):
    low, soft, aux = (_constant(n, fp8) for n in ("kRegsLow", "kRegsSoftmax", "kRegsAux"))
    assert low % 8 == soft % 8 == aux % 8 == 0
    assert low + 2 * soft + aux <= 4 * _constant("kRegsLaunch", fp8)


def test_code_shared_by_two_warpgroups_has_one_limit():
    shared = re.search(r"if constexpr \(!kFp8\) \{[^\n]*\n\s*if \(warp == (\d+) \|\| warp == (\d+)\)", SOURCE)
    assert shared, "the copy loop that two warps share is not where it was"
    groups = {int(w) // 4 for w in shared.groups()}
    limit = {0: "kRegsLow", 3: "kRegsAux"}
    assert len({_constant(limit[g], False) for g in groups}) == 1
