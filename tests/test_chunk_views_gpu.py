"""Tables of unusual strides: a matrix of one row has any row stride, and rows
that overlap are refused."""
import pytest
import torch

from test_chunk_gpu import FMT, SCALE, call, check, make
from test_chunk_fp8_gpu import check8

pytestmark = pytest.mark.gpu


def _one_row(cuda, fmt):
    """A sequence whose table is its matrix' only row."""
    c = make(cuda, [3], [100], 12, 2, fmt, seed=3)
    c["tables"] = c["tables"][c["rows"][0].item():][:1].contiguous()
    c["rows"] = torch.zeros(1, dtype=torch.int32, device=cuda)
    return c


@FMT
def test_one_row_as_a_turned_column(cuda, fmt):
    c = _one_row(cuda, fmt)
    c["tables"] = c["tables"][0][:, None].T
    assert c["tables"].shape[0] == 1 and c["tables"].stride(0) == 1
    (check8 if fmt == "fp8" else check)(c)


@FMT
def test_rows_that_overlap_are_refused(cuda, fmt):
    c = _one_row(cuda, fmt)
    for tables in (c["tables"].expand(3, -1), c["tables"].reshape(-1).as_strided((2, 4), (2, 1))):
        with pytest.raises(ValueError, match="overlap"):
            call(dict(c, tables=tables))


def test_moves_take_a_turned_column_too(cuda):
    import pagedkv

    pool = torch.arange(8 * 16 * 2 * 128, device=cuda).view(1, 128, 2, 128).to(torch.bfloat16)
    want = pool.clone()
    want[0, 16:32] = want[0, 96:112]
    tables = torch.tensor([[6], [0], [6], [3]], dtype=torch.int32, device=cuda).T
    ids = torch.tensor([6, 1], dtype=torch.int32, device=cuda)
    pagedkv.move_blocks(pool, ids[:1], ids[1:], tables)
    assert torch.equal(pool, want) and tables.tolist() == [[1, 0, 1, 3]]
    with pytest.raises(ValueError, match="overlap"):
        pagedkv.move_blocks(pool, ids[:1], ids[1:], tables.expand(2, -1))
