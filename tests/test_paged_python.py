"""The Python helpers that describe a paged cache and a batch: what they refuse (no GPU needed)."""
import pytest

import turbo_b200 as T

torch = pytest.importorskip("torch")

LENS = torch.zeros(4, dtype=torch.int32)


@pytest.mark.parametrize("table", [
    torch.zeros((1, 6), dtype=torch.int32).expand(4, 6),           # one row for all: its next row is not 6 entries on
    torch.zeros(24, dtype=torch.int32).as_strided((4, 6), (2, 1)),  # rows that overlap
    torch.zeros(24, dtype=torch.int32).as_strided((4, 6), (5, 1)),
])
def test_tables_whose_rows_overlap_are_refused(table):
    with pytest.raises(ValueError, match="rows"):
        T.paged_batch(LENS, table)


def test_tensors_in_host_memory_are_refused():
    pool = torch.zeros((3, 16, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        T.paged_cache(pool, pool.clone())
    with pytest.raises(ValueError, match="GPU"):
        T.paged_batch(LENS, torch.zeros((4, 6), dtype=torch.int32))
