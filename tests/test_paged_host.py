"""Limits and host arithmetic of the paged cache's entry points, no GPU needed."""
import ctypes
import os
import random

import pytest

import turbo_b200 as T
from test_paged_abi import append, batch, cache, decode, refused, shared

pytestmark = pytest.mark.skipif(not os.path.exists(T.LIB_PATH), reason="library not built")

MOST = 2 ** 31 - 1 - 65536  # tokens of a sequence that a table describes


@pytest.mark.parametrize("page", [1, 16, 1 << 16, 1 << 30])
def test_tables_of_nearly_2_to_the_31_tokens(page):
    """Lengths are rounded up to whole tiles in 32 bits: a table of all 2^31 - 1 tokens would leave no room for that."""
    c = cache(page_size=page, n_pages=1, kv_heads=1, page_stride=64, token_stride=64)
    for f in (append, decode, shared):
        for pages in ((2 ** 31 - 1) // page, MOST // page + 1):
            if pages * page > MOST:
                refused(f, c=c, b=batch(batch=1, max_pages=pages, table_stride=pages))
    # a call of no tokens: checked in full, launched never
    append(c=c, b=batch(batch=0, max_pages=MOST // page, table_stride=MOST // page), tokens=0)
    decode(c=c, b=batch(batch=0, max_pages=MOST // page, table_stride=MOST // page))


def selfcheck(name, *args):
    lib = ctypes.CDLL(os.path.join(os.path.dirname(T.LIB_PATH), "libturbo_b200_selfcheck.so"))
    fn = getattr(lib, name)
    fn.argtypes, fn.restype = [ctypes.c_int64] * len(args), ctypes.c_int64
    return fn(*args)


def test_prefix_splits_finish_first():
    """Against every number of splits: waves of CTAs times a share's tiles and a start, within 2 %."""
    r = random.Random(5)
    for _ in range(600):
        items, tiles = r.choice([1, 2, 8, 12, 100, 147, 148, 149, 300, r.randint(1, 2000)]), r.randint(1, 3000)
        ctas, most = r.choice([148, 296, 444, r.randint(1, 500)]), r.randint(1, 4000)

        def time(n):
            return -(-items * n // ctas) * (-(-tiles // n) + 6)

        n = selfcheck("tb_selfcheck_prefix_splits", items, tiles, ctas, most)
        assert 1 <= n <= min(most, tiles)
        assert time(n) <= 1.02 * min(time(m) for m in range(1, min(most, tiles) + 1))
        assert all(time(m) > time(n) for m in range(1, n))


def test_prefix_splits_look_at_few():
    """The choice is made at every call: its cost must not grow with the prefix (rows and most as a call has them)."""
    for rows in (1, 2, 8, 16, 64, 300, 4096, 1 << 17):
        most = (2 * rows + 2 * 148 * 128 + (2 * rows if rows < 1 << 17 else 1 << 18)) // rows - 1
        for items in {max(1, rows // 256), max(1, rows // 8), max(1, rows)}:
            for tiles in (512, 2048, 16384, 1 << 24):
                assert selfcheck("tb_selfcheck_prefix_splits_looks", items, tiles, 148, most) <= 16


def test_rows_of_the_pools_that_the_kernels_get():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(T.LIB_PATH), "libturbo_b200_selfcheck.so"))
    row = lib.tb_selfcheck_paged_row_of
    row.argtypes = [ctypes.POINTER(T.PagedCache)] + [ctypes.c_int64] * 3
    row.restype = ctypes.c_int64
    for c in (cache(), cache(dtype=T.F32), cache(token_stride=64, head_stride=1024),
              cache(n_pages=0x7FFFFFFF, page_stride=1 << 20), cache(n_pages=1, page_stride=-7),
              cache(page_size=1, token_stride=-7, page_stride=128), cache(kv_heads=1, head_stride=-7, token_stride=64)):
        size = 4 if c.dtype == T.F32 else 2
        for page in {0, c.n_pages // 2, c.n_pages - 1}:
            for t in (0, 1, c.page_size - 1, c.page_size, 12345, MOST - 1):
                for h in (0, c.kv_heads - 1):
                    want = (page * c.page_stride if c.n_pages > 1 else 0) + t % c.page_size * c.token_stride + (
                        h * c.head_stride)
                    assert row(c, page, t, h) == size * want
        for bad in (-1, -2 ** 31, c.n_pages, 2 ** 31 - 1):
            assert row(c, bad, 5, 0) == -1


def test_lists_of_integers_are_aligned():
    """A list at an odd address would fault the kernels."""
    for f in (append, decode, shared):
        refused(f, b=batch(lens=(1 << 20) + 2))
        refused(f, b=batch(table=(1 << 20) + 1))
    refused(append, starts=(1 << 20) + 2)
    refused(shared, prefix=(1 << 20) + 3)
