"""Limits and host arithmetic of the paged cache's entry points, no GPU needed."""
import os

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
