"""The paged cache's entry points without a GPU: every refusal is made by the
host before anything is launched, page ids outside the pool never become an
address, and the workspace size is host arithmetic."""
import ctypes
import os

import pytest

import turbo_b200 as T

pytestmark = pytest.mark.skipif(not os.path.exists(T.LIB_PATH), reason="library not built")

A = 1 << 20  # an aligned address; no call here gets as far as reading it


def cache(**kw):
    c = T.PagedCache()
    d = dict(k=A, v=A, dtype=T.F16, page_size=16, n_pages=8, kv_heads=2, head_dim=64, page_stride=2048,
             token_stride=128, head_stride=64)
    d.update(kw)
    for n, v in d.items():
        setattr(c, n, v)
    return c


def batch(**kw):
    b = T.PagedBatch()
    d = dict(batch=3, lens=A, table=A, max_pages=4, table_stride=4)
    d.update(kw)
    for n, v in d.items():
        setattr(b, n, v)
    return b


APPEND = dict(act=T.F32, q=A, ldq=512, k=A, ldk=128, v=A, ldv=128, tokens=3, heads=8, starts=None, cos=A, sin=A,
              rope=100, q_out=A, ldqo=512)
ATTN = dict(act=T.F32, q=A, ldq=512, heads=8, out=A, ldo=512, ws=A, ws_bytes=1 << 40)


def append(c=None, b=None, **kw):
    a = dict(APPEND, **kw)
    T.call("tb_rope_paged_append", c if c is not None else cache(), b if b is not None else batch(), a["act"], a["q"],
           a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["tokens"], a["heads"], a["starts"], a["cos"], a["sin"],
           a["rope"], a["q_out"], a["ldqo"], None)


def decode(c=None, b=None, **kw):
    a = dict(ATTN, **kw)
    T.call("tb_paged_attention_decode", c if c is not None else cache(), b if b is not None else batch(), a["act"],
           a["q"], a["ldq"], a["heads"], 0.125, a["out"], a["ldo"], a["ws"], a["ws_bytes"], None)


def shared(c=None, b=None, prefix=A, n=100, **kw):
    a = dict(ATTN, **kw)
    T.call("tb_paged_attention_shared", c if c is not None else cache(), b if b is not None else batch(), prefix, n,
           a["act"], a["q"], a["ldq"], a["heads"], 0.125, a["out"], a["ldo"], a["ws"], a["ws_bytes"], None)


def refused(f, *args, **kw):
    with pytest.raises(T.TbError) as e:
        f(*args, **kw)
    assert e.value.status == T.EINVAL, str(e.value)


BAD_CACHE = [dict(dtype=T.I32), dict(dtype=T.Q8_0), dict(page_size=0), dict(page_size=-16), dict(page_size=24),
             dict(n_pages=-1), dict(n_pages=1 << 31), dict(kv_heads=0), dict(head_dim=0), dict(k=None), dict(v=None),
             dict(k=A + 8), dict(v=A + 2), dict(page_stride=2044), dict(token_stride=60), dict(token_stride=0),
             dict(head_stride=68), dict(head_stride=-64), dict(page_stride=1 << 41), dict(head_dim=40)]
BAD_BATCH = [dict(batch=-1), dict(batch=1 << 21), dict(lens=None), dict(table=None), dict(max_pages=-1),
             dict(max_pages=1 << 28), dict(table_stride=3)]


@pytest.mark.parametrize("f", [append, decode, shared])
def test_descriptors_are_checked(f):
    for kw in BAD_CACHE:
        refused(f, c=cache(**kw))
    for kw in BAD_BATCH:
        refused(f, b=batch(**kw))
    refused(f, c=ctypes.POINTER(T.PagedCache)())
    refused(f, b=ctypes.POINTER(T.PagedBatch)())
    for act, ct in [(T.F16, T.BF16), (T.BF16, T.F32), (T.I32, T.F16)]:
        refused(f, c=cache(dtype=ct), act=act)


def test_append_refusals():
    for kw in [dict(tokens=2), dict(tokens=-1), dict(heads=-1), dict(cos=None), dict(sin=None), dict(rope=0),
               dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(ldk=127), dict(ldv=64), dict(ldq=511),
               dict(ldqo=500), dict(q=A + 4), dict(k=A + 8), dict(ldk=129), dict(ldq=514), dict(cos=A + 4),
               dict(q_out=A + 2)]:
        refused(append, **kw)
    for d in (8, 24, 272):
        refused(append, c=cache(head_dim=d, head_stride=272, token_stride=544, page_stride=544 * 16), ldk=2 * d,
                ldv=2 * d, ldq=8 * d, ldqo=8 * d)


@pytest.mark.parametrize("f", [decode, shared])
def test_attention_refusals(f):
    for kw in [dict(heads=0), dict(heads=7), dict(q=None), dict(out=None), dict(ws=None), dict(ldq=504), dict(ldo=504),
               dict(q=A + 8), dict(out=A + 4), dict(ldq=514), dict(ldo=513), dict(ws=A + 128), dict(ws_bytes=1000)]:
        refused(f, **kw)
    for d in (32, 96, 256):
        refused(f, c=cache(head_dim=d, head_stride=256, token_stride=512, page_stride=512 * 16), ldq=8 * d, ldo=8 * d)
    refused(f, b=batch(batch=1 << 20), heads=32, ldq=2048, ldo=2048)  # more rows than the grid's arithmetic takes


def test_shared_refusals():
    refused(shared, prefix=None)
    refused(shared, n=-1)
    refused(shared, n=1 << 31)


def test_empty_calls_need_no_device():
    append(b=batch(batch=0), tokens=0)
    append(tokens=0, starts=A)
    decode(b=batch(batch=0, lens=None, table=None))
    shared(b=batch(batch=0))


def test_workspace_size_needs_no_device():
    def size(*a):
        n = ctypes.c_size_t(0)
        T.call("tb_paged_attention_workspace_bytes", *a, ctypes.byref(n))
        return n.value

    assert size(0, 32, 8, 64) > 0 and size(0, 32, 8, 64) % 256 == 0
    assert size(64, 32, 8, 64) < size(64, 32, 8, 128) < size(128, 32, 8, 128)
    for bad in [(-1, 32, 8, 64), (4, 0, 8, 64), (4, 32, 0, 64), (4, 30, 8, 64), (4, 32, 8, 96), (1 << 20, 32, 8, 64)]:
        with pytest.raises(T.TbError) as e:
            size(*bad)
        assert e.value.status == T.EINVAL
    with pytest.raises(T.TbError):
        T.call("tb_paged_attention_workspace_bytes", 4, 32, 8, 64, None)


def test_page_ids_outside_the_pool_have_no_address():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(T.LIB_PATH), "libturbo_b200_selfcheck.so"))
    row = lib.tb_selfcheck_paged_row
    row.argtypes = [ctypes.POINTER(T.PagedCache), ctypes.c_int32, ctypes.c_int, ctypes.c_int64]
    row.restype = ctypes.c_int64
    for c in [cache(), cache(n_pages=1), cache(n_pages=0), cache(n_pages=0x7FFFFFFF, page_stride=1 << 20),
              cache(page_size=1, page_stride=128), cache(token_stride=64, head_stride=1024)]:
        for bad in (-1, -2147483648, 2147483647, c.n_pages, c.n_pages + 1):
            if 0 <= bad < c.n_pages or bad > 2147483647:
                continue
            assert row(c, bad, 5, 0) == -1
        for page in {0, c.n_pages // 2, c.n_pages - 1}:
            if not 0 <= page < c.n_pages:
                continue
            for t in (0, 1, c.page_size - 1, c.page_size, 12345):
                for h in (0, c.kv_heads - 1):
                    want = 2 * (page * c.page_stride + t % c.page_size * c.token_stride + h * c.head_stride)
                    assert row(c, page, t, h) == want
