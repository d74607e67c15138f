"""The paged key/value cache on the GPU: the rotating append, the batched decode
attention and the attention behind a shared prefix, against plain 64-bit
implementations.

Tolerances.  A rounding to a type is off by at most eps/2 of the value.
 append: y = x0 c -+ x1 s as one multiplication and one fused multiply-add: at
   most (|x0 c| + |x1 s|) 2 2^-24 off, then one rounding to the output's type.
 attention: with A = scale max_t sum_d |q_d k_td|, a score is off by ds <= A
   (2 2^-22 + (D/4 + 8) 2^-23): 22-bit operands on both sides, D/8 (fp32 caches
   2 D/8) accumulations inside the tensor core, each off by at most one unit of
   2^-23, and the additions and multiplications around them.  A probability is
   off by 2 ds + 2^-20 relative (numerator and maximum; exp2 to 2^-22, joins), the
   weighted sum by that, 2^-22 for p's parts, 4 2^-23 inside the tensor core and
   one unit of 2^-24 per addition to a running sum, at most (keys / 8 + 200)
   of them; all relative to sum p |v|.  Then one rounding to the output's type.
   16-bit activations behind a prefix may round each p to the cache's type: eps/2
   of p, numerator and denominator alike."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import turbo_b200 as T  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.fixture(autouse=True)
def _no_errors_left():
    yield
    torch.cuda.synchronize()
    T.take_device_errors()


def pools(pages, page, kvh, dim, dtype, layout, fill=float("nan")):
    """K and V pools [pages, page, kvh, dim] full of `fill`."""
    out = []
    for _ in range(2):
        if layout == "token":
            t = torch.full((pages, page, kvh, dim), fill, dtype=dtype, device="cuda")
        elif layout == "head":
            t = torch.full((pages, kvh, page, dim), fill, dtype=dtype, device="cuda").permute(0, 2, 1, 3)
        else:  # gaps between heads, tokens and pages
            t = torch.full((pages, page + 1, kvh + 1, dim + 16), fill, dtype=dtype, device="cuda")[:, :page, :kvh, :dim]
        out.append(t)
    return out


def tables(lens, page, pages, seed, spare=2):
    """Scattered page ids for the lengths (numpy [batch, max_pages]); unused
    entries hold an id outside any pool."""
    r = np.random.default_rng(seed)
    ids = r.permutation(pages)
    width = max((max(lens) + page - 1) // page, 1) + spare
    table = np.full((len(lens), width), 2 ** 31 - 1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        k = (n + page - 1) // page
        table[b, :k] = ids[at:at + k]
        at += k
    assert at <= pages
    return table, ids[at:]


def cuda_i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def put_rows(pool, table_row, page, rows):
    """Writes rows [n, kvh, dim] at positions 0 .. n - 1."""
    n = rows.shape[0]
    if n:
        t = torch.arange(n)
        ids = torch.from_numpy(table_row.astype(np.int64))[t // page].cuda()
        pool[ids, (t % page).cuda()] = rows.to(pool.dtype)


def get_rows(pool, table_row, page, n):
    t = torch.arange(n)
    ids = torch.from_numpy(table_row.astype(np.int64))[t // page].cuda()
    return pool[ids, (t % page).cuda()]


def workspace(batch, heads, kvh, dim):
    n = ctypes.c_size_t(0)
    T.call("tb_paged_attention_workspace_bytes", batch, heads, kvh, dim, ctypes.byref(n))
    return torch.zeros(n.value, dtype=torch.uint8, device="cuda")


def randn(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


# ------------------------------------------------------------------- append --

def rope_tables(n, dim):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) * 2 /
                                                                    dim)[None]
    return a.cos().float().cuda(), a.sin().float().cuda()


def rotated(x, cos, sin):
    """x [tokens, n, dim], tables [tokens, dim / 2]: the rotation and |x0 c| + |x1 s|, in 64 bits."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return (torch.cat((a * c - b * s, a * s + b * c), -1),
            torch.cat((a.abs() * c.abs() + b.abs() * s.abs(), a.abs() * s.abs() + b.abs() * c.abs()), -1))


def near(got, want, mag, dtype):
    tol = mag * 2 ** -23 + (want.abs() + mag * 2 ** -23) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), "%d of %d off, first at %s" % (bad.sum(), bad.numel(), bad.nonzero()[0].tolist())


def append_call(kp, vp, lens, table, q, k, v, starts, cos, sin, q_out, stream=None):
    heads = 0 if q is None else q.shape[1]
    c, b = T.paged_cache(kp, vp), T.paged_batch(lens, table)
    T.call("tb_rope_paged_append", T.byref(c), T.byref(b), T.dtype_code(k), T.ptr(q) if heads else None,
           q.stride(0) if heads else 0, T.ptr(k), k.stride(0), T.ptr(v), v.stride(0), k.shape[0], heads,
           T.ptr(starts) if starts is not None else None, T.ptr(cos) if cos is not None else None,
           T.ptr(sin) if sin is not None else None, cos.shape[0] if cos is not None else 0,
           T.ptr(q_out) if heads else None, q_out.stride(0) if heads else 0, T.stream_handle(stream))


APPEND = [
    # (group, kv_heads, dim, page, layout, held, new): new None: one token each, held[b] = -1 an empty slot
    (4, 8, 64, 16, "token", [0, 500, 15, 16, 31], None),
    (4, 8, 128, 32, "head", [7, -1, 0, 300, -1, 63], None),
    (1, 1, 16, 1, "token", [3, 0, 9], None),
    (3, 2, 80, 8, "gaps", [5, 11], [9, 1]),
    (7, 5, 256, 4, "head", [0, 3, 2], [1, 0, 14]),
    (0, 2, 64, 16, "token", [0, 17], [33, 5]),
    (4, 8, 64, 16, "token", [0, 1, 0, 100, 7] * 9, [0, 1, 40, 3, 0] * 9),
    (2, 1, 128, 64, "gaps", list(range(70)), [b % 3 for b in range(70)]),
    (1, 2, 64, 16, "token", [5] * 1100, [b % 2 for b in range(1100)]),
]


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case, act, ct):
    group, kvh, dim, page, layout, held, new = APPEND[case]
    heads = group * kvh
    one_each = new is None
    if one_each:
        new = [0 if h < 0 else 1 for h in held]
    lens = [max(h, 0) + n if h >= 0 else 0 for h, n in zip(held, new)]
    pages = sum((n + page - 1) // page for n in lens) + 3
    table, _ = tables(lens, page, pages, case)
    kp, vp = pools(pages, page, kvh, dim, TYPES[ct], layout, fill=7.0)
    tokens = len(held) if one_each else sum(new)
    pad = 0 if one_each else 3  # rows behind the last sequence
    q = randn((tokens + pad, heads * dim + 8), case + 1).to(TYPES[act]).cuda()[:, :heads * dim].unflatten(1, (heads, dim)) if heads else None
    kv = randn((tokens + pad, 2, kvh, dim), case + 2).to(TYPES[act]).cuda()
    q_out = torch.full((tokens + pad, heads, dim), 5.0, dtype=TYPES[act], device="cuda") if heads else None
    starts = None if one_each else cuda_i32(np.concatenate(([0], np.cumsum(new))))
    cos, sin = rope_tables(max(lens), dim)
    append_call(kp, vp, cuda_i32(lens), cuda_i32(table), q, kv[:, 0], kv[:, 1], starts, cos, sin, q_out)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    want_k, want_v = pools(pages, page, kvh, dim, TYPES[ct], layout, fill=7.0)
    touched = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
    rows, t = [], 0
    for b, n in enumerate(new):
        for i in range(n):
            pos = lens[b] - n + i
            rows.append((b if one_each else t + i, pos, int(table[b, pos // page]), pos % page))
        t += n
    row, pos, pg, slot = (torch.tensor(x).cuda() for x in zip(*rows))
    touched[pg, slot] = True
    assert torch.equal(kp[~touched], want_k[~touched]) and torch.equal(vp[~touched], want_v[~touched])
    assert torch.equal(vp[pg, slot], kv[row, 1].to(TYPES[ct]))
    want, mag = rotated(kv[row, 0], cos[pos], sin[pos])
    near(kp[pg, slot], want, mag, TYPES[ct])
    if heads:
        left = torch.ones(tokens + pad, dtype=torch.bool, device="cuda")
        left[row] = False
        assert (q_out[left] == 5.0).all()
        want, mag = rotated(q[row], cos[pos], sin[pos])
        near(q_out[row], want, mag, TYPES[act])
        # in place, and the same bits
        if not one_each:
            append_call(kp, vp, cuda_i32(lens), cuda_i32(table), q, kv[:, 0], kv[:, 1], starts, cos, sin, q)
            assert torch.equal(q[row], q_out[row])


def test_append_equals_rope_and_copy_bit_for_bit():
    kvh, heads, dim, page, n, at = 2, 8, 64, 16, 40, 21
    table, _ = tables([at + n], page, 6, 3)
    kp, vp = pools(6, page, kvh, dim, torch.float32, "token")
    q, k, v = (randn((n, h, dim), s).cuda() for h, s in ((heads, 1), (kvh, 2), (kvh, 3)))
    cos, sin = rope_tables(at + n, dim)
    q_out = torch.empty_like(q)
    append_call(kp, vp, cuda_i32([at + n]), cuda_i32(table), q, k, v, cuda_i32([0, n]), cos, sin, q_out)
    for x, got in ((q, q_out), (k, torch.stack([kp[int(table[0, p // page]), p % page] for p in range(at, at + n)]))):
        y = x.clone()
        w = T.view(y, 0, (1, x.shape[1], n, dim), (y.numel(), dim, x.shape[1] * dim, 1))
        T.call("tb_rope", T.byref(w), T.ptr(cos), T.ptr(sin), dim, at + n, at, T.stream_handle())
        assert torch.equal(got, y)


def test_append_without_rotation():
    table, _ = tables([9, 4], 4, 6, 3)
    kp, vp = pools(6, 4, 2, 64, torch.float16, "head")
    k, v = randn((2, 2, 64), 1).cuda(), randn((2, 2, 64), 2).cuda()
    append_call(kp, vp, cuda_i32([9, 4]), cuda_i32(table), None, k, v, None, None, None, None)
    for b, pos in ((0, 8), (1, 3)):
        assert torch.equal(kp[int(table[b, pos // 4]), pos % 4], k[b].half())
        assert torch.equal(vp[int(table[b, pos // 4]), pos % 4], v[b].half())


def test_append_bad_positions_and_pages():
    """Each bad token is left out and reported; the others are written."""
    page, kvh, dim = 8, 1, 64
    kp, vp = pools(9, page, kvh, dim, torch.float32, "token", fill=0.0)
    table = np.array([[0, 1], [-1, 2], [3, 9], [4, 5], [6, 7], [2 ** 31 - 1, 8]], np.int32)
    lens = [16, 3, 12, 17, -4, 1]  # fine; page -1; page 9 of 9; past the table's pages; negative; far page id
    k, v = randn((6, 1, dim), 1).cuda(), randn((6, 1, dim), 2).cuda()
    q = randn((6, 2, dim), 3).cuda()
    cos, sin = rope_tables(20, dim)
    q_out = torch.full_like(q, 5.0)
    append_call(kp, vp, cuda_i32(lens), cuda_i32(table), q, k, v, None, cos, sin, q_out)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2
    want = torch.zeros_like(vp)
    want[1, 7] = v[0]
    assert torch.equal(vp, want) and (kp[1, 7] != 0).all() and (kp != 0).sum() == dim
    assert (q_out[1:] == 5.0).all() and (q_out[0] != 5.0).any()
    append_call(kp, vp, cuda_i32(lens[:1]), cuda_i32(table[:1]), q[:1], k[:1], v[:1], None, cos[:15], sin[:15], q_out)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2  # position 15 of a table of 15
    # fewer keys than new tokens: the tokens at negative positions are left out
    append_call(kp, vp, cuda_i32([1]), cuda_i32(table[3:4]), q[:2], k[:2], v[:2], cuda_i32([0, 2]), cos, sin, q_out)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2
    assert torch.equal(vp[4, 0], v[1])


# ---------------------------------------------------------------- attention --

def exact(q, k, v, scale, p_eps=0.0):
    """One sequence: q [heads, dim], k and v [n, kvh, dim].  The output and its
    tolerance before the rounding to a type."""
    heads, dim = q.shape
    n, kvh = k.shape[:2]
    if n == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    q, k, v = q.double().view(kvh, -1, dim), k.double().transpose(0, 1), v.double().transpose(0, 1)
    p = torch.softmax(q @ k.transpose(1, 2) * scale, -1)
    a = (q.abs() @ k.abs().transpose(1, 2)).max(-1, keepdim=True).values * abs(scale)
    ds = a * (2 * 2 ** -22 + (dim / 4 + 8) * 2 ** -23)
    rel = 2 * ds + 2 ** -20 + 2 ** -22 + 4 * 2 ** -23 + (n / 8 + 200) * 2 ** -24 + 2 * p_eps
    return (p @ v).reshape(heads, dim), (p @ v.abs() * rel).reshape(heads, dim)


def check_rows(got, want, tol, dtype):
    got = got.double()
    assert not got.isnan().any()
    lim = tol + (want.abs() + tol) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
    bad = (got - want).abs() > lim
    assert not bad.any(), "%d of %d off, worst %.3g of its limit" % (bad.sum(), bad.numel(), ((got - want).abs() / lim).max())


class Batch:
    """A paged cache with random keys and values for sequences of `lens` keys
    behind `prefix` common ones; everything else in the pools is NaN."""

    def __init__(self, act, ct, group, kvh, dim, page, layout, lens, prefix=0, seed=0, qscale=1.0):
        self.act, self.ct, self.dim, self.page, self.kvh = TYPES[act], TYPES[ct], dim, page, kvh
        self.heads, self.lens, self.n_prefix = group * kvh, list(lens), prefix
        pages = sum((n + page - 1) // page for n in lens) + (prefix + page - 1) // page + 2
        self.table, rest = tables(self.lens, page, pages, seed)
        self.prefix = rest[:(prefix + page - 1) // page].astype(np.int32)
        self.kp, self.vp = pools(pages, page, kvh, dim, self.ct, layout)
        for b, n in enumerate(self.lens):
            put_rows(self.kp, self.table[b], page, randn((n, kvh, dim), seed * 1000 + b).cuda())
            put_rows(self.vp, self.table[b], page, randn((n, kvh, dim), seed * 1000 + b + 500).cuda())
        put_rows(self.kp, self.prefix, page, randn((prefix, kvh, dim), seed + 71).cuda())
        put_rows(self.vp, self.prefix, page, randn((prefix, kvh, dim), seed + 72).cuda())
        self.ldq = self.heads * dim + 16
        self.q = (randn((len(lens), self.ldq), seed + 9) * qscale).to(self.act).cuda()
        self.scale = dim ** -0.5
        self.d_lens, self.d_table, self.d_prefix = cuda_i32(self.lens), cuda_i32(self.table), cuda_i32(self.prefix)
        self.ws = workspace(len(lens), self.heads, kvh, dim)
        self.cache, self.batch = T.paged_cache(self.kp, self.vp), T.paged_batch(self.d_lens, self.d_table)

    def rows(self):
        return self.q[:, :self.heads * self.dim].unflatten(1, (self.heads, self.dim))

    def run(self, shared=False, out=None, ws=None, stream=None):
        ldo = self.heads * self.dim + 8
        if out is None:
            out = torch.full((len(self.lens), ldo), 9.0, dtype=self.act, device="cuda")
        ws = self.ws if ws is None else ws
        if shared:
            T.call("tb_paged_attention_shared", T.byref(self.cache), T.byref(self.batch), T.ptr(self.d_prefix),
                   self.n_prefix, T.dtype_code(self.q), T.ptr(self.q), self.ldq, self.heads, self.scale, T.ptr(out), ldo,
                   T.ptr(ws), ws.numel(), T.stream_handle(stream))
        else:
            T.call("tb_paged_attention_decode", T.byref(self.cache), T.byref(self.batch), T.dtype_code(self.q),
                   T.ptr(self.q), self.ldq, self.heads, self.scale, T.ptr(out), ldo, T.ptr(ws), ws.numel(),
                   T.stream_handle(stream))
        return out

    def check(self, out, lens=None):
        torch.cuda.synchronize()
        assert T.take_device_errors() == 0
        assert (out[:, self.heads * self.dim:] == 9.0).all()
        p_eps = torch.finfo(self.ct).eps / 2 if self.n_prefix and self.act != torch.float32 else 0.0
        pk, pv = (get_rows(p, self.prefix, self.page, self.n_prefix) for p in (self.kp, self.vp))
        for b, n in enumerate(self.lens if lens is None else lens):
            k, v = (torch.cat((x, get_rows(p, self.table[b], self.page, n))) for x, p in ((pk, self.kp), (pv, self.vp)))
            want, tol = exact(self.rows()[b], k, v, self.scale, p_eps)
            got = out[b, :self.heads * self.dim].view(self.heads, self.dim)
            if k.shape[0] == 0:
                assert (got == 0).all()
            check_rows(got, want, tol, self.act)


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 0, 200, 511]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("act,ct", PAIRS)
def test_decode_types(act, ct, dim):
    x = Batch(act, ct, 4, 2, dim, 16, "token", EDGES, seed=dim)
    x.check(x.run())


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 9, 16, 17, 32, 33, 64, 71])
@pytest.mark.parametrize("ct,dim", [("f16", 64), ("f32", 128)])
def test_decode_groups(group, ct, dim):
    x = Batch("f32", ct, group, 2, dim, 8, "head", [1, 0, 77, 300], seed=group)
    x.check(x.run())


@pytest.mark.parametrize("page,layout", [(1, "token"), (2, "gaps"), (16, "gaps"), (64, "head"), (1024, "token")])
def test_decode_pages(page, layout):
    x = Batch("bf16", "bf16", 5, 3, 128, page, layout, [130, 1, 0, 65, 400], seed=page)
    x.check(x.run())


@pytest.mark.parametrize("lens,kvh,act,ct,dim", [
    ([40000], 1, "f32", "f16", 64),         # one item over every CTA
    ([100003, 1, 0, 7], 2, "bf16", "bf16", 128),
    ([9000, 8191, 12], 8, "f32", "f32", 64),
    ([257] * 300, 1, "f16", "f16", 64),     # more sequences than threads of a CTA
    ([3] * 999 + [5000] + [0] * 100, 2, "f32", "bf16", 64),
])
def test_decode_long_and_many(lens, kvh, act, ct, dim):
    x = Batch(act, ct, 4, kvh, dim, 32, "head", lens, seed=len(lens))
    out = x.run()
    x.check(out)
    assert torch.equal(out, x.run())  # the same order of sums every time


def test_decode_large_scores():
    """Scores of some thousands: all weight on few keys, exponents far below the range of fp32."""
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [1, 130, 700], seed=5, qscale=500.0)
    x.check(x.run())


def test_decode_one_dominant_key_per_tile():
    x = Batch("f32", "bf16", 2, 1, 64, 16, "token", [600], seed=6)
    k = get_rows(x.kp, x.table[0], 16, 600)
    k[::64] *= 12
    put_rows(x.kp, x.table[0], 16, k)
    x.check(x.run())


def test_decode_infinite_scores():
    """A key of -inf scores takes no weight; a sequence of nothing else is NaN, as softmax of it is."""
    x = Batch("f32", "f32", 1, 1, 64, 16, "token", [300, 40], seed=7)
    x.q[:, :64] = 3e38
    k = torch.full((300, 1, 64), -3e38, device="cuda")
    k[250] = 0.0
    put_rows(x.kp, x.table[0], 16, k)
    put_rows(x.kp, x.table[1], 16, k[:40])
    out = x.run()
    torch.cuda.synchronize()
    # p = 1 for key 250 alone: an fp32 value v goes through as hi + lo, |v - hi - lo| <= 2^-22 |v| (the documented 22
    # bits), and the two products' sum inside the tensor core is off by at most 2 units of 2^-23 of |v|: 2^-21 |v|
    v = get_rows(x.vp, x.table[0], 16, 300)[250, 0]
    assert ((out[0, :64] - v).abs() <= v.abs() * 2 ** -21).all()
    assert out[1, :64].isnan().all()


def test_decode_bad_lengths_and_pages():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [100, 50, 40, 30], seed=8)
    x.d_lens.copy_(cuda_i32([100, -1, x.table.shape[1] * 16 + 1, 30]))
    out = x.run()
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2
    n = x.heads * x.dim
    assert (out[1:3, :n] == 0).all()
    for bad in (-1, x.kp.shape[0], 2 ** 31 - 1, -2 ** 31):
        y = Batch("f32", "f16", 4, 2, 64, 16, "token", [100, 50], seed=8)
        y.table[1, 1] = bad
        y.d_table.copy_(cuda_i32(y.table))
        out = y.run()
        torch.cuda.synchronize()
        assert T.take_device_errors() == 2
        k, v = get_rows(y.kp, y.table[0], 16, 100), get_rows(y.vp, y.table[0], 16, 100)
        want, tol = exact(y.rows()[0], k, v, y.scale)
        check_rows(out[0, :n].view(8, 64), want, tol, y.act)
        y.table[1, 1] = 0  # the page reads as zeros
        k, v = (get_rows(p, y.table[1], 16, 50).clone() for p in (y.kp, y.vp))
        k[16:32], v[16:32] = 0, 0
        want, tol = exact(y.rows()[1], k, v, y.scale)
        check_rows(out[1, :n].view(8, 64), want, tol, y.act)


def test_decode_far_offsets():
    """Rows past 2^31 elements and 2^32 bytes of a pool."""
    pages, page, kvh, dim = 40, 1 << 20, 1, 64
    kp, vp = (torch.empty((pages, page, kvh, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    table = np.array([[39, 0], [0, 38]], np.int32)
    lens = [700, page + 130]
    for b in range(2):
        for i in range(2):
            n = min(max(lens[b] - i * page, 0), page)
            for p, s in ((kp, 3), (vp, 4)):
                p[int(table[b, i]), :n] = (torch.randn((n, kvh, dim), generator=torch.Generator("cuda").manual_seed(s + b + 2 * i), device="cuda") if b == 1 else torch.randn((n, kvh, dim), generator=torch.Generator("cuda").manual_seed(90 + s), device="cuda")).half()
    q = randn((2, 4 * dim), 5).cuda()
    out = torch.zeros_like(q)
    ws = workspace(2, 4, 1, dim)
    lens_d, table_d = cuda_i32(lens), cuda_i32(table)
    c, bt = T.paged_cache(kp, vp), T.paged_batch(lens_d, table_d)
    T.call("tb_paged_attention_decode", T.byref(c), T.byref(bt), T.F32, T.ptr(q), 4 * dim, 4, 0.125, T.ptr(out), 4 * dim,
           T.ptr(ws), ws.numel(), T.stream_handle())
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    for b in range(2):
        k = torch.cat([kp[int(table[b, i]), :min(max(lens[b] - i * page, 0), page)] for i in range(2)])
        v = torch.cat([vp[int(table[b, i]), :min(max(lens[b] - i * page, 0), page)] for i in range(2)])
        want, tol = exact(q[b].view(4, dim), k, v, 0.125)
        check_rows(out[b].view(4, dim), want, tol, torch.float32)


def test_many_sequences():
    """More sequences than rows of one grid dimension, one key each; then all of them behind a prefix."""
    batch, heads, dim = 150000, 2, 64
    gen = torch.Generator("cuda").manual_seed(3)
    kp, vp = (torch.randn((batch + 5, 16, 1, dim), generator=gen, device="cuda").bfloat16() for _ in range(2))
    table = torch.randperm(batch, generator=gen, device="cuda").int()[:, None].contiguous()
    lens = torch.ones(batch, dtype=torch.int32, device="cuda")
    q = torch.randn((batch, heads * dim), generator=gen, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    ws = workspace(batch, heads, 1, dim)
    c, b = T.paged_cache(kp, vp), T.paged_batch(lens, table)
    T.call("tb_paged_attention_decode", T.byref(c), T.byref(b), T.BF16, T.ptr(q), heads * dim, heads, 0.125, T.ptr(out),
           heads * dim, T.ptr(ws), ws.numel(), T.stream_handle())
    own = vp[table[:, 0].long(), 0, 0]
    assert torch.equal(out.view(batch, heads, dim), own[:, None].expand(batch, heads, dim))
    prefix = torch.arange(batch, batch + 5, dtype=torch.int32, device="cuda")
    T.call("tb_paged_attention_shared", T.byref(c), T.byref(b), T.ptr(prefix), 77, T.BF16, T.ptr(q), heads * dim, heads,
           0.125, T.ptr(out), heads * dim, T.ptr(ws), ws.numel(), T.stream_handle())
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    pk, pv = (p[batch:].reshape(80, 1, dim)[:77] for p in (kp, vp))
    for i in (0, 1, 127, 128, 65535, 65536, 99999, batch - 1):
        k, v = (torch.cat((x, p[table[i, 0].long(), :1])) for x, p in ((pk, kp), (pv, vp)))
        want, tol = exact(q[i].view(heads, dim), k, v, 0.125, torch.finfo(torch.bfloat16).eps / 2)
        check_rows(out[i].view(heads, dim), want, tol, torch.bfloat16)


def test_first_use_is_captured():
    """In a new process: the first calls of all are captured, then replayed."""
    code = """
import ctypes, torch, turbo_b200 as T
torch.manual_seed(1)
kp, vp = (torch.randn((20, 16, 2, 64), device="cuda").half() for _ in range(2))
table = torch.arange(18, dtype=torch.int32, device="cuda").view(2, 9)
lens = torch.tensor([140, 3], dtype=torch.int32, device="cuda")
q, kv = torch.randn((2, 512), device="cuda"), torch.randn((2, 2, 128), device="cuda")
cos, sin = torch.ones((200, 32), device="cuda"), torch.zeros((200, 32), device="cuda")
out, again, turned = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
prefix = torch.tensor([18, 19], dtype=torch.int32, device="cuda")
c, b = T.paged_cache(kp, vp), T.paged_batch(lens, table)
n = ctypes.c_size_t()
T.call("tb_paged_attention_workspace_bytes", 2, 8, 2, 64, ctypes.byref(n))
ws = torch.zeros(n.value, dtype=torch.uint8, device="cuda")
def step(s, out):
    T.call("tb_rope_paged_append", T.byref(c), T.byref(b), T.F32, T.ptr(q), 512, T.ptr(kv), 256, kv.data_ptr() + 512, 256, 2,
           8, None, T.ptr(cos), T.ptr(sin), 200, T.ptr(turned), 512, s)
    T.call("tb_paged_attention_shared", T.byref(c), T.byref(b), T.ptr(prefix), 25, T.F32, T.ptr(turned), 512, 8, 0.125,
           T.ptr(out), 512, T.ptr(ws), n.value, s)
s, g = ctypes.c_void_p(), ctypes.c_void_p()
T.call("tb_init", 0)
T.call("tb_stream_create", ctypes.byref(s))
torch.cuda.synchronize()
T.call("tb_capture_begin", s)
step(s, out)
T.call("tb_capture_end", s, ctypes.byref(g))
for _ in range(3):
    T.call("tb_graph_launch", g, s)
T.call("tb_sync", s)
step(s, again)
T.call("tb_sync", s)
assert torch.equal(out, again) and out.abs().sum() > 0 and T.take_device_errors() == 0
T.call("tb_graph_destroy", g)
print("captured")
"""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, env=env)
    assert "captured" in r.stdout, r.stdout + r.stderr


SHARED = [
    # (act, cache, group, kv_heads, dim, page, layout, lens, prefix)
    ("f32", "f32", 4, 8, 64, 16, "token", [1, 60, 0, 33], 1001),
    ("f32", "f16", 4, 2, 64, 16, "token", [0], 1),
    ("f32", "f16", 1, 2, 64, 1, "token", [5, 0, 9], 127),
    ("f32", "bf16", 3, 1, 128, 32, "head", [7, 129], 128),
    ("f16", "f16", 8, 2, 128, 32, "head", [0, 3, 200, 1, 77], 129),
    ("bf16", "bf16", 4, 2, 64, 64, "gaps", list(range(17)), 640),
    ("f32", "f16", 4, 2, 64, 16, "token", [b % 5 for b in range(37)], 2049),
    ("bf16", "bf16", 7, 1, 128, 16, "head", [0] * 41, 333),
    ("f16", "f16", 4, 3, 64, 16, "token", [b * 7 % 90 for b in range(65)], 4100),
    ("f32", "bf16", 16, 1, 128, 64, "head", [b % 3 for b in range(20)], 1500),
    ("f32", "f32", 5, 2, 128, 8, "gaps", [b % 4 for b in range(30)], 700),
    ("bf16", "bf16", 4, 8, 128, 64, "head", [1, 2, 300] * 11, 9000),
    ("f32", "f16", 2, 1, 128, 32, "head", [3] * 300, 515),
    ("f32", "f32", 1, 1, 64, 16, "token", [2], 50000),
    # many key tiles per CTA, one row tile and two, every number of operand parts
    ("bf16", "bf16", 4, 8, 64, 64, "head", [b % 3 for b in range(17)], 30011),
    ("bf16", "bf16", 4, 8, 128, 64, "head", [b % 3 for b in range(33)], 20003),
    ("f16", "f16", 4, 8, 128, 16, "token", [b % 3 for b in range(64)], 20000),
    ("f16", "f16", 8, 8, 64, 16, "token", [b % 3 for b in range(40)], 20001),
    ("f32", "f16", 4, 8, 64, 16, "token", [b % 3 for b in range(20)], 15000),
    ("f32", "f16", 4, 8, 128, 16, "token", [b % 3 for b in range(40)], 15000),
    ("f32", "bf16", 4, 8, 64, 16, "token", [b % 3 for b in range(70)], 15000),
    ("f32", "bf16", 4, 8, 128, 16, "token", [b % 3 for b in range(20)], 15000),
]


@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared(case):
    *a, lens, prefix = SHARED[case]
    x = Batch(*a, lens, prefix, seed=case + 40)
    out = x.run(shared=True)
    x.check(out)
    assert torch.equal(out, x.run(shared=True))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 8, 9, 31, 64, 65, 127, 128, 129, 300])
def test_shared_rows(rows, dim, act, ct):
    for prefix in (259, 643):  # read by the decode kernel, and by kernels of its own
        x = Batch(act, ct, 1, 1, dim, 16, "token", [b % 2 for b in range(rows)], prefix, seed=rows)
        x.check(x.run(shared=True))


@pytest.mark.parametrize("lens", [[0, 3, 64, 65, 200], [5, 0]])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 128, 500])
@pytest.mark.parametrize("act,ct,dim", [("f32", "f16", 64), ("bf16", "bf16", 128), ("f32", "f32", 128)])
def test_shared_short_prefix(act, ct, dim, prefix, lens):
    x = Batch(act, ct, 4, 2, dim, 16, "head", lens * 40, prefix, seed=prefix)
    x.check(x.run(shared=True))


def test_shared_without_prefix_is_decode():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [100, 0, 3], seed=2)
    assert torch.equal(x.run(shared=True), x.run())


def test_shared_large_scores():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [3] * 40, 500, seed=5, qscale=500.0)
    x.check(x.run(shared=True))
    y = Batch("bf16", "bf16", 4, 2, 128, 16, "token", [3] * 40, 500, seed=5, qscale=100.0)
    y.check(y.run(shared=True))


@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-30])
@pytest.mark.parametrize("act,ct,dim", [("f32", "f16", 64), ("bf16", "bf16", 128), ("f32", "f32", 64)])
def test_other_scales(act, ct, dim, scale):
    x = Batch(act, ct, 4, 2, dim, 16, "token", [0, 5, 100] * 4, 300, seed=9)
    x.scale = scale
    x.check(x.run(shared=True))
    x.n_prefix = 0  # the sequences' own keys alone
    x.check(x.run())


def test_queries_of_other_rows_do_not_matter():
    """Empty slots of a padded batch hold whatever they hold: NaN, infinities, the largest numbers."""
    for act, ct, dim, rows in (("f32", "f16", 64, 40), ("f32", "bf16", 128, 40), ("f16", "f16", 64, 40), ("f32", "f32", 64, 4)):
        x = Batch(act, ct, 4, 1, dim, 16, "token", [7] * rows, 200, seed=10)
        good = x.run(shared=True).clone(), x.run().clone()
        for b, v in ((1, float("nan")), (2, float("inf")), (3, torch.finfo(TYPES[act]).max)):
            x.q[b] = v
        for was, now in zip(good, (x.run(shared=True), x.run())):
            assert torch.equal(was[0], now[0]) and torch.equal(was[4:], now[4:])


def test_shared_bad_prefix_page():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [3] * 40, 100, seed=3)
    x.d_prefix[2] = x.kp.shape[0]
    x.run(shared=True)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2


# --------------------------------------------------- streams, graphs, in a run --

def test_two_streams_with_a_workspace_each():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [5000, 1, 700, 0], seed=1)
    y = Batch("bf16", "bf16", 8, 4, 128, 32, "head", [9, 4000, 333], 1000, seed=2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.full((len(z.lens), z.heads * z.dim + 8), 9.0, dtype=z.act, device="cuda") for z in (x, y)]
            for _ in range(20)]
    torch.cuda.synchronize()  # the fills ran on another stream
    for a, b in outs:
        x.run(out=a, stream=streams[0])
        y.run(shared=True, out=b, stream=streams[1])
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1])
    x.check(outs[0][0])
    y.check(outs[0][1])


def test_one_workspace_for_calls_of_other_shapes():
    xs = [Batch("f32", "f16", 4, 2, 64, 16, "token", [3000, 1], seed=1),
          Batch("bf16", "bf16", 33, 1, 128, 32, "head", [9, 900], 500, seed=2),
          Batch("f32", "f32", 1, 8, 64, 8, "token", [700] * 20, 64, seed=3)]
    ws = max((x.ws for x in xs), key=lambda w: w.numel())
    for _ in range(2):
        for x in xs:
            x.check(x.run(shared=x.n_prefix > 0, ws=ws))


def test_captured_calls_follow_the_lengths():
    """Two graphs that share a workspace, replayed in turn while the lengths change."""
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [900, 900, 900], 700, seed=4)
    outs, graphs = [], []
    s = ctypes.c_void_p()
    T.call("tb_stream_create", ctypes.byref(s))
    torch.cuda.synchronize()
    for shared in (False, True):
        out = torch.full((3, x.heads * x.dim + 8), 9.0, device="cuda")
        torch.cuda.synchronize()
        T.call("tb_capture_begin", s)
        x.run(shared=shared, out=out, stream=type("S", (), {"cuda_stream": s.value})())
        g = ctypes.c_void_p()
        T.call("tb_capture_end", s, ctypes.byref(g))
        outs.append(out)
        graphs.append(g)
    for lens in ([900, 900, 900], [0, 1, 2], [128, 899, 0], [500, 0, 640]):
        x.d_lens.copy_(cuda_i32(lens))
        torch.cuda.synchronize()
        for _ in range(2):
            for g in graphs:
                T.call("tb_graph_launch", g, s)
        T.call("tb_sync", s)
        prefix, x.n_prefix = x.n_prefix, 0
        x.check(outs[0], lens)
        x.n_prefix = prefix
        x.check(outs[1], lens)
    for g in graphs:
        T.call("tb_graph_destroy", g)
    T.call("tb_stream_destroy", s)


@pytest.mark.parametrize("act,ct,dim", [("f32", "f16", 64), ("bf16", "bf16", 128)])
def test_a_server_s_run(act, ct, dim):
    """A shared prompt and the sequences' own prompts enter the cache, then
    tokens are decoded one by one: append, attention behind the prefix, and the
    same over a batch whose prefix is copied into each sequence's own pages."""
    page, kvh, group, batch, steps, prefix = 16, 2, 4, 5, 6, 45
    heads, dt = group * kvh, TYPES[ct]
    own = [3, 0, 17, 1, 30]
    total = [n + steps for n in own]
    whole = [prefix + n for n in total]
    pages = sum((n + page - 1) // page for n in total + whole) + (prefix + page - 1) // page + 1
    table, rest = tables(total, page, pages, 5)
    wide = (max(whole) + page - 1) // page
    full, at = np.zeros((batch, wide), np.int32), 0
    for b, n in enumerate(whole):
        k = (n + page - 1) // page
        full[b, :k] = rest[at:at + k]
        at += k
    pre = rest[at:at + (prefix + page - 1) // page].astype(np.int32)
    kp, vp = pools(pages, page, kvh, dim, dt, "token")
    cos, sin = rope_tables(max(whole) + 1, dim)
    ws = workspace(batch, heads, kvh, dim)
    new = lambda n, h, s: randn((n, h, dim), s).to(TYPES[act]).cuda()
    pk, pv = new(prefix, kvh, 1), new(prefix, kvh, 2)
    mk, mv = new(sum(own), kvh, 3), new(sum(own), kvh, 4)
    # the common prompt
    append_call(kp, vp, cuda_i32([prefix]), cuda_i32(pre[None]), None, pk, pv, cuda_i32([0, prefix]), cos, sin, None)
    starts = np.concatenate(([0], np.cumsum(own)))
    t_pos = [prefix + i for n in own for i in range(n)]
    # the sequences' own prompts: their positions follow the prefix, so their angles are looked up from there
    own_starts, d_table = cuda_i32(starts), cuda_i32(table)
    append_call(kp, vp, cuda_i32(own), d_table, None, mk, mv, own_starts, cos[prefix:], sin[prefix:], None)
    # the same, every sequence with the prefix in its own pages
    rows_k = torch.cat([torch.cat((pk, mk[starts[b]:starts[b + 1]])) for b in range(batch)])
    rows_v = torch.cat([torch.cat((pv, mv[starts[b]:starts[b + 1]])) for b in range(batch)])
    d_full = cuda_i32(full)
    append_call(kp, vp, cuda_i32([prefix + n for n in own]), d_full, None, rows_k, rows_v,
                cuda_i32(starts + prefix * np.arange(batch + 1)), cos, sin, None)
    ks, vs = [], []
    for b in range(batch):
        n = prefix + own[b]
        kr, _ = rotated(rows_k[starts[b] + prefix * b:starts[b] + prefix * b + n], cos[:n], sin[:n])
        ks.append(kr.to(dt))
        vs.append(rows_v[starts[b] + prefix * b:starts[b] + prefix * b + n].to(dt))
    lens, d_pre = cuda_i32(own), cuda_i32(pre)
    lens_full = lens + prefix
    c = T.paged_cache(kp, vp)
    p_eps = torch.finfo(dt).eps / 2 if act != "f32" else 0.0
    slack = torch.finfo(dt).eps  # the reference's rounded keys may lie one step off the cache's
    for step in range(steps):
        q, k, v = new(batch, heads, 10 + step), new(batch, kvh, 20 + step), new(batch, kvh, 30 + step)
        lens += 1
        lens_full += 1
        qa, qb = torch.empty_like(q), torch.empty_like(q)
        append_call(kp, vp, lens, d_table, q, k, v, None, cos[prefix:], sin[prefix:], qa)
        append_call(kp, vp, lens_full, d_full, q, k, v, None, cos, sin, qb)
        assert torch.equal(qa, qb)
        oa, ob = torch.zeros_like(q), torch.zeros_like(q)
        ba, bb = T.paged_batch(lens, d_table), T.paged_batch(lens_full, d_full)
        code = T.dtype_code(q)
        T.call("tb_paged_attention_shared", T.byref(c), T.byref(ba), T.ptr(d_pre), prefix, code, T.ptr(qa), heads * dim,
               heads, dim ** -0.5, T.ptr(oa), heads * dim, T.ptr(ws), ws.numel(), T.stream_handle())
        T.call("tb_paged_attention_decode", T.byref(c), T.byref(bb), code, T.ptr(qb), heads * dim, heads, dim ** -0.5,
               T.ptr(ob), heads * dim, T.ptr(ws), ws.numel(), T.stream_handle())
        torch.cuda.synchronize()
        assert T.take_device_errors() == 0
        for b in range(batch):
            pos = prefix + own[b] + step
            ks[b] = torch.cat((ks[b], rotated(k[b][None], cos[pos:pos + 1], sin[pos:pos + 1])[0].to(dt)))
            vs[b] = torch.cat((vs[b], v[b][None].to(dt)))
            want, tol = exact(qa[b], ks[b], vs[b], dim ** -0.5, p_eps)
            mag = (dim ** -0.5) * (qa[b].double().abs().view(kvh, group, dim) @ ks[b].double().abs().permute(1, 2, 0)).max()
            tol = tol + 2 * slack * mag * vs[b].double().abs().max()
            check_rows(oa[b], want, tol, TYPES[act])
            check_rows(ob[b], want, tol, TYPES[act])
