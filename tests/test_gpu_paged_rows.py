"""Attention over the paged cache, held to what single keys and single bits add.

Tolerances as in test_gpu_paged.py, with these for 16-bit activations: a
probability is two parts of the cache's type, each to nearest, so it is off by
at most (eps/2)^2 of itself; a tensor core's accumulator is read out after 512
steps at most, each off by at most one unit of 2^-23."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import turbo_b200 as T  # noqa: E402
from test_gpu_paged import (PAIRS, SHARED, TYPES, Batch, _no_errors_left, check_rows, cuda_i32, exact,  # noqa: E402,F401
                            get_rows, put_rows, randn, workspace)

STEPS = 512 * 2 ** -23


def rows_of(x, out, lens=None):
    """Each sequence's keys and values (the prefix first) and its output rows."""
    pk, pv = (get_rows(p, x.prefix, x.page, x.n_prefix) for p in (x.kp, x.vp))
    for b, n in enumerate(x.lens if lens is None else lens):
        k, v = (torch.cat((y, get_rows(p, x.table[b], x.page, n))) for y, p in ((pk, x.kp), (pv, x.vp)))
        yield b, k, v, out[b, :x.heads * x.dim].view(x.heads, x.dim)


def check_two_parts(x, out):
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    p_eps = (torch.finfo(x.ct).eps / 2) ** 2
    off, least = [], []
    for b, k, v, got in rows_of(x, out):
        want, tol = exact(x.rows()[b], k, v, x.scale, p_eps)
        off.append(got.double() - want)
        least.append(want.to(x.act).double() - want)
        if k.shape[0]:  # the steps, relative to sum p |v|
            tol = tol + exact(x.rows()[b], k, v.abs(), x.scale)[0] * STEPS
        check_rows(got, want, tol, x.act)
    # The roundings of parts are independent of each other, so that they add up like the outputs themselves and stay
    # below (eps/2)^2 of them; the steps take up to 2^-15 of them off.  Beside the output's own rounding, an eighth of a
    # step of fp16 and 0.3 of it in the mean, that is a few per cent.  (One part: 39 % more.)
    assert torch.cat(off).norm() <= 1.1 * torch.cat(least).norm()


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [1, 32, 33, 128, 129, 300])
def test_16_bit_activations_keep_two_parts(rows, dim, act):
    """However many rows a batch has, and whichever kernel reads its prefix."""
    for prefix in (259, 643, 5000):
        x = Batch(act, act, 1, 1, dim, 16, "token", [b % 2 for b in range(rows)], prefix, seed=rows)
        check_two_parts(x, x.run(shared=True))


@pytest.mark.parametrize("lens", [[0, 3, 64, 65, 200], [5, 0]])
@pytest.mark.parametrize("prefix", [1, 65, 500])
@pytest.mark.parametrize("act,dim", [("f16", 64), ("bf16", 128)])
def test_16_bit_activations_behind_a_short_prefix_keep_two_parts(act, dim, prefix, lens):
    x = Batch(act, act, 4, 2, dim, 16, "head", lens * 40, prefix, seed=prefix)
    check_two_parts(x, x.run(shared=True))


@pytest.mark.parametrize("act,dim", [("f16", 64), ("f16", 128), ("bf16", 64)])
def test_many_rows_behind_a_very_long_prefix(act, dim):
    """So many rows that one CTA takes 2^20 keys (one page, again and again) by itself."""
    page, times, group, batch = 1024, 1024, 64, 592
    kp, vp = (torch.zeros((1, page, 1, dim), dtype=TYPES[act], device="cuda") for _ in range(2))
    kp[0] = randn((page, 1, dim), 1).cuda().to(TYPES[act])
    vp[0] = (1 + torch.rand((page, 1, dim), generator=torch.Generator().manual_seed(2))).cuda().to(TYPES[act])
    q = randn((batch, group * dim), 3, 0.25).cuda().to(TYPES[act])
    lens, table = cuda_i32([0] * batch), cuda_i32(np.zeros((batch, 1)))
    prefix = cuda_i32([0] * times)
    ws, out = workspace(batch, group, 1, dim), torch.zeros_like(q)
    c, b = T.paged_cache(kp, vp), T.paged_batch(lens, table)
    scale = dim ** -0.5
    T.call("tb_paged_attention_shared", T.byref(c), T.byref(b), T.ptr(prefix), page * times, T.dtype_code(q), T.ptr(q),
           group * dim, group, scale, T.ptr(out), group * dim, T.ptr(ws), ws.numel(), T.stream_handle())
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    rows = q.view(-1, dim)  # equal keys: the softmax over one page is the softmax over all of them
    want, tol = exact(rows, kp[0], vp[0], scale, (torch.finfo(TYPES[act]).eps / 2) ** 2)
    # read-outs: 2^20 keys are 16384 tiles, 64 at a time added in fp32
    check_rows(out.view(-1, dim), want, tol + want * (STEPS + 16384 / 64 * 2 ** -24), TYPES[act])


def test_rows_of_a_wider_table():
    x = Batch("f32", "f16", 4, 2, 64, 16, "token", [100, 0, 3, 40], seed=2)
    want = x.run().clone()
    wide = torch.full((4, x.table.shape[1] + 5), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + x.table.shape[1]] = x.d_table
    x.batch = T.paged_batch(x.d_lens, wide[:, 2:2 + x.table.shape[1]])
    assert torch.equal(x.run(), want)
    x.check(want)


def run_out(x, shared):
    """A call whose waits all give up: it ends, says so, and leaves the context and what lies beside its rows alone."""
    want = x.run(shared=shared)
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    T.call("tb_set_wait_limit_ns", 0)
    try:
        out = x.run(shared=shared)
        torch.cuda.synchronize()
    finally:
        T.call("tb_set_wait_limit_ns", 2000000000)
    assert T.take_device_errors() == 1
    assert (out[:, x.heads * x.dim:] == 9.0).all()
    x.ws.zero_()
    assert torch.equal(x.run(shared=shared), want)
    x.check(want)


@pytest.mark.parametrize("act,ct,group,kvh,dim,lens,prefix", [
    ("f32", "f32", 1, 1, 64, [5], 0),
    ("f32", "f16", 4, 2, 64, [3000, 1, 0, 700], 0),       # long items over many CTAs
    ("bf16", "bf16", 4, 8, 128, [300] * 200, 0),          # many short ones per CTA
    ("f32", "bf16", 33, 1, 64, [2000, 64, 5], 0),
    ("f16", "f16", 4, 2, 64, [0, 65, 3] * 40, 200),       # a short prefix
    ("f32", "f32", 4, 8, 64, [1, 60, 0, 33], 1001),       # few rows: joined by the kernel of their own keys
    ("f32", "f16", 4, 2, 128, [300, 5], 9000),            # few rows, joined by a kernel of its own
    ("f32", "f32", 4, 2, 64, [40] * 70, 2000),
])
def test_waits_that_run_out(act, ct, group, kvh, dim, lens, prefix):
    run_out(Batch(act, ct, group, kvh, dim, 16, "token", lens, prefix, seed=3), prefix > 0)


@pytest.mark.parametrize("act,ct,group,kvh,dim,batch,prefix", [
    ("bf16", "bf16", 4, 8, 128, 100, 9000),  # two row tiles a CTA
    ("f16", "f16", 4, 2, 64, 20, 3000),      # one, alternate keys
    ("f32", "f16", 4, 8, 64, 64, 5000),
    ("f32", "f16", 4, 1, 128, 64, 700),
    ("f32", "bf16", 4, 2, 128, 64, 2000),    # one buffer of scores
])
def test_waits_that_run_out_on_tcgen05(act, ct, group, kvh, dim, batch, prefix):
    run_out(Batch(act, ct, group, kvh, dim, 16, "token", [b % 3 for b in range(batch)], prefix, seed=4), True)


@pytest.mark.parametrize("act,ct,group,kvh,batch,prefix,room", [
    ("f16", "f16", 4, 2, 20, 1500, 8),     # 33 and more rows: the prefix on tcgen05
    ("bf16", "bf16", 4, 8, 80, 3000, 20),
    ("f32", "f16", 2, 2, 9, 4000, 30),     # fewer
    ("f32", "f32", 4, 2, 3, 900, 2),       # few short sequences: joined by the kernel of their own keys
    ("f32", "f32", 4, 2, 30, 100, 9),      # a short prefix
])
def test_steps_in_one_stream_without_a_host_wait(act, ct, group, kvh, batch, prefix, room):
    """Each step changes queries and lengths in place, appends, and attends; nothing waits for the host in between."""
    steps, dim, page = 24, 64, 16
    own = [b % 5 for b in range(batch)]
    x = Batch(act, ct, group, kvh, dim, page, "token", [n + steps + room for n in own], prefix, seed=batch)
    new = [[randn((batch, h, dim), 100 * s + i).to(TYPES[act]).cuda() for i, h in enumerate((group * kvh, kvh, kvh))]
           for s in range(steps)]
    start = cuda_i32(own)
    q = torch.empty_like(new[0][0])
    cos, sin = torch.ones((64, dim // 2), device="cuda"), torch.zeros((64, dim // 2), device="cuda")
    width = group * kvh * dim

    def chain(wait):
        sync = torch.cuda.synchronize if wait else lambda: None
        outs = [torch.zeros_like(q) for _ in range(steps)]
        x.d_lens.copy_(start)
        sync()
        for s in range(steps):
            x.d_lens += 1
            sync()
            q.copy_(new[s][0])
            sync()
            T.call("tb_rope_paged_append", T.byref(x.cache), T.byref(x.batch), T.dtype_code(q), T.ptr(q), width,
                   T.ptr(new[s][1]), kvh * dim, T.ptr(new[s][2]), kvh * dim, batch, group * kvh, None, T.ptr(cos),
                   T.ptr(sin), 64, T.ptr(q), width, T.stream_handle())
            sync()
            T.call("tb_paged_attention_shared", T.byref(x.cache), T.byref(x.batch), T.ptr(x.d_prefix), prefix,
                   T.dtype_code(q), T.ptr(q), width, group * kvh, x.scale, T.ptr(outs[s]), width, T.ptr(x.ws),
                   x.ws.numel(), T.stream_handle())
            sync()
        torch.cuda.synchronize()
        assert T.take_device_errors() == 0
        return outs

    want = chain(True)
    assert not torch.equal(want[0], want[1])
    for _ in range(5):
        for a, b in zip(chain(False), want):
            assert torch.equal(a, b)


def test_append_lowest_length():
    """A length so far below zero that the positions of a long prompt would come out above it."""
    tokens, page, pages = (1 << 20) + 5000, 1 << 20, 2047
    kp, vp = (torch.full((1, page, 1, 16), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = torch.ones((tokens, 1, 16), dtype=torch.float16, device="cuda")
    q_out = torch.full_like(rows, 5.0)
    starts, lens, table = cuda_i32([0, tokens]), cuda_i32([-2 ** 31]), cuda_i32(np.zeros((1, pages)))
    c, b = T.paged_cache(kp, vp), T.paged_batch(lens, table)
    T.call("tb_rope_paged_append", T.byref(c), T.byref(b), T.F16, T.ptr(rows), 16, T.ptr(rows), 16, T.ptr(rows), 16,
           tokens, 1, T.ptr(starts), None, None, 0, T.ptr(q_out), 16, T.stream_handle())
    torch.cuda.synchronize()
    assert T.take_device_errors() == 2
    assert (kp == 7.0).all() and (vp == 7.0).all() and (q_out == 5.0).all()


def selective(x):
    """Row r of a key/value head's rows takes the keys t with (t + head) % dim == r % dim, each with the same weight, and
    key t's value is a one in column (t // dim) % dim: an output counts a share of the keys, a dim-th of a dim-th of
    them, and one left out or taken twice changes it by one of few.  With dim rows every key is counted, with fewer some of
    every dim keys in a row."""
    c = 64.0  # c c scale > 360: the other keys' weights are 0 in 32 bits
    eye = torch.eye(x.dim, device="cuda")
    head = torch.arange(x.kvh, device="cuda")

    def put(table_row, n, first):
        t = first + torch.arange(n, device="cuda")
        put_rows(x.kp, table_row, x.page, c * eye[(t[:, None] + head) % x.dim])
        put_rows(x.vp, table_row, x.page, eye[(t // x.dim) % x.dim][:, None].expand(n, x.kvh, x.dim))

    put(x.prefix, x.n_prefix, 0)
    for b, n in enumerate(x.lens):
        put(x.table[b], n, x.n_prefix)
    group = x.heads // x.kvh
    r = torch.arange(len(x.lens) * group, device="cuda").view(len(x.lens), 1, group)
    x.rows().copy_(c * eye[r.expand(len(x.lens), x.kvh, group).reshape(len(x.lens), x.heads) % x.dim])


def check_counts(x, out):
    torch.cuda.synchronize()
    assert T.take_device_errors() == 0
    for b, k, v, got in rows_of(x, out):
        if k.shape[0] == 0:
            assert (got == 0).all()
            continue
        # The taken keys' weights are the same number, off by (eps/2)^2 once rounded to parts (bf16 2^-16); the sums by
        # STEPS = 2^-14, or by one unit of 2^-24 for each of (keys / 8 + 200) additions.
        want, _ = exact(x.rows()[b], k, v, x.scale)
        rel = 2 ** -16 + STEPS + (k.shape[0] / 8 + 200) * 2 ** -24
        check_rows(got, want, want * rel, x.act)
        # one key more or less would be seen
        assert 1 / (k.shape[0] // x.dim ** 2 + 1) > 2 * (rel + torch.finfo(x.act).eps)


@pytest.mark.parametrize("case", range(len(SHARED)))
def test_every_key_behind_a_prefix_counts_once(case):
    *a, lens, prefix = SHARED[case]
    x = Batch(*a, lens, prefix, seed=case)
    selective(x)
    check_counts(x, x.run(shared=True))


@pytest.mark.parametrize("act,ct", PAIRS)
@pytest.mark.parametrize("group,kvh,dim,lens", [
    (4, 8, 64, [0, 1, 16, 63, 64, 65, 700, 4096, 4097]),
    (16, 2, 128, [12000, 3, 0, 130]),
    (33, 1, 64, [9000, 257, 40]),
    (2, 1, 128, [300] * 700),
])
def test_every_key_of_a_batch_counts_once(group, kvh, dim, lens, act, ct):
    x = Batch(act, ct, group, kvh, dim, 16, "token", lens, seed=group)
    selective(x)
    check_counts(x, x.run())


@pytest.mark.parametrize("act,ct,group,kvh,batch,prefix,room", [
    ("f16", "f16", 4, 2, 20, 1500, 8),
    ("f32", "f32", 4, 2, 3, 900, 2),
    ("bf16", "bf16", 2, 2, 9, 4000, 30),
    ("f32", "f16", 4, 2, 5, 0, 40),
])
def test_a_captured_step_follows_its_inputs(act, ct, group, kvh, batch, prefix, room):
    """One captured step, replayed while queries and lengths change in place ahead of it, without a host wait."""
    steps, dim = 20, 128
    x = Batch(act, ct, group, kvh, dim, 16, "head", [b % 7 + steps + room for b in range(batch)], prefix, seed=batch)
    qs = [randn(x.q.shape, 50 + s).to(x.act).cuda() for s in range(steps)]
    start = cuda_i32([b % 7 for b in range(batch)])
    out = torch.zeros((batch, x.heads * dim + 8), dtype=x.act, device="cuda")
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    T.call("tb_stream_create", ctypes.byref(s))
    stream = torch.cuda.ExternalStream(s.value)
    torch.cuda.synchronize()
    T.call("tb_capture_begin", s)
    x.run(shared=True, out=out, stream=stream)
    T.call("tb_capture_end", s, ctypes.byref(g))

    def replay(wait):
        sync = torch.cuda.synchronize if wait else lambda: None
        outs = [torch.zeros_like(out) for _ in range(steps)]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            x.d_lens.copy_(start)
            for i in range(steps):
                x.d_lens += 1
                x.q.copy_(qs[i])
                sync()
                T.call("tb_graph_launch", g, s)
                sync()
                outs[i].copy_(out)
        torch.cuda.synchronize()
        assert T.take_device_errors() == 0
        return outs

    want = replay(True)
    assert not torch.equal(want[0], want[1])
    for _ in range(5):
        for a, b in zip(replay(False), want):
            assert torch.equal(a, b)
    T.call("tb_graph_destroy", g)
    T.call("tb_stream_destroy", s)


@pytest.mark.parametrize("act,ct,group,kvh,dim,lens,prefix", [
    ("f32", "f16", 4, 2, 64, [3000, 1, 0, 700], 0),
    ("bf16", "bf16", 4, 8, 128, [300] * 200, 0),
    ("f32", "f32", 4, 8, 64, [1, 60, 0, 33], 1001),
    ("bf16", "bf16", 4, 8, 128, [3, 70] * 50, 9000),
    ("f16", "f16", 4, 2, 64, [5] * 20, 3000),
    ("f32", "bf16", 4, 2, 128, [5] * 64, 2000),
])
def test_waits_that_may_run_out(act, ct, group, kvh, dim, lens, prefix):
    """The shortest limit there is: some waits end in time and some do not."""
    x = Batch(act, ct, group, kvh, dim, 16, "token", lens, prefix, seed=6)
    want = x.run(shared=prefix > 0)
    torch.cuda.synchronize()
    T.call("tb_set_wait_limit_ns", 1)
    try:
        for _ in range(3):
            out = x.run(shared=prefix > 0)
            torch.cuda.synchronize()
            assert T.take_device_errors() in (0, 1)
            assert (out[:, x.heads * x.dim:] == 9.0).all()
            x.ws.zero_()
    finally:
        T.call("tb_set_wait_limit_ns", 2000000000)
    assert torch.equal(x.run(shared=prefix > 0), want)
    x.check(want)
