"""The paged key/value cache and the attention that reads it: what is measured.

Three operators of a server that decodes a batch of sequences:
  append   new keys and values into the pages of a paged cache, the position
           rotation of queries and keys applied on the way
           (tb_rope_paged_append)
  decode   one query token per sequence against the keys and values of its
           pages (tb_paged_attention_decode)
  shared   the same for a batch whose sequences begin with one common prefix,
           held once in the cache (tb_paged_attention_shared)

A cache page holds `page` tokens of every key/value head, laid out token by
token ("token": [page, kv_heads, dim]) or head by head ("head": [kv_heads,
page, dim]).  `act` is the type of queries, new keys, new values and outputs,
`cache` that of the pages.  Pages of a sequence are scattered over the pool.

`run` with `own` false is the plain form: elementary torch operations in 32
bits.  With `own` true it makes the library's calls.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


# ------------------------------------------------------------------- cases --

def _case(name, op, act, cache, group, kv_heads, dim, page, layout, batch, low, high, new=0, prefix=0, mix=0):
    """low..high: the range of the sequences' lengths (for `shared` without
    the prefix, for `append` before the call); new: for `append`, the most new
    tokens of a sequence (0: exactly one each); mix: picks the lengths."""
    return {"name": name, "op": op, "act": act, "cache": cache, "group": group, "kv_heads": kv_heads, "dim": dim,
            "page": page, "layout": layout, "batch": batch, "low": low, "high": high, "new": new, "prefix": prefix,
            "mix": mix}


def listed():
    return [
        # One decode step of one sequence of the 1B-shaped model (32 query heads, 8 key/value heads of 64): latency.
        _case("append_step_1", "append", "f32", "f16", 4, 8, 64, 16, "token", 1, 500, 500),
        # The same step for a full batch of a model with heads of 128.
        _case("append_step_256", "append", "bf16", "bf16", 4, 8, 128, 32, "head", 256, 0, 300, mix=1),
        # Prompts of uneven lengths entering the cache behind what their sequences hold already.
        _case("append_prompts_ragged", "append", "f32", "bf16", 4, 8, 64, 16, "token", 16, 0, 200, new=1023, mix=2),
        # A prefill batch: 64 prompts of up to 1024 tokens, 16-bit activations.
        _case("append_prompts_large", "append", "f16", "f16", 4, 8, 128, 64, "token", 64, 0, 0, new=1024, mix=3),
        # One sequence of 511 keys of the 1B-shaped model in a 32-bit cache: latency.
        _case("decode_1_short", "decode", "f32", "f32", 4, 8, 64, 16, "token", 1, 511, 511),
        # A serving batch of the 1B-shaped model with 16-bit pages, lengths up to its prompt plus answer.
        _case("decode_32_ragged", "decode", "f32", "f16", 4, 8, 64, 16, "token", 32, 1, 4096, mix=4),
        # One sequence with a long document.
        _case("decode_1_long", "decode", "bf16", "bf16", 4, 8, 128, 32, "head", 1, 131071, 131071),
        # A large serving batch, uneven lengths up to 8192.
        _case("decode_128_ragged", "decode", "bf16", "bf16", 4, 8, 128, 32, "head", 128, 1, 8192, mix=5),
        # A few sequences behind a system prompt of 1001 tokens, 32-bit cache: latency.
        _case("shared_4_short", "shared", "f32", "f32", 4, 8, 64, 16, "token", 4, 1, 60, prefix=1001, mix=6),
        # A serving batch of the 1B-shaped model behind a prompt of 8192 tokens.
        _case("shared_64", "shared", "f32", "f16", 4, 8, 64, 16, "token", 64, 0, 512, prefix=8192, mix=7),
        # Eight query heads to a key/value head, an odd prefix and an odd batch.
        _case("shared_17_odd", "shared", "f16", "f16", 8, 4, 128, 32, "head", 17, 0, 777, prefix=16387, mix=8),
        # Many samples of one long document: the matrix products bound it.
        _case("shared_128_long", "shared", "bf16", "bf16", 4, 8, 128, 64, "head", 128, 1, 256, prefix=32768, mix=9),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "decode", "shared"])
    act, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    layout = rng.choice(["token", "head"])
    mix = rng.randrange(1 << 30)
    row = kv_heads * dim * SIZES[cache]  # bytes of a token's keys
    if op == "append":
        batch = _log(rng, 1, 256)
        new = rng.choice([0, _log(rng, 1, 4096)])
        most = 200000000 // (kv_heads * dim * (2 * group + 4) * SIZES[act])
        if new:
            new = max(1, min(new, 2 * most // batch))
        high = _log(rng, 1, 512)
        return _case("", op, act, cache, group, kv_heads, dim, page, layout, batch, 0 if new else 1, high, new=new,
                     mix=mix)
    if op == "decode":
        batch = _log(rng, 1, 128)
        high = min(_log(rng, 1, 131072), 400000000 // (row * batch))
        return _case("", op, act, cache, group, kv_heads, dim, page, layout, batch, min(1, high), max(1, high), mix=mix)
    batch = _log(rng, 2, 128)
    high = min(_log(rng, 1, 1024), 100000000 // (row * batch))
    prefix = _log(rng, 16, 32768)
    # no more rows times prefix keys than the largest listed case has
    prefix = max(1, min(prefix, 128 * 32 * 32768 * 128 // (batch * group * kv_heads * dim)))
    return _case("", op, act, cache, group, kv_heads, dim, page, layout, batch, 0, max(1, high), prefix=prefix, mix=mix)


def _lens(case):
    """(held, new): keys each sequence holds before the call, and new tokens.
    Fixed by the case alone, so that its work is known."""
    r = random.Random(case["mix"])
    b = case["batch"]
    held = [r.randint(case["low"], case["high"]) for _ in range(b)]
    if case["op"] == "append":
        new = [r.randint(1, case["new"]) if case["new"] else 1 for _ in range(b)]
        if case["new"] and b >= 8:
            new[1] = 0  # a sequence that takes no token in this call
            new[2] = 1
        return held, new
    if b >= 8 and case["low"] < case["high"]:
        held[1] = 0  # an empty sequence, and one with a single key
        held[2] = 1
    return held, [0] * b


def work(case):
    heads = case["group"] * case["kv_heads"]
    act, size, dim = SIZES[case["act"]], SIZES[case["cache"]], case["dim"]
    row = case["kv_heads"] * dim
    held, new = _lens(case)
    b, page = case["batch"], case["page"]
    if case["op"] == "append":
        t = sum(new)
        pages = sum((h + n + page - 1) // page - h // page for h, n in zip(held, new) if n)
        angles = len({p for h, n in zip(held, new) for p in range(h, h + n)}) * dim * 4  # cos and sin, dim / 2 each
        moved = t * (2 * heads * dim * act + 2 * row * act + 2 * row * size) + angles + 4 * (pages + 2 * b)
        return {"bytes": moved, "flops": 3 * t * (heads * dim + row)}
    tokens = sum(held)
    pages = sum((h + page - 1) // page for h in held) + (case["prefix"] + page - 1) // page
    moved = 2 * (tokens + case["prefix"]) * row * size + 2 * b * heads * dim * act + 4 * (pages + b)
    return {"bytes": moved, "flops": 4 * heads * dim * (tokens + b * case["prefix"])}


# ------------------------------------------------------------------- inputs --

def _pool(case, pages, gen):
    """A pool of `pages` pages with values in it; returned as [pages, page,
    kv_heads, dim] whatever the layout in memory."""
    p, k, d = case["page"], case["kv_heads"], case["dim"]
    shape = (pages, p, k, d) if case["layout"] == "token" else (pages, k, p, d)
    t = torch.empty(shape, dtype=DTYPES[case["cache"]], device=DEV)
    for i in range(0, pages, 4096):  # in parts: the 32-bit numbers of a large pool take no room at once
        part = t[i:i + 4096]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    return t if case["layout"] == "token" else t.permute(0, 2, 1, 3)


def _rows(n, width, case, gen):
    return torch.randn((n, width), generator=gen, device=DEV).to(DTYPES[case["act"]])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    host = random.Random(seed)
    b, page, dim = case["batch"], case["page"], case["dim"]
    heads = case["group"] * case["kv_heads"]
    held, new = _lens(case)
    total = [h + n for h, n in zip(held, new)]
    need = [(t + page - 1) // page for t in total]
    prefix_pages = (case["prefix"] + page - 1) // page
    pages = sum(need) + prefix_pages + 3
    order = list(range(pages))
    host.shuffle(order)
    max_pages = max(max(need), 1)
    table = torch.zeros((b, max_pages), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    st = {"case": case, "held": held, "new": new, "k": _pool(case, pages, gen), "v": _pool(case, pages, gen),
          "table": table.to(DEV), "lens": torch.tensor(total, dtype=torch.int32).to(DEV)}
    if case["op"] == "append":
        tokens = sum(new)
        st["q"] = _rows(tokens, heads * dim, case, gen)
        # the output of one fused projection: a token's keys and values side by side
        st["kv"] = _rows(tokens, 2 * case["kv_heads"] * dim, case, gen)
        st["q_out"] = torch.zeros((tokens, heads * dim), dtype=DTYPES[case["act"]], device=DEV)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        st["starts"] = torch.tensor(starts, dtype=torch.int32).to(DEV) if case["new"] else None
        far = max(total)
        angle = torch.arange(far, dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) * 2 / dim))[None, :]
        st["cos"], st["sin"] = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
        # where each token goes: its sequence and its position there
        seq = [i for i, n in enumerate(new) for _ in range(n)]
        pos = [h + j for h, n in zip(held, new) for j in range(n)]
        st["seq"], st["pos"] = torch.tensor(seq).to(DEV), torch.tensor(pos).to(DEV)
    else:
        st["q"] = _rows(b, heads * dim, case, gen)
        st["out"] = torch.zeros_like(st["q"])
        st["scale"] = dim ** -0.5
        st["prefix_table"] = torch.tensor(order[at:at + prefix_pages], dtype=torch.int32).to(DEV)
    if own:
        _library_state(st)
    return st


# --------------------------------------------------------- the library's calls --

def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "turbo.cpp_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import turbo_b200
    return turbo_b200


def _library_state(st):
    """The handles that a server keeps: the cache's and the batch's
    descriptions, and a workspace."""
    T, case = _library(), st["case"]
    st["T"] = T
    st["paged"] = T.paged_cache(st["k"], st["v"])
    st["batch"] = T.paged_batch(st["lens"], st["table"])
    if case["op"] != "append":
        n = ctypes.c_size_t(0)
        T.call("tb_paged_attention_workspace_bytes", case["batch"], case["group"] * case["kv_heads"], case["kv_heads"],
               case["dim"], ctypes.byref(n))
        st["workspace"] = torch.zeros(n.value, dtype=torch.uint8, device=DEV)


def _run_library(st):
    T, case = st["T"], st["case"]
    heads, dim = case["group"] * case["kv_heads"], case["dim"]
    act = T.dtype_code(st["q"])
    stream = T.stream_handle()
    if case["op"] == "append":
        q, kv = st["q"], st["kv"]
        k_at, width = kv.data_ptr(), kv.shape[1]
        v_at = k_at + width // 2 * kv.element_size()
        starts = st["starts"].data_ptr() if st["starts"] is not None else None
        T.call("tb_rope_paged_append", T.byref(st["paged"]), T.byref(st["batch"]), act, q.data_ptr(), heads * dim,
               k_at, width, v_at, width, q.shape[0], heads, starts, st["cos"].data_ptr(), st["sin"].data_ptr(),
               st["cos"].shape[0], st["q_out"].data_ptr(), heads * dim, stream)
        return st["q_out"], st["k"], st["v"]
    q, out, ws = st["q"], st["out"], st["workspace"]
    if case["op"] == "decode":
        T.call("tb_paged_attention_decode", T.byref(st["paged"]), T.byref(st["batch"]), act, q.data_ptr(), heads * dim,
               heads, st["scale"], out.data_ptr(), heads * dim, ws.data_ptr(), ws.numel(), stream)
    else:
        T.call("tb_paged_attention_shared", T.byref(st["paged"]), T.byref(st["batch"]), st["prefix_table"].data_ptr(),
               case["prefix"], act, q.data_ptr(), heads * dim, heads, st["scale"], out.data_ptr(), heads * dim,
               ws.data_ptr(), ws.numel(), stream)
    return out


# ------------------------------------------------------------- the plain form --

def _rotate(x, cos, sin):
    """x [tokens, n, dim] in 32 bits; the first half of dim paired with the second."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def _plain_append(st):
    case = st["case"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    heads = case["group"] * kv
    q, x = st["q"].float().view(-1, heads, dim), st["kv"].float().view(-1, 2 * kv, dim)
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    where = st["table"][st["seq"], st["pos"] // page].long(), st["pos"] % page
    st["q_out"].copy_(_rotate(q, cos, sin).view(-1, heads * dim))
    st["k"][where] = _rotate(x[:, :kv], cos, sin).to(st["k"].dtype)
    st["v"][where] = x[:, kv:].to(st["v"].dtype)
    return st["q_out"], st["k"], st["v"]


def _gather(pool, ids, n):
    """The first n tokens of the pages `ids`, [kv_heads, n, dim] in 32 bits."""
    t = pool[ids.long()]
    return t.reshape(-1, t.shape[2], t.shape[3])[:n].float().transpose(0, 1)


def _attend(q, k, v, scale):
    """q [kv_heads, rows, dim]: softmax(scale q k^T) v over all keys."""
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    e = torch.exp(s - s.max(-1, keepdim=True).values)
    return torch.matmul(e, v) / e.sum(-1, keepdim=True)


def _plain_attention(st):
    case = st["case"]
    kv, g, dim, page = case["kv_heads"], case["group"], case["dim"], case["page"]
    q = st["q"].float().view(-1, kv, g, dim)
    n = case["prefix"]
    if n:
        pk, pv = _gather(st["k"], st["prefix_table"], n), _gather(st["v"], st["prefix_table"], n)
    out = torch.zeros_like(q)
    for b, length in enumerate(st["held"]):
        if length:
            ids = st["table"][b, :(length + page - 1) // page]
            k, v = _gather(st["k"], ids, length), _gather(st["v"], ids, length)
            if n:
                k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
        elif n:
            k, v = pk, pv
        else:
            continue  # no key: the row stays zero
        out[b] = _attend(q[b], k, v, st["scale"])
    st["out"].copy_(out.view(st["out"].shape))
    return st["out"]


def run(state):
    if own:
        return _run_library(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attention(state)


# --------------------------------------------------- the definition in 64 bits --

def exact(case, seed):
    st = prepare(case, seed)
    kv, g, dim, page = case["kv_heads"], case["group"], case["dim"], case["page"]
    heads = g * kv
    if case["op"] == "append":
        half = dim // 2
        x = st["kv"].double()
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"]]  # [tokens, half]

        def rotated(part):
            part = part.reshape(part.shape[0], -1, 2, half)
            z = torch.complex(part[:, :, 0], part[:, :, 1]) * turn[:, None]
            return torch.stack((z.real, z.imag), 2).reshape(part.shape[0], -1, dim)

        q, k = rotated(st["q"].double()), rotated(x[:, :kv * dim])
        v = x[:, kv * dim:].reshape(-1, kv, dim)
        pools = []
        for pool, rows in ((st["k"], k), (st["v"], v)):
            full = pool.double().reshape(-1, kv, dim)
            full[st["table"].long()[st["seq"], st["pos"] // page] * page + st["pos"] % page] = rows
            pools.append(full.view(pool.shape))
        return q.reshape(-1, heads * dim), pools[0], pools[1]
    out = torch.zeros((case["batch"], heads, dim), dtype=torch.float64, device=DEV)
    q = st["q"].double().view(case["batch"], heads, dim)
    prefix = torch.arange(case["prefix"], device=DEV)
    first = st["prefix_table"].long()[prefix // page]
    for h in range(kv):  # one key/value head at a time
        mine = slice(h * g, (h + 1) * g)
        pk, pv = st["k"][first, prefix % page, h].double(), st["v"][first, prefix % page, h].double()
        for b, length in enumerate(st["held"]):
            if length + case["prefix"] == 0:
                continue
            t = torch.arange(length, device=DEV)
            ids = st["table"][b].long()[t // page]
            k = torch.cat((pk, st["k"][ids, t % page, h].double()))
            v = torch.cat((pv, st["v"][ids, t % page, h].double()))
            p = torch.softmax(st["scale"] * (q[b, mine] @ k.T), -1)
            out[b, mine] = p @ v
    return out.view(case["batch"], heads * dim)
