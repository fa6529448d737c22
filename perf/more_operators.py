"""Operators around a key-value cache: rotary positions, writing to and reading from a paged cache, attention of new tokens over it.

`listed()` names the calls by which they are judged, `draw()` gives further ones from the same ranges.  `run()` makes a call: through
the public entry points of `cutile_b200` where `own` is true, else in plain torch operations in f32 (angles in f64).  `exact()` gives the
same outputs in f64 from the definitions.  Slots and page tables are 1-based and 0 stands for "none", as everywhere in the package.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "int8": 1}
LARGEST = {"e4m3": 448.0, "int8": 127.0}  # magnitude of an 8-bit code


def listed():
    return [
        # Queries and keys of one decoding step of a few sequences. Latency counts.
        dict(name="rope_step", kind="rope", dtype="bf16", tokens=8, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             first=4000, scaling="none", train=False),
        # A prompt deep inside a long context: interleaved pairs, a part of the head, frequencies scaled for the length.
        dict(name="rope_prompt", kind="rope", dtype="f16", tokens=4001, heads=16, kv_heads=16, dim=64, rotary=32, interleaved=True,
             first=900000, scaling="parts", train=False),
        # A training step, forward and backward.
        dict(name="rope_train", kind="rope", dtype="bf16", tokens=16384, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             first=0, scaling="none", train=True),
        # One decoding step of a full batch: rotated and written in 16 bits.
        dict(name="cache_step", kind="cache", dtype="bf16", store="bf16", batch=64, longest=256, new=1, heads=32, kv_heads=8, dim=128,
             page=16, rotary=128, interleaved=False, read=False),
        # Prompts of a few sequences, rotated, stored in 8 bits, and read back for the attention of the next chunk.
        dict(name="cache_prompt", kind="cache", dtype="bf16", store="e4m3", batch=4, longest=4096, new=4096, heads=32, kv_heads=8, dim=128,
             page=64, rotary=128, interleaved=False, read=True),
        # A further chunk of long prompts, behind what is in the cache already; pages of a size that the lengths do not fit.
        dict(name="cache_chunk", kind="cache", dtype="f16", store="int8", batch=7, longest=12001, new=500, heads=16, kv_heads=16, dim=64,
             page=32, rotary=64, interleaved=True, read=True),
        # A few short conversations. Latency counts.
        dict(name="attend_few", kind="attend", dtype="bf16", store="bf16", batch=4, longest=500, idle=0, heads=32, kv_heads=8, dim=128,
             page=16, lse=False),
        # One very long context.
        dict(name="attend_long", kind="attend", dtype="f16", store="f16", batch=1, longest=131072, idle=0, heads=32, kv_heads=8, dim=128,
             page=64, lse=False),
        # A full batch of unlike lengths, some places of it unused; the log of the sums for a join with another part.
        dict(name="attend_batch", kind="attend", dtype="bf16", store="bf16", batch=64, longest=8000, idle=3, heads=64, kv_heads=8, dim=128,
             page=32, lse=True),
        # A large batch over a cache in 8 bits.
        dict(name="attend_8bit", kind="attend", dtype="bf16", store="e4m3", batch=128, longest=4096, idle=0, heads=32, kv_heads=8, dim=128,
             page=16, lse=False),
        # Small heads, each with keys of its own, in 8-bit integers.
        dict(name="attend_heads", kind="attend", dtype="f16", store="int8", batch=32, longest=2001, idle=0, heads=16, kv_heads=16, dim=64,
             page=16, lse=False),
        # A layer's decoding step: rotate, write, attend.
        dict(name="step", kind="step", dtype="bf16", store="bf16", batch=32, longest=4000, new=1, heads=32, kv_heads=8, dim=128, page=16,
             rotary=128, interleaved=False, read=False),
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_ELEMENTS = 59 * 8000 // 2 * 8 * 128  # of keys in a cache: those of the largest listed case


def _draw_rope(rng):
    dim = rng.choice((64, 80, 96, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
    rotary = rng.choice((dim, dim, dim // 2, dim // 4))
    dtype = rng.choice(("f32", "f16", "bf16"))
    tokens = max(1, min(_log(rng, 1, 16384), 16384 * 40 * 128 * 2 // ((heads + kv_heads) * dim * BYTES[dtype])))
    return dict(kind="rope", dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                interleaved=rng.random() < 0.5, first=_log(rng, 1, 1000000), scaling=rng.choice(("none", "linear", "base", "parts")),
                train=rng.random() < 0.5)


def _draw_heads(rng):
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    return dict(dtype=rng.choice(("f16", "bf16")), heads=kv_heads * rng.choice((1, 2, 4, 5, 7, 8, 16)), kv_heads=kv_heads,
                dim=rng.choice((64, 128)), page=rng.choice((16, 32, 64, 128, 256)))


def _longest(rng, c, batch, least, most):
    return max(least, min(_log(rng, least, most), 2 * _MOST_ELEMENTS // (c["kv_heads"] * c["dim"] * (batch + 1))))


def _draw_cache(rng, kind="cache"):
    c = _draw_heads(rng)
    batch = _log(rng, 1, 128)
    read = kind == "cache" and rng.random() < 0.7
    new = 1 if kind == "step" or rng.random() < 0.3 else _log(rng, 1, 4096)
    longest = _longest(rng, c, batch * (4 if read else 1), 1, 16384)
    new = min(new, longest, max(1, 16384 * 24 // (batch * (c["heads"] + 2 * c["kv_heads"]))))
    return dict(c, kind=kind, store=rng.choice((c["dtype"], "e4m3", "int8")) if read else c["dtype"], batch=batch, longest=longest, new=new,
                rotary=rng.choice((c["dim"], c["dim"], c["dim"] // 2, 0)) if kind == "cache" else c["dim"],
                interleaved=rng.random() < 0.5, read=read)


def _draw_attend(rng):
    c = _draw_heads(rng)
    batch = _log(rng, 1, 256)
    return dict(c, kind="attend", store=rng.choice((c["dtype"], "e4m3", "int8")), batch=batch, longest=_longest(rng, c, batch, 1, 131072),
                idle=rng.choice((0, 0, batch // 8)), lse=rng.random() < 0.5)


def draw(rng):
    return rng.choice((_draw_rope, _draw_cache, _draw_attend, _draw_attend, lambda r: _draw_cache(r, "step")))(rng)


# ------------------------------------------------------------------ shared
def _package():
    path = os.path.abspath("cutile.jl_b200")  # the package of the tree that is the working folder
    if path not in sys.path:
        sys.path.insert(0, path)
    import cutile_b200
    return cutile_b200


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _lengths(c):
    """Lengths of the sequences, spread evenly up to the longest, in an order of chance; the places without a sequence have 0."""
    batch, idle = c["batch"], c.get("idle", 0)
    live = batch - idle
    lengths = [0] * idle + [max(1, c["longest"] * (i + 1) // live) for i in range(live)]
    random.Random(batch * 7 + c["longest"]).shuffle(lengths)
    return lengths


def _frequencies(rotary, scaling):
    f = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if scaling == "linear":
        f = f / 4
    elif scaling == "base":
        f = (10000.0 * 8 ** (rotary / max(rotary - 2, 1))) ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    elif scaling == "parts":  # as it is where a turn is short beside the original length, by the factor where it is long
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f.cuda()


def _codes(x, store):
    """Codes and scales of rows in 8 bits: the row's largest magnitude gets the largest code."""
    peak = x.abs().amax(-1)
    live = peak >= 2.0 ** -100
    code = torch.where(live[..., None], x * LARGEST[store] / peak[..., None], 0.0).clamp(-LARGEST[store], LARGEST[store])
    return (code.round() if store == "int8" else code).to(DTYPES[store]), torch.where(live, peak / LARGEST[store], 0.0)


def _fill(g, c, pages):
    """One of the two sides of a cache: pages [pages, kv_heads, page, dim], and scales with 8 bits."""
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    x = _normal(g, *shape)
    if c["store"] not in LARGEST:
        return x.to(DTYPES[c["store"]]), None
    x.mul_(torch.exp(0.5 * _normal(g, *shape[:3]))[..., None])
    return _codes(x, c["store"])


def _prepare_cache(c, g):
    """A cache with its page table: pages in an order of chance, a spare one for every sixteen."""
    lengths = _lengths(c)
    used = [-(-n // c["page"]) for n in lengths]
    width = -(-c["longest"] // c["page"])
    pages = sum(used) + sum(used) // 16 + 1
    order = (torch.randperm(pages, device="cuda", generator=g) + 1).int()
    used = torch.tensor(used, device="cuda")
    column = torch.arange(width, device="cuda")
    at = (torch.cumsum(used, 0) - used)[:, None] + column[None]
    table = torch.where(column[None] < used[:, None], order[at.clamp(max=pages - 1)], 0)
    k, ks = _fill(g, c, pages)
    v, vs = _fill(g, c, pages)
    return dict(k=k, v=v, ks=ks, vs=vs, table=table.contiguous(), lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32))


def _own_cache(s):
    return _package().kvcache.KvCache(s["k"], s["v"], s["ks"], s["vs"])


def _rotated(x, angle, interleaved, scale=1.0):
    """Rows [tokens, heads, dim] rotated by angles [tokens, pairs]: in the precision of x, cosines from f64."""
    pairs = angle.shape[1]
    cos, sin = ((t * scale).to(x.dtype)[:, None] for t in (torch.cos(angle), torch.sin(angle)))
    a, b = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., 2 * pairs:]), -1)


# ------------------------------------------------------------------ rotary positions
ATTENTION_FACTOR = 1.2  # of scaled frequencies


def _split(x, c, v=True):
    """q, k and v of a projection that makes them side by side."""
    n, h, kv, d = x.shape[0], c["heads"], c["kv_heads"], c["dim"]
    return x[:, :h * d].view(n, h, d), x[:, h * d:(h + kv) * d].view(n, kv, d), x[:, (h + kv) * d:].view(n, kv, d) if v else None


def _prepare_rope(c, g):
    n, dtype = c["tokens"], DTYPES[c["dtype"]]
    q, k, _ = _split(_normal(g, n, (c["heads"] + c["kv_heads"]) * c["dim"]).to(dtype), c, v=False)
    positions = (torch.arange(n, device="cuda") + c["first"]).int()
    if c["first"] > 1:
        positions = positions + torch.randint(0, 1000, (1,), device="cuda", generator=g).int()
    return dict(q=q, k=k, dq=_normal(g, *q.shape).to(dtype) if c["train"] else None, dk=_normal(g, *k.shape).to(dtype) if c["train"] else None,
                positions=positions, frequencies=_frequencies(c["rotary"], c["scaling"]), interleaved=c["interleaved"],
                scale=ATTENTION_FACTOR if c["scaling"] == "parts" else 1.0, train=c["train"])


def _own_rope(s):
    ops = _package().rope
    out = list(ops.rope_fwd(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=s["interleaved"], scale=s["scale"]))
    if s["train"]:
        out += ops.rope_bwd(s["dq"], s["dk"], s["positions"], s["frequencies"], interleaved=s["interleaved"], scale=s["scale"])
    return out


def _plain_rope(s):
    angle = s["positions"].double()[:, None] * s["frequencies"][None]
    out = [_rotated(x.float(), angle, s["interleaved"], s["scale"]).to(x.dtype) for x in (s["q"], s["k"])]
    if s["train"]:
        out += [_rotated(x.float(), -angle, s["interleaved"], s["scale"]).to(x.dtype) for x in (s["dq"], s["dk"])]
    return out


def _exact_turn(x, s):
    """The same as a product of complex numbers in f64."""
    angle = s["positions"].double()[:, None] * s["frequencies"][None]
    unit = torch.polar(torch.full_like(angle, s.get("scale", 1.0)), angle)[:, None]
    pairs, x = angle.shape[1], x.double()
    head = x[..., :2 * pairs]
    z = torch.view_as_complex(head.reshape(*head.shape[:-1], pairs, 2)) if s["interleaved"] else torch.complex(head[..., :pairs], head[..., pairs:])
    z = z * unit
    head = torch.view_as_real(z).flatten(-2) if s["interleaved"] else torch.cat((z.real, z.imag), -1)
    return torch.cat((head, x[..., 2 * pairs:]), -1)


def _exact_rope(s):
    x = [s[n].double().requires_grad_(s["train"]) for n in ("q", "k")]
    out = [_exact_turn(t, s) for t in x]
    if not s["train"]:
        return out
    return [t.detach() for t in out] + list(torch.autograd.grad(out, x, [s["dq"].double(), s["dk"].double()]))


def _work_rope(c):
    n = c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"] * (2 if c["train"] else 1)
    return {"bytes": 2 * n * BYTES[c["dtype"]] + 4 * c["tokens"], "flops": 3 * n}


# ------------------------------------------------------------------ writing to a cache and reading it
def _prepare_write(c, g):
    s = _prepare_cache(c, g)
    lengths = _lengths(c)
    which = [(b, p) for b, n in enumerate(lengths) for p in range(max(0, n - c["new"]), n)]
    which = torch.tensor(which, device="cuda")
    page = s["table"][which[:, 0], which[:, 1] // c["page"]].long()
    q, k, v = _split(_normal(g, len(which), (c["heads"] + 2 * c["kv_heads"]) * c["dim"]).to(DTYPES[c["dtype"]]), c)
    return dict(s, q=q, k_new=k, v_new=v, positions=which[:, 1].int(), slots=((page - 1) * c["page"] + which[:, 1] % c["page"] + 1).int(),
                frequencies=_frequencies(c["rotary"], "none") if c["rotary"] else None, interleaved=c["interleaved"], store=c["store"],
                read=c["read"], longest=c["longest"])


def _own_write(s):
    return _package().kvcache.kv_write(_own_cache(s), s["slots"], s["k_new"], s["v_new"], q=s["q"] if s["frequencies"] is not None else None,
                                       positions=s["positions"], frequencies=s["frequencies"], interleaved=s["interleaved"])


def _own_cached(s):
    q = _own_write(s)
    if not s["read"]:
        return [q, s["k"], s["v"]]
    k, v = _package().kvcache.kv_read(_own_cache(s), s["table"], s["lengths"], s["longest"], dtype=s["q"].dtype)
    return [q, k, v, s["ks"], s["vs"]]


def _plain_write(s):
    q, k, v = s["q"], s["k_new"].float(), s["v_new"].float()
    if s["frequencies"] is not None:
        angle = s["positions"].double()[:, None] * s["frequencies"][None]
        q, k = _rotated(q.float(), angle, s["interleaved"]).to(q.dtype), _rotated(k, angle, s["interleaved"])
    else:
        q = None
    at, page = s["slots"].long() - 1, s["k"].shape[2]
    at = at // page, slice(None), at % page
    if s["ks"] is None:
        s["k"][at], s["v"][at] = k.to(s["k"].dtype), v.to(s["v"].dtype)
    else:
        s["k"][at], s["ks"][at] = _codes(k, s["store"])
        s["v"][at], s["vs"][at] = _codes(v, s["store"])
    return q


def _pages(s, side, dtype):
    """What the sequences have of one side, [batch, kv_heads, width * page, dim], as values."""
    at = (s["table"].long() - 1).clamp(min=0)
    x = s[side][at].to(dtype)
    if s["ks"] is not None:
        x = x * s[side + "s"][at].to(dtype)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_cached(s):
    q = _plain_write(s)
    if not s["read"]:
        return [q, s["k"], s["v"]]
    here = torch.arange(s["longest"], device="cuda")[None] < s["lengths"][:, None]
    k, v = (torch.where(here[:, None, :, None], _pages(s, side, torch.float32)[:, :, :s["longest"]], 0.0).to(s["q"].dtype) for side in "kv")
    return [q, k, v, s["ks"], s["vs"]]


def _rounded(x, store):
    """x in the steps of a code: whole numbers, or three bits behind the leading one and no exponent below -6."""
    if store == "int8":
        return x.round()
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).double() - 3)
    return (x / step).round() * step


def _exact_write(s):
    """(q, sides): the sides as f64 values [pages, kv_heads, page, dim], with their scales."""
    q = _exact_turn(s["q"], s) if s["frequencies"] is not None else None
    rows = {"k": _exact_turn(s["k_new"], s) if q is not None else s["k_new"].double(), "v": s["v_new"].double()}
    page = s["k"].shape[2]
    where = torch.div(s["slots"].long() - 1, page, rounding_mode="floor"), slice(None), (s["slots"].long() - 1) % page
    sides = {}
    for side, x in rows.items():
        values, scales = s[side].double(), None
        if s["ks"] is not None:
            scales = s[side + "s"].double()
            values = values * scales[..., None]
            peak = x.abs().amax(-1, keepdim=True)
            scales[where] = peak[..., 0] / LARGEST[s["store"]]
            x = _rounded(x * LARGEST[s["store"]] / peak, s["store"]) * peak / LARGEST[s["store"]]
        values[where] = x
        sides[side] = values, scales
    return q, sides


def _exact_cached(s):
    q, sides = _exact_write(s)
    if not s["read"]:
        return [q, sides["k"][0], sides["v"][0]]
    out = []
    for side in "kv":
        dense = torch.zeros(len(s["lengths"]), s["k"].shape[1], s["longest"], s["k"].shape[3], device="cuda", dtype=torch.float64)
        for b, n in enumerate(s["lengths"].tolist()):
            pages = sides[side][0][s["table"][b, :-(-n // s["k"].shape[2])].long() - 1]
            dense[b, :, :n] = pages.transpose(0, 1).flatten(1, 2)[:, :n]
        out.append(dense)
    return [q] + out + [sides["k"][1], sides["v"][1]]


def _work_cache(c):
    lengths = _lengths(c)
    new = sum(min(n, c["new"]) for n in lengths)
    h, kv, d, e = c["heads"], c["kv_heads"], c["dim"], BYTES[c["store"]]
    rows = 2 * kv * (d * e + (4 if e == 1 else 0))  # of a token, stored
    nbytes = new * (2 * kv * d * 2 + rows + 4 + (4 + 4 * h * d if c["rotary"] else 0))
    flops = new * (h + kv) * d * 3 + new * 2 * kv * d * 3
    if c["read"]:
        nbytes += sum(lengths) * rows + 2 * c["batch"] * kv * c["longest"] * d * 2
        flops += 2 * sum(lengths) * kv * d
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ attention of new tokens over a cache
def _prepare_attend(c, g):
    s = _prepare_cache(c, g)
    return dict(s, q=(1.5 * _normal(g, c["batch"], c["heads"], c["dim"])).to(DTYPES[c["dtype"]]), lse=c["lse"])


def _own_attend(s):
    out = _package().fmha.fmha_paged(s["q"], _own_cache(s), s["table"], s["lengths"], return_lse=s["lse"])
    return list(out) if s["lse"] else [out]


def _attend(s, q, k, v):
    """o and lse from q [batch, heads, dim] and dense k, v, in their precision."""
    batch, heads, dim = q.shape
    kv_heads, longest = k.shape[1:3]
    grouped = q.view(batch, kv_heads, heads // kv_heads, dim)
    score = torch.matmul(grouped, k.transpose(2, 3)) / math.sqrt(dim)
    here = (torch.arange(longest, device="cuda")[None] < s["lengths"][:, None])[:, None]
    score = torch.where(here[:, None], score, -math.inf)
    peak = score.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(score - peak)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, torch.where(here[..., None], v, 0.0)) / torch.where(total > 0, total, 1.0)
    return o.reshape(q.shape), (peak + torch.log(total)).reshape(batch, heads)


def _plain_attend(s):
    o, lse = _attend(s, s["q"].float(), _pages(s, "k", torch.float32), _pages(s, "v", torch.float32))
    return [o.to(s["q"].dtype)] + ([lse] if s["lse"] else [])


def _exact_sequence(q, k, v):
    """q [heads, dim] against k, v [kv_heads, length, dim], f64."""
    group = q.shape[0] // k.shape[0]
    logits = torch.einsum("hgd,hnd->hgn", q.view(k.shape[0], group, -1), k) / math.sqrt(q.shape[1])
    return torch.einsum("hgn,hnd->hgd", torch.softmax(logits, -1), v).reshape(q.shape), torch.logsumexp(logits, -1).reshape(-1)


def _exact_attend(s, q=None, sides=None):
    q = s["q"].double() if q is None else q
    o, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    page = s["k"].shape[2]
    for b, n in enumerate(s["lengths"].tolist()):
        if n:
            at = s["table"][b, :-(-n // page)].long() - 1
            kv = []
            for side in "kv":
                x = s[side][at].double() if sides is None else sides[side][0][at]
                x = x * s[side + "s"][at].double()[..., None] if sides is None and s["ks"] is not None else x
                kv.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
            o[b], lse[b] = _exact_sequence(q[b], *kv)
    return [o] + ([lse] if s.get("lse") else [])


def _work_attend(c):
    keys = sum(_lengths(c))
    e = BYTES[c["store"]]
    nbytes = keys * 2 * c["kv_heads"] * (c["dim"] * e + (4 if e == 1 else 0)) + 4 * c["batch"] * c["heads"] * c["dim"]
    nbytes += 4 * sum(-(-n // c["page"]) for n in _lengths(c)) + 4 * c["batch"] * (1 + (c["heads"] if c.get("lse") else 0))
    return {"bytes": nbytes, "flops": 4 * keys * c["heads"] * c["dim"]}


# ------------------------------------------------------------------ a layer's decoding step
def _own_step(s):
    q = _own_write(s)
    return [_package().fmha.fmha_paged(q, _own_cache(s), s["table"], s["lengths"]), s["k"], s["v"]]


def _plain_step(s):
    q = _plain_write(s).float()
    o, _ = _attend(s, q, _pages(s, "k", torch.float32), _pages(s, "v", torch.float32))
    return [o.to(s["q"].dtype), s["k"], s["v"]]


def _exact_step(s):
    """The query is rounded as it is handed on, and new rows as they are stored."""
    q, sides = _exact_write(s)
    stored = {side: (x.to(s["k"].dtype).double(), None) for side, (x, _) in sides.items()}
    return _exact_attend(s, q.to(s["q"].dtype).double(), stored) + [sides["k"][0], sides["v"][0]]


def _work_step(c):
    a, b = _work_cache(c), _work_attend(c)
    return {k: a[k] + b[k] for k in a}


# ------------------------------------------------------------------ the interface
_PREPARE = {"rope": _prepare_rope, "cache": _prepare_write, "attend": _prepare_attend, "step": _prepare_write}
_OWN = {"rope": _own_rope, "cache": _own_cached, "attend": _own_attend, "step": _own_step}
_PLAIN = {"rope": _plain_rope, "cache": _plain_cached, "attend": _plain_attend, "step": _plain_step}
_EXACT = {"rope": _exact_rope, "cache": _exact_cached, "attend": _exact_attend, "step": _exact_step}
_WORK = {"rope": _work_rope, "cache": _work_cache, "attend": _work_attend, "step": _work_step}


def prepare(case, seed):
    return dict(_PREPARE[case["kind"]](case, _generator(seed)), kind=case["kind"])


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def work(case):
    return _WORK[case["kind"]](case)


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))
