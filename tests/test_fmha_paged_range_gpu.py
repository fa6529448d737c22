"""Attention over a paged cache where one tile's contents or layout say little about the next one's.  Bounds as in test_fmha_paged_gpu,
with probabilities as two 16-bit numbers for every type (2^-17)."""
import math

import pytest

from test_fmha_paged_gpu import Case, same

pytestmark = pytest.mark.gpu

EIGHT = ("float8_e4m3fn", "int8")
SIXTEEN = ("float16", "bfloat16")


def case(*args, **kw):
    """A Case without the NaN that its e4m3 codes of numbers beyond 4.64 are: in long sequences every row would have one."""
    import torch
    c = Case(*args, **kw)
    if c.store == torch.float8_e4m3fn:
        for i, (x, s) in enumerate(((c.cache.k, c.cache.k_scale), (c.cache.v, c.cache.v_scale))):
            x.copy_(x.float().nan_to_num(448.0).to(c.store))
            c.values[i] = x.float().double() * s.double()[..., None]
    return c


def bound_of(c, b, k, v, keys=None):
    """(o, what it may be off by, lse, what that may be off by) of sequence b over its keys k and values v (f64), of which `keys` (a mask) are meant."""
    import torch
    D, info = c.q.shape[2], torch.finfo(c.dtype)
    q = c.q[b].double().view(k.shape[0], -1, D)
    if keys is not None:
        k, v = k[:, keys], v[:, keys]
    s = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(D)
    S = (torch.einsum("hgd,hnd->hgn", q.abs(), k.abs()).amax(-1) / math.sqrt(D))[..., None]
    p = torch.softmax(s, -1)
    o, W = torch.einsum("hgn,hnd->hgd", p, v), torch.einsum("hgn,hnd->hgd", p, v.abs())
    F = torch.zeros_like(o)
    if c.cache.v_scale is not None:
        n = int(c.lengths[b])
        at = c.table[b, :-(-n // c.page)].long() - 1
        codes = c.cache.v[at].float().double().transpose(0, 1).flatten(1, 2)[:, :n].abs()
        each = c.cache.v_scale[at].double().transpose(0, 1).flatten(1, 2)[:, :n].abs()
        if keys is not None:
            codes, each = codes[:, keys], each[:, keys]
        F = 2.0 ** -33 * (p * each[:, None]).amax(-1)[..., None] * codes.sum(1)[:, None]
    elif c.store == torch.float16:
        F = 2.0 ** -33 * p.amax(-1)[..., None] * v.abs().sum(1)[:, None]
    off = info.eps / 2 * o.abs() + W * (2 * (S * 2.0 ** -18 + 2.0 ** -22) + 2.0 ** -17 + 2.0 ** -17) + F + info.smallest_normal * info.eps / 2
    lse = torch.logsumexp(s, -1)
    return o, off, lse, S[..., 0] * 2.0 ** -18 + 2.0 ** -20 * (1 + lse.abs())


def check(c, got, keys=None, sequences=None):
    for b in range(c.q.shape[0]) if sequences is None else sequences:
        o, off, lse, lse_off = bound_of(c, b, *c.sequence(b), None if keys is None else keys[b])
        err = (got[0][b].double().view(o.shape) - o).abs()
        assert (err <= off).all(), (b, float((err / off).max()))
        err = (got[1][b].double().view(lse.shape) - lse).abs()
        assert (err <= lse_off).all(), (b, float((err / lse_off).max()))


def slots_of(c, b, keys):
    """(pages, places) of keys of sequence b."""
    return c.table[b].long()[keys // c.page] - 1, keys % c.page


def runs(c, b, first, length, every):
    """Keys of sequence b in runs: `length` of every `every` keys, from `first` on."""
    import torch
    n = torch.arange(int(c.lengths[b]), device="cuda")
    return n[((n - first) % every < length) & (n >= first)]


@pytest.mark.parametrize("store", EIGHT)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", SIXTEEN)
@pytest.mark.parametrize("lead", [32, 64, 100])
def test_runs_of_zero_values(cuda, store, D, dtype, lead):
    """Values whose scales are zero, as an untouched cache has them and rows below 2^-100 are stored, before small ones: in the first tiles of a
    sequence (whole items), and in stretches (items in parts)."""
    for lengths, heads, kv_heads, every in (([400, lead + 1, lead + 90], 8, 1, 10 ** 6), ([300, 220], 6, 2, 10 ** 6), ([9000] * 8, 16, 8, 2 * lead)):
        for size in (1.0, 1e-3, 1e-6, 1e-9):
            c = case(cuda, lengths, heads, kv_heads, D, 16, store, dtype, seed=lead)
            c.cache.v_scale.mul_(size)
            for b in range(len(lengths)):
                pages, places = slots_of(c, b, runs(c, b, 0, lead, every))
                c.cache.v_scale[pages, :, places] = 0
            c.values[1] = c.cache.v.float().double() * c.cache.v_scale.double()[..., None]
            check(c, c.run(), sequences=range(min(len(lengths), 3)))


@pytest.mark.parametrize("store", EIGHT)
@pytest.mark.parametrize("dtype", SIXTEEN)
def test_negative_scales(cuda, store, dtype):
    """A value is code * scale, whatever the scale's sign: all of them negative, or the large ones only, later than small positive ones."""
    import torch
    for every in (True, False):
        c = case(cuda, [500, 70], 8, 1, 64, 16, store, dtype, seed=23)
        c.cache.v_scale.mul_(-1e-4 if every else 1e-4)
        if not every:
            for b in (0, 1):
                pages, places = slots_of(c, b, torch.arange(64, int(c.lengths[b]), device="cuda"))
                c.cache.v_scale[pages, :, places] *= -1e5
        c.values[1] = c.cache.v.float().double() * c.cache.v_scale.double()[..., None]
        check(c, c.run())


@pytest.mark.parametrize("store", EIGHT)
def test_large_scales_of_keys_that_do_not_count(cuda, store):
    """Tiny values, and huge ones whose probabilities are zero in every row of the operand."""
    import torch
    c = case(cuda, [4000], 8, 1, 64, 16, store, "bfloat16", seed=29)
    c.q.abs_()
    c.cache.v_scale.mul_(1e-30)
    keys = runs(c, 0, 150, 1, 200)
    pages, places = slots_of(c, 0, keys)
    c.cache.v_scale[pages, 0, places] = 1e12
    c.cache.k[pages, 0, places] = -100
    c.cache.k_scale[pages, 0, places] = 1.0  # scores of -100 sum |q| / 8, below -400
    for i, (x, s) in enumerate(((c.cache.k, c.cache.k_scale), (c.cache.v, c.cache.v_scale))):
        c.values[i] = x.float().double() * s.double()[..., None]
    check(c, c.run(), keys=[torch.ones(4000, device="cuda", dtype=torch.bool).index_fill_(0, keys, False)])  # e^-400 1e14 is nothing beside 1e-30


@pytest.mark.parametrize("store", EIGHT)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [4, 16])
def test_values_that_cancel(cuda, store, D, heads):
    """Neighbouring keys alike, their values opposite, from other codes and scales: what is left is small beside the terms, so that bf16 results
    show how probabilities were rounded."""
    import torch
    c = case(cuda, [2, 64, 500], heads, 1, D, 16, store, "bfloat16", seed=31, q_size=0.01)  # scores add little to the bound
    k, v, ks, vs = c.cache
    first, second = slice(0, None, 2), slice(1, None, 2)
    k[:, :, second], ks[:, :, second] = k[:, :, first], ks[:, :, first]
    sign = torch.where(torch.rand(v[:, :, first].shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.5, -1.0, 1.0)
    v[:, :, first], v[:, :, second] = (44 * sign).to(v.dtype), (-32 * sign).to(v.dtype)
    vs[:, :, second] = vs[:, :, first] * (44 / 32)
    for i, (x, s) in enumerate(((k, ks), (v, vs))):
        c.values[i] = x.float().double() * s.double()[..., None]
    check(c, c.run())


@pytest.mark.parametrize("store", SIXTEEN)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lead", [16, 32, 100])
@pytest.mark.parametrize("shift", [0.0, -300.0])
def test_runs_of_keys_of_minus_infinity(cuda, store, D, lead, shift):
    """Keys that score -inf throughout the first tiles of an item or a part do not count, before ordinary scores and before very low ones."""
    import torch
    for lengths, heads, kv_heads, every in (([400, lead + 1, lead + 90], 8, 1, 10 ** 6), ([300, 220], 6, 2, 10 ** 6), ([5000] * 8, 16, 8, 2 * lead)):
        c = case(cuda, lengths, heads, kv_heads, D, 16, store, seed=lead + 1)
        c.q.abs_().clamp_(min=0.25)
        if shift:  # by shift or so: every query has 8 in one dimension
            c.q[..., 0] = 8.0
            c.cache.k[..., 0] += shift / 8 * math.sqrt(D)
            c.values[0] = c.cache.k.double()
        keep = []
        for b, n in enumerate(lengths):
            keys = runs(c, b, 0, lead, every)
            pages, places = slots_of(c, b, keys)
            c.cache.k[pages, :, places] = -math.inf
            keep.append(torch.ones(n, device="cuda", dtype=torch.bool).index_fill_(0, keys, False))
        out, lse = c.run()
        check(c, (out, lse), keys=keep, sequences=range(min(len(lengths), 3)))
    c = case(cuda, [lead, lead + 3000], 8, 1, D, 16, store, seed=2)  # all of one sequence's
    c.q.abs_()
    pages, places = slots_of(c, 0, torch.arange(lead, device="cuda"))
    clean = c.run()
    c.cache.k[pages, :, places] = -math.inf
    out, lse = c.run()
    assert out[0].isnan().all() and (lse[0] == -math.inf).all() and same(out[1], clean[0][1]) and same(lse[1], clean[1][1])


@pytest.mark.parametrize("store", SIXTEEN)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([100, 37], 8, 1), ([9000], 4, 2), ([3000] * 3, 32, 2)])
def test_infinite_values(cuda, store, D, lengths, heads, kv_heads):
    """An infinite value makes its dimension infinite, infinities of both signs and a NaN make it NaN, and nothing else changes."""
    import torch
    c = case(cuda, lengths, heads, kv_heads, D, 16, store, seed=37)
    clean = c.run()
    inf, nan = math.inf, math.nan
    b, h = len(lengths) - 1, kv_heads - 1
    n = lengths[b]
    marks = {0: [(3, inf)], 9: [(n - 1, -inf)], 17: [(0, inf), (n // 2, inf)], 25: [(1, inf), (n - 2, -inf)], 33: [(5, inf), (20, nan)], D - 1: [(n // 3, -inf)]}
    for dim, at in marks.items():
        for key, x in at:
            (page,), (place,) = slots_of(c, b, torch.tensor([key], device="cuda"))
            c.cache.v[page, h, place, dim] = x
    out, lse = c.run()
    group = heads // kv_heads
    want = clean[0].clone()
    for dim, at in marks.items():
        want[b, h * group:(h + 1) * group, dim] = sum(x for _, x in at)
    assert same(out, want) and same(lse, clean[1])


def test_strides_of_one_element(cuda):
    """Strides along a dimension of one element mean nothing."""
    import torch
    c = case(cuda, [40], 4, 2, 64, 16, "float16", seed=41)
    q = c.q.as_strided((1, 4, 64), (4 * 64 + 1, 64, 1))
    want = c.run()
    got = cuda.fmha.fmha_paged(q, c.cache, c.table, c.lengths, return_lse=True)
    assert got[0].equal(want[0]) and got[1].equal(want[1])
    assert cuda.fmha.fmha_paged(q, c.cache, c.table, c.lengths, occupancy=1).equal(want[0])
    c = case(cuda, [40, 3], 1, 1, 64, 16, "bfloat16", seed=43)
    q = c.q.as_strided((2, 1, 64), (64, 3, 1))
    assert cuda.fmha.fmha_paged(q, c.cache, c.table, c.lengths).equal(c.run()[0])


def test_no_scratch_where_none_is_used(cuda):
    """A page table too narrow for items that several CTAs share takes no scratch: neither a stream's nor a graph's."""
    import torch
    c = case(cuda, [700, 20], 8, 2, 128, 16, "bfloat16", seed=47)
    want = c.run()
    side, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    out = None

    def capture():
        nonlocal out
        graph = torch.cuda.CUDAGraph()
        out = None  # its place in the pool is the next one's
        with torch.cuda.graph(graph, stream=side, pool=pool):
            out = c.run()
        return graph
    graphs = [capture() for _ in range(4)]
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    graphs += [capture() for _ in range(60)]
    assert free - torch.cuda.mem_get_info()[0] < 64 << 20  # 60 slots of 2.5 MB would be 150
    graphs[-1].replay()
    torch.cuda.synchronize()
    assert out[0].equal(want[0]) and out[1].equal(want[1])


def test_scale_refused(cuda):
    """A scale that is no f32 number in powers of two."""
    c = case(cuda, [20], 2, 1, 64, 16, "float16")
    with pytest.raises(cuda.CtbError, match="not finite"):
        c.run(qk_scale=3e38)
