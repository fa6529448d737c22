"""Attention of new tokens over a paged cache against f64.

With c the scale, S = c max_j sum_i |q_i k_ji| and W = sum_j p_j |v_j| (for one output): a score is off by what D f32 products and their
sums lose, 2^-19 S at most (sums of 16 products at a time, each rounded or cut off to 24 bits), and by the roundings of its scale, its 8-bit
scale and its distance from the reference (2^-21 of the score, again below S); queries in bf16 over 8-bit keys lose 2^-33 of a row's
largest element.  Probabilities are therefore off by 2^-18 S + 2^-22 (ex2) relative to each other, which moves o by twice that of W; they
enter as two 16-bit numbers (2^-17), in bf16 beside 8-bit values as one f16 (2^-11), and the sums over keys and over parts take 24-bit roundings, 2^-17 W for up to 2^7 of them in a
row (a tile of a part adds one; longer parts are averages).  Pairs of f16 numbers, where the type or the cache's eight bits ask for them, have a
smallest step, 2^-24, and hold numbers whose largest is brought to 2^8 or more: a probability (with its value's scale) is off by 2^-33 of
the largest of the row besides, F = 2^-33 max_j (p_j s_j) sum_j |v_j| / s_j, s = 1 without scales.  One rounding to the type at the end.  lse: the scores' part, and 2^-20 of
1 + |lse|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

STORES = ("float16", "bfloat16", "float8_e4m3fn", "int8")


def same(x, y):
    return bool(((x == y) | (x.isnan() & y.isnan())).all())


class Case:
    """A cache in which everything that the sequences do not have is NaN, and the dense f64 keys and values of every sequence."""

    def __init__(self, cuda, lengths, heads, kv_heads, D, page, store, dtype=None, seed=0, q_size=1.0, spread=0.5):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cuda, self.store = cuda, getattr(torch, store)
        self.dtype = self.store if store.endswith("float16") else getattr(torch, dtype or "bfloat16")
        B = len(lengths)
        used = [-(-max(n, 0) // page) for n in lengths]
        width, total = max(max(used), 1), sum(used)
        pages = total + 2
        order = (torch.randperm(pages, device="cuda", generator=g) + 1).int()
        self.table = torch.zeros(B, width, device="cuda", dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.lengths = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        self.q = (torch.randn(B, heads, D, device="cuda", generator=g) * q_size).to(self.dtype)
        live = torch.zeros(pages * page, device="cuda", dtype=torch.bool)
        for b, n in enumerate(lengths):
            slots = ((self.table[b].long() - 1)[:, None] * page + torch.arange(page, device="cuda")).flatten()
            live[slots[:max(n, 0)]] = True
        live = live.view(pages, 1, page)
        self.cache, self.values = [], []
        scales = []
        for _ in range(2):
            x = torch.randn(pages, kv_heads, page, D, device="cuda", generator=g)
            if store.endswith("float16"):
                x = x.to(self.store)
                self.values.append(x.double())
                self.cache.append(torch.where(live[..., None], x, float("nan")))
                scales.append(None)
            else:
                scale = torch.exp(spread * torch.randn(pages, kv_heads, page, device="cuda", generator=g))
                code = (x * 30).round().clamp(-127, 127).to(torch.int8) if store == "int8" else (x * 100).to(self.store)
                scale = scale / (30 if store == "int8" else 100)
                self.values.append(code.float().double() * scale.double()[..., None])
                self.cache.append(code)
                scales.append(torch.where(live, scale, float("nan")))
        self.cache = cuda.kvcache.KvCache(*self.cache, *scales)
        self.page = page

    def run(self, **kw):
        return self.cuda.fmha.fmha_paged(self.q, self.cache, self.table, self.lengths, return_lse=True, **kw)

    def sequence(self, b):
        n = max(int(self.lengths[b]), 0)
        at = self.table[b, :-(-n // self.page)].long() - 1
        return [x[at].transpose(0, 1).flatten(1, 2)[:, :n] for x in self.values]

    def check(self, got, scale=None, sequences=None):
        import torch
        out, lse = got
        B, H, D = self.q.shape
        scale = 1 / math.sqrt(D) if scale is None else scale
        info = torch.finfo(self.dtype)
        for b in range(B) if sequences is None else sequences:
            k, v = self.sequence(b)
            if k.shape[1] == 0:
                assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
                continue
            q = self.q[b].double().view(k.shape[0], -1, D)
            s = torch.einsum("hgd,hnd->hgn", q, k) * scale
            S = (torch.einsum("hgd,hnd->hgn", q.abs(), k.abs()).amax(-1) * abs(scale))[..., None]
            p = torch.softmax(s, -1)
            o, W = torch.einsum("hgn,hnd->hgd", p, v), torch.einsum("hgn,hnd->hgd", p, v.abs())
            F, P = torch.zeros_like(o), 2.0 ** -17 if self.cache.v_scale is None or self.dtype == torch.float16 else 2.0 ** -11
            if self.cache.v_scale is not None:
                at = self.table[b, :-(-k.shape[1] // self.page)].long() - 1
                codes = self.cache.v[at].float().double().transpose(0, 1).flatten(1, 2)[:, :k.shape[1]].abs().sum(1)
                each = self.cache.v_scale[at].double().transpose(0, 1).flatten(1, 2)[:, :k.shape[1]]
                F = 2.0 ** -33 * (p * each[:, None]).amax(-1)[..., None] * codes[:, None]
            elif self.store == torch.float16:
                F = 2.0 ** -33 * p.amax(-1)[..., None] * v.abs().sum(1)[:, None]
            mine = out[b].double().view(o.shape)
            err = (mine - o).abs()
            bound = info.eps / 2 * o.abs() + W * (2 * (S * 2.0 ** -18 + 2.0 ** -22) + P + 2.0 ** -17) + F + info.smallest_normal * info.eps / 2
            assert ((err <= bound) | (mine.isnan() & o.isnan())).all(), (b, float((err / bound).max()))  # codes beyond 448 are NaN
            want = torch.logsumexp(s, -1)
            mine = lse[b].double().view(want.shape)
            off = (mine - want).abs()
            assert ((off <= S[..., 0] * 2.0 ** -18 + 2.0 ** -20 * (1 + want.abs())) | (mine.isnan() & want.isnan())).all(), (b, float(off.max()))


@pytest.mark.parametrize("lengths,heads,kv_heads,D,page", [
    ([1], 1, 1, 64, 16), ([1], 8, 1, 128, 16), ([15, 16, 17], 4, 2, 128, 16), ([0, 1, 33, 0, 64, 65], 6, 3, 64, 32), ([500, 3, 77, 250], 32, 8, 128, 16),
    ([1000], 7, 1, 128, 64), ([2000, 1999], 16, 2, 64, 128), ([130, 4000], 20, 2, 128, 256), ([300, 5], 17, 1, 64, 16), ([700, 0, 9], 40, 1, 128, 1024),
    ([9000], 8, 8, 128, 16), ([0, 0, 0], 2, 1, 64, 16), (list(range(1, 200)), 4, 4, 64, 16), ([777] * 31, 10, 2, 128, 32)])
@pytest.mark.parametrize("store", STORES)
def test_attention(cuda, lengths, heads, kv_heads, D, page, store):
    import torch
    for dtype in (None,) if store.endswith("float16") else ("float16", "bfloat16"):
        c = Case(cuda, lengths, heads, kv_heads, D, page, store, dtype, seed=len(lengths) + heads)
        got = c.run()
        assert got[0].dtype == c.dtype and got[0].shape == c.q.shape and got[1].dtype == torch.float32
        c.check(got)
        again = c.run()
        without = cuda.fmha.fmha_paged(c.q, c.cache, c.table, c.lengths)
        for x, y in ((got[0], again[0]), (got[1], again[1]), (got[0], without)):
            assert same(x, y)
    cuda.check_device_status(0)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("D", [64, 128])
def test_sharp_and_growing_scores(cuda, store, D):
    """Scores that rise along the sequence, scores of one key far above the others, negative and zero scales."""
    import torch
    c = Case(cuda, [900, 130], 8, 2, D, 16, store, seed=3, q_size=4.0)
    c.check(c.run())
    for scale in (-0.3, 0.0, 1e-4):
        c.check(c.run(qk_scale=scale), scale)
    ramp = torch.linspace(-1, 1, c.table.shape[1] * 16, device="cuda")
    for b in (0, 1):  # keys along the queries' mean, longer and longer
        at = c.table[b, :-(-int(c.lengths[b]) // 16)].long() - 1
        d = c.q[b].float().view(2, 4, D).mean(1)
        k = ramp[:len(at) * 16].view(len(at), 1, 16, 1) * d[None, :, None, :] * 2
        if store.endswith("float16"):
            k = k.to(c.store)
            c.cache.k[at] = k
            c.values[0][at] = k.double()
        else:
            most = 127 if store == "int8" else 448
            s = k.abs().amax(-1).clamp(min=1e-6) / most
            code = (k / s[..., None]).round().clamp(-most, most).to(c.store)
            c.cache.k[at], c.cache.k_scale[at] = code, s
            c.values[0][at] = code.float().double() * s.double()[..., None]
    c.check(c.run())


@pytest.mark.parametrize("store", ["float8_e4m3fn", "int8"])
def test_scales_of_any_size(cuda, store):
    """Scales of values that differ by many powers of ten, also those of the keys that matter most; rows of zeros."""
    import torch
    c = Case(cuda, [600, 50, 1], 4, 1, 64, 16, store, "bfloat16", seed=5, q_size=3.0)
    g = torch.Generator(device="cuda").manual_seed(1)
    f = 10.0 ** torch.randint(-28, 3, c.cache.v_scale.shape, device="cuda", generator=g)
    f[torch.rand(f.shape, device="cuda", generator=g) < 0.1] = 0
    c.cache.v_scale.mul_(f)
    c.values[1] = c.cache.v.float().double() * c.cache.v_scale.double()[..., None]
    c.check(c.run())
    c.cache.v_scale[c.cache.v_scale > 1e-20] *= 1e-25  # small values throughout: the outputs are below them
    c.values[1] = c.cache.v.float().double() * c.cache.v_scale.double()[..., None]
    c.check(c.run())


def test_many_sequences(cuda):
    """More than fit one launch's table of lengths."""
    import random
    r = random.Random(1)
    lengths = [r.randint(0, 40) for _ in range(4500)]
    c = Case(cuda, lengths, 2, 1, 64, 16, "float16", seed=7)
    c.check(c.run(), sequences=list(range(0, 4500, 97)) + [4095, 4096, 4499])


@pytest.mark.parametrize("store", STORES)
def test_infinities_and_nan(cuda, store):
    """What a key or value that counts has spreads over its heads' rows only; keys of -inf do not count."""
    import torch
    c = Case(cuda, [100, 100], 4, 2, 64, 16, store, seed=11)
    clean = c.run()
    page, place = int(c.table[0, 2]) - 1, 5
    target = c.cache.v if store.endswith("float16") else c.cache.v_scale
    target[page, 1, place] = float("nan")
    out, lse = c.run()
    assert out[0, 2:].isnan().all() and same(out[0, :2], clean[0][0, :2]) and same(out[1], clean[0][1]) and same(lse, clean[1])
    target = c.cache.k if store.endswith("float16") else c.cache.k_scale
    target[page, 0, place] = float("nan")
    out, lse = c.run()
    assert out[0].isnan().all() and lse[0, :2].isnan().all() and same(out[1], clean[0][1])
    if store.endswith("float16"):
        c = Case(cuda, [100, 3], 2, 1, 64, 16, store, seed=12)
        c.q.abs_()
        c.cache.k[int(c.table[0, 2]) - 1, 0, place] = -float("inf")
        out, lse = c.run()
        k, v = c.sequence(0)
        keep = torch.arange(100, device="cuda") != 32 + place
        s = (c.q[0].double() @ k[0, keep].T) / 8
        o = torch.softmax(s, -1) @ v[0, keep]
        assert ((out[0].double() - o).abs() <= 2.0 ** -8 * o.abs() + 2.0 ** -12).all()  # bf16's half step, and |q||k| < 100 in 2^-18


@pytest.mark.parametrize("store", ["bfloat16", "int8"])
def test_bad_pages_and_lengths(cuda, store):
    """They are reported and make their own rows NaN; nothing is read for them."""
    import torch
    for page_id in (0, -3, 10 ** 6):
        c = Case(cuda, [100, 40, 300], 4, 2, 128, 16, store, seed=13)
        clean = c.run()
        c.table[2, 7] = page_id
        out, lse = c.run()
        with pytest.raises(cuda.CtbError, match="out-of-range"):
            cuda.check_device_status(0)
        assert out[2].isnan().all() and lse[2].isnan().all() and out[:2].equal(clean[0][:2]) and lse[:2].equal(clean[1][:2])
    width = c.table.shape[1] * 16
    c.table[2, 7] = 1
    for n in (-1, width + 1, 2 ** 31 - 1, -2 ** 31):
        c.lengths[1] = n
        c.table[1] = 1
        out, lse = c.run()
        with pytest.raises(cuda.CtbError, match="out-of-range"):
            cuda.check_device_status(0)
        assert out[1].isnan().all() and lse[1].isnan().all()
        c.check((out, lse), sequences=[0])  # another length moves the ends of the parts, and with them the last bits
    c.lengths[:] = 5
    out, lse = cuda.fmha.fmha_paged(c.q, c.cache, c.table[:, :0], c.lengths, return_lse=True)
    with pytest.raises(cuda.CtbError, match="out-of-range"):
        cuda.check_device_status(0)
    assert out.isnan().all()
    cuda.check_device_status(0)


def test_views(cuda):
    """Queries of a fused projection, tables with room, pages of k and v in one allocation."""
    import torch
    c = Case(cuda, [90, 200, 17], 6, 2, 64, 16, "bfloat16", seed=15)
    want = c.run()
    fused = torch.randn(3, 10, 64, device="cuda").bfloat16()
    fused[:, 2:8] = c.q
    both = torch.stack((c.cache.k, c.cache.v), 1)
    wide = torch.full((3, c.table.shape[1] + 5), -1, device="cuda", dtype=torch.int32)
    wide[:, :c.table.shape[1]] = c.table
    cache = cuda.kvcache.KvCache(both[:, 0], both[:, 1])
    for table in (wide, wide[:, :c.table.shape[1]]):
        got = cuda.fmha.fmha_paged(fused[:, 2:8], cache, table, c.lengths, return_lse=True)
        assert got[0].equal(want[0]) and got[1].equal(want[1])
    got = cuda.fmha.fmha_paged(c.q, c.cache, c.table, c.lengths, return_lse=True, occupancy=1)  # launch keywords
    assert got[0].equal(want[0])


def test_offsets_beyond_32_bits(cuda):
    """A cache of more than 2^31 elements, of which a short sequence has the first and the last pages."""
    import torch
    pages = 2 ** 31 // (64 * 16) + 40
    k = torch.empty(pages, 1, 16, 64, device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    ids = [1, pages, pages - 1, 2, pages - 17]
    at = torch.tensor(ids, device="cuda") - 1
    x, y = torch.randn(5, 1, 16, 64, device="cuda").half(), torch.randn(5, 1, 16, 64, device="cuda").half()
    k[at], v[at] = x, y
    q = torch.randn(1, 2, 64, device="cuda").half()
    n = torch.tensor([75], device="cuda", dtype=torch.int32)
    table = torch.tensor([ids], device="cuda", dtype=torch.int32)
    out = cuda.fmha.fmha_paged(q, cuda.kvcache.KvCache(k, v), table, n)
    small = torch.tensor([[1, 2, 3, 4, 5]], device="cuda", dtype=torch.int32)
    assert out.equal(cuda.fmha.fmha_paged(q, cuda.kvcache.KvCache(x, y), small, n))
    K, V = cuda.kvcache.kv_read(cuda.kvcache.KvCache(k, v), table, n, 75)
    assert K[0, 0].equal(x.flatten(0, 2)[:75]) and V[0, 0].equal(y.flatten(0, 2)[:75])
    new = torch.randn(2, 1, 64, device="cuda").half()
    slots = torch.tensor([pages * 16, (pages - 17) * 16 + 3], device="cuda")
    cuda.kvcache.kv_write(cuda.kvcache.KvCache(k, v), slots, new, -new)
    assert k[pages - 1, 0, 15].equal(new[0, 0]) and v[pages - 17, 0, 2].equal(-new[1, 0])


def test_streams_and_graphs(cuda):
    """Calls on several streams at once and captured ones, replayed while others run: each gives what it gives alone."""
    import torch
    cases = [Case(cuda, n, 16, 2, 128, 16, s, seed=i) for i, (n, s) in enumerate((([3000, 100, 5], "bfloat16"), ([70, 9000], "float16"), ([2500] * 3, "int8")))]
    want = [c.run() for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(6)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                if i < 3:
                    got.append((i, cases[i].run()))
                else:
                    graphs[i - 3].replay()
    torch.cuda.synchronize()
    for i, (o, l) in got + list(enumerate(outs)):
        assert o.equal(want[i][0]) and l.equal(want[i][1])
    c = cases[0]
    c.lengths.copy_(torch.tensor([1, 0, 5], dtype=torch.int32))  # a graph goes by the lengths at its replay
    graphs[0].replay()
    torch.cuda.synchronize()
    c.check(outs[0])


@pytest.mark.parametrize("store", STORES)
def test_decoding_as_it_is_used(cuda, store):
    """A prompt by kv_write, kv_read and cutile_fmha, then single tokens by kv_write and fmha_paged: every row is near what attention over
    all of the stored keys in f64 gives (f16: test_fmha_gpu's tolerance of 2e-3 for the prompt)."""
    import torch
    dtype = torch.bfloat16 if store == "bfloat16" else torch.float16
    B, H, KVH, D, page, prompt, steps = 2, 8, 2, 64, 16, 70, 5
    kc, f = cuda.kvcache, cuda.rope.rope_frequencies(64, scaling="linear", factor=2.0).cuda()
    cache = kc.kv_cache(20, KVH, page, D, getattr(torch, store))
    table = (torch.randperm(20, device="cuda")[:2 * 6] + 1).int().view(2, 6)

    def slots(first, n):
        at = torch.arange(first, first + n, device="cuda").repeat(B, 1)
        return ((table.gather(1, at // page).long() - 1) * page + at % page + 1).flatten(), at.flatten()

    def stored(n):
        K, V = kc.kv_read(cache, table, torch.full((B,), n, device="cuda", dtype=torch.int32), n, dtype=dtype)
        if cache.k_scale is None:
            return K.double(), V.double()
        at = table.long() - 1
        return [(c[at].float().double() * s[at].double()[..., None]).transpose(1, 2).flatten(2, 3)[:, :, :n] for c, s in zip(cache[:2], cache[2:])]

    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(B * prompt, H + 2 * KVH, D, device="cuda", generator=g).to(dtype)
    q, k, v = qkv.split((H, KVH, KVH), 1)
    where, positions = slots(0, prompt)
    q = kc.kv_write(cache, where, k, v, q=q, positions=positions, frequencies=f)
    K, V = kc.kv_read(cache, table, torch.full((B,), prompt, device="cuda", dtype=torch.int32), prompt, dtype=dtype)
    Q = q.view(B, prompt, H, D).transpose(1, 2).contiguous()
    out = cuda.fmha.cutile_fmha(Q, K, V, causal=True, query_group_size=H // KVH)
    Kd, Vd = (x.double().repeat_interleave(H // KVH, 1) for x in (K, V))
    s = (Q.double() @ Kd.transpose(2, 3)) / 8
    s = s.masked_fill(torch.ones(prompt, prompt, device="cuda", dtype=torch.bool).triu(1), -math.inf)
    want = torch.softmax(s, -1) @ Vd
    assert (out.double() - want).norm() / want.norm() <= (2e-3 if dtype == torch.float16 else 1.6e-2)
    for i in range(steps):
        n = prompt + i + 1
        qkv = torch.randn(B, H + 2 * KVH, D, device="cuda", generator=g).to(dtype)
        q, k, v = qkv.split((H, KVH, KVH), 1)
        where, positions = slots(n - 1, 1)
        q = kc.kv_write(cache, where, k, v, q=q, positions=positions, frequencies=f)
        out, _ = cuda.fmha.fmha_paged(q, cache, table, torch.full((B,), n, device="cuda", dtype=torch.int32), return_lse=True)
        K, V = (x.repeat_interleave(H // KVH, 1) for x in stored(n))
        want = (torch.softmax((q.double()[:, :, None] @ K.transpose(2, 3)) / 8, -1) @ V)[:, :, 0]
        assert ((out.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -11).all()
        # the new token's own keys: turned by its position
        from test_rope_gpu import reference
        turned_k = reference(k, positions, f.cpu())[0]
        row = stored(n)[0][:, :, -1]
        step = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float8_e4m3fn": 2.0 ** -4, "int8": 0.0}[store]
        least = turned_k.abs().amax(-1, keepdim=True) * (0.5 / 127 * 1.01 if store == "int8" else 2.0 ** -10 / 448 * 1.01)
        assert ((row - turned_k).abs() <= step * 1.01 * turned_k.abs() + least + 1e-6).all()
    cuda.check_device_status(0)


def test_refusals(cuda):
    import torch
    c = Case(cuda, [20, 30], 4, 2, 64, 16, "float16")
    fp = cuda.fmha.fmha_paged
    q, cache, table, n = c.q, c.cache, c.table, c.lengths
    odd = torch.zeros(2 * 4 * 64 + 1, device="cuda", dtype=torch.float16)[1:].view(2, 4, 64)
    calls = [(lambda: fp(q.float(), cache, table, n), "f16 or bf16"), (lambda: fp(q.bfloat16(), cache, table, n), "type of the queries"),
             (lambda: fp(q[:, :3], cache, table, n), "multiple of kv_heads"), (lambda: fp(q[..., :32], cache, table, n), "Q must be"),
             (lambda: fp(q[:1], cache, table, n), "Q must be"), (lambda: fp(q, cache, table.long(), n), "int32"), (lambda: fp(q, cache, table, n.long()), "lengths"),
             (lambda: fp(q, cache, table, n[:1]), "lengths"), (lambda: fp(q, cache, table, n, qk_scale=float("nan")), "not finite"),
             (lambda: fp(odd, cache, table, n), "16-byte aligned"), (lambda: fp(q.cpu(), cache, table, n), "CUDA tensor"),
             (lambda: fp(q.transpose(1, 2), cache, table, n), "Q must be"), (lambda: fp(q[0], cache, table, n), "Q must be")]
    for call, word in calls:
        with pytest.raises(cuda.CtbError, match=word):
            call()
    assert fp(q[:0], cache, table[:0], n[:0]).shape == (0, 4, 64)
