"""The paged key-value cache against f64: what is stored, what is read back, and what stays as it was.

16 bits: rows that are not turned are stored bit for bit, turned ones within the bound of test_rope_gpu.  8 bits, with a the largest
magnitude and c the largest code: y = x c / a in f32 (a product, a quotient to an ulp: 2^-22 of y at most, besides c / a times what a turn is
off by), and the code is the number nearest to it: at most half a step (1/2, or 2^-4 of y, and 2^-10 below 2^-6) away.
"""
import pytest

pytestmark = pytest.mark.gpu

STORES = ("float16", "bfloat16", "float8_e4m3fn", "int8")


def places(pages, page, n, seed=0):
    """n slots (1-based) of a cache in an order of chance."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randperm(pages * page, device="cuda", generator=g)[:n].int() + 1


def rows_at(t, slots):
    page = t.shape[2]
    return t[(slots.long() - 1) // page, :, (slots.long() - 1) % page]


def filled(cuda, pages, heads, page, D, store):
    """A cache whose contents a test can tell from what it writes."""
    import torch
    c = cuda.kvcache.kv_cache(pages, heads, page, D, getattr(torch, store))
    for t in c[:2]:
        t.view(torch.uint8).random_(0, 100)
    for t in c[2:]:
        if t is not None:
            t.uniform_(1, 2)
    return c


def untouched(before, after, slots):
    import torch
    for b, a in zip(before, after):
        if b is None:
            continue
        used = torch.zeros(b.shape[0] * b.shape[2], dtype=torch.bool, device="cuda")
        used[slots.long() - 1] = True
        keep = ~used.view(b.shape[0], 1, b.shape[2])
        x, y = (t.reshape(*t.shape[:3], -1).view(torch.uint8) for t in (b, a))
        assert ((x == y) | ~keep[..., None]).all()


def stored_close(code, scale, x, off=0.0):
    """Codes and scales of f64 rows x, which the kernel has within `off` of each element."""
    import torch
    c = 127.0 if code.dtype == torch.int8 else 448.0
    a = x.abs().amax(-1)
    small = a < 2.0 ** -100
    off = torch.zeros_like(x) + off
    assert ((scale.double() - a / c).abs() <= a / c * 2.0 ** -23 + off.amax(-1) / c)[~small].all() and (scale[small] == 0).all()
    y = x * c / a.clamp(min=2.0 ** -100)[..., None]
    step = torch.ones_like(y) if c == 127 else torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    got = code.double() if c == 127 else code.float().double()
    bound = step / 2 * (1 + 2.0 ** -20) + y.abs() * 2.0 ** -22 + 2 * off * c / a.clamp(min=2.0 ** -100)[..., None]
    assert ((got - y).abs() <= bound)[~small].all() and (got[small] == 0).all()


def turned(x, positions, f, interleaved):
    from test_rope_gpu import reference
    if f is None:
        return x.double(), 0.0
    want, size = reference(x, positions, f, interleaved=interleaved, scale=0.75)
    return want, size * 2.0 ** -21


@pytest.mark.parametrize("T,H,KVH,D,page,R,interleaved", [(1, 4, 1, 64, 16, 64, False), (7, 0, 2, 128, 16, 0, False), (33, 5, 5, 64, 32, 32, True),
                                                          (64, 32, 8, 128, 16, 128, False), (130, 3, 3, 128, 128, 64, False), (9, 2, 1, 64, 64, 24, False),
                                                          (40, 8, 2, 128, 256, 6, True), (2500, 4, 2, 64, 1024, 16, False)])
@pytest.mark.parametrize("store", STORES)
def test_write(cuda, T, H, KVH, D, page, R, interleaved, store):
    import torch

    from test_rope_gpu import close
    dtype = getattr(torch, store) if store.endswith("float16") else (torch.bfloat16 if T % 2 else torch.float16)
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, H + 2 * KVH, D, device="cuda", generator=g).to(dtype)
    q, k, v = qkv.split((H, KVH, KVH), 1)
    pages = -(-2 * T // page)
    cache = filled(cuda, pages, KVH, page, D, store)
    before = [None if t is None else t.clone() for t in cache]
    slots = places(pages, page, T)
    f = cuda.rope.rope_frequencies(R) if R else None
    positions = torch.randint(0, 100000, (T,), device="cuda", generator=g)
    more = dict(positions=positions, frequencies=f.cuda(), interleaved=interleaved, scale=0.75, q=q if H else None) if R else {}
    out = cuda.kvcache.kv_write(cache, slots if T % 2 else slots.long(), k, v, **more)
    untouched(before, cache, slots)
    if H and R:
        close(out, q, positions, f, interleaved=interleaved, scale=0.75)
    else:
        assert out is None
    for i, x in enumerate((k, v)):
        got = rows_at(cache[i], slots)
        want, off = turned(x, positions, f if i == 0 else None, interleaved)
        if cache.k_scale is not None:
            stored_close(got, rows_at(cache[2 + i], slots), want, off)
        elif i == 1 or not R:
            assert got.equal(x)
        else:
            close(got, x, positions, f, interleaved=interleaved, scale=0.75)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_anywhere_and_in_place(cuda, store, shift):
    """Heads that start at any element; queries turned in place; slots of 0."""
    import torch

    from test_rope_gpu import close
    dtype = getattr(torch, store) if store.endswith("float16") else torch.float16
    T, H, KVH, D, page = 19, 3, 2, 64, 16
    base = torch.randn(T, (H + 2 * KVH) * D + 8 + shift, device="cuda").to(dtype)
    part = base[:, shift:shift + (H + 2 * KVH) * D].unflatten(1, (H + 2 * KVH, D))
    q, k, v = part.split((H, KVH, KVH), 1)
    cache = filled(cuda, 4, KVH, page, D, store)
    before = [None if t is None else t.clone() for t in cache]
    slots = places(4, page, T, 1)
    slots[::3] = 0
    live = slots > 0
    for R, interleaved in ((64, False), (12, False), (12, True)):
        f, positions = cuda.rope.rope_frequencies(R), torch.arange(T, device="cuda") + 3
        was, kept = q.clone(), base.clone()
        out = cuda.kvcache.kv_write(cache, slots, k, v, q=q, positions=positions, frequencies=f.cuda(), interleaved=interleaved, scale=0.75, out_q=q)
        assert out is q
        close(q, was, positions, f, interleaved=interleaved, scale=0.75)
        q.copy_(was)
        assert base.equal(kept)
        untouched(before, cache, slots[live])
        want, off = turned(k, positions, f, interleaved)
        got = rows_at(cache.k, slots[live])
        if cache.k_scale is None:
            close(got, k[live], positions[live], f, interleaved=interleaved, scale=0.75)
        else:
            stored_close(got, rows_at(cache.k_scale, slots[live]), want[live], off[live])


@pytest.mark.parametrize("store", ["float8_e4m3fn", "int8"])
def test_rounding_to_codes(cuda, store):
    """Ties go to even, the largest element gets the largest code, and rows of zeros, tiny and huge numbers, infinities and NaN."""
    import torch
    c = 127 if store == "int8" else 448
    x = torch.zeros(8, 1, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 0, :5] = torch.tensor([c / 2 if c == 448 else 63.5, 0.5, 1.5, -2.5, 0.75])
    x[0, 0, 5] = float(c)
    if c == 448:
        x[0, 0, :5] = torch.tensor([17.0, 19.0, -21.0, 2.0 ** -9 * 0.5, 2.0 ** -9 * 1.5])  # between 16, 18, 20, 22; between 0, 2^-9, 2^-8
    x[2, 0, :3] = torch.tensor([2.0 ** -101, -(2.0 ** -102), 2.0 ** -110])
    x[3, 0, :3] = torch.tensor([2.0 ** -100, -(2.0 ** -101), 0.0])
    x[4, 0, :3] = torch.tensor([3e38, -1.5e38, 1e30])
    x[5, 0, 7] = float("inf")
    x[6, 0, 9] = float("nan")
    x[6, 0, 10] = float("inf")
    x[7, 0] = torch.linspace(-3, 3, 64).bfloat16()
    cache = cuda.kvcache.kv_cache(1, 1, 16, 64, getattr(torch, store))
    slots = torch.arange(1, 9, device="cuda", dtype=torch.int32)
    cuda.kvcache.kv_write(cache, slots, x, x)
    code, scale = rows_at(cache.k, slots).float()[:, 0], rows_at(cache.k_scale, slots)[:, 0]
    assert code[:5].equal(rows_at(cache.v, slots).float()[:5, 0]) and cache.k_scale[0, 0, :5].equal(cache.v_scale[0, 0, :5])
    if c == 127:  # the scale is 1
        assert code[0, :6].tolist() == [64.0, 0.0, 2.0, -2.0, 1.0, 127.0] and float(scale[0]) == 1.0
    else:
        assert code[0, :6].tolist() == [16.0, 20.0, -20.0, 0.0, 2.0 ** -8, 448.0] and float(scale[0]) == 1.0
    assert (code[1] == 0).all() and scale[1] == 0 and (code[2] == 0).all() and scale[2] == 0
    assert code[3, 0] == c and float(scale[3]) > 0
    assert code[4, 0] == c and abs(float(code[4, 1]) + c / 2) <= (1 if c == 127 else 8)
    assert scale[5] == float("inf") and scale[6].isnan() and (code[5] == 0).all() and (code[6] == 0).all()
    stored_close(rows_at(cache.k, slots)[3:5], rows_at(cache.k_scale, slots)[3:5], x[3:5].double())
    stored_close(rows_at(cache.k, slots)[7:], rows_at(cache.k_scale, slots)[7:], x[7:].double())
    table, lengths = torch.ones(1, 1, device="cuda", dtype=torch.int32), torch.tensor([8], device="cuda", dtype=torch.int32)
    K, _ = cuda.kvcache.kv_read(cache, table, lengths, 8, dtype=torch.bfloat16)
    assert K[0, 0, 5].isnan().all() and K[0, 0, 6].isnan().all() and (K[0, 0, 1:3] == 0).all()


@pytest.mark.parametrize("B,KVH,D,page,lengths,seq", [(1, 1, 64, 16, [1], 1), (3, 2, 64, 16, [0, 17, 40], 40), (2, 3, 128, 64, [64, 65], 130),
                                                      (4, 8, 128, 32, [500, 1, 31, 33], 500), (2, 1, 64, 1024, [1024, 1500], 1400), (2, 2, 128, 16, [0, 0], 5)])
@pytest.mark.parametrize("store", STORES)
def test_read(cuda, B, KVH, D, page, lengths, seq, store):
    import torch
    width = -(-max(max(lengths), 1) // page)
    pages = B * width + 2
    cache = filled(cuda, pages, KVH, page, D, store)
    table = (torch.randperm(pages, device="cuda")[:B * width] + 1).int().view(B, width)
    for b, n in enumerate(lengths):
        table[b, -(-n // page):] = 0  # pages that are not needed have no number
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    dtypes = [getattr(torch, store)] if cache.k_scale is None else [torch.float16, torch.bfloat16]
    for dtype in dtypes:
        got = cuda.kvcache.kv_read(cache, table, n, seq, dtype=dtype)
        for i in range(2):
            assert got[i].shape == (B, KVH, seq, D) and got[i].dtype == dtype
            for b in range(B):
                m = min(lengths[b], seq)
                at = table[b, :-(-m // page)].long() - 1
                x = cache[i][at]
                if cache.k_scale is not None:
                    x = (x.float() * cache[2 + i][at][..., None]).to(dtype)
                x = x.transpose(0, 1).flatten(1, 2)[:, :m]
                assert got[i][b, :, :m].equal(x) and (got[i][b, :, m:] == 0).all()
    cuda.check_device_status(0)


def test_bad_indices(cuda):
    """Slots, pages and lengths out of range are reported, and nothing else is written or read for them."""
    import torch
    cache = filled(cuda, 3, 1, 16, 64, "float16")
    before = [t.clone() for t in cache[:2]]
    k = torch.randn(4, 1, 64, device="cuda").half()
    for bad in (-1, 49, 2 ** 31 - 1, -2 ** 31):
        slots = torch.tensor([bad, 5, 0, bad], device="cuda", dtype=torch.int64)
        cuda.kvcache.kv_write(cache, slots, k, k)
        with pytest.raises(cuda.CtbError, match="out-of-range"):
            cuda.check_device_status(0)
        untouched(before, cache[:2], torch.tensor([5], device="cuda"))
        assert rows_at(cache.k, torch.tensor([5], device="cuda"))[0].equal(k[1])
    cuda.check_device_status(0)
    for ids, length, nan in (([1, 4], 32, slice(16, 32)), ([0, 2], 20, slice(0, 16)), ([-7, 2], 32, slice(0, 16)), ([1, 2], 33, slice(32, 40)),
                             ([1, 2], -1, slice(0, 40))):
        K, V = cuda.kvcache.kv_read(cache, torch.tensor([ids], device="cuda", dtype=torch.int32), torch.tensor([length], device="cuda", dtype=torch.int32), 40)
        with pytest.raises(cuda.CtbError, match="out-of-range"):
            cuda.check_device_status(0)
        assert K[0, 0, nan].isnan().all() and V[0, 0, nan].isnan().all() and not K[0, 0].isnan().all(-1)[list(set(range(40)) - set(range(40)[nan]))].any()


def test_pages_of_one_allocation(cuda):
    """k and v as views of one array; pages lie apart."""
    import torch
    both = torch.zeros(6, 2, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    cache = cuda.kvcache.KvCache(both[:, 0], both[:, 1])
    k, v = torch.randn(30, 2, 64, device="cuda").bfloat16(), torch.randn(30, 2, 64, device="cuda").bfloat16()
    slots = places(6, 16, 30, 3)
    cuda.kvcache.kv_write(cache, slots, k, v)
    assert rows_at(cache.k, slots).equal(k) and rows_at(cache.v, slots).equal(v)
    scales = torch.zeros(6, 2, 2, 16, device="cuda")
    codes = torch.zeros(6, 2, 2, 16, 64, device="cuda", dtype=torch.int8)
    cache = cuda.kvcache.KvCache(codes[:, 0], codes[:, 1], scales[:, 0], scales[:, 1])
    cuda.kvcache.kv_write(cache, slots, k, v)
    stored_close(rows_at(cache.k, slots), rows_at(cache.k_scale, slots), k.double())
    stored_close(rows_at(cache.v, slots), rows_at(cache.v_scale, slots), v.double())
    table = torch.arange(1, 7, device="cuda", dtype=torch.int32)[None]
    K, V = cuda.kvcache.kv_read(cache, table, torch.tensor([96], device="cuda", dtype=torch.int32), 96, dtype=torch.bfloat16)
    want = (codes[:, 1].float() * scales[:, 1][..., None]).bfloat16().transpose(0, 1).flatten(1, 2)
    assert V[0].equal(want)


def test_one_token_of_any_stride(cuda):
    import torch
    from test_rope_gpu import close
    x = torch.randn(1, 3, 64, device="cuda").half()
    far = x.as_strided((1, 3, 64), (2 ** 40, 64, 1))
    cache = cuda.kvcache.kv_cache(1, 3, 16, 64, torch.float16)
    f, one = cuda.rope.rope_frequencies(64).cuda(), torch.ones(1, device="cuda", dtype=torch.int32)
    out = cuda.kvcache.kv_write(cache, one, far, far, q=far, positions=one, frequencies=f)
    close(out, x, one, f.cpu())
    close(cache.k[0, :, 0][None], x, one, f.cpu())
    assert cache.v[0, :, 0].equal(x[0])


@pytest.mark.parametrize("store", STORES)
def test_streams_and_graphs(cuda, store):
    """Writes and reads of caches of their own on several streams, captured ones among them: each gives what it gives alone."""
    import torch
    f = cuda.rope.rope_frequencies(128).cuda()
    cases = []
    for T in (5, 900, 2100):
        q, k, v = (torch.randn(T, h, 128, device="cuda").bfloat16() for h in (8, 2, 2))
        pages = -(-T // 32)
        cache = cuda.kvcache.kv_cache(pages, 2, 32, 128, getattr(torch, store if store != "float16" else "bfloat16"))
        args = dict(slots=torch.arange(1, T + 1, device="cuda"), k=k, v=v, q=q, positions=torch.arange(T, device="cuda"), frequencies=f, out_q=torch.empty_like(q))
        cases.append((cache, args, torch.arange(1, pages + 1, device="cuda", dtype=torch.int32)[None], torch.tensor([T], device="cuda", dtype=torch.int32), T))

    def run(cache, args, table, length, T):
        out = cuda.kvcache.kv_write(cache, **args)
        return (out, *cuda.kvcache.kv_read(cache, table, length, T, dtype=torch.bfloat16))

    want = [[t.clone() for t in run(*c)] for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(*c))
        graphs.append(g)
    for cache, args, *_ in cases:
        for t in (*cache, args["out_q"]):
            if t is not None:
                t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                got.append((i, run(*cases[i])))
    torch.cuda.synchronize()
    for i, parts in got + list(enumerate(outs)):
        assert all(a.equal(b) for a, b in zip(parts, want[i]))
    cases[0][1]["k"].normal_()  # a graph goes by what its inputs hold at its replay
    cases[0][1]["positions"].add_(100)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(a.equal(b) for a, b in zip([t.clone() for t in outs[0]], run(*cases[0])))


def test_refusals(cuda):
    import torch
    kc = cuda.kvcache
    cache = kc.kv_cache(3, 2, 16, 64, torch.float16)
    k = torch.randn(4, 2, 64, device="cuda").half()
    slots, f = torch.arange(1, 5, device="cuda"), cuda.rope.rope_frequencies(64).cuda()
    pos = torch.arange(4, device="cuda")
    n8 = torch.zeros(3, 2, 16, 64, device="cuda", dtype=torch.int8)
    n16 = torch.zeros(3, 2, 16, 64, device="cuda", dtype=torch.float16)
    scale = torch.zeros(3, 2, 16, device="cuda")
    odd = torch.zeros(3 * 2 * 16 * 64 + 1, device="cuda", dtype=torch.float16)[1:].view(3, 2, 16, 64)
    calls = [(lambda: kc.kv_write(cache, slots, k.float(), k.float()), "implemented"), (lambda: kc.kv_write(cache, slots, k.bfloat16(), k.bfloat16()), "own type"),
             (lambda: kc.kv_write(cache, slots, k, k[:, :1]), "v: expected"), (lambda: kc.kv_write(cache, slots, k[:3], k), "v: expected"),
             (lambda: kc.kv_write(cache, slots[:3], k, k), "slots"), (lambda: kc.kv_write(cache, slots.float(), k, k), "int32 or int64"),
             (lambda: kc.kv_write(cache, slots, k[..., :32], k[..., :32]), "k: expected"), (lambda: kc.kv_write(cache, slots, k, k, q=k), "positions"),
             (lambda: kc.kv_write(cache, slots, k, k, positions=pos), "come together"), (lambda: kc.kv_write(cache, slots, k, k, out_q=k), "comes with q"),
             (lambda: kc.kv_write(cache, slots, k, k, q=k, positions=pos, frequencies=f.float()), "float64"),
             (lambda: kc.kv_write(cache, slots, k, k, positions=pos, frequencies=torch.cat((f, f))), "rotary"),
             (lambda: kc.kv_write(cache, slots, k, k, positions=pos, frequencies=f, scale=float("inf")), "not finite"),
             (lambda: kc.kv_write(kc.KvCache(n16, n16[:2]), slots, k, k), "alike"), (lambda: kc.kv_write(kc.KvCache(n8, n8), slots, k, k), "f32 tensor"),
             (lambda: kc.kv_write(kc.KvCache(n16, n16, scale, scale), slots, k, k), "no scales"),
             (lambda: kc.kv_write(kc.KvCache(n8, n8, scale, scale[:, :1]), slots, k, k), "Pages"),
             (lambda: kc.kv_write(kc.KvCache(odd, odd), slots, k, k), "16-byte aligned"),
             (lambda: kc.kv_write(kc.KvCache(n16.transpose(1, 2), n16.transpose(1, 2)), slots, k, k), "page must be dense"),
             (lambda: kc.kv_write(kc.kv_cache(3, 2, 24, 64, torch.float16), slots, k, k), "page_size"),
             (lambda: kc.kv_write(kc.kv_cache(3, 2, 8, 64, torch.float16), slots, k, k), "page_size"),
             (lambda: kc.kv_write(kc.kv_cache(3, 2, 16, 96, torch.float16), slots, k[..., :1].expand(4, 2, 96).contiguous(), k[..., :1].expand(4, 2, 96).contiguous()),
              "64 and 128"),
             (lambda: kc.kv_write(cache, slots, k.cpu(), k.cpu()), "CUDA tensor"), (lambda: kc.kv_cache(3, 2, 16, 64, torch.float32), "elements of"),
             (lambda: kc.kv_cache(0, 2, 16, 64, torch.float16), "non-positive")]
    table, lengths = torch.ones(2, 3, device="cuda", dtype=torch.int32), torch.ones(2, device="cuda", dtype=torch.int32)
    eight = kc.KvCache(n8, n8.clone(), scale, scale.clone())
    calls += [(lambda: kc.kv_read(cache, table.long(), lengths, 4), "int32"), (lambda: kc.kv_read(cache, table, lengths[:1], 4), "lengths"),
              (lambda: kc.kv_read(cache, table, lengths, -1), "negative"), (lambda: kc.kv_read(cache, table.t(), lengths, 4), "contiguous rows"),
              (lambda: kc.kv_read(eight, table, lengths, 4), "needs a dtype"), (lambda: kc.kv_read(eight, table, lengths, 4, dtype=torch.float32), "implemented"),
              (lambda: kc.kv_read(cache, table, lengths, 4, dtype=torch.bfloat16), "own type"), (lambda: kc.kv_read(cache, table, lengths.cpu(), 4), "expected a tensor on")]
    for call, word in calls:
        with pytest.raises(cuda.CtbError, match=word):
            call()
    assert (cache.k == 0).all()
    empty = k[:0]
    assert kc.kv_write(cache, slots[:0], empty, empty) is None
    assert kc.kv_read(cache, table, lengths, 0)[0].shape == (2, 2, 0, 64) and kc.kv_read(cache, table[:0], lengths[:0], 4)[0].shape == (0, 2, 4, 64)
    K, _ = kc.kv_read(cache, table, lengths, 4, occupancy=2)
    assert K.shape == (2, 2, 4, 64)
