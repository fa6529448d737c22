"""Token log probabilities, entropies, alternatives and their gradient against f64.

Tolerances.  An exponent t = (x - max) log2(e) / temperature carries three f32 roundings, |t| 2^-22.4 in all, and ex2.approx a relative 2^-22:
a power e^z is off by 2^-22 (1 + |z|) relative, sums of powers by no more than the mean of that (and 2^-22 for the additions, pairwise over
threads), a logarithm of a sum by the same amount absolutely.  With |z| <= 64 in these tests and two roundings of the result:
    lse, log probabilities, entropy:  |error| <= 2^-18 + 2^-23 |result|        (an entropy has 2^-18 for w / s once more)
A probability in the gradient comes from t = x c - lse log2(e), off by 2^-23 (|x| c + |lse| log2(e)) <= 2^-16 in the exponent for |z|, |lse| <=
64: |error| <= 2^-16 p (|G| + |g_H| (|log p| + H)) / temperature + 2^-22 |sum of the gradients that meet at v| / temperature + half a
step of the type.  That counts what the exponent's error does to p; log p in the bracket has the same error absolutely, which adds 2^-16 p |g_H| /
temperature (with one element p = 1, log p = H = 0, and t = 2^-24 |x| c alone is left of it).  G and what meets at v are f32 sums of up to 33
gradients that may cancel: off by 33 2^-24 < 2^-18 of the sum of their magnitudes.
"""
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")


def make(T, V, dtype, seed=0, shift=0, ld=None, scale=3.0):
    """[T, V] rows with stride ld (V) that start `shift` elements behind a 16-byte boundary."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or V
    flat = torch.full((T * ld + 16,), float("nan"), device="cuda", dtype=getattr(torch, dtype))
    x = flat[shift:shift + T * ld].view(T, ld)[:, :V]
    x.copy_(torch.randn(T, V, device="cuda", generator=g) * scale)
    return x


def reference(x, tokens, top, temperature):
    """(logprobs, entropy, lse, top_logprobs, top_ids) in f64, rows with token 0 as 0."""
    import torch
    z = x.double() / temperature
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, p).sum(1)
    live = torch.ones(len(x), dtype=torch.bool, device=x.device) if tokens is None else tokens != 0
    zero = lambda t: torch.where(live.view(-1, *[1] * (t.dim() - 1)), t, torch.zeros_like(t))  # noqa: E731
    lp = None if tokens is None else zero(logp.gather(1, (tokens.long() - 1).clamp(min=0)[:, None])[:, 0])
    ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
    return lp, zero(entropy), zero(torch.logsumexp(z, 1)), zero(logp.gather(1, ids)), zero(ids + 1).int()


def close(got, want):
    import torch
    assert got.dtype == torch.float32 and got.shape == want.shape
    same = (got.double() == want) | (got.isnan() & want.isnan())
    err = (got.double() - want).abs()
    assert (same | (err <= 2.0 ** -17 + 2.0 ** -23 * want.abs())).all(), err[~same].max()


def check(cuda, x, tokens, top, temperature=1.0):
    r = cuda.logprobs.token_logprobs(x, tokens, top=top, temperature=temperature)
    want = reference(x, tokens, top, temperature)
    for got, w in zip(r[:3], want[:3]):
        if w is not None:
            close(got, w)
    if top:
        assert r.top_ids.equal(want[4])
        close(r.top_logprobs, want[3])
    return r


SHAPES = [(1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (3, 33), (700, 100), (2, 1000), (1, 4097), (600, 4096), (3, 8191), (9, 8192), (2, 8193),
          (7, 20000), (1, 50001), (40, 50001), (700, 9001), (2, 131072), (1, 262147), (150, 33000)]


@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward(cuda, T, V, dtype):
    import torch
    for k, (shift, temperature) in enumerate(((0, 1.0), (1, 0.7), (5, 1.9))):
        x = make(T, V, dtype, seed=T + V + k, shift=shift, ld=V + 3 * (k == 2))
        tokens = torch.randint(1, V + 1, (T,), device="cuda", dtype=torch.int32 if k == 1 else torch.int64)
        if k == 2 and T > 2:
            tokens[::3] = 0
        for top in (0, min(V, 1), min(V, 20), min(V, 32)):
            check(cuda, x, tokens if k < 2 or top else None, top, temperature)
    cuda.check_device_status(0)


@pytest.mark.parametrize("V", [40, 1000, 8200, 50001, 200003])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_and_equal_values(cuda, V, dtype):
    """Rows with nearly all masked, by -inf or by the lowest value, with equal values throughout or in runs, all masked, with NaN and infinity;
    few rows, which are cut into parts, and many."""
    import torch
    inf = float("inf")
    low = torch.finfo(getattr(torch, dtype)).min
    for T in (12, 700 if V < 60000 else 12):
        x = make(T, V, dtype, seed=V, shift=3)
        x[0] = 1.5
        x[1] = -inf
        x[1, 3::V // 4] = 0.5
        x[2] = low
        x[2, V - 5:] = 0.0
        x[3] = -inf
        x[3, V // 2] = 2.0
        x[4] = torch.round(x[4])
        x[5] = low
        x[6] = torch.clamp(x[6], max=0.0)
        x[7, :V // 2] = -inf
        x[8, V // 3:] = -inf
        tokens = torch.randint(1, V + 1, (T,), device="cuda")
        tokens[1], tokens[3] = 4, V // 2 + 1
        tokens[7] = V
        check(cuda, x, tokens, min(V, 32))
        check(cuda, x, tokens, 5)
        x[9, 0] = inf
        x[10] = -inf
        x[11, V // 2] = float("nan")
        r = cuda.logprobs.token_logprobs(x, tokens, top=7)
        for t in (r.logprobs, r.entropy, r.lse, r.top_logprobs):
            assert t[[9, 11]].isnan().all() and not t[:9].isnan().any()
        assert r.logprobs[10].isnan() and r.entropy[10].isnan() and r.lse[10] == -inf and r.top_logprobs[10].isnan().all()
        assert (r.top_ids >= 0).all() and (r.top_ids <= V).all()
    cuda.check_device_status(0)


@pytest.mark.parametrize("V", [9000, 50001, 150000])
@pytest.mark.parametrize("dtype", TYPES)
def test_ordered_rows(cuda, V, dtype):
    """Ascending and descending rows and saw teeth: every element above all before it, lists that overflow."""
    import torch
    for T in (4, 640):
        up = torch.linspace(-20, 20, V, device="cuda")
        x = torch.stack([up, -up, up[torch.arange(V, device="cuda") * 7919 % V], up.abs()]).to(getattr(torch, dtype)).repeat(T // 4, 1)
        tokens = torch.randint(1, V + 1, (T,), device="cuda")
        for top in (1, 20, 32):
            check(cuda, x, tokens, top)


def gradients(x, tokens, ids, g0, gh, gt, temperature):
    """(gradient, tolerance without the type's rounding) by the formula in f64; x [T, V] f64."""
    import torch
    live = tokens != 0
    at = (tokens.long() - 1).clamp(min=0)[:, None]
    logp = torch.log_softmax(x / temperature, 1)
    p = logp.exp()
    logp = torch.where(p > 0, logp, torch.zeros_like(p))
    h = -(p * logp).sum(1, keepdim=True)
    total, direct = torch.zeros_like(h), torch.zeros_like(p)
    sizes, meeting = torch.zeros_like(h), torch.zeros_like(p)
    if g0 is not None:
        sizes = sizes + g0.double().abs()[:, None]
        meeting.scatter_add_(1, at, g0.double().abs()[:, None])
        total = total + g0.double()[:, None]
        direct.scatter_add_(1, at, g0.double()[:, None])
    if gt is not None:
        total = total + gt.double().sum(1, keepdim=True)
        sizes = sizes + gt.double().abs().sum(1, keepdim=True)
        meeting.scatter_add_(1, (ids.long() - 1).clamp(min=0), gt.double().abs())
        direct.scatter_add_(1, (ids.long() - 1).clamp(min=0), gt.double())
    ge = torch.zeros_like(h) if gh is None else gh.double()[:, None]
    d = (direct - p * (total + ge * (logp + h))) / temperature
    tol = 2.0 ** -16 * p * (total.abs() + ge.abs() * (logp.abs() + h + 1)) + 2.0 ** -22 * direct.abs()
    tol = (tol + 2.0 ** -18 * (p * sizes + meeting)) / temperature
    return torch.where(live[:, None], d, torch.zeros_like(d)), tol


def close_gradient(got, want, tol):
    import torch
    info = torch.finfo(got.dtype)
    step = info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2  # half a step, also below the normal numbers
    err = (got.double() - want).abs()
    assert (err <= tol + step + info.eps * tol).all(), (err - tol - step).max()


@pytest.mark.parametrize("T,V", [(1, 1), (3, 7), (2, 1000), (300, 129), (5, 8193), (2, 50001), (170, 50001), (1, 262147)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient(cuda, T, V, dtype):
    import torch
    ops = cuda.logprobs
    for k, temperature in enumerate((1.0, 0.7)):
        x = make(T, V, dtype, seed=T + V, shift=k * 3, ld=V + 5 * k)
        tokens = torch.randint(1, V + 1, (T,), device="cuda")
        if k and T > 2:
            tokens[1::3] = 0
            x[1] = float("nan")  # padding is not read
        top = min(V, 5)
        r = ops.token_logprobs(x, tokens, top=top, temperature=temperature)
        tokens = torch.where((torch.arange(T, device="cuda") % 4 == 3) & (tokens != 0), r.top_ids[:, 0], tokens)  # an alternative is the token
        g0, gh, gt = torch.randn(T, device="cuda"), torch.randn(T, device="cuda"), torch.randn(T, top, device="cuda")
        x64 = torch.where((tokens != 0)[:, None], x.double(), 0.0)
        for a, b, c in ((g0, gh, gt), (g0, None, None), (None, gh, None), (None, None, gt), (None, None, None)):
            want, tol = gradients(x64, tokens, r.top_ids, a, b, c, temperature)
            got = ops.token_logprobs_bwd(x, tokens, r.lse, r.entropy, a, b, r.top_ids, c, temperature)
            assert got.dtype == x.dtype
            close_gradient(got, want, tol)
        # into columns of a larger array, and over the logits
        want = ops.token_logprobs_bwd(x, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature)
        wide = torch.full((T, V + 9), 7.0, device="cuda", dtype=x.dtype)
        ops.token_logprobs_bwd(x, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature, out=wide[:, 2:2 + V])
        assert wide[:, 2:2 + V].equal(want) and (wide[:, :2] == 7).all() and (wide[:, 2 + V:] == 7).all()
        over = make(T, V, dtype, seed=T + V, shift=k * 3, ld=V + 5 * k)
        assert ops.token_logprobs_bwd(over, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature, out=over).equal(want)
    cuda.check_device_status(0)


def test_gradient_against_differences(cuda):
    import torch
    T, V, step = 4, 37, 1e-5
    x = make(T, V, "float32", seed=3)
    tokens = torch.tensor([1, 37, 5, 9], device="cuda")
    ops, top, tau = cuda.logprobs, 3, 0.8
    r = ops.token_logprobs(x, tokens, top=top, temperature=tau)
    g0, gh, gt = torch.randn(T, device="cuda"), torch.randn(T, device="cuda"), torch.randn(T, top, device="cuda")
    got = ops.token_logprobs_bwd(x, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, tau)

    def value(x64):
        lp, h, _, _, _ = reference(x64, tokens, top, tau)
        alternatives = torch.log_softmax(x64 / tau, 1).gather(1, r.top_ids.long() - 1)
        return lp * g0 + h * gh + (alternatives * gt).sum(1)
    for v in range(V):
        e = torch.zeros(V, device="cuda", dtype=torch.float64)
        e[v] = step
        slope = (value(x.double() + e) - value(x.double() - e)) / (2 * step)
        # a central difference is off by step^2 / 6 of the third derivative (< 100 here) and 2^-52 |value| / step
        assert ((got[:, v].double() - slope).abs() <= 1e-8 + 2.0 ** -16 * (1 + slope.abs())).all()


def test_masked_gradient(cuda):
    """Masked elements get 0; a masked row gives NaN as in the forward pass, and only there."""
    import torch
    inf = float("inf")
    x = make(6, 5000, "bfloat16", seed=1)
    x[:, ::2] = -inf
    x[3] = -inf
    tokens = torch.full((6,), 2, device="cuda")
    r = cuda.logprobs.token_logprobs(x, tokens)
    one = torch.ones(6, device="cuda")
    d = cuda.logprobs.token_logprobs_bwd(x, tokens, r.lse, r.entropy, one, one)
    keep = [0, 1, 2, 4, 5]
    assert (d[keep][:, ::2] == 0).all() and d[keep].isfinite().all() and d[3].isnan().any()
    want, tol = gradients(x[keep].double(), tokens[keep], None, one[keep], one[keep], None, 1.0)
    close_gradient(d[keep], want, tol)


def test_bad_tokens_are_reported(cuda):
    import torch
    x = make(4, 1000, "float32")
    tokens = torch.tensor([1, 1001, -1, 7], device="cuda")
    r = cuda.logprobs.token_logprobs(x, tokens, top=2)
    with pytest.raises(cuda.CtbError, match="out-of-range index"):
        cuda.check_device_status(0)
    assert r.logprobs[1:3].isnan().all() and not r.logprobs[[0, 3]].isnan().any() and not r.lse.isnan().any()
    d = cuda.logprobs.token_logprobs_bwd(x, tokens, r.lse, r.entropy, torch.ones(4, device="cuda"))
    with pytest.raises(cuda.CtbError, match="out-of-range index"):
        cuda.check_device_status(0)
    assert (d[1:3] == 0).all() and (d[[0, 3]] != 0).any()
    cuda.check_device_status(0)


def test_offsets_beyond_32_bits(cuda):
    import torch
    T, V = 16500, 131072
    x = torch.zeros(T, V, device="cuda", dtype=torch.bfloat16)
    last = make(2, V, "bfloat16", seed=5)
    x[-2:] = last
    tokens = torch.zeros(T, device="cuda", dtype=torch.int64)
    tokens[-2:] = torch.tensor([5, V], device="cuda")
    tokens[0] = 3
    r = cuda.logprobs.token_logprobs(x, tokens, top=4)
    want = reference(last, tokens[-2:], 4, 1.0)
    close(r.logprobs[-2:], want[0])
    close(r.entropy[-2:], want[1])
    assert r.top_ids[-2:].equal(want[4]) and (r.top_ids[1:-2] == 0).all() and r.top_ids[0].tolist() == [1, 2, 3, 4]
    g = torch.ones(T, device="cuda")
    cuda.logprobs.token_logprobs_bwd(x, tokens, r.lse, r.entropy, g, out=x)
    want, tol = gradients(last.double(), tokens[-2:], None, g[-2:], None, None, 1.0)
    close_gradient(x[-2:], want, tol)
    assert x[1:-2].abs().max() == 0


def test_repeatable_and_on_streams(cuda):
    """Bitwise the same on every call, on several streams at once and from replayed graphs beside eager calls."""
    import torch
    ops = cuda.logprobs
    xs = [make(3, 120001, "bfloat16", seed=1), make(64, 30000, "float32", seed=2), make(700, 5000, "float16", seed=3)]
    tokens = [torch.randint(1, x.shape[1] + 1, (len(x),), device="cuda") for x in xs]

    def run(i):
        r = ops.token_logprobs(xs[i], tokens[i], top=20)
        return list(r) + [ops.token_logprobs_bwd(xs[i], tokens[i], r.lse, r.entropy, r.lse, r.entropy)]
    want = [run(i) for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(6)]
    graphs, captured = [], []
    for i in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured.append(run(i))
        graphs.append(g)
    got = []
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                if k < 3:
                    got.append((k, run(k)))
                else:
                    graphs[k - 3].replay()
    torch.cuda.synchronize()
    for k, r in got + list(enumerate(captured)):
        assert all(a.equal(b) for a, b in zip(r, want[k]))
    cuda.check_device_status(0)


@pytest.mark.parametrize("top", [0, 5])
def test_more_rows_than_counters(cuda, top):
    """Beyond 4096 rows there is no counter per row: rows in several launches, or whole."""
    import torch
    T, V = 4100, 17001
    x = make(T, V, "bfloat16", seed=8, shift=1)
    tokens = torch.randint(0, V + 1, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    tokens[::7] = 0
    check(cuda, x, tokens, top)
    x = make(9000, 40, "float32", seed=9)
    check(cuda, x, tokens[:1].clamp(min=1, max=40).expand(9000).contiguous(), top)


@pytest.mark.parametrize("T,V", [(1, 262144), (8, 131073), (40, 33333)])
@pytest.mark.parametrize("top", [1, 19, 31, 32])
def test_lists_of_parts(cuda, T, V, top):
    """Rows cut into many parts: the best elements in one part, in the last elements, spread, alike, or fewer than `top` at all."""
    import torch
    for dtype in TYPES:
        x = make(T, V, dtype, seed=top, shift=3)
        tokens = torch.full((T,), V, device="cuda", dtype=torch.int32)
        check(cuda, x, tokens, top)
        x[:, V // 2:V // 2 + 40] += 16
        x[0, -7:] += 40
        check(cuda, x, tokens, top)
        x[:, ::V // 64] = 60.0  # alike, in every part
        check(cuda, x, tokens, top)
        x.fill_(-float("inf"))
        x[:, V - 3:] = 1.0
        check(cuda, x, tokens, top)


def test_refusals(cuda):
    import torch
    ops, lib = cuda.logprobs, cuda._lib
    x = make(4, 1000, "float32")
    tokens = torch.ones(4, device="cuda", dtype=torch.int64)

    def refused(status, word, f):
        with pytest.raises(cuda.CtbError, match=word) as e:
            f()
        assert e.value.status == status
    refused(lib.UNSUPPORTED, "top must lie", lambda: ops.token_logprobs(x, tokens, top=33))
    refused(lib.BAD_ARG, "top must lie", lambda: ops.token_logprobs(x[:, :5], tokens, top=6))
    refused(lib.BAD_ARG, "top must lie", lambda: ops.token_logprobs(x, tokens, top=-1))
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-7):
        refused(lib.BAD_ARG, "temperature", lambda: ops.token_logprobs(x, tokens, temperature=t))
    refused(lib.BAD_ARG, "int32 or int64", lambda: ops.token_logprobs(x, tokens.float()))
    refused(lib.BAD_ARG, "shape", lambda: ops.token_logprobs(x, tokens[:3]))
    refused(lib.BAD_ARG, "contiguous rows", lambda: ops.token_logprobs(x.t(), tokens))
    refused(lib.BAD_ARG, "element type", lambda: ops.token_logprobs(x.double(), tokens))
    refused(lib.BAD_ARG, "expected a tensor on", lambda: ops.token_logprobs(x, tokens.cpu()))
    refused(lib.BAD_ARG, "CUDA tensor", lambda: ops.token_logprobs(x.cpu(), tokens))
    r = ops.token_logprobs(x, tokens, top=3)
    g = torch.ones(4, device="cuda")
    refused(lib.BAD_ARG, "d_logprobs without tokens", lambda: ops.token_logprobs_bwd(x, None, r.lse, r.entropy, g))
    refused(lib.BAD_ARG, "needs entropy", lambda: ops.token_logprobs_bwd(x, tokens, r.lse, None, g, g))
    refused(lib.BAD_ARG, "needs top_ids", lambda: ops.token_logprobs_bwd(x, tokens, r.lse, None, d_top_logprobs=r.top_logprobs))
    refused(lib.BAD_ARG, "dense", lambda: ops.token_logprobs_bwd(x, tokens, r.lse, None, g[:1].expand(4)))
    refused(lib.BAD_ARG, "out must have", lambda: ops.token_logprobs_bwd(x, tokens, r.lse, None, g, out=x.half()))
    buf = torch.zeros(5, 1000, device="cuda")
    refused(lib.BAD_ARG, "not overlap", lambda: ops.token_logprobs_bwd(buf[:4], tokens, r.lse, None, g, out=buf[1:]))
    flat = torch.zeros(8000, device="cuda")
    refused(lib.BAD_ARG, "not overlap", lambda: ops.token_logprobs_bwd(flat[:4000].view(4, 1000), tokens, r.lse, None, g,
                                                                       out=flat[500:4500].view(4, 1000)))
    side = torch.zeros(4, 2000, device="cuda")
    ops.token_logprobs_bwd(side[:, :1000], tokens, r.lse, None, g, out=side[:, 1000:])  # columns side by side
    empty = ops.token_logprobs(x[:0], tokens[:0], top=3)
    assert empty.lse.shape == (0,) and empty.top_ids.shape == (0, 3)
    assert ops.token_logprobs_bwd(x[:0], tokens[:0], empty.lse, empty.entropy, g[:0]).shape == (0, 1000)
    cuda.check_device_status(0)
