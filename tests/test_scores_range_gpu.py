"""Operators over rows of logits at the ends of their range: rows that start anywhere, large logits, small temperatures, rows that a mask
of any kind leaves empty.

Temperatures here are powers of two, the same number in f32 and f64.  What a row's shift or a temperature does to the exponents cancels
in differences from the row's maximum, which f32 holds to 2^-24 of themselves: the tolerances of test_logprobs_gpu.py and
test_distill_gpu.py hold whatever the magnitude.  Results beyond f32 are its infinities.
"""
import pytest

pytestmark = pytest.mark.gpu

from test_distill_gpu import close_loss, teacher  # noqa: E402
from test_logprobs_gpu import TYPES, check, close, close_gradient, gradients, make, reference  # noqa: E402


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("dtype", TYPES)
def test_lists_made_again_from_rows_that_start_anywhere(cuda, shift, dtype):
    """Ascending rows, whose list overflows, and rows of equal values: their first and last vectors are read element by element."""
    import torch
    V = 9003
    x = make(4, V, dtype, shift=shift, ld=V + 1)
    x[:2] = torch.linspace(-20, 20, V, device="cuda").to(x.dtype)
    x[2:] = 1.5
    check(cuda, x, torch.tensor([1, V, 1, V], device="cuda"), 32)


MAGNITUDES = (3e4, 1e9, 1e10, 3e12, 1e20, 1e29, 2e30, 3e38)


def shifted_rows(T, V, dtype, seed=0, shift=0):
    """Rows whose maximum is a large number: equal throughout, one element or half of the row above the rest, random but for a shift."""
    import torch
    x = make(T, V, dtype, seed=seed, shift=shift)
    most = torch.finfo(x.dtype).max
    row = 0
    for m in MAGNITUDES:
        for a in (m, -m):
            if m > most:
                a = most if a > 0 else -most
            x[row] = a
            x[row + 1] = -abs(a)
            x[row + 1, V // 3] = a
            x[row + 2] = a
            x[row + 2, V // 2:] = a * 2 if a < 0 and abs(a) * 2 < most else -abs(a)
            row += 3
    for a in (1e3, 1e4, -1e3, -1e4):
        x[row] += a
        row += 1
    x[row] = -float("inf")
    x[row, V // 2:] = -1e4
    x[row + 1] = -float("inf")
    x[row + 1, V - 1] = most
    return x, row + 2


@pytest.mark.parametrize("T,V", [(54, 1), (54, 70), (54, 9001), (900, 1025), (54, 70001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(cuda, T, V, dtype):
    import torch
    for temperature in (1.0, 2.0 ** -5, 2.0 ** -19, 2.0 ** 19):
        x, rows = shifted_rows(T, V, dtype, seed=V, shift=1)
        assert rows <= T
        tokens = torch.randint(1, V + 1, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
        for top in (0, min(V, 5)):
            r = cuda.logprobs.token_logprobs(x, tokens, top=top, temperature=temperature)
            want = reference(x, tokens, top, temperature)
            for got, w in zip(r[:3 if top == 0 else 4], want):
                inside = w.abs() < 3.4e38
                close(torch.where(inside, got, torch.zeros_like(got)), torch.where(inside, w, torch.zeros_like(w)))
                assert (inside | (got == torch.sign(w) * float("inf")) | (got.double().abs() > 3.3e38)).all()
            if top:
                assert r.top_ids.equal(want[4])
    cuda.check_device_status(0)


@pytest.mark.parametrize("shift", [3e3, -2e4, 1e5, 3e5, -6e5, 7e5, 1e6])
def test_shifted_rows_whose_maximum_rises(cuda, shift):
    """A thread's sums follow its maximum: what they are relative to is off by the rounding of a large product, and must be so throughout."""
    import torch
    for T, V in ((24, 39812), (700, 12001)):
        x = make(T, V, "float32", seed=5, scale=3.0) + shift
        x[::3] = x[::3].sort(dim=1).values
        tokens = torch.argmax(x, 1) + 1
        check(cuda, x, tokens, 0)
        check(cuda, x, tokens, 7)
        ids = torch.topk(x, 20, 1).indices.int() + 1
        values = torch.zeros(T, 20, device="cuda")
        for lse in (None, torch.full((T,), 4.0, device="cuda")):
            want = distillation(x, ids, values, lse, 1.0, tokens.float())[0]
            close_loss(cuda.distill.distill_fwd(x, ids, values, lse)[0], want)


def distillation(x, ids, values, lse, temperature, d_loss):
    """(loss, gradient, tolerance of the gradient) in f64; what the teacher's list leaves over by logarithms."""
    import torch
    used = ids > 0
    at = (ids.long() - 1).clamp(min=0)
    z = x.double() / temperature
    u = torch.where(used, values.double() / temperature, -float("inf"))
    log_q = u - (torch.logsumexp(u, 1, keepdim=True) if lse is None else lse.double()[:, None])
    q = log_q.exp()
    log_p = torch.log_softmax(z, 1)
    p = log_p.exp()
    loss = torch.where(q > 0, q * (log_q - log_p.gather(1, at)), 0.0).sum(1)
    g = (d_loss.double() / temperature)[:, None]
    qv = torch.zeros_like(p).scatter_add_(1, at, q)
    whole = torch.ones_like(g)
    rest = torch.zeros_like(p)
    if lse is not None:
        listed = torch.zeros_like(p).scatter_add_(1, at, used.double()) > 0
        left = (1 - q.sum(1, keepdim=True)).clamp(min=0)
        whole = q.sum(1, keepdim=True) + left
        others = z.masked_fill(listed, -float("inf"))
        most = others.amax(1, keepdim=True)  # apart from the sum, which f64 would lose beside 1e38 as well
        log_rest = (most - z.amax(1, keepdim=True)) + (others - most).exp().sum(1, keepdim=True).log() - (z - z.amax(1, keepdim=True)).exp().sum(1, keepdim=True).log()
        loss = loss + (torch.xlogy(left, left) - torch.where(left > 0, left * log_rest, 0.0))[:, 0]
        rest = left * torch.softmax(others, 1).nan_to_num(0.0)
    d = g * (whole * p - rest - qv)
    # see test_distill_gpu.py; and a power below 2^-126 counts as 0, of which the gradient takes at most g whole
    tol = g.abs() * (2.0 ** -16 * (whole * p + rest) + 2.0 ** -22 * qv + 2.0 ** -125 * whole)
    return loss, d, tol


def check_distillation(cuda, x, ids, values, lse, temperature):
    """By two calls, by one, and over the logits."""
    import torch
    ops = cuda.distill
    g = torch.rand(len(x), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) + 0.1
    want_loss, want, tol = distillation(x, ids, values, lse, temperature, g)
    loss, saved = ops.distill_fwd(x, ids, values, lse, temperature)
    close_loss(loss, want_loss)
    d = ops.distill_bwd(x, ids, values, saved, g, temperature)
    close_gradient(d, want, tol)
    both_loss, both = ops.distill_fwd_bwd(x, ids, values, g, lse, temperature)
    close_loss(both_loss, want_loss)
    close_gradient(both, want, tol)
    over = x.clone()
    want = ops.distill_bwd(over, ids, values, saved, g, temperature)
    assert ops.distill_bwd(over, ids, values, saved, g, temperature, out=over).equal(want)
    over = x.clone()
    want = ops.distill_fwd_bwd(over, ids, values, g, lse, temperature)[1]
    assert ops.distill_fwd_bwd(over, ids, values, g, lse, temperature, out=over)[1].equal(want)


@pytest.mark.parametrize("T,V", [(54, 3), (54, 9001), (900, 20003), (54, 70001), (160, 70001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_of_large_logits(cuda, T, V, dtype):
    """Loss and gradient where the logarithm of a row's sum is large beside what the sum's last digit says."""
    import torch
    inf = float("inf")
    for temperature in (1.0, 2.0 ** -5, 2.0 ** (-13 if dtype == "float16" else -19)):  # f16 does not hold 2^19 times a gradient
        x, rows = shifted_rows(T, V, dtype, seed=V + 1, shift=3)
        x[x == -inf] = -1.0  # what a list gives to a masked id is an infinite loss
        ids, values, _ = teacher(T, V, min(V, 30), dtype, seed=V)
        ids[:, 0] = V // 3 + 1
        z = x.double() / temperature
        small = (torch.logsumexp(z, 1) - z.gather(1, ids.long() - 1).amin(1)) < 1e30  # or the loss is beyond f32
        x, ids, values = x[small], ids[small], values[small] * temperature
        assert len(x) >= 30
        check_distillation(cuda, x, ids, values.to(x.dtype), None, temperature)
    cuda.check_device_status(0)


@pytest.mark.parametrize("T,V,K", [(12, 1000, 4), (12, 9001, 256), (700, 20003, 20), (12, 70001, 30)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rest_that_is_far_below_the_list(cuda, T, V, K, dtype):
    """A student whose listed logits stand above all else by more than an f32 power holds: the loss is finite, and what the teacher leaves
    over still pulls at all else."""
    import torch
    for k, (gap, temperature) in enumerate(((20, 1.0), (80, 1.0), (86, 1.0), (87, 1.0), (90, 1.0), (103, 1.0), (1000, 1.0), (10000, 1.0), (4.5, 2.0 ** -4),
                                            (6, 2.0 ** -4), (30000, 2.0 ** -7), (-90, 1.0), (-1000, 1.0))):
        x = make(T, V, dtype, seed=V + k, shift=k % 8, scale=1.0)
        ids, values, all_values = teacher(T, V, K, seed=K)
        ids[1, K // 2:] = 0
        ids[2, 1:] = ids[2, :1]
        values[2, 1:] = -float("inf")
        x.scatter_(1, (ids.long() - 1).clamp(min=0), (x.gather(1, (ids.long() - 1).clamp(min=0)).float() + gap).to(x.dtype))
        x[3] = x[3].round()
        for over in (1.0, 1e-3, 0.0, -1.0):  # in logarithms, of what the list leaves over: much, little, next to nothing, less than nothing
            lse = torch.logsumexp(values.double() / temperature, 1).float() + over
            check_distillation(cuda, x, ids, values, lse, temperature)
    cuda.check_device_status(0)


@pytest.mark.parametrize("T,V,K", [(8, 40, 5), (8, 9001, 256), (600, 20003, 40)])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_values_of_the_teacher(cuda, T, V, K, dtype):
    """A list is a distribution whatever its values' magnitude: equal ones of any size, a large shift, a small temperature."""
    import torch
    x = make(T, V, "float32", seed=V)
    ids, values, _ = teacher(T, V, K, dtype, seed=K)
    low = torch.finfo(values.dtype).min
    values[0] = low
    values[1] = -low
    values[2] = low
    values[2, K // 2:] = 0.5
    values[3] += 6e4 if dtype == "float16" else 1e5
    values[4] = 0.0 if dtype == "float16" else -1e30
    for temperature in (1.0, 2.0 ** -5, 2.0 ** -19, 2.0 ** 19):
        u = values.double() / temperature
        got, saved = cuda.distill.distill_fwd(x, ids, values, None, temperature)
        q = torch.softmax(u - u.amax(1, keepdim=True), 1)
        log_p = torch.log_softmax(x.double() / temperature, 1)
        want = (torch.xlogy(q, q) - q * log_p.gather(1, ids.long() - 1)).sum(1)
        close_loss(got, want)
        g = torch.ones(T, device="cuda")
        d = (log_p.exp().scatter_add(1, ids.long() - 1, -q)) / temperature
        tol = (2.0 ** -16 * log_p.exp() + torch.zeros_like(log_p).scatter_add(1, ids.long() - 1, 2.0 ** -22 * q) + 2.0 ** -125) / temperature
        close_gradient(cuda.distill.distill_bwd(x, ids, values, saved, g, temperature), d, tol)
        loss, both = cuda.distill.distill_fwd_bwd(x, ids, values, g, None, temperature)
        close_loss(loss, want)
        close_gradient(both, d, tol)


@pytest.mark.parametrize("T,V", [(54, 1), (54, 70), (54, 9001), (900, 1025), (54, 70001), (160, 70001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_large_logits(cuda, T, V, dtype):
    """Gradients where half a step of an f32 lse is much of an exponent, or all of it; also over the logits, and into other columns."""
    import torch
    ops = cuda.logprobs
    for k, temperature in enumerate((1.0, 2.0 ** -5, 2.0 ** (-13 if dtype == "float16" else -19), 8.0)):  # f16 does not hold 2^19 times a gradient
        x, rows = shifted_rows(T, V, dtype, seed=V + 2, shift=k)
        generator = torch.Generator(device="cuda").manual_seed(V)
        tokens = torch.randint(1, V + 1, (T,), device="cuda", generator=generator)
        tokens[1::7] = 0
        top = min(V, 5)
        r = ops.token_logprobs(x, tokens, top=top, temperature=temperature)
        g0, gh, gt = (torch.randn(*s, device="cuda", generator=generator) for s in ((T,), (T,), (T, top)))
        for a, b, c in ((g0, gh, gt), (g0, None, None), (None, gh, None)):
            want, tol = gradients(x.double(), tokens, r.top_ids, a, b, c, temperature)
            # a power below 2^-126 (log p of -88) counts as 0
            lost = sum((t.abs() * w).view(T, -1).sum(1) for t, w in ((a, 1), (c, 1), (b, 100 + r.entropy)) if t is not None)
            tol = tol + 2.0 ** -125 * lost.double()[:, None] / temperature
            got = ops.token_logprobs_bwd(x, tokens, r.lse, r.entropy, a, b, r.top_ids, c, temperature)
            close_gradient(got, want, tol)
        over = x.clone()
        want = ops.token_logprobs_bwd(over, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature)
        wide = torch.full((T, V + 9), 7.0, device="cuda", dtype=x.dtype)
        ops.token_logprobs_bwd(over, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature, out=wide[:, 2:2 + V])
        assert wide[:, 2:2 + V].equal(want) and (wide[:, :2] == 7).all() and (wide[:, 2 + V:] == 7).all()
        assert ops.token_logprobs_bwd(over, tokens, r.lse, r.entropy, g0, gh, r.top_ids, gt, temperature, out=over).equal(want)
    cuda.check_device_status(0)


@pytest.mark.parametrize("shift", [0.0, 500.0])
def test_gradient_of_a_part_of_a_vocabulary(cuda, shift):
    """The lse and the entropy of all parts make each part's gradient that of its columns."""
    import torch
    T, V, cut = 30, 5000, 1999
    ops = cuda.logprobs
    x = make(T, V, "float32", seed=3) + shift
    tokens = torch.randint(1, cut + 1, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    r = ops.token_logprobs(x, tokens)
    g0, gh = torch.randn(T, device="cuda"), torch.randn(T, device="cuda")
    want, tol = gradients(x.double(), tokens, None, g0, gh, None, 1.0)
    close_gradient(ops.token_logprobs_bwd(x[:, :cut], tokens, r.lse, r.entropy, g0, gh), want[:, :cut], tol[:, :cut] * 4)  # lse to 2^-15


@pytest.mark.parametrize("V", [400003, 4000003])
def test_long_rows_with_a_rest(cuda, V):
    """As many rows as there are counters: parts are longer than a warp has bits for.  All rows but three are padding, which is not read."""
    import torch
    T, K, live = 4096, 40, [0, 1777, 4095]
    x = torch.empty(T, V, device="cuda", dtype=torch.bfloat16)
    x[live] = make(3, V, "bfloat16", seed=V)
    some_ids, some_values, all_values = teacher(3, V, K, seed=1)
    some_ids[1, 3:] = some_ids[1, :1]
    ids, values = torch.zeros(T, K, device="cuda", dtype=torch.int32), torch.zeros(T, K, device="cuda")
    ids[live], values[live] = some_ids, some_values
    lse = torch.zeros(T, device="cuda")
    lse[live] = torch.logsumexp(all_values, 1) + 1
    g = torch.ones(T, device="cuda")
    want_loss, want, tol = distillation(x[live], some_ids, some_values, lse[live], 1.0, g[live])
    loss, saved = cuda.distill.distill_fwd(x, ids, values, lse)
    close_loss(loss[live], want_loss)
    assert loss.count_nonzero() == 3
    cuda.distill.distill_bwd(x, ids, values, saved, g, out=x)
    close_gradient(x[live], want, tol)
    assert all(not x[r].any() for r in (1, 1776, 4094))
    cuda.check_device_status(0)
