"""Routing and its gradient at the ends of their range."""
import pytest

pytestmark = pytest.mark.gpu


def test_as_many_tokens_as_there_are(cuda):
    """2^31 - 1 tokens: a token's number, and that of the next one of its warp, pass 32 bits."""
    import torch
    T = 2 ** 31 - 1
    x = torch.zeros(T, 1, device="cuda", dtype=torch.float16)
    x[-1], x[-20000], x[0] = 2.0, -1.0, 1.0  # the last round of the grid, and the one before
    w, ids = cuda.moe.moe_route(x, 1, score="sigmoid", renormalize=False)
    at = [0, 1, T // 2, T - 20000, T - 2, T - 1]
    want = torch.sigmoid(x[at].double())
    assert ((w[0, at, None].double() - want).abs() <= 2.0 ** -10 * want).all() and ids.min() == 1 and ids.max() == 1
    assert int((w != 0.5).sum()) == 3
    cuda.moe.moe_route_bwd(x, ids, w, score="sigmoid", renormalize=False, out=x)
    want = w[0, at, None].double() * want * (1 - want)
    assert ((x[at].double() - want).abs() <= 2.0 ** -10 * want).all()
    assert int((x != 0.125).sum()) == 3
    cuda.check_device_status(0)


TYPES = ("float32", "float16", "bfloat16")


@pytest.mark.parametrize("E,topk", [(4, 1), (30, 3), (64, 8), (128, 4), (250, 6), (512, 32)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_large_sigmoid_logits(cuda, E, topk, dtype):
    """s (1 - s) where s is near 1 and near 0.  An exponential is off by 2^-22, its sum with 1, the quotient and four products by 2^-24 each: 2^-20."""
    import torch
    T = 40
    generator = torch.Generator(device="cuda").manual_seed(E)
    x = ((torch.rand(T, E, device="cuda", generator=generator) - 0.5) * 60).to(getattr(torch, dtype))
    dw = torch.randn(topk, T, device="cuda", generator=generator)
    ids = cuda.moe.moe_route(x, topk, score="sigmoid", renormalize=False)[1]
    got = cuda.moe.moe_route_bwd(x, ids, dw, score="sigmoid", renormalize=False, scale=2.5)
    want = torch.sigmoid(x.double()) * torch.sigmoid(-x.double()) * 2.5
    want = want * torch.zeros_like(want).scatter_(1, ids.long().t() - 1, dw.double().t())
    info = torch.finfo(got.dtype)
    assert ((got.double() - want).abs() <= (2.0 ** -20 + info.eps / 2) * want.abs() + info.smallest_normal * info.eps).all()


def gradient(x, ids, dw, score, renormalize, scale):
    """(gradient, tolerance without the type's rounding) in f64, from sums in which nothing cancels:
        dx_v = scale f_v / T sum_w s_w (dw_v - dw_w) / T,  f = s (softmax), s (1 - s) (sigmoid),
    over all experts (softmax, T = 1) or the chosen ones (renormalised; T the sum of their s); sigmoid: scale f_v dw_v.
    An exponential is off by 2^-22 (and a softmax's by 2^-24 of its argument's size, whose difference is rounded), s and f by 2^-24 for each of up to four
    operations more, and so is what they are multiplied by: 2^-19 of the sum of the terms' sizes.  The difference of sums in which the kernel
    takes them, each rounded to f32 twice, adds (2 topk + 1) 2^-23 of that sum, renormalised, and 17 * 2^-23 otherwise (where more than 7/8 are
    chosen, f64 instead: 54 additions, 2^-47 of the largest dw)."""
    import torch
    x, dw = x.double(), dw.double().t()
    chosen = torch.zeros_like(x).scatter_(1, ids.long().t() - 1, 1.0)
    dw = torch.zeros_like(x).scatter_(1, ids.long().t() - 1, dw)
    if score == "softmax":
        s = f = torch.softmax(x, 1)
    else:
        s, f = torch.sigmoid(x), torch.sigmoid(x) * torch.sigmoid(-x)
    if renormalize or score == "softmax":
        w = s * chosen / (s * chosen).sum(1, keepdim=True) if renormalize else s
        apart = dw[:, :, None] - dw[:, None, :]
        mean, size = (w[:, None, :] * apart).sum(2), (w[:, None, :] * apart.abs()).sum(2)
        f = f / (s * chosen).sum(1, keepdim=True) * chosen if renormalize else f
    else:
        mean, size = dw, dw.abs()
    reach = (x.amax(1, keepdim=True) - x).amax(1, keepdim=True) if score == "softmax" else 0
    part = 2.0 ** -19 + (2 * len(ids) + 1 if renormalize else 17) * 2.0 ** -23 + 2.0 ** -22 * reach
    return scale * f * mean, scale * f * (size * part + 2.0 ** -47 * dw.abs().amax(1, keepdim=True))


def close(got, want, tol):
    import torch
    info = torch.finfo(got.dtype)
    err = (got.double() - want).abs()
    assert (err <= tol * (1 + info.eps) + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2).all(), (err / want.abs()).max()


@pytest.mark.parametrize("E,topk", [(4, 1), (30, 3), (64, 8), (128, 4), (250, 6), (512, 32)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_sure_choices(cuda, E, topk, dtype):
    """Scores near 1 and near 0, one expert that has nearly all of the probability, two that share it, gradients that are alike: what is
    left of the differences counts."""
    import torch
    T = 40
    generator = torch.Generator(device="cuda").manual_seed(E)
    x = torch.randn(T, E, device="cuda", generator=generator)
    x[:10] = (torch.rand(10, E, device="cuda", generator=generator) - 0.5) * 60
    x[10:20, E // 3] += torch.arange(6, 26, 2, device="cuda")
    x[20:30, 1] += torch.arange(6, 26, 2, device="cuda")
    x[20:30, E - 1] = x[20:30, 1]
    x = x.to(getattr(torch, dtype))
    for k in range(3):
        dw = torch.randn(topk, T, device="cuda", generator=generator)
        if k == 1:
            dw[:] = 1.0
        if k == 2:
            dw = 0.7 + dw * 2.0 ** -20
        for score in ("softmax", "sigmoid"):
            for renormalize in (False, True):
                ids = cuda.moe.moe_route(x, topk, score=score, renormalize=renormalize)[1]
                got = cuda.moe.moe_route_bwd(x, ids, dw, score=score, renormalize=renormalize, scale=2.5)
                close(got, *gradient(x, ids, dw, score, renormalize, 2.5))
    cuda.check_device_status(0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_of_a_sum_that_is_held(cuda, score):
    """Chosen scores whose sum is below 1e-20 are divided by 1e-20: no gradient flows through that sum, and all else stays."""
    import torch
    T, E, topk, scale = 6, 16, 3, 1.5
    x = torch.randn(T, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    bias = torch.zeros(E, device="cuda")
    bias[[2, 7, 11]] = 4.0
    x[:, bias > 0] -= 55
    w, ids = cuda.moe.moe_route(x, topk, bias=bias, score=score, scale=scale, weights_dtype=torch.float32)
    dw = torch.randn(topk, T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    x64 = x.double().requires_grad_()
    s = torch.softmax(x64, 1) if score == "softmax" else torch.sigmoid(x64)
    s = s.gather(1, ids.long().t() - 1)
    assert (s.sum(1) < 1e-20).all()
    (s / s.sum(1, keepdim=True).clamp(min=1e-20) * scale * dw.double().t()).sum().backward()
    got = cuda.moe.moe_route_bwd(x, ids, dw, score=score, scale=scale)
    # a sum of three products that may cancel, each off by 2^-22 and by 2^-24 of an argument of up to 60
    size = (s.detach() * 1e20 * scale * dw.double().t().abs()).sum(1, keepdim=True)
    assert ((got.double() - x64.grad).abs() <= 2.0 ** -17 * size).all()
    assert (x64.grad[:, bias == 0].abs() > 2.0 ** -10 * size).any() == (score == "softmax")
