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
