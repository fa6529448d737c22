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
