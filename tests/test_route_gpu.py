"""Routing to experts and its gradient against f64.

Ids are compared one by one: the kernel compares selection values in f64, and so does the reference.  Weights are rounded once to their
type from values that are off by at most a few f32 roundings (2^-21 relative).  The gradient's scores come from f32 exponentials (2^-22) and
sums over at most 512 experts in a tree (2^-22): its terms are off by 2^-20 of their size, and half a step of the type.  What the f64
reference itself rounds (2^-50 of the largest gradient) shows where the gradient is 0: experts that renormalised weights do not reach.
"""
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")
LOWEST = -1.7976931348623157e308


def reference(x, topk, bias=None, score="softmax", groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    """(weights [topk, T] f64, ids [topk, T])"""
    import torch
    T, E = x.shape
    x = x.double()
    s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    c = s if bias is None else s + bias.double()
    c = torch.where(c > LOWEST, c, torch.full_like(c, LOWEST))
    if topk_groups < groups:
        g = torch.sort(c.view(T, groups, -1), dim=2, descending=True).values[:, :, :group_top].sum(2)
        best = torch.sort(g, dim=1, descending=True, stable=True).indices[:, :topk_groups]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        c = torch.where(keep.repeat_interleave(E // groups, 1), c, -float("inf"))
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :topk]
    w = s.gather(1, ids)
    if renormalize:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-20)
    return (w * scale).t(), (ids + 1).int().t()


def close(got, want, relative=2.0 ** -21):
    import torch
    info = torch.finfo(got.dtype)
    same = (got.isnan() & want.isnan()) | (got.double() == want)
    err = (got.double() - want).abs()
    assert (same | (err <= (relative + info.eps / 2) * want.abs() + info.smallest_normal * info.eps / 2)).all(), err[~same].max()


def check(cuda, x, topk, weights_dtype=None, **kw):
    import torch
    w, ids = cuda.moe.moe_route(x, topk, weights_dtype=weights_dtype or torch.float16, **kw)
    want_w, want_ids = reference(x, topk, **kw)
    assert ids.equal(want_ids)
    close(w, want_w)
    return w, ids


def logits(T, E, dtype, seed=0, ld=None):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.full((T, ld or E), float("nan"), device="cuda", dtype=getattr(torch, dtype))
    x[:, :E] = torch.randn(T, E, device="cuda", generator=g) * 1.5
    return x[:, :E]


@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (3, 2, 2), (5, 8, 2), (1, 32, 8), (257, 33, 5), (64, 60, 4), (1000, 64, 8), (33, 100, 32), (129, 128, 6),
                                      (4096, 256, 8), (65, 257, 3), (700, 512, 16)])
@pytest.mark.parametrize("dtype", TYPES)
def test_route(cuda, T, E, topk, dtype):
    import torch
    x = logits(T, E, dtype, seed=T + E, ld=E + 3)
    bias = torch.randn(E, device="cuda") * 0.1
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            check(cuda, x, topk, bias=b, score=score)
            check(cuda, x, topk, torch.float32, bias=b, score=score, renormalize=False, scale=2.5)
    check(cuda, x, topk, torch.bfloat16)


@pytest.mark.parametrize("E,groups,kept,topk", [(8, 4, 1, 2), (64, 8, 3, 8), (60, 5, 2, 6), (256, 8, 4, 8), (256, 32, 5, 8), (160, 16, 9, 6), (512, 2, 1, 4),
                                                (384, 8, 4, 32), (64, 32, 31, 1)])
@pytest.mark.parametrize("group_top", [1, 2])
def test_groups(cuda, E, groups, kept, topk, group_top):
    import torch
    bias = torch.randn(E, device="cuda") * 0.2
    for dtype in TYPES:
        x = logits(333, E, dtype, seed=E + groups)
        for score in ("softmax", "sigmoid"):
            check(cuda, x, topk, bias=bias, score=score, groups=groups, topk_groups=kept, group_top=group_top, scale=1.5)
            check(cuda, x, topk, score=score, groups=groups, topk_groups=kept, group_top=group_top, renormalize=False)
        check(cuda, x, topk, groups=groups, topk_groups=groups, group_top=group_top)


def test_ties_and_masks(cuda):
    """Equal logits, a bias that shuts experts out, masked logits, near ties that f32 cannot tell apart."""
    import torch
    inf = float("inf")
    E = 64
    x = torch.round(logits(500, E, "float32", seed=1))
    bias = torch.round(torch.randn(E, device="cuda") * 2) / 4
    for score in ("softmax", "sigmoid"):
        for kw in (dict(), dict(groups=8, topk_groups=3, group_top=2)):
            check(cuda, x, 8, score=score, **kw)
            check(cuda, x, 8, score=score, bias=bias, **kw)
            shut = bias.clone()
            shut[::3] = -inf
            check(cuda, x, 8, score=score, bias=shut, **kw)
            y = x.clone()
            y[:, 5:] = -inf  # fewer than topk are left
            y[1] = 0.25
            check(cuda, y, 8, score=score, **kw)
            check(cuda, y, 8, score=score, bias=bias, **kw)
    g = torch.Generator(device="cuda").manual_seed(3)
    near = 0.5 + torch.randint(0, 40, (2000, E), device="cuda", generator=g).float() * 2.0 ** -24
    for score in ("softmax", "sigmoid"):
        check(cuda, near, 8, score=score)
        check(cuda, near, 8, score=score, bias=torch.randint(0, 40, (E,), device="cuda", generator=g).float() * 2.0 ** -27)
        check(cuda, near, 8, score=score, bias=bias, groups=4, topk_groups=2, group_top=2)
    far = logits(300, E, "float32", seed=9) * 30  # scores down to e^-100, differences below any f32 of the sum
    check(cuda, far, 8, score="sigmoid", bias=torch.full((E,), 1.0, device="cuda"))
    check(cuda, far, 8, score="softmax", bias=torch.full((E,), 1.0, device="cuda"))
    y = logits(6, E, "float32", seed=4)
    y[0] = float("nan")
    y[1, 3] = float("nan")
    y[2] = -inf
    y[3, 7] = inf
    for score in ("softmax", "sigmoid"):
        w, ids = cuda.moe.moe_route(y, 8, score=score, groups=8, topk_groups=4, group_top=2)
        assert (ids >= 1).all() and (ids <= E).all() and all(len(set(c)) == 8 for c in ids.t().tolist()) and w[:, 4:].isfinite().all()
    cuda.check_device_status(0)


def gradient(x, ids, dw, score, renormalize, scale):
    import torch
    x = x.double().requires_grad_()
    s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    w = s.gather(1, ids.long().t() - 1)
    size = (s / x.shape[1]).detach()
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    (w * scale * dw.double().t()).sum().backward()
    chosen = torch.zeros_like(s).scatter_(1, ids.long().t() - 1, 1.0).detach()
    biggest = dw.double().abs().amax(0)[:, None] * scale
    top = s.detach().gather(1, ids.long().t() - 1).sum(1, keepdim=True) if renormalize else torch.ones_like(size[:, :1])
    terms = 3 * biggest * s.detach() * (chosen / top + (0 if renormalize or score == "sigmoid" else 1))
    return x.grad, terms


@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (5, 8, 2), (257, 33, 5), (1000, 64, 8), (33, 100, 32), (2000, 256, 8), (700, 512, 16)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient(cuda, T, E, topk, dtype):
    import torch
    ops = cuda.moe
    x = logits(T, E, dtype, seed=T, ld=E + 1)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            w, ids = ops.moe_route(x, topk, score=score, renormalize=renormalize, scale=1.5)
            dw = torch.randn(topk, T, device="cuda")
            want, terms = gradient(x, ids, dw, score, renormalize, 1.5)
            got = ops.moe_route_bwd(x, ids, dw, score=score, renormalize=renormalize, scale=1.5)
            info = torch.finfo(got.dtype)
            err = (got.double() - want).abs()
            assert (err <= 2.0 ** -20 * terms + 2.0 ** -50 * dw.abs().max() * 1.5 + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2).all(), err.max()
            half = ops.moe_route_bwd(x, ids.long(), dw.half(), score=score, renormalize=renormalize, scale=1.5)
            assert half.equal(ops.moe_route_bwd(x, ids, dw.half().float(), score=score, renormalize=renormalize, scale=1.5))
            wide = torch.full((T, E + 7), 7.0, device="cuda", dtype=x.dtype)
            ops.moe_route_bwd(x, ids, dw, score=score, renormalize=renormalize, scale=1.5, out=wide[:, 3:3 + E])
            assert wide[:, 3:3 + E].equal(got) and (wide[:, :3] == 7).all() and (wide[:, 3 + E:] == 7).all()
            over = logits(T, E, dtype, seed=T, ld=E + 1)
            assert ops.moe_route_bwd(over, ids, dw, score=score, renormalize=renormalize, scale=1.5, out=over).equal(got)
    cuda.check_device_status(0)


def test_gradient_against_differences(cuda):
    import torch
    T, E, topk, step = 3, 12, 3, 1e-5
    x = logits(T, E, "float32", seed=8)
    dw = torch.randn(topk, T, device="cuda")
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            _, ids = cuda.moe.moe_route(x, topk, score=score)
            got = cuda.moe.moe_route_bwd(x, ids, dw, score=score, renormalize=renormalize, scale=2.0)

            def value(x64):
                s = torch.softmax(x64, 1) if score == "softmax" else torch.sigmoid(x64)
                w = s.gather(1, ids.long().t() - 1)
                return (2.0 * (w / w.sum(1, keepdim=True) if renormalize else w) * dw.double().t()).sum(1)
            for e in range(E):
                h = torch.zeros(E, device="cuda", dtype=torch.float64)
                h[e] = step
                slope = (value(x.double() + h) - value(x.double() - h)) / (2 * step)
                assert ((got[:, e].double() - slope).abs() <= 1e-8 + 2.0 ** -20 * 8).all()


def test_no_choice_and_repeated_ids(cuda):
    import torch
    x = logits(4, 16, "float32", seed=2)
    ids = torch.tensor([[3, 0, 5, 2], [4, 1, 5, 17]], device="cuda", dtype=torch.int32)
    dw = torch.randn(2, 4, device="cuda")
    d = cuda.moe.moe_route_bwd(x, ids, dw, score="sigmoid", renormalize=False)
    with pytest.raises(cuda.CtbError, match="out-of-range index"):
        cuda.check_device_status(0)
    s = torch.sigmoid(x.double())
    want = torch.zeros(4, 16, dtype=torch.float64, device="cuda")
    for j in range(2):
        for t in range(4):
            if 1 <= ids[j, t] <= 16:
                want[t, ids[j, t].long() - 1] += dw[j, t].double()
    want *= s * (1 - s)
    assert ((d.double() - want).abs() <= 2.0 ** -20 * dw.abs().sum()).all()
    cuda.check_device_status(0)


def test_router_of_an_expert_layer(cuda):
    """The run that belongs together: logits of the existing router's product, grouped sigmoid routing, the experts, in a graph too; plain
    softmax routing chooses and weighs as moe_router does."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    T, H, E, I, topk = 300, 256, 16, 128, 4
    x = torch.randn(T, H, device="cuda", generator=g).half()
    wr, w1, w2 = (torch.randn(*s, device="cuda", generator=g).half() * 0.05 for s in ((E, H), (E, 2 * I, H), (E, H, I)))
    gates, ids, scores = cuda.moe.moe_router(x, wr, topk, return_logits=True)
    mine, my_ids = cuda.moe.moe_route(scores, topk)
    assert my_ids.equal(ids)
    assert ((mine.float() - gates.float()).abs() <= 2.0 ** -10 * gates.float()).all()  # one f16 step: either may round the other way
    bias = torch.randn(E, device="cuda", generator=g) * 0.05

    def layer():
        _, _, s = cuda.moe.moe_router(x, wr, topk, return_logits=True)
        w, i = cuda.moe.moe_route(s, topk, bias=bias, score="sigmoid", groups=4, topk_groups=2, group_top=2, scale=2.5)
        return w, i, cuda.moe.cutile_moe(x, w1, w2, w, i, 128, 128, 64)
    w, i, out = layer()
    want_w, want_i = reference(scores, topk, bias, "sigmoid", 4, 2, 2, True, 2.5)
    assert i.equal(want_i)
    close(w, want_w)
    e = (i - 1).long()
    expect = torch.zeros(T, H, device="cuda", dtype=torch.float64)
    for j in range(topk):
        for k in range(E):
            rows = (e[j] == k).nonzero()[:, 0]
            h = x[rows].double() @ w1[k].double().t()
            h = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
            expect[rows] += (h @ w2[k].double().t()) * w[j, rows].double()[:, None]
    assert (out.double() - expect).norm() <= 2e-3 * expect.norm()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = layer()
    graph.replay()
    assert all(a.equal(b) for a, b in zip(again, (w, i, out)))
    cuda.check_device_status(0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_doubtful_orders(cuda, score):
    """Scores with a bias so close that f32 cannot order them, next to each other, at the last choice and at the last group; scores beyond f32."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(11)
    for T, E, topk, kw in ((3000, 256, 8, dict(groups=8, topk_groups=4, group_top=2)), (3000, 64, 30, dict()), (3000, 64, 31, dict()),
                           (500, 60, 32, dict()), (3000, 384, 6, dict(groups=8, topk_groups=3, group_top=1))):
        x = torch.randn(T, E, device="cuda", generator=g)
        bias = torch.randn(E, device="cuda", generator=g) * 0.1
        scores = torch.softmax(x.double(), 1) if score == "softmax" else torch.sigmoid(x.double())
        a, b = torch.randperm(E, device="cuda", generator=g)[:2]
        step = torch.randint(-3, 4, (E,), device="cuda", generator=g) * 2.0 ** -25
        bias[b] = 0.7
        bias[a] = (scores[0, b] + 0.7 - scores[0, a]).float()  # the two best of the first token, a rounding apart
        check(cuda, x, topk, torch.float32, score=score, bias=bias, **kw)
        close_x = x.clone()
        close_x[:, 1::2] = close_x[:, ::2]
        check(cuda, close_x, topk, torch.float32, score=score, bias=bias, **kw)
        check(cuda, close_x, topk, torch.float32, score=score, bias=(bias.view(-1, 2)[:, :1].expand(-1, 2).reshape(-1) + step).float(), **kw)
        check(cuda, close_x, topk, torch.float32, score=score, bias=(bias.view(-1, 2)[:, :1].expand(-1, 2).reshape(-1) + step).float() * 1e4, **kw)
        check(cuda, x * 12, topk, torch.float32, score=score, renormalize=False, **kw)
        check(cuda, x * 12, topk, torch.float32, score=score, bias=bias, renormalize=False, **kw)
        check(cuda, x * 12 + 18, topk, torch.float32, score=score, bias=bias, **kw)


@pytest.mark.parametrize("topk", [1, 29, 30, 31, 32])
def test_doubt_at_the_last_choice(cuda, topk):
    """Every score within a few f32 roundings of every other, whatever the number of choices."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(topk)
    for E in (40, 64, 250):
        x = 0.5 + torch.randint(0, 40, (400, E), device="cuda", generator=g).float() * 2.0 ** -24
        bias = 0.25 + torch.randint(0, 40, (E,), device="cuda", generator=g).float() * 2.0 ** -25
        for score in ("softmax", "sigmoid"):
            check(cuda, x, topk, torch.float32, score=score, bias=bias)
            check(cuda, x, topk, torch.float32, score=score)


def test_refusals(cuda):
    import torch
    ops, lib = cuda.moe, cuda._lib
    x = logits(4, 64, "float32")

    def refused(status, word, **kw):
        topk = kw.pop("topk", 4)
        with pytest.raises(cuda.CtbError, match=word) as e:
            ops.moe_route(kw.pop("x", x), topk, **kw)
        assert e.value.status == status
    refused(lib.BAD_ARG, "topk", topk=0)
    refused(lib.BAD_ARG, "topk", topk=65)
    refused(lib.UNSUPPORTED, "32 experts per token", topk=33)
    refused(lib.UNSUPPORTED, "512 experts", x=logits(2, 513, "float32"))
    refused(lib.BAD_ARG, "score must be", score="relu")
    refused(lib.BAD_ARG, "cannot be cut", groups=7)
    refused(lib.UNSUPPORTED, "32 groups", groups=64)
    refused(lib.BAD_ARG, "topk_groups", groups=8, topk_groups=9)
    refused(lib.BAD_ARG, "topk_groups", groups=8, topk_groups=0)
    refused(lib.BAD_ARG, "hold fewer", groups=32, topk_groups=1)
    refused(lib.BAD_ARG, "group_top", groups=8, topk_groups=2, group_top=3)
    refused(lib.BAD_ARG, "two experts", x=logits(2, 32, "float32"), groups=32, topk_groups=8, group_top=2)
    refused(lib.BAD_ARG, "finite", scale=float("nan"))
    refused(lib.BAD_ARG, "bias", bias=torch.zeros(63, device="cuda"))
    refused(lib.BAD_ARG, "bias", bias=torch.zeros(64, device="cuda", dtype=torch.float16))
    refused(lib.BAD_ARG, "element type", weights_dtype=torch.float64)
    w, ids = ops.moe_route(x[:0], 4)
    assert w.shape == (4, 0) and ids.shape == (4, 0)
    assert ops.moe_route_bwd(x[:0], ids, w).shape == (0, 64)
    w, ids = ops.moe_route(x, 4)
    for f in (lambda: ops.moe_route_bwd(x, ids.float(), w), lambda: ops.moe_route_bwd(x, ids, w[:3]), lambda: ops.moe_route_bwd(x, ids[:, :3], w[:, :3]),
              lambda: ops.moe_route_bwd(x[:3], ids[:, :3].contiguous(), w[:, :3].contiguous(), out=x[1:])):
        with pytest.raises(cuda.CtbError):
            f()
    cuda.check_device_status(0)
