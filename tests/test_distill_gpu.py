"""Distillation from a teacher's top logits, loss and gradient, against f64.

Tolerances.  The teacher's side and the products of the loss are computed in f64 from f32 statistics of the student's row, whose sum of
powers is off by at most 2^-18 relative for |z| <= 64 (see test_logprobs_gpu.py): the loss, whose q sum to 1, by 2^-18, with the
rest's probability once more, and 2^-24 of its value.  A gradient p outside or (all p - q) is off by 2^-16 p (|all| + |outside|) from p and by 2^-22
of `outside` and q, times g / temperature, and half a step of the type.
"""
import pytest

pytestmark = pytest.mark.gpu

from test_logprobs_gpu import TYPES, close_gradient, make  # noqa: E402


def teacher(T, V, K, dtype="float32", seed=0, spread=2.0):
    """(ids [T, K] int32 without repeats, values, lse of all the teacher's values at temperature 1)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(T, V, device="cuda", generator=g) * spread
    v, i = torch.topk(t, K, 1)
    return (i + 1).int(), v.to(getattr(torch, dtype)), t


def reference(x, ids, values, lse, temperature, d_loss):
    """(loss, gradient, tolerance of the gradient) in f64."""
    import torch
    T, V = x.shape
    used = ids > 0
    at = (ids.long() - 1).clamp(min=0)
    live = used.any(1)
    u = torch.where(used, values.double() / temperature, -float("inf"))
    norm = torch.logsumexp(u, 1, keepdim=True) if lse is None else lse.double()[:, None]
    q = torch.where(used & live[:, None], (u - norm).exp(), 0.0)
    logp = torch.log_softmax(torch.where(live[:, None], x.double(), 0.0) / temperature, 1)
    p = logp.exp()
    loss = (torch.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, at), q)).sum(1)
    total, outside = torch.ones(T, 1, device=x.device, dtype=torch.float64), torch.ones(T, 1, device=x.device, dtype=torch.float64)
    mask = torch.zeros(T, V, dtype=torch.float64, device=x.device).scatter_add_(1, at, used.double()) > 0
    if lse is not None:
        left = (1 - q.sum(1, keepdim=True)).clamp(min=0)
        total = q.sum(1, keepdim=True) + left
        rest = torch.where(mask, 0.0, p).sum(1, keepdim=True)
        log_rest = torch.logsumexp(logp.masked_fill(mask, -float("inf")), 1, keepdim=True)
        loss = loss + torch.where(left > 0, left * (left.log() - log_rest), left)[:, 0]
        outside = torch.where(rest > 0, total - left / rest, total)
    qv = torch.zeros_like(p).scatter_add_(1, at, q)
    g = (d_loss.double() / temperature)[:, None]
    d = torch.where(mask, total * p - qv, outside * p) * g
    tol = g.abs() * (p * (2.0 ** -16 * (total.abs() + outside.abs()) + 2.0 ** -17 * (total - outside).abs()) + 2.0 ** -22 * qv)
    zero = torch.zeros_like
    return torch.where(live, loss, zero(loss)), torch.where(live[:, None], d, zero(d)), tol


def close_loss(got, want):
    err = (got.double() - want).abs()
    same = (got.double() == want) | (got.isnan() & want.isnan())
    assert (same | (err <= 2.0 ** -17 + 2.0 ** -23 * want.abs())).all(), err.max()


def check(cuda, x, ids, values, lse=None, temperature=1.0, seed=0):
    import torch
    ops = cuda.distill
    g = torch.rand(len(x), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) + 0.1
    want_loss, want, tol = reference(x, ids, values, lse, temperature, g)
    loss, saved = ops.distill_fwd(x, ids, values, lse, temperature)
    close_loss(loss, want_loss)
    d = ops.distill_bwd(x, ids, values, saved, g, temperature)
    close_gradient(d, want, tol)
    both_loss, both = ops.distill_fwd_bwd(x, ids, values, g, lse, temperature)
    close_loss(both_loss, want_loss)
    close_gradient(both, want, tol)
    return loss, d


@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (3, 2, 2), (5, 9, 3), (2, 33, 32), (700, 130, 64), (2, 1000, 256), (400, 4097, 16), (3, 8193, 50),
                                   (1, 50001, 100), (310, 50001, 17), (2, 262147, 33)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_loss_and_gradient(cuda, T, V, K, dtype, tail):
    import torch
    for k, temperature in enumerate((1.0, 2.0)):
        x = make(T, V, dtype, seed=T + V, shift=3 * k, ld=V + 5 * k, scale=2.0)
        ids, values, all_values = teacher(T, V, K, dtype if k else "float32", seed=V)
        lse = torch.logsumexp(all_values / temperature, 1) if tail else None
        if k:
            ids = ids.long()
            ids[:, K - K // 3:] = 0
            if T > 2:
                ids[2] = 0
                x[2] = float("nan")  # padding is not read
        check(cuda, x, ids, values, lse, temperature)
    cuda.check_device_status(0)


@pytest.mark.parametrize("T", [5, 400])
@pytest.mark.parametrize("tail", [False, True])
def test_repeated_ids(cuda, T, tail):
    import torch
    V, K = 9000, 40
    x = make(T, V, "float32", seed=2)
    ids, values, all_values = teacher(T, V, K, seed=1)
    ids[:, 7] = ids[:, 3]
    ids[:, 39] = ids[:, 3]
    ids[:, 20] = ids[:, 19]
    lse = torch.logsumexp(all_values, 1) + 1.0 if tail else None
    check(cuda, x, ids, values, lse)


@pytest.mark.parametrize("T", [6, 400])
def test_masks(cuda, T):
    """A student that masks what the teacher lists, or all else; a teacher with masked entries, one that lists all of its probability."""
    import torch
    inf = float("inf")
    V, K = 20001, 30
    x = make(T, V, "float32", seed=4)
    ids, values, all_values = teacher(T, V, K, seed=5)
    values[1, 4:] = -inf
    keep = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep[ids[2].long() - 1] = True
    x[2, ~keep] = -inf          # nothing outside of the list
    x[3, 1000:] = -inf
    x[3, ids[3].long() - 1] = 0.5
    for lse in (None, torch.logsumexp(all_values, 1), torch.logsumexp(values, 1) - 1e-3):  # the last: more than 1, nothing is left
        rows = [r for r in range(T) if not (r == 2 and lse is not None)]
        check(cuda, x[rows], ids[rows], values[rows], None if lse is None else lse[rows])
    x[0, ids[0, 0].long() - 1] = -inf  # likely for the teacher, impossible for the student
    loss, saved = cuda.distill.distill_fwd(x, ids, values)
    assert loss[0] == inf and loss[1:].isfinite().all()
    loss, d = cuda.distill.distill_fwd_bwd(x, ids, values, torch.ones(T, device="cuda"), torch.logsumexp(all_values, 1))
    assert loss[0] == inf and loss[2] == inf and loss[3:].isfinite().all() and d.isfinite().all()  # row 2: the teacher's rest
    cuda.check_device_status(0)


def test_gradient_against_differences(cuda):
    import torch
    T, V, K, step, tau = 3, 29, 6, 1e-5, 1.5
    x = make(T, V, "float32", seed=3)
    ids, values, all_values = teacher(T, V, K, seed=6)
    ids[1, 5] = 0
    ids[2, 4] = ids[2, 1]
    g = torch.tensor([0.5, 1.0, -2.0], device="cuda")
    for lse in (None, torch.logsumexp(all_values / tau, 1) + 0.2):
        _, saved = cuda.distill.distill_fwd(x, ids, values, lse, tau)
        got = cuda.distill.distill_bwd(x, ids, values, saved, g, tau)
        for v in range(V):
            e = torch.zeros(V, device="cuda", dtype=torch.float64)
            e[v] = step
            up, down = (reference(x.double() + s * e, ids, values, lse, tau, g)[0] for s in (1, -1))
            slope = (up - down) / (2 * step) * g
            assert ((got[:, v].double() - slope).abs() <= 1e-8 + 2.0 ** -16 * (1 + slope.abs())).all()


def test_over_the_logits_and_into_columns(cuda):
    import torch
    for T, V in ((7, 5003), (400, 5003)):
        ids, values, all_values = teacher(T, V, 20, seed=1)
        lse, g = torch.logsumexp(all_values, 1), torch.rand(T, device="cuda")
        for l in (None, lse):
            x = make(T, V, "bfloat16", seed=9, shift=1)
            loss, want = cuda.distill.distill_fwd_bwd(x, ids, values, g, l)
            wide = torch.full((T, V + 9), 7.0, device="cuda", dtype=x.dtype)
            cuda.distill.distill_fwd_bwd(x, ids, values, g, l, out=wide[:, 4:4 + V])
            assert wide[:, 4:4 + V].equal(want) and (wide[:, :4] == 7).all() and (wide[:, 4 + V:] == 7).all()
            _, saved = cuda.distill.distill_fwd(x, ids, values, l)
            again = x.clone()
            assert cuda.distill.distill_bwd(again, ids, values, saved, g, out=again).equal(
                cuda.distill.distill_bwd(x, ids, values, saved, g))
            again, out = cuda.distill.distill_fwd_bwd(x, ids, values, g, l, out=x)
            assert out is x and x.equal(want) and again.equal(loss)


def test_bad_ids_are_reported(cuda):
    import torch
    for T in (4, 400):
        x = make(T, 3000, "float32")
        ids, values, _ = teacher(T, 3000, 8)
        ids[1, 2], ids[2, 0] = 3001, -4
        for f in (lambda: cuda.distill.distill_fwd_bwd(x, ids, values, torch.ones(T, device="cuda")),):
            loss, d = f()
            with pytest.raises(cuda.CtbError, match="out-of-range index"):
                cuda.check_device_status(0)
            assert loss[1:3].isnan().all() and (d[1:3] == 0).all() and loss[[0, 3]].isfinite().all() and (d[3] != 0).any()
    cuda.check_device_status(0)


def test_teacher_from_token_logprobs(cuda):
    """The run that belongs together: the teacher's alternatives and lse, the student's loss and gradient at a temperature."""
    import torch
    T, V, K, tau = 40, 12001, 20, 2.0
    tl, x = make(T, V, "bfloat16", seed=1), make(T, V, "bfloat16", seed=2)
    r = cuda.logprobs.token_logprobs(tl, None, top=K, temperature=tau, entropy=False)
    assert r.logprobs is None and r.entropy is None
    values = r.top_logprobs * tau  # log probabilities at the temperature: with an lse of 0 they stand for themselves
    zero = torch.zeros(T, device="cuda")
    loss, d = check(cuda, x, r.top_ids, values, zero, tau)
    also, _ = check(cuda, x, r.top_ids, tl.gather(1, r.top_ids.long() - 1), r.lse, tau)
    assert ((loss - also).abs() <= 1e-5).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r2 = cuda.logprobs.token_logprobs(tl, None, top=K, temperature=tau, entropy=False)
        l2, d2 = cuda.distill.distill_fwd_bwd(x, r2.top_ids, r2.top_logprobs * tau, zero + 1, zero, tau)
    eager = cuda.distill.distill_fwd_bwd(x, r.top_ids, values, zero + 1, zero, tau)
    for _ in range(3):
        l2.zero_(), d2.zero_()
        g.replay()
        assert l2.equal(eager[0]) and d2.equal(eager[1])
    cuda.check_device_status(0)


@pytest.mark.parametrize("T,V,K", [(1, 70001, 256), (70, 9001, 256), (5, 40001, 256), (149, 70001, 40), (4100, 17001, 33)])
def test_many_entries_and_rows(cuda, T, V, K):
    """Long lists with ids many times over (more alike than a small table keeps apart), and more rows than there are counters."""
    import torch
    x = make(T, V, "bfloat16", seed=3, shift=5)
    ids, values, all_values = teacher(T, V, K, seed=4)
    ids[:, K // 2:] = ids[:, :K - K // 2]
    ids[0, 1:] = ids[0, :1]
    if T > 60:
        ids[50:] = 0
    for lse in (None, torch.logsumexp(all_values, 1) + 2.0):
        check(cuda, x, ids, values, lse)


@pytest.mark.parametrize("V,dtype", [(17001, "bfloat16"), (8300, "float32"), (9000, "float16")])
def test_padding_and_bad_rows_between(cuda, V, dtype):
    """Several rows per CTA, some of them padding (not read), some with a bad id; loss and gradient in one call and in two."""
    import torch
    T, K = 1900, 9
    x = make(T, V, dtype, seed=6, shift=1)
    ids, values, all_values = teacher(T, V, K, seed=7)
    kind = torch.randint(0, 5, (T,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ids[kind == 0] = 0
    x[kind == 0] = float("nan")
    check(cuda, x, ids, values)
    lse = torch.logsumexp(all_values, 1) + 0.25
    check(cuda, x, ids, values, lse)
    cuda.check_device_status(0)
    ids[kind == 1, 4] = V + 1
    loss, d = cuda.distill.distill_fwd_bwd(x, ids, values, torch.ones(T, device="cuda"), lse)
    with pytest.raises(cuda.CtbError, match="out-of-range index"):
        cuda.check_device_status(0)
    assert loss[kind == 1].isnan().all() and (loss[kind == 0] == 0).all() and loss[kind > 1].isfinite().all()
    assert (d[kind < 2] == 0).all() and d.isfinite().all()


def test_repeatable_and_on_streams(cuda):
    """Bitwise the same on every call, on several streams at once and from replayed graphs beside eager calls."""
    import torch
    ops = cuda.distill
    cases = []
    for T, V, K, dtype in ((2, 120001, 60, "bfloat16"), (64, 30000, 256, "float32"), (700, 5000, 17, "float16")):
        x = make(T, V, dtype, seed=T)
        ids, values, all_values = teacher(T, V, K, seed=V)
        ids[:, K // 2] = ids[:, 0]
        cases.append((x, ids, values, torch.logsumexp(all_values, 1) + 0.5, torch.rand(T, device="cuda")))

    def run(i):
        x, ids, values, lse, g = cases[i]
        loss, saved = ops.distill_fwd(x, ids, values)
        return [loss, saved, ops.distill_bwd(x, ids, values, saved, g), *ops.distill_fwd_bwd(x, ids, values, g, lse)]
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


def test_refusals(cuda):
    import torch
    ops, lib = cuda.distill, cuda._lib
    x = make(4, 1000, "float32")
    ids, values, _ = teacher(4, 1000, 8)
    g = torch.ones(4, device="cuda")

    def refused(status, word, f):
        with pytest.raises(cuda.CtbError, match=word) as e:
            f()
        assert e.value.status == status
    many = torch.ones(4, 257, device="cuda", dtype=torch.int32)
    refused(lib.UNSUPPORTED, "1 to 256 entries", lambda: ops.distill_fwd(x, many, many.float()))
    refused(lib.UNSUPPORTED, "1 to 256 entries", lambda: ops.distill_fwd(x, ids[:, :0], values[:, :0]))
    refused(lib.BAD_ARG, "shape", lambda: ops.distill_fwd(x, ids[:3], values[:3]))
    refused(lib.BAD_ARG, "shape", lambda: ops.distill_fwd(x, ids, values[:, :7]))
    refused(lib.BAD_ARG, "int32 or int64", lambda: ops.distill_fwd(x, ids.float(), values))
    refused(lib.BAD_ARG, "element type", lambda: ops.distill_fwd(x, ids, values.double()))
    refused(lib.BAD_ARG, "teacher_lse", lambda: ops.distill_fwd(x, ids, values, g.half()))
    refused(lib.BAD_ARG, "temperature", lambda: ops.distill_fwd(x, ids, values, temperature=0))
    refused(lib.BAD_ARG, "saved", lambda: ops.distill_bwd(x, ids, values, torch.zeros(4, 3, device="cuda"), g))
    refused(lib.BAD_ARG, "d_loss", lambda: ops.distill_fwd_bwd(x, ids, values, g[:2]))
    refused(lib.BAD_ARG, "not overlap", lambda: ops.distill_fwd_bwd(x[:3], ids[:3], values[:3], g[:3], out=x[1:]))
    loss, d = ops.distill_fwd_bwd(x[:0], ids[:0], values[:0], g[:0])
    assert loss.shape == (0,) and d.shape == (0, 1000)
    cuda.check_device_status(0)
