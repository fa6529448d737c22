"""Rotary positions and their gradient against f64.

A result is x1 cos - x2 sin (or x1 sin + x2 cos), times the scale.  Cosines and sines are within 2^-22 (the angle's half turns are
rounded to f32, pi 2^-25, and sincospif is good to 2 ulp), the product with the scale, the two products and the sum take one f32 rounding (2^-24) each at most:
(|x1| + |x2|) |scale| (2^-22 + 3 2^-24) <= 2^-21 of that together, and one rounding to the type, eps / 2 of the result or half of its
smallest step.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "float16", "bfloat16")


def reference(x, positions, f, interleaved=False, scale=1.0, inverse=False):
    """(turned, the sizes of its terms), f64; x [..., heads, D], positions [...]"""
    import torch
    x = x.double()
    a = (positions.double()[..., None] * f.to(x.device))[..., None, :]
    cos, sin = scale * torch.cos(a), scale * torch.sin(a) * (-1 if inverse else 1)
    n = f.numel()
    out, size = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    x1, x2 = x[..., one], x[..., two]
    out[..., one], out[..., two] = x1 * cos - x2 * sin, x1 * sin + x2 * cos
    size[..., one] = size[..., two] = (x1.abs() + x2.abs()) * abs(scale)
    return out, size


def close(got, x, positions, f, **kw):
    import torch
    want, size = reference(x, positions, f, **kw)
    info = torch.finfo(got.dtype)
    err = (got.double() - want).abs()
    bound = size * 2.0 ** -21 + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2
    bound[..., 2 * f.numel():] = 0
    assert (err <= bound).all(), (err - bound).max()


def make(T, heads, D, dtype, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, heads, D, device="cuda", generator=g).to(getattr(torch, dtype))


@pytest.mark.parametrize("T,Hq,Hk,D,R", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 5, 5, 64, 64), (33, 4, 2, 64, 32), (129, 3, 1, 80, 80), (40, 2, 2, 96, 24),
                                         (257, 8, 1, 256, 256), (19, 3, 3, 66, 6), (5, 2, 1, 31, 30), (3001, 4, 4, 128, 64), (2, 1, 1, 4096, 4096)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_and_gradient(cuda, T, Hq, Hk, D, R, dtype, interleaved):
    import torch
    q, k = make(T, Hq, D, dtype, 1), make(T, Hk, D, dtype, 2)
    f = cuda.rope.rope_frequencies(R)
    positions = torch.arange(T, device="cuda", dtype=torch.int32) * 37 + 5
    for fn, inverse in ((cuda.rope.rope_fwd, False), (cuda.rope.rope_bwd, True)):
        oq, ok = fn(q, k, positions, f.cuda(), interleaved=interleaved, scale=1.25)
        assert oq.shape == q.shape and ok.shape == k.shape and oq.dtype == q.dtype
        close(oq, q, positions, f, interleaved=interleaved, scale=1.25, inverse=inverse)
        close(ok, k, positions, f, interleaved=interleaved, scale=1.25, inverse=inverse)
        alone, none = fn(q, None, positions.long(), f.cuda(), interleaved=interleaved, scale=1.25)
        assert none is None and alone.equal(oq)


@pytest.mark.parametrize("first", [0, 1 << 20, 2 ** 31 - 1000, -5, -(2 ** 31 - 1000)])
def test_far_positions(cuda, first):
    import torch
    q = make(64, 2, 128, "float32", 3)
    f = cuda.rope.rope_frequencies(128)
    positions = torch.arange(64, device="cuda") + first
    close(cuda.rope.rope_fwd(q, None, positions, f.cuda())[0], q, positions, f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_views_and_in_place(cuda, dtype, shift):
    """Heads of a fused projection, at any element, with padding between tokens, and in place; what stands between stays as it is."""
    import torch
    T, Hq, Hk, D = 21, 6, 2, 64
    base = torch.full((T, (Hq + 2 * Hk) * D + 8 + shift), 7.0, device="cuda", dtype=getattr(torch, dtype))
    q = base[:, shift:shift + Hq * D].unflatten(1, (Hq, D))
    k = base[:, shift + Hq * D:shift + (Hq + Hk) * D].unflatten(1, (Hk, D))
    q.copy_(make(T, Hq, D, dtype, 4))
    k.copy_(make(T, Hk, D, dtype, 5))
    before = base.clone()
    f, positions = cuda.rope.rope_frequencies(32), torch.arange(T, device="cuda")
    oq, ok = cuda.rope.rope_fwd(q, k, positions, f.cuda())
    assert base.equal(before)
    close(oq, q, positions, f)
    close(ok, k, positions, f)
    rq, rk = cuda.rope.rope_fwd(q, k, positions, f.cuda(), out_q=q, out_k=k)
    assert rq is q and rk is k and q.equal(oq) and k.equal(ok)
    rest = before.clone()
    rest[:, shift:shift + (Hq + Hk) * D] = base[:, shift:shift + (Hq + Hk) * D]
    assert base.equal(rest)


@pytest.mark.parametrize("dtype", TYPES)
def test_arrays_of_attention(cuda, dtype):
    """[Batch, Heads, SeqLen, D] by transposed views; one position for many tokens; expanded inputs."""
    import torch
    Q = make(3 * 4 * 11, 1, 64, dtype, 6).view(3, 4, 11, 64)
    f = cuda.rope.rope_frequencies(64)
    positions = torch.randint(0, 5000, (3, 11), device="cuda")
    out, _ = cuda.rope.rope_fwd(Q.transpose(1, 2), None, positions, f.cuda())
    assert out.transpose(1, 2).is_contiguous()
    close(out, Q.transpose(1, 2), positions, f)
    row = make(1, 1, 64, dtype, 7)
    many = row.expand(40, 3, 64)
    positions = torch.arange(40, device="cuda")
    out, _ = cuda.rope.rope_fwd(many, None, positions, f.cuda())
    close(out, many, positions, f)
    with pytest.raises(cuda.CtbError, match="rows of a result overlap"):
        cuda.rope.rope_fwd(many, None, positions, f.cuda(), out_q=many)


def test_copied_elements_are_copied(cuda):
    import torch
    q = make(5, 2, 64, "float32", 8)
    q[..., 32:] = float("nan")
    q[0, 0, 40] = float("inf")
    out, _ = cuda.rope.rope_fwd(q, None, torch.arange(5, device="cuda"), cuda.rope.rope_frequencies(32).cuda())
    assert out[..., 32:].view(torch.int32).equal(q[..., 32:].contiguous().view(torch.int32)) and out[..., :32].isfinite().all()


def test_gradient_by_differences(cuda):
    """The turn is linear: a difference of two results is the turn of the difference, and <fwd(x), d> = <x, bwd(d)>."""
    import torch
    x, d = make(9, 3, 64, "float32", 9), make(9, 3, 64, "float32", 10)
    f, positions = cuda.rope.rope_frequencies(48).cuda(), torch.arange(9, device="cuda") * 1000
    y = cuda.rope.rope_fwd(x, None, positions, f, scale=0.5)[0]
    g = cuda.rope.rope_bwd(d, None, positions, f, scale=0.5)[0]
    size = float((x.double().abs().sum() + 1) * d.abs().max())
    assert abs(float((y.double() * d.double()).sum() - (x.double() * g.double()).sum())) <= size * 2.0 ** -20
    h = 2.0 ** -6  # exact in f32 beside these values to 2^-18
    for at in ((0, 0, 0), (4, 1, 30), (8, 2, 63)):
        z = x.clone()
        z[at] += h
        step = float(z[at].double() - x[at].double())
        slope = ((cuda.rope.rope_fwd(z, None, positions, f, scale=0.5)[0].double() - y.double()) * d.double()).sum() / step
        assert abs(float(slope - g[at])) <= 8 * float(d.abs().max()) * float(x.abs().max()) * 2.0 ** -21 / h


def test_empty(cuda):
    import torch
    f = cuda.rope.rope_frequencies(64).cuda()
    q = torch.empty(0, 4, 64, device="cuda")
    assert cuda.rope.rope_fwd(q, q, torch.empty(0, device="cuda", dtype=torch.int32), f)[0].shape == q.shape


def test_captured(cuda):
    import torch
    q, k = make(50, 4, 128, "bfloat16", 11), make(50, 2, 128, "bfloat16", 12)
    f, positions = cuda.rope.rope_frequencies(128).cuda(), torch.arange(50, device="cuda")
    oq, ok = torch.empty_like(q), torch.empty_like(k)
    cuda.rope.rope_fwd(q, k, positions, f, out_q=oq, out_k=ok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda.rope.rope_fwd(q, k, positions, f, out_q=oq, out_k=ok)
    positions += 100
    q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    close(oq, q, positions, f.cpu())
    close(ok, k, positions, f.cpu())


def test_large_strides(cuda):
    """Sequences more than 2^31 elements apart, and strides along dimensions of one element, which mean nothing."""
    import torch
    apart = 2 ** 31 + 64
    f, positions = cuda.rope.rope_frequencies(64).cuda(), torch.tensor([[3, 4], [70, 5]], device="cuda")
    store = torch.empty(apart + 2 * 3 * 64, device="cuda", dtype=torch.float16)
    q = store.as_strided((2, 2, 3, 64), (apart, 3 * 64, 64, 1))
    q.copy_(make(4, 3, 64, "float16", 3).view(2, 2, 3, 64))
    before = q.clone()
    close(cuda.rope.rope_fwd(q, None, positions, f)[0], before, positions, f.cpu())
    cuda.rope.rope_fwd(q, None, positions, f, out_q=q)
    close(q, before, positions, f.cpu())
    one = before[:1, :1].as_strided((1, 1, 3, 64), (2 ** 40, 2 ** 40, 64, 1))
    close(cuda.rope.rope_fwd(one, None, positions[:1, :1], f)[0], before[:1, :1], positions[:1, :1], f.cpu())
    with pytest.raises(cuda.CtbError, match="strides too large"):
        cuda.rope.rope_fwd(store.as_strided((1, 2, 3, 64), (apart, apart, 64, 1)), None, positions[:1], f)


def test_refusals(cuda):
    import torch
    q, k = make(4, 2, 64, "float16"), make(4, 1, 64, "float16")
    f, positions = cuda.rope.rope_frequencies(64).cuda(), torch.arange(4, device="cuda")
    big = torch.zeros(8, 2, 64, device="cuda", dtype=torch.float16)
    calls = [(dict(q=q.double()), "element type"), (dict(q=q[:, 0]), "expected"), (dict(q=q.transpose(1, 2)), "contiguous heads"), (dict(k=k.float()), "type and device"),
             (dict(k=k[:2]), "tokens"), (dict(positions=positions[:3]), "positions"), (dict(positions=positions.float()), "int32 or int64"),
             (dict(frequencies=f.float()), "float64"), (dict(frequencies=f.cpu()), "expected a tensor on"), (dict(frequencies=f[None]), "one dimension"),
             (dict(frequencies=torch.cat((f, f)).contiguous()), "rotary"), (dict(frequencies=f[:0]), "rotary"), (dict(scale=float("nan")), "not finite"),
             (dict(out_q=q.float()), "out_q"), (dict(q=big[:4], out_q=big[2:6]), "must lie where"), (dict(q=q.cpu()), "CUDA tensor")]
    for change, word in calls:
        args = dict(dict(q=q, k=None, positions=positions, frequencies=f), **change)
        with pytest.raises(cuda.CtbError, match=word):
            cuda.rope.rope_fwd(**args)
    assert math.isfinite(float(cuda.rope.rope_fwd(q, k, positions, f, occupancy=2)[0].sum()))  # launch keywords
