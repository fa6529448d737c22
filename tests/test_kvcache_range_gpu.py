"""Cache writes and rotary positions of large calls, whose kernels take several rows and units at a time, against f64 as in test_kvcache_gpu and
test_rope_gpu; calls that their documentation allows and those tests do not make."""
import pytest

from test_kvcache_gpu import STORES, filled, places, rows_at, stored_close, turned, untouched
from test_rope_gpu import close, make

pytestmark = pytest.mark.gpu


# Tokens * heads * D is above what 148 SMs take one group per warp for (2.42 M elements); two groups per warp up to 512 elements of keys per token,
# then four.  Heads that do not fill the groups of a task, tokens that do not fill the last CTA, and queries that are few or many beside the keys.
@pytest.mark.parametrize("T,H,KVH,D,page,R,interleaved,shift", [
    (2501, 8, 4, 128, 16, 128, False, 0), (10001, 0, 2, 64, 32, 64, False, 0), (4003, 3, 8, 64, 64, 32, True, 0), (3001, 40, 1, 128, 16, 24, False, 0),
    (2000, 5, 5, 128, 128, 64, False, 1), (1701, 32, 8, 128, 16, 128, False, 0), (3001, 1, 9, 64, 1024, 64, True, 0), (2003, 0, 8, 128, 16, 0, False, 0),
    (1999, 9, 9, 128, 32, 12, True, 1), (8200, 0, 9, 64, 16, 6, False, 0), (5003, 2, 5, 128, 64, 2, True, 0)])
@pytest.mark.parametrize("store", STORES)
def test_large_writes(cuda, T, H, KVH, D, page, R, interleaved, shift, store):
    import torch
    assert T * (H + 2 * KVH) * D >= 256 * 4 * 16 * 148
    dtype = getattr(torch, store) if store.endswith("float16") else (torch.bfloat16 if T % 3 else torch.float16)
    g = torch.Generator(device="cuda").manual_seed(T)
    base = torch.randn(T, (H + 2 * KVH) * D + 8 * shift + shift, device="cuda", generator=g).to(dtype)
    q, k, v = base[:, shift:shift + (H + 2 * KVH) * D].unflatten(1, (H + 2 * KVH, D)).split((H, KVH, KVH), 1)
    pages = -(-T // page) + 3
    cache = filled(cuda, pages, KVH, page, D, store)
    before = [None if t is None else t.clone() for t in cache]
    slots = places(pages, page, T, T)
    slots[::7] = 0
    live = slots > 0
    f = cuda.rope.rope_frequencies(R) if R else None
    positions = torch.randint(0, 100000, (T,), device="cuda", generator=g)
    more = dict(positions=positions, frequencies=f.cuda(), interleaved=interleaved, scale=0.75, q=q if H else None) if R else {}
    out = cuda.kvcache.kv_write(cache, slots, k, v, **more)
    untouched(before, cache, slots[live])
    if H and R:
        close(out, q, positions, f, interleaved=interleaved, scale=0.75)
        was, kept = q.clone(), base.clone()
        assert cuda.kvcache.kv_write(cache, slots, k, v, out_q=q, **more) is q  # in place
        assert q.equal(out)
        q.copy_(was)
        assert base.equal(kept)
    else:
        assert out is None
    for i, x in enumerate((k, v)):
        got = rows_at(cache[i], slots[live])
        want, off = turned(x, positions, f if i == 0 else None, interleaved)
        if cache.k_scale is not None:
            stored_close(got, rows_at(cache[2 + i], slots[live]), want[live], off[live] if torch.is_tensor(off) else off)
        elif i == 1 or not R:
            assert got.equal(x[live])
        else:
            close(got, x[live], positions[live], f, interleaved=interleaved, scale=0.75)


# Two units per thread: from 4.85 M elements in 16-bit vectors, 2.42 M in f32 ones, 0.61 M off the grid of 16 bytes (148 SMs).
@pytest.mark.parametrize("T,Hq,Hk,D,R,shift", [(4099, 8, 2, 128, 128, 0), (20001, 3, 1, 64, 32, 0), (16001, 2, 2, 80, 80, 0), (1201, 16, 1, 256, 64, 0),
                                               (3001, 3, 1, 64, 64, 1), (1201, 5, 3, 66, 6, 0), (5001, 7, 0, 128, 24, 0), (150, 1, 1, 4096, 4096, 1)])
@pytest.mark.parametrize("dtype", ("float32", "float16", "bfloat16"))
@pytest.mark.parametrize("interleaved", [False, True])
def test_large_turns(cuda, T, Hq, Hk, D, R, shift, dtype, interleaved):
    import torch
    vector = 4 if dtype == "float32" else 8
    assert T * (Hq + Hk) * D >= 2 * (vector if D % vector == 0 and R % (2 * vector) == 0 and not shift else 1) * 256 * 2 * 4 * 148
    base = make(T, Hq + Hk + (1 if shift else 0), D, dtype, T).flatten(1)
    q, k = base[:, shift:shift + (Hq + Hk) * D].unflatten(1, (Hq + Hk, D)).split((Hq, Hk), 1)
    f = cuda.rope.rope_frequencies(R)
    positions = torch.arange(T, device="cuda", dtype=torch.int32) * 37 + 5
    for fn, inverse in ((cuda.rope.rope_fwd, False), (cuda.rope.rope_bwd, True)):
        oq, ok = fn(q, k if Hk else None, positions, f.cuda(), interleaved=interleaved, scale=1.25)
        close(oq, q, positions, f, interleaved=interleaved, scale=1.25, inverse=inverse)
        if Hk:
            close(ok, k, positions, f, interleaved=interleaved, scale=1.25, inverse=inverse)
    kept = base.clone()
    rq, rk = cuda.rope.rope_bwd(q, k if Hk else None, positions, f.cuda(), interleaved=interleaved, scale=1.25, out_q=q, out_k=k if Hk else None)
    assert rq is q and q.equal(oq) and (not Hk or k.equal(ok))
    base[:, shift:shift + (Hq + Hk) * D] = kept[:, shift:shift + (Hq + Hk) * D]
    assert base.equal(kept)


def test_frequencies_of_no_pairs(cuda):
    """An empty array, whose address is null, is not the same as none."""
    import torch
    cache = cuda.kvcache.kv_cache(1, 2, 16, 64, torch.float16)
    k, positions = torch.ones(3, 2, 64, device="cuda").half(), torch.arange(1, 4, device="cuda")
    none = torch.empty(0, device="cuda", dtype=torch.float64)
    for more in ({}, dict(q=k), dict(occupancy=1)):
        with pytest.raises(cuda.CtbError, match="rotary"):
            cuda.kvcache.kv_write(cache, positions, k, k, positions=positions, frequencies=none, **more)
    with pytest.raises(cuda.CtbError, match="rotary"):
        cuda.rope.rope_fwd(k, None, positions, none)
    assert (cache.k == 0).all()


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("bits", ["int32", "int64"])
def test_rows_that_are_not_turned(cuda, store, bits):
    """Positions beside frequencies of None, as of a model without rotary positions: rows are stored as they are."""
    import torch
    k, v = (torch.randn(9, 2, 64, device="cuda").to(torch.bfloat16 if store != "float16" else torch.float16) for _ in range(2))
    slots, positions = places(2, 16, 9), torch.arange(9, device="cuda").to(getattr(torch, bits))
    caches = [cuda.kvcache.kv_cache(2, 2, 16, 64, getattr(torch, store)) for _ in range(3)]
    for cache, more in zip(caches, ({}, dict(positions=positions, frequencies=None), dict(positions=positions, frequencies=None, occupancy=1))):
        assert cuda.kvcache.kv_write(cache, slots, k, v, q=None, interleaved=True, **more) is None
    for other in caches[1:]:
        for x, y in zip(caches[0], other):
            assert x is y is None or x.view(torch.uint8).equal(y.view(torch.uint8))
    for bad, word in ((positions[:8], "positions"), (positions.float(), "int32 or int64"), (positions.cpu(), "positions")):
        with pytest.raises(cuda.CtbError, match=word):
            cuda.kvcache.kv_write(caches[0], slots, k, v, positions=bad, frequencies=None)
    with pytest.raises(cuda.CtbError, match="positions and frequencies"):
        cuda.kvcache.kv_write(caches[0], slots, k, v, q=k, positions=positions, frequencies=None)


def test_results_whose_rows_overlap(cuda):
    """Strides that are each as long as a row, but too short together."""
    import torch
    f, positions = cuda.rope.rope_frequencies(64).cuda(), torch.arange(3, device="cuda")
    q = make(3, 2, 64, "float16")
    store = torch.zeros(4096, device="cuda", dtype=torch.float16)
    cache = cuda.kvcache.kv_cache(1, 2, 16, 64, torch.float16)
    for strides in ((64, 64, 1), (96, 64, 1), (64, 96, 1), (64, 191, 1)):
        out = store.as_strided((3, 2, 64), strides)
        with pytest.raises(cuda.CtbError, match="rows of a result overlap"):
            cuda.rope.rope_fwd(q, None, positions, f, out_q=out)
        with pytest.raises(cuda.CtbError, match="rows of a result overlap"):
            cuda.kvcache.kv_write(cache, positions, q, q, q=q, positions=positions, frequencies=f, out_q=out)
    assert (store == 0).all() and (cache.k == 0).all()
    for strides in ((128, 64, 1), (64, 192, 1), (200, 72, 1)):
        out = store.as_strided((3, 2, 64), strides)
        cuda.rope.rope_fwd(q, None, positions, f, out_q=out)
        close(out, q, positions, f.cpu())
    out = store.as_strided((1, 3, 2, 64), (1, 128, 64, 1))  # the batch of one has no stride
    cuda.rope.rope_fwd(q[None], None, positions[None], f, out_q=out)
    close(out[0], q, positions, f.cpu())
