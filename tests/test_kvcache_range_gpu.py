"""Cache writes and rotary positions of large calls, whose kernels take several rows and units at a time, against f64 as in test_kvcache_gpu and
test_rope_gpu; calls that their documentation allows and those tests do not make."""
import pytest

from test_kvcache_gpu import STORES, places
from test_rope_gpu import close, make

pytestmark = pytest.mark.gpu


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
