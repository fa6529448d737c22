"""Rotary positions and the paged cache without a GPU: frequencies, and what is refused before any device call."""
import ctypes as C
import math

import pytest


def test_null_context():
    from cutile_b200 import _lib
    for name in ("ctb_rope", "ctb_kv_write", "ctb_kv_read", "ctb_fmha_paged"):
        args = [0 if t.__name__ in ("c_int", "c_long", "c_longlong") else 1.0 if t.__name__ == "c_float" else None for t in _lib.SIGNATURES[name]]
        assert getattr(_lib.lib, name)(*args) == _lib.BAD_ARG and "null context" in _lib.last_error()


def test_cache_layout_matches_header(tmp_path):
    import os
    import subprocess

    from cutile_b200 import _lib
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    src = tmp_path / "layout.c"
    names = [n for n, _ in _lib.KvCacheArrays._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cutile_b200.h"\nint main(void) { printf("%zu", sizeof(ctb_kv_cache));\n' +
                   "".join(f'printf(" %zu", offsetof(ctb_kv_cache, {n}));\n' for n in names) + "return 0; }\n")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    said = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert said == [C.sizeof(_lib.KvCacheArrays)] + [getattr(_lib.KvCacheArrays, n).offset for n in names]


def test_frequencies():
    import torch

    import cutile_b200 as ctb
    freq = ctb.rope.rope_frequencies
    f = freq(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and not f.is_cuda
    for i in (0, 1, 17, 31):
        assert abs(float(f[i]) - 10000.0 ** (-2 * i / 64)) <= 1e-15 * float(f[i])
    assert torch.equal(freq(64, scaling="linear", factor=4.0), f / 4)
    g = freq(64, scaling="base", factor=8.0)
    assert abs(float(g[0]) - 1) < 1e-15 and abs(float(g[31] / f[31]) - 1 / 8) < 1e-12  # the last pair is divided by the factor
    h = freq(64, scaling="parts", factor=8.0, original_length=8192, low=1.0, high=4.0)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(h[turns >= 4], f[turns >= 4]) and torch.allclose(h[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (h[mid] < f[mid]).all() and (h[mid] > f[mid] / 8).all()
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=64, base=0.0), dict(rotary_dim=64, factor=-1.0), dict(rotary_dim=64, scaling="other"),
                dict(rotary_dim=2, scaling="base"), dict(rotary_dim=64, scaling="parts"), dict(rotary_dim=64, scaling="parts", original_length=10, low=2.0, high=2.0)):
        with pytest.raises(ctb.CtbError) as e:
            freq(**bad)
        assert e.value.status == ctb._lib.BAD_ARG


def test_host_arrays():
    import torch

    import cutile_b200 as ctb
    x, one = torch.zeros(2, 2, 64), torch.ones(2, dtype=torch.int32)
    table, f = torch.ones(2, 1, dtype=torch.int32), ctb.rope.rope_frequencies(64)
    cache = ctb.kvcache.kv_cache(2, 2, 16, 64, torch.float16, device="cpu")
    calls = [lambda: ctb.rope.rope_fwd(x, x, one, f), lambda: ctb.rope.rope_bwd(x, None, one, f), lambda: ctb.kvcache.kv_write(cache, one, x.half(), x.half()),
             lambda: ctb.kvcache.kv_read(cache, table, one, 4), lambda: ctb.fmha.fmha_paged(x.half(), cache, table, one)]
    for call in calls:
        with pytest.raises(ctb.CtbError, match="CUDA tensor") as e:
            call()
        assert e.value.status == ctb._lib.BAD_ARG


def test_argument_helpers():
    """The checks of the Python side on tensors of the host, which they take for arrays of one device."""
    import torch

    import cutile_b200 as ctb
    from cutile_b200.kvcache import KvCache, cache_struct, page_table_of
    like = torch.zeros(1)
    cache = ctb.kvcache.kv_cache(3, 2, 16, 64, torch.int8, device="cpu")
    s = cache_struct(cache, like)
    assert (s.pages, s.kv_heads, s.page_size, s.head_dim, s.dtype) == (3, 2, 16, 64, ctb._lib.I8)
    assert (s.k_page_stride, s.k_scale_page_stride) == (2 * 16 * 64, 2 * 16) and s.v == cache.v.data_ptr() and s.v_scale == cache.v_scale.data_ptr()
    both = torch.zeros(3, 2, 2, 16, 64, dtype=torch.float16)
    s = cache_struct(KvCache(both[:, 0], both[:, 1]), like)
    assert s.k_page_stride == s.v_page_stride == 2 * 2 * 16 * 64 and s.v - s.k == 2 * 16 * 64 * 2 and not s.k_scale
    table = torch.ones(4, 7, dtype=torch.int32)
    assert page_table_of(table[:, :5], torch.ones(4, dtype=torch.int32), like) == (4, 5, 7)
    assert page_table_of(table[:1, :0], torch.ones(1, dtype=torch.int32), like)[:2] == (1, 0)
    h = torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    for bad in (KvCache(h, h[:2]), KvCache(h, h.bfloat16()), KvCache(h.float(), h.float()), KvCache(h, None), KvCache(h, h, cache.k_scale, cache.v_scale),
                KvCache(cache.k, cache.v), KvCache(cache.k, cache.v, cache.k_scale, cache.v_scale.half()), KvCache(h.transpose(2, 3), h.transpose(2, 3))):
        with pytest.raises(ctb.CtbError) as e:
            cache_struct(bad, like)
        assert e.value.status == ctb._lib.BAD_ARG
    for t, n in ((table.long(), torch.ones(4, dtype=torch.int32)), (table, torch.ones(3, dtype=torch.int32)), (table, torch.ones(4)), (table.t(), torch.ones(7, dtype=torch.int32))):
        with pytest.raises(ctb.CtbError):
            page_table_of(t, n, like)
