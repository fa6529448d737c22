"""Operators over rows of scores without a GPU: what is refused before any device call."""
import pytest


def test_null_context():
    from cutile_b200 import _lib
    for name in ("ctb_token_logprobs", "ctb_token_logprobs_bwd", "ctb_distill_fwd", "ctb_distill_bwd", "ctb_distill_fwd_bwd", "ctb_moe_route",
                 "ctb_moe_route_bwd"):
        args = [0 if t.__name__ in ("c_int", "c_long", "c_longlong") else 1.0 if t.__name__ == "c_float" else None
                for t in _lib.SIGNATURES[name]]
        assert getattr(_lib.lib, name)(*args) == _lib.BAD_ARG and "null context" in _lib.last_error()


def test_host_arrays_and_bad_options():
    import torch

    import cutile_b200 as ctb
    x, ids, one = torch.zeros(2, 8), torch.ones(2, 3, dtype=torch.int32), torch.ones(2)
    calls = [lambda: ctb.logprobs.token_logprobs(x), lambda: ctb.logprobs.token_logprobs_bwd(x, None, one, one),
             lambda: ctb.distill.distill_fwd(x, ids, ids.float()), lambda: ctb.distill.distill_bwd(x, ids, ids.float(), one, one),
             lambda: ctb.distill.distill_fwd_bwd(x, ids, ids.float(), one), lambda: ctb.moe.moe_route(x, 2),
             lambda: ctb.moe.moe_route_bwd(x, ids, one)]
    for f in calls:
        with pytest.raises(ctb.CtbError, match="CUDA tensor") as e:
            f()
        assert e.value.status == ctb._lib.BAD_ARG


def test_argument_helpers():
    import torch

    import cutile_b200 as ctb
    from cutile_b200._util import dense, gradient_of, ids_bits
    x = torch.zeros(4, 6)
    assert ids_bits(torch.zeros(1, dtype=torch.int32), "ids") == 32 and ids_bits(torch.zeros(1, dtype=torch.int64), "ids") == 64
    assert dense(x, (4, 6), "x", x, torch.float32) is x
    out, ld = gradient_of(x[:, :3], None)
    assert out.shape == (4, 3) and ld == 3
    wide = torch.zeros(4, 10)
    assert gradient_of(x, wide[:, 2:8])[1] == 10
    for f, word in ((lambda: ids_bits(x, "ids"), "int32 or int64"), (lambda: dense(x[:, :3], (4, 3), "x", x), "dense"),
                    (lambda: dense(x, (6, 4), "x", x), "dense"), (lambda: dense(x, (4, 6), "x", x, torch.float16), "float16"),
                    (lambda: dense(None, (4, 6), "x", x), "expected a tensor"), (lambda: gradient_of(x, x.half()), "out must"),
                    (lambda: gradient_of(x, x.t().contiguous().t()), "contiguous rows")):
        with pytest.raises(ctb.CtbError, match=word) as e:
            f()
        assert e.value.status == ctb._lib.BAD_ARG
    with pytest.raises(ctb.CtbError, match="score must be"):
        ctb.moe._score("relu")
