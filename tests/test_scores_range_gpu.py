"""Operators over rows of logits at the ends of their range: rows that start anywhere, large logits, small temperatures, rows that a mask
of any kind leaves empty."""
import pytest

pytestmark = pytest.mark.gpu

from test_logprobs_gpu import TYPES, check, make  # noqa: E402


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("dtype", TYPES)
def test_lists_made_again_from_rows_that_start_anywhere(cuda, shift, dtype):
    """Ascending rows, whose list overflows, and rows of equal values: their first and last vectors are read element by element."""
    import torch
    V = 9003
    x = make(4, V, dtype, shift=shift, ld=V + 1)
    x[:2] = torch.linspace(-20, 20, V, device="cuda").to(x.dtype)
    x[2:] = 1.5
    check(cuda, x, torch.tensor([1, V, 1, V], device="cuda"), 32)
