"""Log probabilities and their gradient at the ends of what they take: the
largest temperatures, and rows that answer with NaN."""
import numpy as np
import pytest

from test_log_probs_gpu import backward, check_backward, check_forward, grads_in, logits, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,t", [(np.float32, 1e29), (np.float32, 5e30), (np.float32, 3e37), (np.float32, 1e38),
                                     (np.float64, 1e292), (np.float64, 1e307), (np.float64, 1e308)])
@pytest.mark.parametrize("v", [5, 1000, 9001])
def test_temperatures_near_the_largest_number(kx, torch_cuda, dtype, t, v):
    """lse is log V there, T lse may not be finite in the type; incoming
    gradients of the temperature's size make results that can be seen.  A mask
    of the type's lowest value in one row still is a token of some probability
    at the largest temperatures."""
    x, tokens = logits(101 + v, 4, v, dtype)
    x[1, ::3] = -np.inf
    x[2, 0] = np.finfo(dtype).min
    x[3] = -np.inf
    check_forward(run(kx, torch_cuda, x, tokens, t, 3), x, tokens, t, dtype, 3)
    g, gh, gl = [(a * dtype(t / 4)).astype(dtype) for a in grads_in(49, 4, dtype)]
    for a in ((g, None, None), (None, None, gl), (g, gh, gl)):
        got = backward(kx, torch_cuda, x, tokens, t, *a)
        assert np.isfinite(got).all() and (got[:3] != 0).any()
        check_backward(got, x, tokens, t, dtype, *a)
