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


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,v", [(9, 5), (9, 1003), (9, 5001), (3, 50_021)])
def test_masked_logits_of_a_row_that_is_nan(kx, torch_cuda, dtype, rows, v):
    """A NaN or +inf makes its row's gradient NaN, but for the logits of -inf,
    whose gradient is 0 in each row; in rows aligned like their gradient and
    not, and with a stride."""
    torch = torch_cuda
    x, tokens = logits(111 + v, rows, v, dtype)
    x[:, 1::2] = -np.inf
    x[0, 0], x[1, v - 1 - (v - 1) % 2], x[2, 2] = np.nan, np.inf, np.inf
    gone = np.isneginf(x)
    a = grads_in(59, rows, dtype)
    dev = [torch.from_numpy(b).cuda() for b in a]
    dt = torch.from_numpy(tokens).cuda()
    wide = torch.full((rows, v + 3), 7.0, dtype=dev[0].dtype, device="cuda")
    wide[:, 1:v + 1] = torch.from_numpy(x).cuda()
    plain = wide[:, 1:v + 1].contiguous()
    for view in (plain, wide[:, 1:v + 1], plain.t().contiguous().t()):
        res = kx.token_log_probs(view, dt, entropy=True)
        got = kx.token_log_probs_backward(view, dt, lse=res.lse, entropy=res.entropy, grad_log_probs=dev[0],
                                          grad_entropy=dev[1], grad_lse=dev[2]).cpu().numpy()
        assert (got[gone] == 0).all()
        assert np.isnan(got[:3][~gone[:3]]).all() and np.isfinite(got[3:]).all()
