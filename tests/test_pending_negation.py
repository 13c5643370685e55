"""Tensors whose negation torch has left to their readers: the memory holds the
other sign, so they are refused rather than read, in each place that describes
an operand (host), and by every kind of call (device)."""
import pytest
import torch as _torch

import kernix_b200 as kernix


def pending(device="cpu", dtype=_torch.complex64, shape=(4, 4)):
    x = _torch.randn(*shape, dtype=dtype, device=device).conj().imag
    assert x.is_neg()
    return x


def test_descriptors_refuse():
    x = pending()
    buf = kernix.C.create_string_buffer(kernix._SIZE)
    flat = pending(shape=(16,))
    for describe in (lambda: kernix._descriptor(x), lambda: kernix._pack(buf, 0, x),
                     lambda: kernix._descriptor(kernix.TensorView(flat, (4, 4), (4, 1))),
                     lambda: kernix._descriptors([x.resolve_neg(), x], [1]), lambda: kernix._descriptors([flat])):
        with pytest.raises(kernix.Unsupported, match="resolve_neg"):
            describe()
    kernix._descriptor(x.resolve_neg())
    kernix._descriptors([x.resolve_neg(), _torch.zeros(3)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [_torch.complex64, _torch.complex128])
def test_calls_refuse(kx, torch_cuda, dtype):
    torch = torch_cuda
    x, r = pending("cuda", dtype), pending("cuda", dtype, (4,))
    y, s = x.resolve_neg(), r.resolve_neg()
    t = torch.arange(4, device="cuda")
    lse = kx.token_log_probs(y, t).lse
    out = torch.full_like(y, 5.0)
    for call in (lambda: kx.matmul(x, y), lambda: kx.matmul_into(y, y, x), lambda: kx.softmax(x, -1),
                 lambda: kx.matmul_backward(y, x, y), lambda: kx.token_log_probs(x, t),
                 lambda: kx.token_log_probs_into(y, t, kx.TokenLogProbs(log_probs=r)),
                 lambda: kx.token_log_probs_backward(y, t, lse=lse, grad_log_probs=r),
                 lambda: kx.token_log_probs_backward_into(y, t, x, lse=lse, grad_log_probs=s),
                 lambda: kx.grad_norm([y, x]), lambda: kx.grad_norm([y.t(), x.t()]),
                 lambda: kx.clip_grad_norm([x], 1.0), lambda: kx.clip_grad_norm_into([y], 1.0, [x]),
                 lambda: kx.clip_grad_norm_into([x, y], 1.0, [out, torch.empty_like(y)])):
        with pytest.raises(kx.Unsupported, match="resolve_neg"):
            call()
    assert bool((out == 5).all())
    assert kx.grad_norm([x.resolve_neg()]).item() == kx.grad_norm([y]).item()
