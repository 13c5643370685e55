"""Threads that share the default handle of a device, each on a stream of its
own: products, softmaxes and the operators between logits and an update side by
side, each reading what its thread has written right before."""
import threading

import pytest

pytestmark = pytest.mark.gpu


def test_products_beside_log_probabilities(kx, torch_cuda):
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(96, 2000, generator=gen, device="cuda")
    tokens = torch.arange(96, device="cuda")
    eye = torch.eye(96, device="cuda")
    torch.cuda.synchronize()
    wrong = []

    def scores(x):
        out = kx.token_log_probs(x, tokens, top=2)
        lse = torch.logsumexp(x, -1)
        # sums of 2000 terms in f32: 2000 2^-24 at the very most, of about 8
        return bool(((out.lse - lse).abs() <= 3e-4 * lse.abs()).all()) and torch.equal(out.top_tokens[:, 0], x.argmax(-1))

    def norm(x):
        # 192000 squares: 2e5 2^-24 of the norm at the very most on torch's side
        return abs(float(kx.grad_norm([x])) / float(torch.linalg.vector_norm(x)) - 1) <= 0.012

    def product(x):
        # by the unit matrix: each element once, in two parts that hold 21 bits or more of it
        return bool(((kx.matmul(eye, x) - x).abs() <= x.abs() * 2.0 ** -20).all())

    def softmax(x):
        p = kx.softmax(x, -1)
        return bool(((p - torch.softmax(x, -1)).abs() <= 1e-3 * p).all())

    def work(k, check):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(80):
                    if not check(base * (1 + 0.01 * k) + 0.01 * i):     # written on this stream right before
                        wrong.append((check.__name__, i))
        except Exception as e:  # noqa: BLE001  (reported by the test's thread)
            wrong.append((check.__name__, e))

    threads = [threading.Thread(target=work, args=(k, c)) for k, c in enumerate((scores, norm, product, softmax, scores))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_closed_handle_is_refused(kx, torch_cuda):
    """In every call, through the binding and the general path alike."""
    torch = torch_cuda
    own = kx.Handle(0)
    own.close()
    x, t = torch.zeros(4, 4, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    view = kx.TensorView(x.reshape(-1), (4, 4), (4, 1))
    row = torch.zeros(4, device="cuda")
    with kx.using(own):
        for call in (lambda: kx.matmul(x, x), lambda: kx.softmax(x, -1), lambda: kx.token_log_probs(x, t),
                     lambda: kx.token_log_probs(view, t), lambda: kx.grad_norm([x]), lambda: kx.grad_norm([view]),
                     lambda: kx.token_log_probs_backward(x, t, lse=row, grad_log_probs=row),
                     lambda: kx.clip_grad_norm([x], 1.0)):
            with pytest.raises(kx.InvalidParameter):
                call()
