"""The global gradient norm and clipping (kx_grad_norm_*, kx_clip_grad_norm_*)
against sums in 80-bit arithmetic, and the step from logits to clipped
gradients as a whole.

Bounds, with u half a step of the type (2^-24, 2^-53): squares are added in 64
bits, so the sum is off by at most n 2^-53 of itself and the root by half of
that; the norm then rounds once (u).  A scaled element is g times a factor that
is off by n 2^-53 + 2u, rounded once more: 3u + n 2^-53 of its size, or half a
step of the smallest numbers."""
import gc

import numpy as np
import pytest

from kernix_b200 import rng

pytestmark = pytest.mark.gpu
U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
LD = np.longdouble


def make(torch, seed, shapes, dtype, scale=1.0):
    arrs = [(rng.normal(seed + i, int(np.prod(s)) or 1, scale)[:int(np.prod(s))]).astype(dtype).reshape(s)
            for i, s in enumerate(shapes)]
    return arrs, [torch.from_numpy(a).cuda() for a in arrs]


def true_norm(arrs):
    return np.sqrt(sum((a.astype(LD).ravel() ** 2).sum() for a in arrs))


def check_norm(got, arrs, dtype):
    want, n = true_norm(arrs), sum(a.size for a in arrs)
    assert abs(LD(got.item()) - want) <= want * (U[dtype] + n * 2.0 ** -53), (got.item(), want)
    return want


def check_clip(norm, outs, arrs, max_norm, dtype):
    want = check_norm(norm, arrs, dtype)
    n = sum(a.size for a in arrs)
    by = LD(1) if want <= max_norm else LD(max_norm) / want
    for o, a in zip(outs, arrs):
        assert tuple(o.shape) == a.shape
        got = o.cpu().numpy().astype(LD)
        if by == 1:
            assert np.array_equal(got, a)
            continue
        w = a.astype(LD) * by
        tol = np.abs(w) * (3 * U[dtype] + n * 2.0 ** -53) + np.finfo(dtype).smallest_subnormal
        assert (np.abs(got - w) <= tol).all()


SETS = {
    "one element": [()],
    "one tensor": [(7, 3)],
    "empty among others": [(0, 4), (5,), (0,), (3, 0, 2), (11,)],
    "only empty": [(0,), (4, 0)],
    "odd sizes": [(1,), (2,), (3,), (4,), (5,), (1023,), (1024,), (1025,), (33, 65), (8193,), (3, 5, 7, 11)],
    "many small": [(i % 13 + 1,) for i in range(700)],
    "many": [(17,)] * 2500,
    "large and small": [(1 << 20,), (3,), (1000, 1001), (1,), (400_003,)],
}


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("name", list(SETS))
def test_norm_and_clip(kx, torch_cuda, dtype, name):
    torch = torch_cuda
    arrs, dev = make(torch, 7, SETS[name], dtype)
    norm = check_norm(kx.grad_norm(dev), arrs, dtype)
    for max_norm in (float(norm) * 0.37 or 1.0, float(norm) * 2 or 1.0):
        got, outs = kx.clip_grad_norm(dev, max_norm)
        check_clip(got, outs, arrs, max_norm, dtype)
        assert all(np.array_equal(d.cpu().numpy(), a) for d, a in zip(dev, arrs))
    mine = [d.clone() for d in dev]
    got = kx.clip_grad_norm_into(mine, 0.5, mine)       # in place
    check_clip(got, mine, arrs, 0.5, dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_layouts(kx, torch_cuda, dtype):
    """Transposed and permuted tensors, slices at every alignment with what
    lies beside them left alone, columns of a wider buffer, every second
    element, reversed and broadcast views, outputs of other strides."""
    torch = torch_cuda
    tt = torch.float32 if dtype == np.float32 else torch.float64
    base = rng.normal(3, 40_000, 1.0).astype(dtype)
    dev = torch.from_numpy(base).cuda()
    views = [dev[:1200].reshape(30, 40).t(), dev[1200:3600].reshape(10, 12, 20).permute(2, 0, 1),
             dev[3600:6600].reshape(60, 50)[:, 7:31], dev[6601:9000:2], dev[9000:9001].expand(5, 6)]
    views += [dev[10_000 + 1000 * i + i:10_000 + 1000 * i + 900] for i in range(6)]
    views.append(kx.TensorView(dev, (20, 30), (-40, -1), 39_999))
    arrs = [v.cpu().numpy() if not isinstance(v, kx.TensorView) else base[::-1][:800].reshape(20, 40)[:, :30].copy()
            for v in views]
    check_norm(kx.grad_norm(views), arrs, dtype)
    got, outs = kx.clip_grad_norm(views[:4] + views[5:11], 3.0)
    check_clip(got, outs, arrs[:4] + arrs[5:11], 3.0, dtype)
    # outputs of other strides than their gradients', in one guarded buffer
    buf = torch.full((60_000,), 9.0, dtype=tt, device="cuda")
    outs = [buf[:1200].reshape(30, 40).t(), buf[1200:3600].reshape(20, 10, 12), buf[4000:7000].reshape(60, 50)[:, :24],
            buf[8001:8001 + 2400:2], buf[12_000:12_030].reshape(5, 6)]
    outs += [buf[20_000 + 1000 * i + 2 * i + 1:][:a.size] for i, a in enumerate(arrs[5:11])]
    outs.append(kx.TensorView(buf, (20, 30), (-1, 20), 40_019))
    norm = kx.clip_grad_norm_into(views, 2.5, outs)
    assert torch.equal(norm, kx.grad_norm(views))      # the same bits, whatever the outputs are
    host = buf.cpu().numpy()
    last = np.array([[host[40_019 - i + 20 * j] for j in range(30)] for i in range(20)])
    check_clip(norm, outs[:-1] + [torch.from_numpy(last)], arrs, 2.5, dtype)
    touched = torch.zeros(60_000, dtype=torch.bool, device="cuda")
    marks = [touched[:1200], touched[1200:3600], touched[4000:7000].reshape(60, 50)[:, :24],
             touched[8001:8001 + 2400:2], touched[12_000:12_030]]
    marks += [touched[20_000 + 1000 * i + 2 * i + 1:][:a.size] for i, a in enumerate(arrs[5:11])]
    marks.append(touched[40_000:40_600])
    for m in marks:
        m.fill_(True)
    assert (buf[~touched] == 9).all()
    # in place on transposed and gapped views
    mine = dev.clone()
    place = [mine[:1200].reshape(30, 40).t(), mine[3600:6600].reshape(60, 50)[:, 7:31], mine[6601:9000:2]]
    norm = kx.clip_grad_norm_into(place, 1.5, place)
    check_clip(norm, place, [arrs[0], arrs[2], arrs[3]], 1.5, dtype)
    assert torch.equal(mine[1200:3600], dev[1200:3600]) and torch.equal(mine[6600:9000:2], dev[6600:9000:2])


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_extremes(kx, torch_cuda, dtype):
    """f32 squares beyond the type's range, tiny values, and norms that are
    not finite, which scale nothing."""
    torch = torch_cuda
    tt = torch.float32 if dtype == np.float32 else torch.float64
    big = 1e38 if dtype == np.float32 else 1e150
    x = torch.full((5,), big, dtype=tt, device="cuda")
    got, outs = kx.clip_grad_norm([x], 1.0)
    check_clip(got, outs, [x.cpu().numpy()], 1.0, dtype)
    tiny = torch.full((9,), 1e-30, dtype=tt, device="cuda")
    check_norm(kx.grad_norm([tiny]), [tiny.cpu().numpy()], dtype)
    assert kx.grad_norm([torch.zeros(8, dtype=tt, device="cuda")]).item() == 0
    got, outs = kx.clip_grad_norm([torch.zeros(8, dtype=tt, device="cuda")], 1.0)
    assert got.item() == 0 and (outs[0] == 0).all()
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = torch.arange(6000, dtype=tt, device="cuda")
        y[4321] = bad
        got, outs = kx.clip_grad_norm([x, y], 1.0)
        assert not np.isfinite(got.item()) and np.isnan(got.item()) == np.isnan(bad)
        assert torch.equal(outs[0], x) and np.array_equal(outs[1].cpu().numpy(), y.cpu().numpy(), equal_nan=True)


def test_more_elements_than_32_bits_count(kx, torch_cuda):
    """2^32 + 5 elements: the norm of equal values, and both ends scaled."""
    torch = torch_cuda
    n = 2 ** 32 + 5
    x = torch.full((n,), 0.5, device="cuda")
    norm = kx.clip_grad_norm_into([x, x[:0]], 1.0, [x, x[:0]])
    want = LD(0.5) * np.sqrt(LD(n))
    assert abs(LD(norm.item()) - want) <= want * (2.0 ** -24 + n * 2.0 ** -53)
    by = float(LD(0.5) / want)
    for part in (x[:4], x[-4:], x[2 ** 31 - 2:2 ** 31 + 2], x[2 ** 32 - 2:2 ** 32 + 2]):
        assert (np.abs(part.cpu().numpy() - by) <= by * (3 * 2.0 ** -24 + n * 2.0 ** -53)).all()
    assert float(x.min()) == float(x.max())


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("megabytes", [45, 47, 100, 191, 193])
def test_lists_of_the_size_of_the_cache(kx, torch_cuda, dtype, megabytes):
    """Lists that the second-level cache holds partly, with unaligned and tiny
    members: copies apart and in place have the same bits, and every element is
    its gradient's, scaled."""
    torch = torch_cuda
    ty = torch.float32 if dtype == np.float32 else torch.float64
    size = 4 if dtype == np.float32 else 8
    gen = torch.Generator(device="cuda").manual_seed(megabytes)
    each = megabytes * 2 ** 20 // size // 4
    base = [torch.randn(each + 3, generator=gen, device="cuda", dtype=ty) for _ in range(4)]
    grads = [base[0][:each], base[1][1:each], base[2][3:], base[3][:each - 2], base[0][each:], base[3][each:each + 1]]
    outs = [torch.full((g.numel() + 9,), 7.0, device="cuda", dtype=ty) for g in grads]
    views = [o[4:4 + g.numel()] if i != 2 else o[:g.numel()] for i, (o, g) in enumerate(zip(outs, grads))]
    norm = kx.clip_grad_norm_into(grads, 2.5, views)
    n = sum(g.numel() for g in grads)
    want = float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt())
    # n squares added up here and there, in any order: each sum is off by n 2^-53 of itself
    assert abs(float(norm) - want) <= want * (U[dtype] + 2 * n * 2.0 ** -53)
    by = 2.5 / want
    for i, (g, v, o) in enumerate(zip(grads, views, outs)):
        error = (v.double() - g.double() * by).abs()
        assert bool((error <= g.double().abs() * by * (3 * U[dtype] + 2 * n * 2.0 ** -53)).all())
        rest = [o[:4], o[4 + g.numel():]] if i != 2 else [o[g.numel():]]
        assert all(bool((r == 7.0).all()) for r in rest)
    assert torch.equal(kx.clip_grad_norm_into(grads, 2.5, grads), norm)
    assert all(torch.equal(g, v) for g, v in zip(grads, views))


@pytest.mark.parametrize("count,rows", [(6, 1100), (45, 1100), (300, 3)])
def test_many_tensors_with_gaps(kx, torch_cuda, count, rows):
    """Lists whose partial sums are folded before the scaling, and on the way."""
    torch = torch_cuda
    shapes = [(rows, 1000)] * count
    arrs, dev = make(torch, 23, shapes, np.float32)
    views, hosts = [d[:, :999] for d in dev], [a[:, :999] for a in arrs]
    check_norm(kx.grad_norm(views), hosts, np.float32)
    before = [d[:, 999].clone() for d in dev]
    norm = kx.clip_grad_norm_into(views, 0.25, views)
    check_clip(norm, views, hosts, 0.25, np.float32)
    assert all(torch.equal(d[:, 999], b) for d, b in zip(dev, before))


def test_gaps_among_more_than_2_31_elements(kx, torch_cuda):
    """2^31 elements of a gapped tensor, and as many places of one element."""
    torch = torch_cuda
    buf = torch.full((65_536, 32_769), 0.25, device="cuda")
    view = buf[:, :32_768]
    n = view.numel()
    want = LD(0.25) * np.sqrt(LD(n))
    wide = torch.full((1, 1), 0.25, device="cuda").expand(65_536, 32_768)
    for got in (kx.grad_norm([wide]), kx.clip_grad_norm_into([view], 2.0, [view])):
        assert abs(LD(got.item()) - want) <= want * (2.0 ** -24 + n * 2.0 ** -53)
    by = float(LD(2.0) / want) * 0.25
    tol = by * (3 * 2.0 ** -24 + n * 2.0 ** -53)
    assert abs(float(view.min()) - by) <= tol and abs(float(view.max()) - by) <= tol
    assert bool((buf[:, 32_768] == 0.25).all())


def test_streams_graphs_and_repetition(kx, torch_cuda):
    """The same bits again, on another stream, and from two captured graphs
    that run side by side on new values."""
    torch = torch_cuda
    arrs, dev = make(torch, 17, [(300, 1000), (77,), (1 << 19,), (5, 5)], np.float32)
    other = [d * 3 + 1 for d in dev]
    want = [[kx.clip_grad_norm(d, 1.0)[0].cpu(), *[o.cpu() for o in kx.clip_grad_norm(d, 1.0)[1]]] for d in (dev, other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kx.clip_grad_norm(dev, 1.0)
    side.synchronize()
    assert torch.equal(got[0].cpu(), want[0][0]) and all(torch.equal(o.cpu(), w) for o, w in zip(got[1], want[0][1:]))
    bufs = [[d.clone() for d in dev] for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kx.clip_grad_norm(b, 1.0))
        graphs.append(g)
    for which in ((0, 1), (1, 0)):
        for b, k in zip(bufs, which):
            for dst, src in zip(b, (dev, other)[k]):
                dst.copy_(src)
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for o, k in zip(outs, which):
            assert torch.equal(o[0].cpu(), want[k][0])
            assert all(torch.equal(a.cpu(), w) for a, w in zip(o[1], want[k][1:]))


def test_refusals_on_the_device(kx, torch_cuda):
    torch = torch_cuda
    x, y = torch.zeros(8, device="cuda"), torch.zeros(2, 4, device="cuda")
    with pytest.raises(kx.InvalidParameter):
        kx.grad_norm([x, y.double()])
    with pytest.raises(kx.NoDevice):
        kx.grad_norm([x, y.cpu()])
    with pytest.raises(kx.Unsupported):
        kx.grad_norm([x.half()])
    with pytest.raises(kx.InvalidParameter):
        kx.clip_grad_norm([x], 0.0)
    with pytest.raises(kx.InvalidParameter):
        kx.clip_grad_norm_into([x, y], 1.0, [x])
    with pytest.raises(kx.LayoutError):
        kx.clip_grad_norm_into([x], 1.0, [y])
    with pytest.raises(kx.OverlappingOutput):
        kx.clip_grad_norm_into([x, x], 1.0, [x, x])
    with pytest.raises(kx.LayoutError):
        kx.grad_norm_into([x], torch.zeros(2, device="cuda"))
    with pytest.raises(kx.InvalidParameter):
        kx.grad_norm_into([x], torch.zeros((), dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_a_training_step_in_double_precision(kx, torch_cuda, temperature):
    """Logits of two layers' products, their loss (log probabilities with an
    entropy bonus over the positions that have a token), its gradient through
    both products, and the clipped update, against the same step written out in
    torch with its own differentiation.  Both run in f64; the sums are at most
    4000 terms long, so each result is off by less than 1e4 2^-53 of the norm
    of what enters it, well inside 1e-11 of the largest value."""
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=torch.float64)  # noqa: E731
    batch, length, width, hidden, vocab = 3, 5, 24, 40, 501
    x, w1, w2 = new(batch, length, width), new(width, hidden) / 5, new(hidden, vocab) / 6
    labels = torch.randint(0, vocab, (batch, length), generator=gen, device="cuda")
    labels[0, 3:] = -1
    n = (labels[:, 1:] >= 0).sum().double()

    a = kx.matmul(x, w1)
    z = kx.matmul(a, w2)
    shifted = z[:, :-1]
    out = kx.token_log_probs(shifted, labels[:, 1:], temperature=temperature, top=3, entropy=True)
    g_lp = (-1.0 / n).expand(batch, length - 1)
    g_h = torch.where(labels[:, 1:] >= 0, -0.01 / n, 0.0)
    gz = torch.zeros_like(z)
    gz[:, :-1] = kx.token_log_probs_backward(shifted, labels[:, 1:], lse=out.lse, entropy=out.entropy,
                                             grad_log_probs=g_lp, grad_entropy=g_h, temperature=temperature)
    ga, gw2 = kx.matmul_backward(a, w2, gz)
    gx, gw1 = kx.matmul_backward(x, w1, ga)
    norm, clipped = kx.clip_grad_norm([gw1, gw2], 0.1)

    px, pw1, pw2 = (t.clone().requires_grad_() for t in (x, w1, w2))
    lq = torch.log_softmax(((px @ pw1) @ pw2)[:, :-1] / temperature, -1)
    has = labels[:, 1:] >= 0
    lp = torch.where(has, lq.gather(-1, labels[:, 1:].clamp_min(0)[..., None])[..., 0], 0.0)
    ent = -(lq.exp() * lq).sum(-1)
    loss = -lp.sum() / n - 0.01 * torch.where(has, ent, 0.0).sum() / n
    loss.backward()
    want_norm = torch.sqrt((pw1.grad ** 2).sum() + (pw2.grad ** 2).sum())
    scale = torch.clamp(0.1 / want_norm, max=1.0)
    got = -out.log_probs.sum() / n + (g_h * out.entropy).sum()
    pairs = [(got, loss.detach()), (out.log_probs, lp.detach()), (out.entropy, ent.detach()), (gx, px.grad),
             (gw1, pw1.grad), (gw2, pw2.grad), (norm, want_norm), (clipped[0], pw1.grad * scale),
             (clipped[1], pw2.grad * scale)]
    for i, (g, w) in enumerate(pairs):
        assert float((g - w).abs().max()) <= 1e-11 * float(w.abs().max()), i
    assert torch.equal(out.top_tokens[..., 0], lq.detach().argmax(-1))


def test_a_serving_step(kx, torch_cuda):
    """Single tokens of a batch: the product's logits, alternatives, a token
    chosen among them and its log probability, which is the alternative's."""
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(4)
    h = torch.randn(6, 128, generator=gen, device="cuda")
    w = torch.randn(128, 5000, generator=gen, device="cuda") / 8
    z = kx.matmul(h, w)
    out = kx.token_log_probs(z, top=8, temperature=0.8)
    pick = torch.tensor([[0], [3], [7], [1], [0], [5]], device="cuda")
    tokens = out.top_tokens.gather(1, pick)[:, 0]
    lp = kx.token_log_probs(z, tokens, temperature=0.8).log_probs
    assert torch.equal(lp, out.top_log_probs.gather(1, pick)[:, 0])
    assert torch.equal(out.top_tokens[:, 0], z.argmax(-1))


def test_calls_of_several_threads(kx, torch_cuda):
    """Threads that share the default handle, each on a stream of its own: what
    each one enqueues runs in its own order."""
    import threading

    torch = torch_cuda
    x0, tokens = torch.randn(40, 3001, device="cuda"), torch.arange(40, device="cuda")
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(60):
                x = x0 * (1 + 0.01 * k) + 0.001 * i     # written on this stream right before it is read
                out = kx.token_log_probs(x, tokens, top=3)
                grad = kx.token_log_probs_backward(x, tokens, lse=out.lse, grad_log_probs=out.lse)
                norm, (clipped,) = kx.clip_grad_norm([grad], 0.5)
                lse = torch.logsumexp(x, -1)
                # sums of 3001 terms in f32: 3001 2^-24 at the very most, of about 8
                if not bool(((out.lse - lse).abs() <= 4e-4 * lse.abs()).all()) or not torch.equal(
                        out.top_tokens[:, 0], x.argmax(-1)):
                    wrong.append((k, i))
                if abs(float(torch.linalg.vector_norm(clipped)) - 0.5) > 1e-3 or float(norm) <= 0.5:
                    wrong.append((k, i, "norm"))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_the_binding_and_the_general_path_agree(kx, torch_cuda, monkeypatch):
    """Every call on torch tensors through csrc/kx_torch.cpp and without it: the
    same bits, the same refusals, and nothing kept after the call."""
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(4, 7, 333, generator=gen, device="cuda").transpose(0, 1)
    t = torch.randint(-1, 333, (7, 4), generator=gen, device="cuda")
    g = torch.randn(4, 7, generator=gen, device="cuda").t()
    grads = [torch.randn(33, 20, generator=gen, device="cuda").t(), torch.randn(0, 4, device="cuda"),
             torch.randn(10_001, generator=gen, device="cuda")[1:], torch.randn(6, 8, device="cuda")[:, ::3]]

    def calls():
        out = kx.token_log_probs(x, t, temperature=0.7, top=5, entropy=True)
        bare = kx.token_log_probs(x)
        back = kx.token_log_probs_backward(x, t, lse=out.lse, entropy=out.entropy, grad_log_probs=g, grad_entropy=g,
                                           grad_lse=g, temperature=0.7)
        into = torch.empty_like(back)
        kx.token_log_probs_backward_into(x, t, into, lse=out.lse, grad_log_probs=g, temperature=0.7)
        norm, clipped = kx.clip_grad_norm(grads, 0.5)
        mine = [q.clone() for q in grads]
        again = torch.zeros(1, device="cuda")
        kx.clip_grad_norm_into(mine, 0.5, mine, again)
        assert bare.log_probs is None and bare.entropy is None and bare.top_tokens is None
        return [*out, bare.lse, back, into, norm, kx.grad_norm(grads), *clipped, *mine, again]

    def refusals():
        got = []
        for call in (lambda: kx.token_log_probs(x, t[:3]), lambda: kx.token_log_probs(x, t, temperature=-1.0),
                     lambda: kx.token_log_probs(x, t.int()), lambda: kx.token_log_probs(x.half(), t),
                     lambda: kx.token_log_probs_backward(x, t, lse=g.double(), grad_log_probs=g),
                     lambda: kx.token_log_probs_backward_into(x, t, x, lse=g, grad_log_probs=g),
                     lambda: kx.grad_norm([x, g.double()]), lambda: kx.grad_norm([x, t]),
                     lambda: kx.clip_grad_norm_into([x, g], 1.0, [x]), lambda: kx.clip_grad_norm_into([x], 1.0, [g]),
                     lambda: kx.clip_grad_norm([x], float("nan")), lambda: kx.clip_grad_norm_into([g, g], 1.0, [g, g]),
                     lambda: kx.grad_norm_into([x], torch.zeros(2, device="cuda"))):
            with pytest.raises(kx.OpsError) as e:
                call()
            got.append((type(e.value), e.value.fields))
        return got

    native, refused = calls(), refusals()
    gc.collect()        # what the refusals' tracebacks hold
    held = torch.cuda.memory_allocated()
    for _ in range(50):
        calls()
        refusals()
    gc.collect()
    assert torch.cuda.memory_allocated() == held

    class Nothing:
        token_log_probs = token_log_probs_backward = grad_norm = staticmethod(lambda *a: None)

    monkeypatch.setattr(kx, "_native", lambda: Nothing)
    general = calls()
    assert all(torch.equal(a, b) and a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()
               for a, b in zip(native, general))
    assert refusals() == refused
