"""Log probabilities of given tokens, entropies, alternatives and their
gradient (kx_token_log_probs_*, kx_token_log_probs_backward_*) against the
formulas in 80-bit arithmetic, and the gradient against differences.

Bounds, with u half a step of the type (2^-24, 2^-53) and R the largest
|z - max z| with a probability that counts.  A term exp((x - m)/T) is off by
at most 3u R (the difference, the scale and the argument's rounding) + 8u (the
exponential, at most 8 half steps); a chain of additions adds u for each link,
and no more than V/32 of them follow one another, since 32 threads or more
share a row, with 16 to join them.  So S is off by ds = u (3R + 8 + V/32 + 16)
relative to itself, log S by ds, and what follows rounds once or twice more.
R is capped at 40 (f32) or 80 (f64): terms further down weigh e^-40 and less.
"""
import ctypes as C

import numpy as np
import pytest

from kernix_b200 import rng

pytestmark = pytest.mark.gpu
U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
CAP = {np.float32: 40.0, np.float64: 80.0}
LD = np.longdouble


def truth(x, tokens, t, top):
    """The five outputs of [rows, V] logits by the definitions."""
    rows, v = x.shape
    z = x.astype(LD) / LD(t)
    out = {k: np.zeros(rows, LD) for k in ("log_probs", "lse", "entropy", "range", "max", "log_sum")}
    out["top_log_probs"], out["top_tokens"] = np.full((rows, top), -np.inf, LD), np.full((rows, top), -1, np.int64)
    for r in range(rows):
        if np.isnan(x[r]).any() or np.isposinf(x[r]).any():
            for k in ("log_probs", "lse", "entropy"):
                out[k][r] = np.nan
            out["top_log_probs"][r] = np.nan
            if tokens is not None and tokens[r] < 0:
                out["log_probs"][r] = 0
            continue
        live = np.nonzero(~np.isneginf(x[r]))[0]
        if len(live) == 0:
            out["lse"][r] = -np.inf
            out["log_probs"][r] = -np.inf
        else:
            zl = z[r, live]
            m = zl.max()
            d = zl - m
            s = np.exp(d).sum()
            logs = np.log(s)
            out["lse"][r], out["max"][r], out["log_sum"][r] = m + logs, m, logs
            out["entropy"][r] = logs - (np.exp(d) * d).sum() / s
            out["range"][r] = -d.min()
            order = live[np.argsort(-x[r, live], kind="stable")][:top]
            out["top_tokens"][r, :len(order)] = order
            out["top_log_probs"][r, :len(order)] = z[r, order] - m - logs
            if tokens is not None:
                out["log_probs"][r] = z[r, tokens[r] if 0 <= tokens[r] < v else 0] - m - logs
        if tokens is not None:
            if tokens[r] < 0:
                out["log_probs"][r] = 0
            elif tokens[r] >= v:
                out["log_probs"][r] = np.nan
    return out


def near(got, want, tol, what):
    got, want = np.asarray(got).astype(LD), np.asarray(want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True), what
    err = np.abs(got[fine] - want[fine])
    tol = np.broadcast_to(tol, want.shape)[fine]
    assert (err <= tol).all(), (what, float(err.max()), float((err / tol).max()))


def check_forward(res, x, tokens, t, dtype, top, entropy=True):
    """res: numpy arrays of [rows, ..]; x [rows, V]."""
    want = truth(x, tokens, t, top)
    # beyond the type's range (the lowest logit beside the largest) a value rounds to infinity
    for k in ("log_probs", "lse", "top_log_probs"):
        far = np.abs(want[k]) > LD(np.finfo(dtype).max) * (1 + U[dtype])
        want[k] = np.where(far, np.copysign(np.inf, want[k]), want[k])
    u, v = U[dtype], x.shape[1]
    ds = u * (3 * np.minimum(want["range"], CAP[dtype]) + 24 + v / 32)
    tiny = np.finfo(dtype).smallest_normal
    size = lambda a: np.where(np.isfinite(a), np.abs(a), 0)  # noqa: E731
    near(res.lse, want["lse"], ds + 2 * u * size(want["lse"]) + tiny, "lse")
    if tokens is not None:
        near(res.log_probs, want["log_probs"], ds + 2 * u * size(want["log_probs"]) + tiny, "log_probs")
    if entropy:
        # E/S of H = log S - E/S: E's terms are off by 2u more than S's
        h = size(want["entropy"])
        near(res.entropy, want["entropy"], ds + h * (2 * ds + 8 * u) + tiny, "entropy")
    if top:
        assert np.array_equal(res.top_tokens, want["top_tokens"])
        near(res.top_log_probs, want["top_log_probs"], ds[:, None] + 2 * u * size(want["top_log_probs"]) + tiny, "top")
    return want


def run(kx, torch, x, tokens, t, top, entropy=True, lead=None):
    """On [rows, V] numpy logits laid out as they are; numpy results."""
    dx = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    dt = None if tokens is None else torch.from_numpy(np.ascontiguousarray(tokens)).cuda()
    if lead is not None:
        dx = dx.reshape(*lead, x.shape[1])
        dt = None if dt is None else dt.reshape(lead)
    return numpy(kx, kx.token_log_probs(dx, dt, temperature=t, top=top, entropy=entropy), x.shape[0])


def numpy(kx, res, rows):
    flat = lambda a, n: None if a is None else a.cpu().numpy().reshape((rows,) + ((a.shape[-1],) if n else ()))  # noqa: E731
    return kx.TokenLogProbs(flat(res.log_probs, 0), flat(res.lse, 0), flat(res.entropy, 0),
                            flat(res.top_log_probs, 1), flat(res.top_tokens, 1))


def logits(seed, rows, v, dtype, std=2.5):
    x = rng.normal(seed, max(1, rows * v), std)[:rows * v].reshape(rows, v).astype(dtype)
    tokens = (rng.uniform(seed + 1, max(1, rows), 0.0, 1.0)[:rows] * v).astype(np.int64)
    return x, np.minimum(tokens, v - 1)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,v,top,t", [
    (1, 1, 1, 1.0), (3, 2, 5, 1.0), (2, 31, 32, 0.7), (5, 32, 32, 1.0), (4, 33, 32, 2.0), (3, 127, 8, 1.0),
    (1, 255, 1, 1.0), (9, 257, 20, 0.5), (7, 1000, 3, 1.0), (2, 1023, 32, 1.0), (300, 1025, 4, 1.3),
    (2, 4099, 32, 1.0), (1, 8191, 20, 1.0), (3, 16385, 20, 0.9), (20, 32000, 5, 1.0), (1, 65537, 32, 1.0),
    (2, 131072, 20, 0.7), (160, 5003, 1, 1.0), (600, 2049, 8, 1.0)])
def test_forward_matches_the_formulas(kx, torch_cuda, dtype, rows, v, top, t):
    x, tokens = logits(11 + rows + v, rows, v, dtype)
    check_forward(run(kx, torch_cuda, x, tokens, t, top), x, tokens, t, dtype, top)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_each_output_alone(kx, torch_cuda, dtype):
    """What is not asked for is not computed, and the rest keeps its bits."""
    torch = torch_cuda
    x, tokens = logits(3, 5, 1501, dtype)
    full = run(kx, torch, x, tokens, 1.0, 6)
    dx, dt = torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda()
    for names in (("log_probs",), ("lse",), ("entropy",), ("top_log_probs", "top_tokens"), ("lse", "entropy")):
        outs = {n: torch.from_numpy(np.zeros_like(getattr(full, n))).cuda() for n in names}
        out = kx.TokenLogProbs(**outs)
        kx.token_log_probs_into(dx, dt if "log_probs" in names else None, out)
        for n in names:
            assert np.array_equal(outs[n].cpu().numpy(), getattr(full, n)), n
    assert run(kx, torch, x, None, 1.0, 0, False).log_probs is None


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("v", [1, 5, 40, 1003, 20001])
def test_masks_ties_and_special_values(kx, torch_cuda, dtype, v):
    """Row by row: nothing masked; most masked; all but one; all; all at the
    type's lowest value; lowest beside ordinary and beside the largest value;
    equal values; few distinct values; rising; falling; both zeros; NaN; +inf;
    -inf beside NaN; a far offset."""
    low, high = np.finfo(dtype).min, np.finfo(dtype).max
    base, _ = logits(5, 16, v, dtype)
    x = base.copy()
    j = np.arange(v)
    x[1][j % 7 != 3] = -np.inf
    x[2] = -np.inf
    x[2, v // 2] = 1.5
    x[3] = -np.inf
    x[4] = low
    x[5][j % 2 == 0] = low
    x[6] = low
    x[6, v - 1] = high
    x[7] = 0.25
    x[8] = np.floor(x[8])
    x[9] = (j / 64).astype(dtype)
    x[10] = (-j / 64).astype(dtype)
    x[11] = np.where(j % 2 == 0, -0.0, 0.0)
    x[12, v // 3] = np.nan
    x[13, v - 1] = np.inf
    x[14] = -np.inf
    x[14, 0] = np.nan
    x[15] += 1000
    tokens = np.array([v // 2] * 16, np.int64)
    for top in (0, 1, 32):
        check_forward(run(kx, torch_cuda, x, tokens, 1.0, top), x, tokens, 1.0, dtype, top)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,v,kernel", [
    (5, 301, "log_probs_warp"), (2100, 77, "log_probs_warp"), (760, 1501, "log_probs_warp"),
    (2050, 2048, "log_probs_warp"), (760, 5001, "log_probs_block4"),
    (760, 16_401, "log_probs_block4_wide"), (150, 9001, "log_probs_block8"),
    (40, 1025, "log_probs_block8"), (200, 40001, "log_probs_cluster"), (3, 300_007, "log_probs_cluster"), (1, 1_300_001, "log_probs_cluster")])
def test_each_kernel_and_strides(kx, torch_cuda, dtype, rows, v, kernel):
    """Rows of every kernel, as rows and with the vocabulary's stride above one;
    the longest make a part of a thread's elements several rounds."""
    torch = torch_cuda
    if dtype == np.float64 and kernel == "log_probs_block4_wide":
        kernel = "log_probs_block4"
    x, tokens = logits(13 + v, rows, v, dtype)
    some = np.unique(np.linspace(0, rows - 1, 12).astype(int))
    dx, dt = torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda()
    for view in (dx, dx.t().contiguous().t()):
        res = kx.token_log_probs(view, dt, top=32, entropy=True)
        assert kx.handle(0).last_kernel == (kernel if view is dx or kernel != "log_probs_block4_wide" else
                                            "log_probs_block4")
        res = numpy(kx, res, rows)
        check_forward(kx.TokenLogProbs(*[a[some] for a in res]), x[some], tokens[some], 1.0, dtype, 32)
        if view is dx:
            first = res
    # a stride changes the order of the sums alone, never the alternatives
    assert np.array_equal(first.top_tokens, res.top_tokens)


@pytest.mark.parametrize("dtype,v,kernel", [
    (np.float64, 24_575, "log_probs_block8"), (np.float64, 24_577, "log_probs_cluster"),
    (np.float32, 32_767, "log_probs_block8"), (np.float32, 32_769, "log_probs_cluster")])
def test_rows_in_two_parts(kx, torch_cuda, dtype, v, kernel):
    """From which length on rows that the SMs have places for twice are cut."""
    rows = torch_cuda.cuda.get_device_properties(0).multi_processor_count + 2
    x, tokens = logits(v, rows, v, dtype)
    res = run(kx, torch_cuda, x, tokens, 0.9, 6)
    assert kx.handle(0).last_kernel == kernel
    some = np.array([0, 1, 73, rows - 1])
    check_forward(kx.TokenLogProbs(*[a[some] for a in res]), x[some], tokens[some], 0.9, dtype, 6)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,v", [(3, 70_001), (770, 4500), (770, 17_003), (2080, 2000), (64, 1500)])
def test_ties_and_masks_in_each_kernel(kx, torch_cuda, dtype, rows, v):
    """Rows of equal values, of few values, with one or no token left, most of
    them masked, in turn."""
    x, tokens = logits(17 + v, rows, v, dtype)
    x[0::6] = 2.0
    x[1::6] = np.floor(x[1::6])
    x[2::6, 1:] = -np.inf
    x[3::6][:, np.arange(v) % 50 != 7] = -np.inf
    x[4::6] = -np.inf
    some = np.unique(np.r_[0:min(rows, 12), rows - 6:rows] % rows)
    res = run(kx, torch_cuda, x, tokens, 0.8, 20)
    check_forward(kx.TokenLogProbs(*[a[some] for a in res]), x[some], tokens[some], 0.8, dtype, 20)


def test_tokens_outside_the_vocabulary(kx, torch_cuda):
    x, _ = logits(8, 6, 50, np.float32)
    tokens = np.array([0, 49, -1, -100, 50, 2 ** 40], np.int64)
    res = run(kx, torch_cuda, x, tokens, 1.0, 2)
    check_forward(res, x, tokens, 1.0, np.float32, 2)
    assert res.log_probs[2] == 0 and res.log_probs[3] == 0 and np.isnan(res.log_probs[4:]).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("v", [37, 1100, 9001])
def test_layouts(kx, torch_cuda, dtype, v):
    """Rows of a wider buffer at every alignment, a vocabulary that is not the
    innermost axis, every second token, reversed axes, one row read by many,
    and labels shifted against their logits."""
    torch = torch_cuda
    tt = torch.float32 if dtype == np.float32 else torch.float64
    rows = 6
    x, tokens = logits(21, rows, v, dtype)
    dx, dt = torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda()

    def check(view, xs, toks, dtok):
        res = numpy(kx, kx.token_log_probs(view, dtok, top=7, entropy=True), xs.shape[0])
        check_forward(res, xs, toks, 1.0, dtype, 7)

    for off in range(5):
        wide = torch.full((rows, v + 9), float("nan"), dtype=tt, device="cuda")
        wide[:, off:off + v] = dx
        check(wide[:, off:off + v], x, tokens, dt)
    check(dx.t().contiguous().t(), x, tokens, dt)
    gaps = torch.full((rows, v, 2), float("nan"), dtype=tt, device="cuda")
    gaps[..., 1] = dx
    check(gaps[..., 1], x, tokens, dt)
    back = kx.TensorView(dx.reshape(-1), (rows, v), (-v, -1), rows * v - 1)
    check(back, x[::-1, ::-1], tokens, dt)
    check(dx[:1].expand(4, v), np.repeat(x[:1], 4, 0), tokens[:4], dt[:4])
    # [2, 3 positions, V]: position i is scored on the token at i + 1
    labels = torch.from_numpy(np.array([[9, 1, 5], [9, 0, 7]], np.int64)).cuda()
    both = dx.reshape(2, 3, v)
    check(both[:, :-1], x.reshape(2, 3, v)[:, :-1].reshape(4, v), np.array([1, 5, 0, 7]), labels[:, 1:])
    # a [3, 2] arrangement of rows and tokens that no single stride walks
    check(both.transpose(0, 1), x.reshape(2, 3, v).transpose(1, 0, 2).reshape(6, v),
          tokens.reshape(2, 3).T.reshape(-1), dt.reshape(2, 3).t())


def test_most_axes_and_another_handle(kx, torch_cuda):
    """Eight axes of which few nest, through a handle of the caller's own."""
    torch = torch_cuda
    x, tokens = logits(33, 24, 130, np.float32)
    shape = (2, 1, 3, 1, 2, 1, 2, 130)
    dx = torch.from_numpy(x).cuda().reshape(shape)
    dt = torch.from_numpy(tokens).cuda().reshape(shape[:-1])
    order = (2, 1, 6, 3, 0, 5, 4)
    rows = np.arange(24).reshape(shape[:-1]).transpose(order).reshape(-1)
    own = kx.Handle(0)
    with kx.using(own):
        res = kx.token_log_probs(dx.permute(*order, 7), dt.permute(order), top=3, entropy=True)
    assert own.launches == 1 and res.top_tokens.shape == tuple(shape[i] for i in order) + (3,)
    check_forward(numpy(kx, res, 24), x[rows], tokens[rows], 1.0, np.float32, 3)
    g = torch.ones(shape[:-1], device="cuda").permute(order)
    got = kx.token_log_probs_backward(dx.permute(*order, 7), dt.permute(order), lse=res.lse, grad_log_probs=g)
    check_backward(got.cpu().numpy().reshape(24, 130), x[rows], tokens[rows], 1.0, np.float32, np.ones(24, np.float32))
    own.synchronize()
    own.close()


def test_shapes_without_rows_or_vocabulary(kx, torch_cuda):
    torch = torch_cuda
    res = kx.token_log_probs(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    assert res.log_probs.shape == (0,) and res.top_tokens.shape == (0, 2)
    res = kx.token_log_probs(torch.zeros(3, 0, device="cuda"), torch.tensor([-1, 0, 4], device="cuda"), top=2,
                             entropy=True)
    assert res.lse.tolist() == [-np.inf] * 3 and res.entropy.tolist() == [0] * 3
    assert res.log_probs[0] == 0 and res.log_probs[1:].isnan().all()
    assert res.top_tokens.tolist() == [[-1, -1]] * 3 and res.top_log_probs.tolist() == [[-np.inf] * 2] * 3
    one = kx.token_log_probs(torch.tensor([1.0, 2.0], device="cuda"), torch.tensor(1, device="cuda"), top=1)
    assert one.log_probs.shape == () and one.top_tokens.tolist() == [1]
    g = kx.token_log_probs_backward(torch.zeros(3, 0, device="cuda"), lse=res.lse, grad_lse=res.entropy)
    assert g.shape == (3, 0)


def test_rows_far_apart(kx, torch_cuda):
    """Offsets beyond 32 bits: three rows 2^31 + 3 elements apart."""
    torch = torch_cuda
    v, apart = 777, 2 ** 31 + 3
    x, tokens = logits(31, 3, v, np.float32)
    buf = torch.empty(2 * apart + v, device="cuda")
    view = buf.as_strided((3, v), (apart, 1))
    view.copy_(torch.from_numpy(x))
    dt = torch.from_numpy(tokens).cuda()
    res = kx.token_log_probs(view, dt, top=5, entropy=True)
    check_forward(numpy(kx, res, 3), x, tokens, 1.0, np.float32, 5)
    g = torch.from_numpy(np.array([1.0, -2.0, 0.5], np.float32)).cuda()
    got = kx.token_log_probs_backward(view, dt, lse=res.lse, grad_log_probs=g)
    check_backward(got.cpu().numpy(), x, tokens, 1.0, np.float32, g.cpu().numpy())


def test_streams_graphs_and_repetition(kx, torch_cuda):
    """The same bits on another stream, from a captured graph with new logits
    in its buffer, and from two graphs that run side by side."""
    torch = torch_cuda
    data = [logits(50 + i, 3, 30011, np.float32) for i in range(2)]
    dev = [(torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()) for x, t in data]

    def step(x, t):
        out = kx.token_log_probs(x, t, top=20, entropy=True)
        return (*out, kx.token_log_probs_backward(x, t, lse=out.lse, entropy=out.entropy, grad_log_probs=out.lse,
                                                  grad_entropy=out.entropy))

    want = [[o.cpu() for o in step(*d)] for d in dev]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(*dev[0])
    side.synchronize()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(again, want[0]))
    bufs = [tuple(t.clone() for t in dev[0]) for _ in range(2)]
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*b))
        graphs.append(g)
    for which in ((0, 1), (1, 0), (1, 1)):
        for b, k in zip(bufs, which):
            for dst, src in zip(b, dev[k]):
                dst.copy_(src)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, k in zip(outs, which):
            assert all(torch.equal(a.cpu(), b) for a, b in zip(o, want[k]))


# --- the gradient -----------------------------------------------------------
def check_backward(got, x, tokens, t, dtype, g=None, gh=None, gl=None):
    """A probability from logits and a rounded lse: its exponent is off by
    u (4 |log p| + |lse| + |z| + 8) at most, and the exponential adds what the
    8 stands for; the entropy that comes in is rounded too."""
    rows, v = x.shape
    u = U[dtype]
    f = truth(x, np.zeros(rows, np.int64), t, 0)
    zero = np.zeros(rows)
    g_, gh_, gl_ = (np.asarray(zero if a is None else a).astype(LD) for a in (g, gh, gl))
    g_ = g_ if tokens is None else np.where(tokens < 0, 0, g_)
    for r in range(rows):
        if np.isnan(f["lse"][r]) or (g is not None and tokens[r] >= v):
            assert np.isnan(got[r][~np.isneginf(x[r])]).all()
            continue
        live = ~np.isneginf(x[r])
        assert (got[r][~live] == 0).all()
        if not live.any():
            continue
        z = x[r].astype(LD)[live] / LD(t)
        lq = z - f["max"][r] - f["log_sum"][r]
        p = np.exp(lq)
        h = f["entropy"][r]
        want = p * (gl_[r] - g_[r] - gh_[r] * (lq + h))
        size = abs(gl_[r]) + abs(g_[r]) + abs(gh_[r]) * (np.abs(lq) + abs(h))
        off = u * (4 * np.abs(lq) + abs(f["lse"][r]) + np.abs(z) + 8)
        if abs(f["lse"][r]) > 250:   # the row's own sums are taken anew
            off = u * (4 * np.abs(lq) + 3 * min(f["range"][r], CAP[dtype]) + 32 + v / 32)
        tol = p * size * (off + 8 * u) + p * abs(gh_[r]) * (off + u * abs(h))
        if tokens is not None and tokens[r] >= 0:
            at = np.zeros(v, bool)
            at[tokens[r]] = True
            want = want + np.where(at[live], g_[r], 0)
            tol = tol + np.where(at[live], 4 * u * abs(g_[r]), 0)
        # results below the smallest normal number may come out as 0
        near(got[r][live], want / LD(t), tol / t + np.finfo(dtype).smallest_normal * (1 + size / t), ("grad", r))


def grads_in(seed, rows, dtype):
    return [rng.normal(seed + i, rows, 1.0).astype(dtype) for i in range(3)]


def backward(kx, torch, x, tokens, t, g=None, gh=None, gl=None, res=None):
    dx, dt = torch.from_numpy(np.ascontiguousarray(x)).cuda(), torch.from_numpy(tokens).cuda()
    res = kx.token_log_probs(dx, dt, temperature=t, entropy=True) if res is None else res
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    return kx.token_log_probs_backward(dx, dt, lse=res.lse, entropy=res.entropy, grad_log_probs=dev(g),
                                       grad_entropy=dev(gh), grad_lse=dev(gl), temperature=t).cpu().numpy()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("rows,v,t", [(1, 1, 1.0), (3, 2, 1.0), (4, 31, 0.6), (2, 130, 1.0), (5, 1000, 1.7),
                                      (33, 1027, 1.0), (2, 4099, 1.0), (1, 32000, 0.8), (3, 50021, 1.0),
                                      (1, 300_007, 1.0)])
def test_gradient_matches_the_formula(kx, torch_cuda, dtype, rows, v, t):
    x, tokens = logits(61 + rows + v, rows, v, dtype)
    g, gh, gl = grads_in(9, rows, dtype)
    for a in ((g, None, None), (None, gh, None), (None, None, gl), (g, gh, gl)):
        check_backward(backward(kx, torch_cuda, x, tokens, t, *a), x, tokens, t, dtype, *a)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("v", [5, 1003, 9000])
def test_gradient_of_masks_and_special_values(kx, torch_cuda, dtype, v):
    low = np.finfo(dtype).min
    x, _ = logits(71, 12, v, dtype)
    j = np.arange(v)
    x[1][j % 3 != 0] = -np.inf
    x[2] = -np.inf
    x[3] = low
    x[4][j % 2 == 0] = low
    x[5, v // 2] = np.nan
    x[6, 0] = np.inf
    x[7] += 1000
    x[8] = -np.inf
    x[8, 1] = 3
    x[9] -= 30000
    tokens = np.array([0, 0, 1, 1, 1, 0, 0, 2, 2, 3, -1, v], np.int64)
    g, gh, gl = grads_in(19, 12, dtype)
    for a in ((g, None, None), (g, gh, gl)):
        check_backward(backward(kx, torch_cuda, x, tokens, 1.0, *a), x, tokens, 1.0, dtype, *a)


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_gradient_of_an_impossible_token_is_nan_everywhere(kx, torch_cuda, dtype):
    """Where probabilities are 0 too, but for masked logits."""
    x, _ = logits(77, 3, 700, dtype)
    x[:, 1::2] -= 3000
    x[:, 5] = -np.inf
    tokens = np.array([700, 0, 10 ** 12], np.int64)
    got = backward(kx, torch_cuda, x, tokens, 1.0, np.ones(3, dtype))
    for r in (0, 2):
        assert got[r, 5] == 0 and np.isnan(np.delete(got[r], 5)).all()
    check_backward(got[1:2], x[1:2], tokens[1:2], 1.0, dtype, np.ones(1, dtype))


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("v", [9, 1100, 5001])
def test_gradient_layouts(kx, torch_cuda, dtype, v):
    """Logits at every alignment against the gradient's, a vocabulary of
    another stride, and row operands with strides of their own."""
    torch = torch_cuda
    tt = torch.float32 if dtype == np.float32 else torch.float64
    rows = 6
    x, tokens = logits(81, rows, v, dtype)
    g, gh, gl = grads_in(29, rows, dtype)
    dx, dt = torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda()
    apart = lambda a: torch.from_numpy(np.repeat(a, 3)).cuda()[1::3]  # noqa: E731
    res = kx.token_log_probs(dx, dt, entropy=True)

    def check(view, xs=x, toks=tokens, dtok=dt, order=slice(None), lead=(rows,)):
        pick = lambda a: apart(a)[order].reshape(lead) if lead == (rows,) else apart(a).reshape(3, 2).t()  # noqa: E731
        r = [pick(a.cpu().numpy()) for a in (res.lse, res.entropy)]
        out = torch.full((*lead, v), 7.0, dtype=tt, device="cuda")
        kx.token_log_probs_backward_into(view, dtok, out, lse=r[0], entropy=r[1], grad_log_probs=pick(g),
                                         grad_entropy=pick(gh), grad_lse=pick(gl))
        perm = np.arange(rows).reshape(3, 2).T.reshape(-1) if lead != (rows,) else np.arange(rows)[order]
        check_backward(out.cpu().numpy().reshape(rows, v), xs, toks, 1.0, dtype, g[perm], gh[perm], gl[perm])

    for off in range(5):
        wide = torch.full((rows, v + 9), float("nan"), dtype=tt, device="cuda")
        wide[:, off:off + v] = dx
        check(wide[:, off:off + v])
    check(dx.t().contiguous().t())
    check(kx.TensorView(dx.reshape(-1), (rows, v), (v, 1), 0))
    by = dx.reshape(3, 2, v).transpose(0, 1)
    tb = dt.reshape(3, 2).t()
    order = np.arange(rows).reshape(3, 2).T.reshape(-1)
    check(by, x[order], tokens[order], tb, lead=(2, 3))
    # an output that starts off 16 bytes, and what lies beside it stays
    buf = torch.full((rows * v + 3,), 5.0, dtype=tt, device="cuda")
    out = buf[1:1 + rows * v].reshape(rows, v)
    kx.token_log_probs_backward_into(dx, dt, out, lse=res.lse, grad_log_probs=torch.from_numpy(g).cuda())
    check_backward(out.cpu().numpy(), x, tokens, 1.0, dtype, g)
    assert buf[0] == 5 and buf[-2:].tolist() == [5, 5]


def test_gradient_against_differences(kx, torch_cuda):
    """Central differences of the f64 forward pass: sum of a lp + b H + c lse.
    With steps of 1e-5 the third derivatives (at most 20 of each unit here)
    leave 1e-10 x weights / 6, and rounding 2^-53 x values (under 100) / 1e-5."""
    torch = torch_cuda
    rows, v, t = 3, 17, 0.8
    x, tokens = logits(91, rows, v, np.float64, 1.0)
    a = grads_in(39, rows, np.float64)
    got = backward(kx, torch, x, tokens, t, *a)
    tol = sum(float(np.abs(w).sum()) for w in a) * (20e-10 / t ** 3 + 100 * 2.0 ** -52 / 1e-5)

    def value(y):
        r = run(kx, torch, y, tokens, t, 0)
        return float((a[0] * r.log_probs + a[1] * r.entropy + a[2] * r.lse).sum())

    for r in range(rows):
        for j in range(v):
            hi, lo = x.copy(), x.copy()
            hi[r, j] += 1e-5
            lo[r, j] -= 1e-5
            assert abs((value(hi) - value(lo)) / 2e-5 - got[r, j]) <= tol


def test_refusals_on_the_device(kx, torch_cuda):
    torch = torch_cuda
    x = torch.zeros(2, 8, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs(x, t.int())
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs(x, t, temperature=0.0)
    with pytest.raises(kx.NoDevice):
        kx.token_log_probs(x, t.cpu())
    with pytest.raises(kx.Unsupported):
        kx.token_log_probs(x.half(), t)
    with pytest.raises(kx.InvalidRank):
        kx.token_log_probs_into(x[0, 0], None, kx.TokenLogProbs(lse=torch.zeros((), device="cuda")))
    lse = torch.zeros(2, device="cuda")
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs_backward(x, t, lse=lse.double(), grad_log_probs=lse)
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs_backward(x, t, lse=lse, grad_entropy=lse)
    with pytest.raises(kx.OverlappingOutput):
        kx.token_log_probs_backward_into(x, t, x, lse=lse, grad_log_probs=lse)
    err = kx.KxError()
    assert kx.lib.kx_token_log_probs_f32(None, None, None, 1.0, None, None, None, None, None, C.byref(err)) != 0


def test_launches_are_counted(kx, torch_cuda):
    torch = torch_cuda
    h = kx.handle(0)
    n = h.launches
    res = kx.token_log_probs(torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert h.launches == n + 1 and h.last_kernel.startswith("log_probs")
    kx.token_log_probs_backward(torch.zeros(2, 8, device="cuda"), lse=res.lse, grad_lse=res.lse)
    assert h.launches == n + 2 and h.last_kernel.startswith("log_probs_backward")
