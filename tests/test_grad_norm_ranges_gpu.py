"""The gradient norm and clipping over the whole range of f64: squares that
leave 64 bits on either side, and among ordinary ones."""
import numpy as np
import pytest

from test_grad_norm_gpu import check_clip, true_norm

pytestmark = pytest.mark.gpu

TINY = np.finfo(np.float64).smallest_normal


def lists(case):
    """Elements of one size, of sizes far apart, both sides of each border."""
    base = np.array([1.0, -0.75, 0.5, 1.5, -1.25, 0.3, 0.9])
    make = {
        "large": lambda: [base * 1e200, base[:3] * 1e200],
        "largest": lambda: [base[2:3] * 1e308, base[1:2] * 1e308],
        "beyond the squares' range by little": lambda: [base * 2.0 ** 512, base * 2.0 ** 511],
        "within the squares' range by little": lambda: [base * 2.0 ** 509, base * 2.0 ** 508],
        "one large among ordinary": lambda: [np.tile(base, 300), np.array([-1e180]), np.tile(base, 11)],
        "one large in each list": lambda: [np.r_[np.tile(base, 5000), 1e160], np.r_[3e159, np.tile(base, 700)]],
        "large and small": lambda: [base * 1e170, base * 1e-170],
        "small": lambda: [base * 1e-200, base[:5] * 1e-200],
        "smallest": lambda: [np.full(9, 5e-324), base * 1e-310],
        "below the squares' range by little": lambda: [base * 2.0 ** -511, base * 2.0 ** -540],
        "where the sums change": lambda: [base * 2.0 ** -475, base * 2.0 ** -476],
        "small among zeros": lambda: [np.r_[np.zeros(3000), 1e-190, np.zeros(5000)], np.zeros(7)],
        "one ordinary among small": lambda: [np.tile(base, 200) * 1e-180, np.array([2.0])],
        "many small": lambda: [np.tile(base, 20_000) * 1e-165] * 2,
        "many large": lambda: [np.tile(base, 20_000) * 1e155] * 2,
    }
    return make[case]()


CASES = ["large", "largest", "beyond the squares' range by little", "within the squares' range by little",
         "one large among ordinary", "one large in each list", "large and small", "small", "smallest",
         "below the squares' range by little", "where the sums change", "small among zeros",
         "one ordinary among small", "many small", "many large"]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("gaps", [False, True])
def test_f64_squares_out_of_range(kx, torch_cuda, case, gaps):
    """Bounds as for ordinary elements: scaling by powers of two is exact, and
    a norm of the smallest numbers rounds to a multiple of one."""
    torch = torch_cuda
    arrs = lists(case)
    dev = [torch.from_numpy(a).cuda() for a in arrs]
    if gaps:
        dev = [torch.stack([d, torch.full_like(d, 7.0)], 1)[:, 0] for d in dev]
    n = sum(a.size for a in arrs)
    want = true_norm(arrs)
    got = kx.grad_norm(dev)
    tol = want * (2.0 ** -53 + n * 2.0 ** -53) + np.longdouble(5e-324)
    assert np.isfinite(float(want)) and abs(np.longdouble(got.item()) - want) <= tol, (got.item(), want)
    if float(want) < TINY:
        return
    for max_norm in (float(want) / 3, float(want) * 2):
        if max_norm < TINY or not np.isfinite(max_norm):
            continue
        norm, outs = kx.clip_grad_norm(dev, max_norm)
        assert torch.equal(norm, got)       # the same sums, whatever becomes of them
        check_clip(norm, outs, arrs, max_norm, np.float64)


def test_f64_squares_out_of_range_in_folded_sums(kx, torch_cuda):
    """Lists so long that partial sums are folded on the way and before the
    scaling."""
    torch = torch_cuda
    base = torch.arange(1, 601 * 1001 + 1, dtype=torch.float64, device="cuda").reshape(601, 1001) / 601_601
    for scale in (1e180, 1e-180, 1.0):
        views = [(base * (scale * (1 + i % 3)))[:, :1000] for i in range(300)]
        host = [v.cpu().numpy() for v in views[:3]]
        want = np.sqrt(np.longdouble(100)) * true_norm(host)
        n = 300 * 601_000
        norm, outs = kx.clip_grad_norm(views, 3.0 * scale)
        # 100 of each: the same sums, off by n 2^-53 of themselves at most
        for got in (norm, kx.grad_norm(views)):
            assert abs(np.longdouble(got.item()) - want) <= want * (2.0 ** -53 + n * 2.0 ** -53)
        by = np.longdouble(3.0 * scale) / want
        got, w = outs[299].cpu().numpy().astype(np.longdouble), host[2].astype(np.longdouble) * by
        assert (np.abs(got - w) <= np.abs(w) * (3 * 2.0 ** -53 + n * 2.0 ** -53)).all()


def test_f64_norms_that_no_number_holds(kx, torch_cuda):
    """Above the largest number, infinite and NaN among large and small."""
    torch = torch_cuda
    big = torch.full((16,), 1e308, dtype=torch.float64, device="cuda")
    norm, (out,) = kx.clip_grad_norm([big], 1.0)
    assert norm.item() == np.inf and torch.equal(out, big)
    for bad in (np.inf, -np.inf, np.nan):
        for other in (1e200, 1e-200):
            x = torch.full((5000,), other, dtype=torch.float64, device="cuda")
            x[4321] = bad
            norm, (out,) = kx.clip_grad_norm([x], 1.0)
            assert np.isnan(norm.item()) if np.isnan(bad) else norm.item() == np.inf
            assert np.array_equal(out.cpu().numpy(), x.cpu().numpy(), equal_nan=True)


@pytest.mark.parametrize("dtype,size,max_norm", [
    (np.float32, 1e12, 1e-30), (np.float32, 3e30, 1e-7), (np.float32, 1e20, 1e-37), (np.float32, 1e38, 1e-12),
    (np.float32, 1.0, 1e-44), (np.float32, 1.0, 1e-60), (np.float64, 1e200, 1e-150), (np.float64, 3e307, 0.7),
    (np.float64, 1e100, 1e-300), (np.float64, 1e-5, 1e-320)])
@pytest.mark.parametrize("apart", [False, True])
def test_factors_below_the_normal_numbers(kx, torch_cuda, dtype, size, max_norm, apart):
    """max_norm / norm need not be a normal number where its products are; into
    copies, in place, at other alignments, and into outputs of other strides.
    A result rounds once more than check_clip counts where it is itself below
    the normal numbers: two of the smallest numbers."""
    torch = torch_cuda
    base = np.array([1.0, -0.75, 0.5, 1.5, -1.25, 0.3, 0.9, 1e-3, -1e-7])
    arrs = [np.tile(base, 41).astype(dtype) * dtype(size) * dtype(0.06), (base * size).astype(dtype)]
    dev = [torch.from_numpy(a).cuda() for a in arrs]
    if apart:
        dev = [torch.stack([d, torch.full_like(d, 7.0)], 1)[:, 0] for d in dev]
    n = sum(a.size for a in arrs)
    want = true_norm(arrs)
    by = np.longdouble(max_norm) / want
    u = 2.0 ** -24 if dtype == np.float32 else 2.0 ** -53
    buf = torch.full((n + 40,), 9.0, dtype=dev[0].dtype, device="cuda")
    odd = [buf[1:1 + arrs[0].size], buf[arrs[0].size + 11:][:arrs[1].size]]
    norm, outs = kx.clip_grad_norm(dev, max_norm)
    kx.clip_grad_norm_into(dev, max_norm, odd)
    kx.clip_grad_norm_into(dev, max_norm, dev)
    assert abs(np.longdouble(norm.item()) - want) <= want * (u + n * 2.0 ** -53)
    for got in (outs, odd, dev):
        for g, a in zip(got, arrs):
            w = a.astype(np.longdouble) * by
            tol = np.abs(w) * (3 * u + n * 2.0 ** -53) + 2 * np.longdouble(np.finfo(dtype).smallest_subnormal)
            assert (np.abs(g.cpu().numpy().astype(np.longdouble) - w) <= tol).all()


def test_a_factor_just_below_the_smallest_number_in_place(kx, torch_cuda):
    """Its first part rounds to 1, which is not the factor 1."""
    torch = torch_cuda
    x = torch.zeros(9, device="cuda")
    x[4] = 1.0
    kx.clip_grad_norm_into([x], 2.0 ** -149 * (1 - 2.0 ** -27), [x])
    assert x.tolist() == [0] * 4 + [2.0 ** -149] + [0] * 4


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_the_order_of_the_sums(kx, torch_cuda, dtype):
    """The same values at the same places against 16 bytes have the same bits,
    wherever they are; at other places the sums' order is another, and the norm
    within the bounds of any order."""
    torch = torch_cuda
    ty = torch.float32 if dtype == np.float32 else torch.float64
    n, size = 30_011, torch.tensor([], dtype=ty).element_size()
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(n, generator=gen, device="cuda", dtype=ty)
    want = true_norm([x.cpu().numpy()])
    u = 2.0 ** -24 if dtype == np.float32 else 2.0 ** -53
    buf = torch.empty(8 * (n + 64), device="cuda", dtype=ty)
    seen = {}
    for start in (0, 4, 64, 1, 5, 17, 2, 3, 7):
        at = buf[start:start + n]
        at.copy_(x)
        norm = kx.grad_norm([at]).item()
        assert abs(np.longdouble(norm) - want) <= want * (u + n * 2.0 ** -53)
        assert seen.setdefault(at.data_ptr() % 16, norm) == norm
    assert len(seen) == 16 // size
