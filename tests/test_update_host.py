"""Host side of the operators between logits and an update (CPU only, no
device calls): what token_log_probs, its gradient, grad_norm and
clip_grad_norm refuse, and in which order, before any device work.  The
stand-in handle is zeroed host memory, as in the sharded product's tests."""
import ctypes as C

import pytest

import kernix_b200 as kx
from kernix_b200 import _abi

NAN, INF = float("nan"), float("inf")


def _tensor(dims, strides=None, origin=0, length=None, data=0x10000):
    t = _abi.KxTensor()
    if strides is None:
        strides, n = [], 1
        for d in reversed(dims):
            strides.insert(0, n)
            n *= d
    span = 1 + sum((d - 1) * s for d, s in zip(dims, strides) if d > 0)
    t.data, t.origin, t.rank = data, origin, len(dims)
    t.storage_len = span + origin if length is None else length
    for i, (d, s) in enumerate(zip(dims, strides)):
        t.dims[i], t.strides[i] = d, s
    return t


FAKE = (C.c_uint8 * 65536)()


def _call(name, *args):
    err = _abi.KxError()
    refs = [C.byref(a) if isinstance(a, _abi.KxTensor) else a for a in args]
    rc = getattr(_abi.lib, name)(C.addressof(FAKE), *refs, C.byref(err))
    return rc, err


def _forward(logits, tokens, t, *outs, kind="f32"):
    return _call(f"kx_token_log_probs_{kind}", logits, tokens, t, *outs)


LOGITS = _tensor([2, 3, 10])
TOKENS = _tensor([2, 3], data=0x20000)
ROWS = [_tensor([2, 3], data=0x30000 + 0x1000 * i) for i in range(3)]
TOP = [_tensor([2, 3, 4], data=0x40000), _tensor([2, 3, 4], data=0x50000)]


@pytest.mark.parametrize("kind", ["f32", "f64"])
@pytest.mark.parametrize("t", [0.0, -1.0, NAN, INF, 5e-324])
def test_log_probs_refuse_a_temperature_before_everything_else(kind, t):
    rc, err = _forward(_tensor([2, 3], data=None), None, t, None, None, None, None, None, kind=kind)
    assert rc == _abi.KX_E_PARAM and err.operation == b"token_log_probs" and b"temperature" in err.parameter
    rc, err = _call(f"kx_token_log_probs_backward_{kind}", LOGITS, None, None, None, None, None, None, t, None)
    assert rc == _abi.KX_E_PARAM and b"temperature" in err.parameter


def test_log_probs_refusals():
    ok = (*ROWS, *TOP)
    rc, err = _forward(_tensor([]), None, 1.0, None, ROWS[0], None, None, None)
    assert rc == _abi.KX_E_INVALID_RANK and (err.values[0], err.values[1]) == (1, 0)
    rc, err = _forward(_tensor([2, 3, 10], length=59), TOKENS, 1.0, *ok)
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "StorageTooSmall"
    rc, err = _forward(_tensor([2, 1 << 31], [0, 0]), None, 1.0, None, _tensor([2], data=0x30000), None, None, None)
    assert rc == _abi.KX_E_UNSUPPORTED
    for args in [(None, *ok), (TOKENS, None, *ok[1:])]:
        rc, err = _forward(LOGITS, args[0], 1.0, *args[1:])
        assert rc == _abi.KX_E_PARAM and err.parameter == b"tokens and log_probs go together"
    rc, err = _forward(LOGITS, TOKENS, 1.0, *ROWS, TOP[0], None)
    assert rc == _abi.KX_E_PARAM and err.parameter == b"top_log_probs and top_tokens go together"
    rc, err = _forward(LOGITS, None, 1.0, None, None, None, None, None)
    assert rc == _abi.KX_E_PARAM and err.parameter == b"no output"
    for bad in ([2], [2, 4], [2, 3, 1], [3, 2]):
        rc, err = _forward(LOGITS, _tensor(bad, data=0x20000), 1.0, *ok)
        assert rc == _abi.KX_E_PARAM and b"tokens" in err.parameter
        for i in range(3):
            outs = list(ok)
            outs[i] = _tensor(bad, data=0x60000)
            rc, err = _forward(LOGITS, TOKENS, 1.0, *outs)
            assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputShapeMismatch"
    rc, err = _forward(LOGITS, TOKENS, 1.0, *ROWS, TOP[0], _tensor([2, 3, 5], data=0x50000))
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputShapeMismatch"
    rc, err = _forward(LOGITS, TOKENS, 1.0, *ROWS, *[_tensor([2, 3, 33], data=d) for d in (0x40000, 0x50000)])
    assert rc == _abi.KX_E_PARAM and b"32" in err.parameter
    rc, err = _forward(LOGITS, TOKENS, 1.0, _tensor([2, 3], [1, 2], data=0x30000), *ok[1:])
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputNotCContiguous"
    for i in range(5):      # each output over the logits, and over another output or the tokens
        for where in (0x10000 + 8 * 20, 0x20000, 0x40000 if i != 3 else 0x50000):
            outs = list(ok)
            outs[i] = _tensor([2, 3] if i < 3 else [2, 3, 4], data=where)
            rc, err = _forward(LOGITS, TOKENS, 1.0, *outs)
            assert rc == _abi.KX_E_ALIAS, (i, hex(where))
    rc, err = _forward(LOGITS, _tensor([2, 3], data=0x20004), 1.0, *ok)     # int64 off its alignment
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "MisalignedPointer"
    # no rows: nothing to do, with and without a vocabulary
    for dims in ([0, 10], [2, 0, 10]):
        lead = dims[:-1]
        rc, _ = _forward(_tensor(dims, data=None), _tensor(lead, data=None), 1.0, _tensor(lead, data=None), None, None,
                         None, None)
        assert rc == _abi.KX_OK


def test_log_probs_backward_refusals():
    name = "kx_token_log_probs_backward_f32"
    lse, ent, g, gh, gl = (_tensor([2, 3], data=0x30000 + 0x1000 * i) for i in range(5))
    out = _tensor([2, 3, 10], data=0x80000)

    def call(logits=LOGITS, tokens=TOKENS, lse=lse, ent=ent, g=g, gh=gh, gl=gl, out=out):
        return _call(name, logits, tokens, lse, ent, g, gh, gl, 1.0, out)

    rc, err = call(g=None, gh=None, gl=None)
    assert rc == _abi.KX_E_PARAM and err.parameter == b"no incoming gradient"
    for missing, word in ((dict(lse=None), b"lse"), (dict(tokens=None), b"tokens"), (dict(ent=None), b"entropy")):
        rc, err = call(**missing)
        assert rc == _abi.KX_E_PARAM and err.parameter.startswith(word)
    for which in ("tokens", "lse", "ent", "g", "gh", "gl"):
        rc, err = call(**{which: _tensor([6], data=0x90000)})
        assert rc == _abi.KX_E_PARAM and b"one for each row" in err.parameter
    rc, err = call(out=_tensor([2, 30], data=0x80000))
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputShapeMismatch"
    rc, err = call(out=_tensor([2, 3, 10], [60, 20, 2], data=0x80000))
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputNotCContiguous"
    for over in (0x10000, 0x20000, 0x30000, 0x31000, 0x32000, 0x33000, 0x34000):
        assert call(out=_tensor([2, 3, 10], data=over))[0] == _abi.KX_E_ALIAS
    rc, _ = call(logits=_tensor([2, 0], data=None), tokens=_tensor([2], data=0x20000),
                 **{k: _tensor([2], data=0x30000 + 0x1000 * i) for i, k in enumerate(("lse", "ent", "g", "gh", "gl"))},
                 out=_tensor([2, 0], data=None))
    assert rc == _abi.KX_OK


def _size():
    size = C.c_uint64()
    assert _abi.lib.kx_grad_norm_workspace(C.byref(size)) == _abi.KX_OK
    return size.value


def _clip(grads, outs=None, max_norm=1.0, norm=None, ws=0x4000000, size=None, count=None, kind="f32"):
    n = len(grads) if count is None else count
    err = _abi.KxError()
    norm = _tensor([], data=0x8000) if norm is None else norm
    size = _size() if size is None else size
    garr = (_abi.KxTensor * max(1, len(grads)))(*grads)
    tail = (C.byref(norm), ws, size, C.byref(err))
    if outs is None:
        rc = getattr(_abi.lib, f"kx_grad_norm_{kind}")(C.addressof(FAKE), garr, n, *tail)
    else:
        oarr = (_abi.KxTensor * max(1, len(outs)))(*outs)
        rc = getattr(_abi.lib, f"kx_clip_grad_norm_{kind}")(C.addressof(FAKE), garr, n, max_norm, oarr, *tail)
    return rc, err


def test_the_workspace_is_small_and_asked_for():
    assert 0 < _size() <= 1 << 20
    assert _abi.lib.kx_grad_norm_workspace(None) == _abi.KX_E_PARAM


def test_norm_and_clip_refusals():
    a, b = _tensor([4, 8], data=0x10000), _tensor([16], data=0x20000)
    oa, ob = _tensor([4, 8], data=0x30000), _tensor([16], data=0x40000)
    for t in (0.0, -1.0, NAN, INF):
        rc, err = _clip([a], [oa], max_norm=t)
        assert rc == _abi.KX_E_PARAM and err.operation == b"clip_grad_norm" and b"max_norm" in err.parameter
    rc, err = _clip([a], norm=_tensor([2], data=0x8000))
    assert rc == _abi.KX_E_LAYOUT and err.operation == b"grad_norm"
    for kw in (dict(size=_size() - 1), dict(ws=None), dict(ws=0x4000004)):
        rc, err = _clip([a], **kw)
        assert rc == _abi.KX_E_PARAM and b"workspace" in err.parameter
    rc, err = _clip([a, _tensor([4, 8], length=31)])
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "StorageTooSmall"
    rc, err = _clip([a, b], [oa, _tensor([15], data=0x40000)])
    assert rc == _abi.KX_E_LAYOUT and _abi.LAYOUT_ERRORS[err.values[0]] == "OutputShapeMismatch"
    alias = [
        ([a, b], [oa, _tensor([16], data=0x30000)]),                    # two outputs meet
        ([a, b], [oa, _tensor([16], data=0x10000)]),                    # an output over another gradient
        ([a, b], [oa, _tensor([16], data=0x20004)]),                    # shifted over its own gradient
        ([a], [_tensor([4, 8], [1, 4], data=0x10000)]),                 # its own gradient in another order
        ([b, b], [b, b]),                                               # the same gradient twice, in place
        ([b], [_tensor([16], [0], data=0x40000)]),                      # elements that share a place
        ([a], [_tensor([4, 8], [4, 1], data=0x40000)]),
        ([b], [_tensor([16], data=0x8000)]),                            # over the norm
        ([b], [_tensor([16], data=0x4000000)]),                         # over the workspace
    ]
    for grads, outs in alias:
        assert _clip(grads, outs)[0] == _abi.KX_E_ALIAS, (grads, outs)
    assert _clip([b], norm=_tensor([1], data=0x20000))[0] == _abi.KX_E_ALIAS
    assert _clip([b], ws=0x20000)[0] == _abi.KX_E_ALIAS
    rc, err = _clip([a], count=(1 << 20) + 1)
    assert rc == _abi.KX_E_UNSUPPORTED
    huge = [_tensor([1 << 40, 1 << 22], [0, 0])] * 3
    rc, err = _clip(huge)
    assert rc == _abi.KX_E_UNSUPPORTED and b"elements" in err.parameter


def test_python_refuses_before_the_library():
    import torch
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs(x, t, top=33)
    with pytest.raises(kx.InvalidParameter):
        kx.token_log_probs(x, t, top=-1)
    with pytest.raises(kx.NoDevice):
        kx.token_log_probs(x, t)
    with pytest.raises(kx.Unsupported):
        kx.token_log_probs(x.half(), t)
    with pytest.raises(kx.InvalidParameter):
        kx.grad_norm([])
    with pytest.raises(kx.NoDevice):
        kx.grad_norm([x])
    with pytest.raises(kx.NoDevice):
        kx.clip_grad_norm([x], 1.0)


def test_lists_describe_contiguous_pairs_by_their_elements():
    """Host only: a contiguous gradient's descriptor is its elements as one
    axis; others keep their strides, in both lists if either needs it."""
    import torch
    g = [torch.zeros(3, 4)[1:], torch.zeros(4, 3).t(), torch.zeros(0, 3), torch.tensor(1.0), torch.zeros(2, 2)]
    o = [torch.zeros(2, 4), torch.zeros(4, 3).t(), torch.zeros(0, 3), torch.tensor(1.0), torch.zeros(2, 2).t()]
    alone = [1, 4]
    arr = kx._descriptors(g, alone)
    assert (arr[0].data, arr[0].rank, arr[0].dims[0], arr[0].strides[0]) == (g[0].data_ptr(), 1, 8, 1)
    assert (arr[0].storage_len, arr[0].origin) == (8, 0)
    assert (arr[1].rank, list(arr[1].dims)[:2], list(arr[1].strides)[:2]) == (2, [3, 4], [1, 3])
    assert (arr[2].rank, arr[2].dims[0]) == (1, 0) and (arr[3].rank, arr[3].dims[0]) == (1, 1)
    arr = kx._descriptors(o, alone)
    assert list(arr[4].strides)[:2] == [1, 2]


def test_the_binding_leaves_what_it_does_not_take():
    """kernix_b200._kx_torch on the host: anything but CUDA tensors of one
    device and dtype is left to the general path, with nothing called."""
    import torch

    native = kx._native()
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    err = _abi.KxError()
    h, e = C.addressof(FAKE), C.addressof(err)
    assert native.token_log_probs(h, 0, x, t, 1.0, 0, False, e) is None
    assert native.token_log_probs(h, 0, "x", t, 1.0, 0, False, e) is None
    view = kx.TensorView(torch.zeros(10), (2, 5), (5, 1))
    assert native.token_log_probs_backward(h, 0, view, None, x, None, x, None, None, 1.0, None, e) is None
    assert native.grad_norm(h, 0, [], None, 0.0, None, e) is None
    assert native.grad_norm(h, 0, [x], None, 0.0, None, e) is None
    assert native.grad_norm(h, 0, (x,), None, 0.0, None, e) is None
    for name, count in (("token_log_probs", 8), ("token_log_probs_backward", 12), ("grad_norm", 7), ("bind", 9)):
        with pytest.raises(TypeError):
            getattr(native, name)(*[0] * (count - 1))
    with pytest.raises(ValueError):
        native.bind(*[0] * 9)
    with pytest.raises(TypeError):
        native.token_log_probs("h", 0, x, t, 1.0, 0, False, e)
