"""Refusals of the training-head operators' C entry points that need no GPU, and what happens without one."""
import ctypes as C
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from alphazero_gomoku_amd import _lib
    return _lib


def dropout_args(lib, **kw):
    a = lib.DropoutArgs()
    a.dtype, a.rows, a.cols, a.x, a.out, a.x_stride, a.out_stride, a.p, a.row_step = lib.F32, 4, 8, 4096, 4096, 8, 8, 0.5, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def ce_args(lib, **kw):
    a = lib.LinearCeArgs()
    a.dtype, a.n, a.hidden, a.classes, a.x, a.w, a.x_stride, a.w_stride, a.target, a.loss = lib.F32, 4, 8, 16, 4096, 4096, 8, 8, 4096, 4096
    a.workspace, a.workspace_bytes, a.reduction = 4096, 1 << 40, lib.REDUCE_MEAN
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(lib, rc, what):
    text = lib.load().azg_last_error(None).decode()
    assert rc == -1 and what in text, (rc, text)


@pytest.mark.parametrize("kw,what", [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(p=1.5), "p must"), (dict(p=-0.1), "p must"),
                                     (dict(p=math.nan), "p must"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"), (dict(x=None), "null"),
                                     (dict(out=None), "null"), (dict(x_stride=7), "stride"), (dict(out_stride=7), "stride"),
                                     (dict(residual=4096, residual_stride=7), "stride"), (dict(rows=1 << 40, cols=1 << 20), "too many")])
def test_dropout_refuses(lib, kw, what):
    refused(lib, lib.load().azg_dropout(C.byref(dropout_args(lib, **kw))), what)


@pytest.mark.parametrize("kw,what", [(dict(dtype=3), "dtype"), (dict(n=-1), "sizes"), (dict(hidden=0), "sizes"), (dict(classes=0), "sizes"),
                                     (dict(n=1 << 40), "too large"), (dict(n=1 << 26), "too large"), (dict(classes=1 << 27), "too large"), (dict(hidden=1 << 23), "too large"), (dict(reduction=3), "reduction"),
                                     (dict(reduction=-1), "reduction"), (dict(x_stride=7), "stride"), (dict(w_stride=7), "stride"),
                                     (dict(x_stride=1 << 23), "too large"), (dict(w_stride=1 << 23), "too large")])
def test_linear_ce_refuses_sizes(lib, kw, what):
    a = ce_args(lib, **kw)
    refused(lib, lib.load().azg_linear_ce(C.byref(a)), what)
    refused(lib, int(lib.load().azg_linear_ce_workspace(C.byref(a))), what)


@pytest.mark.parametrize("kw,what", [(dict(loss=None), "neither"), (dict(loss=None, dx=4096, dx_stride=8), "stats"), (dict(loss=None, dx=4096, entropy=4096, stats=4096, dx_stride=8), "entropy"),
                                     (dict(dx=4096, dx_stride=7), "stride"), (dict(dw=4096, dw_stride=7), "stride"), (dict(x=None), "null"), (dict(w=None), "null"),
                                     (dict(target=None), "either"), (dict(probs=4096, probs_stride=16), "either"), (dict(target=None, probs=4096, probs_stride=15), "stride"),
                                     (dict(stats=4100), "aligned")])
def test_linear_ce_refuses_pointers(lib, kw, what):
    refused(lib, lib.load().azg_linear_ce(C.byref(ce_args(lib, **kw))), what)


def test_null_and_workspace(lib):
    L = lib.load()
    refused(lib, L.azg_dropout(None), "null")
    refused(lib, L.azg_linear_ce(None), "null")
    refused(lib, int(L.azg_linear_ce_workspace(None)), "null")
    a = ce_args(lib)
    small = int(L.azg_linear_ce_workspace(C.byref(a)))
    assert small >= 4 * 16 * 4
    a.dw, a.dw_stride, a.classes, a.probs_stride = 4096, 8, 100000, 0
    large = int(L.azg_linear_ce_workspace(C.byref(a)))
    assert large > small
    a.n = 0
    assert int(L.azg_linear_ce_workspace(C.byref(a))) == 0


def test_workspace_is_bounded(lib):
    """No image of n * classes elements is kept whole: beyond a gigabyte the classes are cut into pieces."""
    a = ce_args(lib, dtype=lib.BF16, n=32768, hidden=4096, classes=131072, x_stride=4096, w_stride=4096, dx=4096, dx_stride=4096,
                dw=4096, dw_stride=4096)
    size = int(lib.load().azg_linear_ce_workspace(C.byref(a)))
    whole = 2 * 32768 * 131072
    rows = 32768 * 4096 * (2 + 4)                                   # X's image and the float32 sum of the pieces' dX
    stats = 8 * (131072 // 128 + 8) * 32768                         # (maximum, sum) pairs
    assert size < whole / 4 + rows + stats + (1 << 24), size


def test_workspace_of_few_features_and_of_single_rows(lib):
    """The logits that small problems keep are bounded whatever the features; the stride of a single row does not matter."""
    a = ce_args(lib, dtype=lib.BF16, n=1 << 22, hidden=1, classes=32, x_stride=1, w_stride=1)
    assert 0 < int(lib.load().azg_linear_ce_workspace(C.byref(a))) < (1 << 22) * (16 + 4 + 4 + 4 + 2 * 8 + 4 * 128)
    a = ce_args(lib, n=1, classes=1, x_stride=1 << 40, w_stride=1 << 40)
    assert int(lib.load().azg_linear_ce_workspace(C.byref(a))) > 0
    a = ce_args(lib, n=(1 << 26) - 1, classes=2)
    assert int(lib.load().azg_linear_ce_workspace(C.byref(a))) > 0


def test_python_forms_need_a_gpu():
    from alphazero_gomoku_amd import ops
    x, w, t = torch.randn(4, 8), torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.dropout(x, 0.1, 1), lambda: ops.dropout_grad(x, 0.1, 1), lambda: ops.linear_cross_entropy(x, w, t),
                 lambda: ops.linear_cross_entropy_grad(x, w, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    if not torch.cuda.is_available():                               # an error code, not a crash
        from alphazero_gomoku_amd import _lib
        assert _lib.load().azg_dropout(C.byref(dropout_args(_lib))) == -2


def test_forward_mode_is_refused_without_a_gpu():
    import torch.autograd.forward_ad as fw
    from alphazero_gomoku_amd import ops
    x, w, t = torch.randn(4, 8), torch.randn(5, 8), torch.zeros(4, dtype=torch.int64)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        assert not d.requires_grad
        for call in (lambda: ops.dropout(d, 0.1, 1), lambda: ops.dropout_grad(d, 0.1, 1), lambda: ops.linear_cross_entropy(d, w, t),
                     lambda: ops.linear_cross_entropy_grad(d, w, t)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda q: ops.dropout(q, 0.1, 1), (x,), (x,))
