"""Operators of the training heads as functions of CUDA tensors: dropout whose mask is never stored, and the
softmax cross entropy of a projection whose logits are not kept (include/azgomoku.h: azg_dropout, azg_linear_ce).
While a call makes gradients it holds one array of rows x classes in place of the logits -- bfloat16 2 bytes an
element, half precision 4, float32 6 -- of at most 1 GiB together with the copies of the weights that it needs, or
of 1024 classes; beyond that it takes the classes in pieces and makes their logits twice.  A loss alone holds
none; small problems hold at most 16 MB of float32 logits.  The operators run on the tensors' device and its
current stream, like PyTorch's own.

dropout() and linear_cross_entropy() take part in autograd.  dropout_grad() and linear_cross_entropy_grad() are
the same without it -- loss and gradients in one call, no graph of nodes -- and are what to capture into a HIP
graph; the autograd forms refuse to be captured when an input wants a gradient (accumulating into leaves that
an eager graph also holds cannot be captured).  Forward-mode differentiation and second derivatives are refused."""
import ctypes as C
from collections import namedtuple

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_MAX_STRIDE = 1 << 22                         # of a projection's operands
_REDUCTIONS = {"none": _lib.REDUCE_NONE, "sum": _lib.REDUCE_SUM, "mean": _lib.REDUCE_MEAN}

LinearCrossEntropyGrad = namedtuple("LinearCrossEntropyGrad", "loss entropy d_hidden d_weight d_bias")


def _check_tensor(name, t, dtype=None, device=None):
    if not torch.is_tensor(t):
        raise TypeError("%s must be a tensor" % name)
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:   # (its tangent would be lost)
        raise NotImplementedError("%s carries a forward-mode tangent: these operators have no forward-mode derivative" % name)
    if not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor: the operators have no CPU form" % name)
    if dtype is None:
        if t.dtype not in _DTYPES:
            raise ValueError("%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    elif t.dtype != dtype:
        raise ValueError("%s must be %s, not %s" % (name, dtype, t.dtype))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))


def _rows(name, t, max_stride=None):
    """t as (rows, columns, row stride in elements) without a copy, or a copy whose rows are contiguous: (t, rows, cols, stride)."""
    if t.dim() == 0:
        raise ValueError("%s must have at least one dimension" % name)
    cols = t.shape[-1]
    rows = t.numel() // cols if cols else 0
    if t.dim() == 2 and (cols <= 1 or t.stride(1) == 1) and (rows <= 1 or cols <= t.stride(0) <= (max_stride or t.stride(0))):
        return t, rows, cols, t.stride(0) if rows > 1 else cols
    if not t.is_contiguous():
        t = t.contiguous()
    return t, rows, cols, cols


def _refuse_capture(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors) and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("autograd through this operator cannot be captured into a graph: capture dropout_grad / "
                           "linear_cross_entropy_grad, or call it under torch.no_grad()")


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)     # torch.cuda.current_stream(device).cuda_stream, without its object


# ---------------------------------------------------------------- dropout
def _word(name, v):
    if isinstance(v, bool) or not isinstance(v, int) or not 0 <= v < 1 << 64:
        raise ValueError("%s must be an integer from 0 to 2**64 - 1" % name)
    return v


def _dropout_raw(x, p, seed, offset, residual, first_row, row_step, out=None):
    xt, rows, cols, xs = _rows("x", x)
    a = _lib.DropoutArgs()
    a.device, a.dtype = x.device.index, _DTYPES[x.dtype]
    if residual is not None:
        rt, _, _, a.residual_stride = _rows("residual", residual)
        a.residual = rt.data_ptr()
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a.rows, a.cols, a.x, a.x_stride = rows, cols, xt.data_ptr(), xs
    a.out, a.out_stride = out.data_ptr(), cols
    a.p, a.seed, a.first_row, a.row_step = p, seed, first_row, row_step
    if torch.is_tensor(offset):
        a.offset_dev = offset.data_ptr()
    else:
        a.offset = offset
    a.stream = _stream(x.device)
    _lib.check(None, _lib.load().azg_dropout(C.byref(a)))
    return out


def _check_dropout(x, p, seed, offset, residual, first_row, row_step):
    _check_tensor("x", x)
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    if not 0.0 <= float(p) <= 1.0:
        raise ValueError("p must lie in [0, 1]")
    _word("seed", seed), _word("first_row", first_row), _word("row_step", row_step)
    if torch.is_tensor(offset):
        _check_tensor("offset", offset, torch.int64, x.device)
        if offset.numel() != 1:
            raise ValueError("offset must hold one element")
    else:
        _word("offset", offset)
    if residual is not None:
        _check_tensor("residual", residual, x.dtype, x.device)
        if residual.shape != x.shape:
            raise ValueError("residual has shape %s, x %s" % (tuple(residual.shape), tuple(x.shape)))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, first_row, row_step):
        # (an offset on the device may move on before the backward pass: the value of this call is kept)
        ctx.args = (p, seed, offset.clone() if torch.is_tensor(offset) else offset, first_row, row_step)
        return _dropout_raw(x, p, seed, offset, residual, first_row, row_step)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, seed, offset, first_row, row_step = ctx.args
        dx = _dropout_raw(dy, p, seed, offset, None, first_row, row_step) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None, None, None


def dropout(x, p, seed, offset=0, *, residual=None, first_row=0, row_step=1):
    """[residual +] x with each element dropped with probability p and the others scaled so that the expectation
    stays.  The mask is a function of (seed, offset, element number): a training step takes a seed for the run and
    its step number as offset, and nothing is stored for the backward pass.

    x         float32, bfloat16 or float16 [..., cols], any strides.
    p         in [0, 1], rounded to a multiple of 1/65536; the scale is exactly one over the rounded keep rate.
    offset    an integer, or an int64 CUDA tensor of one element that is read when the kernel runs (a captured
              graph then draws a new mask at every replay when the program counts it up).
    first_row, row_step
              the rows of x (all leading dimensions flattened) are rows first_row, first_row + row_step, ... of a
              larger batch: ranks that share one batch draw the mask a single process would draw."""
    _check_dropout(x, p, seed, offset, residual, first_row, row_step)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        _refuse_capture(x, residual)
        return _Dropout.apply(x, residual, float(p), seed, offset, first_row, row_step)
    return _dropout_raw(x, float(p), seed, offset, residual, first_row, row_step)


def dropout_grad(dy, p, seed, offset=0, *, first_row=0, row_step=1):
    """The gradient at dropout()'s x from the gradient dy at its result (the residual's gradient is dy itself)."""
    _check_dropout(dy, p, seed, offset, None, first_row, row_step)
    return _dropout_raw(dy.detach(), float(p), seed, offset, None, first_row, row_step)


# ---------------------------------------------------------------- projection + softmax cross entropy
def _check_ce(hidden, weight, target, bias, reduction, ignore_index):
    _check_tensor("hidden", hidden)
    _check_tensor("weight", weight, hidden.dtype, hidden.device)
    if hidden.dim() < 1 or weight.dim() != 2:
        raise ValueError("hidden must be [..., features] and weight [classes, features]")
    if hidden.shape[-1] != weight.shape[1]:
        raise ValueError("hidden has %d features, weight %d" % (hidden.shape[-1], weight.shape[1]))
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("weight must have at least one class and one feature")
    if bias is not None:
        _check_tensor("bias", bias, hidden.dtype, hidden.device)
        if bias.shape != (weight.shape[0],):
            raise ValueError("bias must be [classes]")
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if isinstance(ignore_index, bool) or not isinstance(ignore_index, int) or not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must be an integer")
    if not torch.is_tensor(target):
        raise TypeError("target must be a tensor")
    if target.dtype == torch.int64:
        _check_tensor("target", target, torch.int64, hidden.device)
        if target.shape != hidden.shape[:-1]:
            raise ValueError("target has shape %s, the rows of hidden %s" % (tuple(target.shape), tuple(hidden.shape[:-1])))
        return True
    if target.dtype == torch.float32:
        _check_tensor("target", target, torch.float32, hidden.device)
        if target.shape != hidden.shape[:-1] + (weight.shape[0],):
            raise ValueError("target probabilities must be [..., classes]")
        if target.requires_grad:
            raise ValueError("target probabilities take no gradient")
        return False
    raise ValueError("target must be int64 class numbers or float32 probabilities, not %s" % target.dtype)


class _CeCall:
    """One azg_linear_ce call: the inputs once, then forward, backward or both."""

    def __init__(self, hidden, weight, target, bias, reduction, ignore_index, by_index):
        self.keep = [hidden, weight, target, bias]
        self.device, self.dtype = hidden.device, hidden.dtype
        self.hidden_shape, self.rows_shape = hidden.shape, hidden.shape[:-1]
        x, n, h, xs = _rows("hidden", hidden, _MAX_STRIDE)
        w, v, _, wst = _rows("weight", weight, _MAX_STRIDE)
        a = self.a = _lib.LinearCeArgs()
        a.device, a.dtype, a.reduction = self.device.index, _DTYPES[hidden.dtype], _REDUCTIONS[reduction]
        a.n, a.hidden, a.classes = (n if h else 0), h, v
        a.x, a.x_stride, a.w, a.w_stride = x.data_ptr(), xs, w.data_ptr(), wst
        self.keep += [x, w]
        if bias is not None:
            b = bias.contiguous()
            self.keep.append(b)
            a.bias = b.data_ptr()
        if by_index:
            t = target.contiguous()
            a.target, a.ignore_index = t.data_ptr(), ignore_index
        else:
            t, _, _, a.probs_stride = _rows("target", target)
            a.probs = t.data_ptr()
        self.keep.append(t)
        a.grad_scale = 1.0

    def _f32(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.device)

    def forward(self, with_entropy, with_stats):
        none = self.a.reduction == _lib.REDUCE_NONE
        shape = self.rows_shape if none else ()
        self.loss = self._f32(*shape)
        self.a.loss = self.loss.data_ptr() if self.loss.numel() else self._spare()
        self.entropy = None
        if with_entropy:
            self.entropy = self._f32(*shape)
            self.a.entropy = self.entropy.data_ptr() if self.entropy.numel() else self._spare()
        if with_stats:
            self.stats = self._f32(self.a.n, 4)
            self.a.stats = self.stats.data_ptr()

    def _spare(self):
        t = self._f32(1)                      # (an empty batch's loss has no address; nothing is written there)
        self.keep.append(t)
        return t.data_ptr()

    def backward(self, dloss, scale, want_x, want_w, want_b):
        a = self.a
        if dloss is not None:
            d = dloss.contiguous()
            self.keep.append(d)
            a.dloss = d.data_ptr() if d.numel() else None
        a.grad_scale = scale
        self.dx = self.dw = self.db = None
        if want_x:
            self.dx = torch.empty(self.hidden_shape, dtype=self.dtype, device=self.device)
            a.dx, a.dx_stride = (self.dx.data_ptr() if a.n else None), a.hidden
        if want_w:
            self.dw = torch.empty((a.classes, a.hidden), dtype=self.dtype, device=self.device)
            a.dw, a.dw_stride = self.dw.data_ptr(), a.hidden
        if want_b:
            self.db = torch.empty(a.classes, dtype=self.dtype, device=self.device)
            a.db = self.db.data_ptr()

    def run(self):
        lib, a = _lib.load(), self.a
        if not (a.loss or a.dx or a.dw or a.db):
            return self                       # the gradient at the rows of an empty batch
        size = lib.azg_linear_ce_workspace(C.byref(a))
        if size < 0:
            _lib.check(None, int(size))
        ws = torch.empty(max(int(size), 1), dtype=torch.uint8, device=self.device)
        a.workspace, a.workspace_bytes, a.stream = ws.data_ptr(), size, _stream(self.device)
        _lib.check(None, lib.azg_linear_ce(C.byref(a)))
        return self


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, reduction, ignore_index, by_index, with_entropy):
        c = _CeCall(hidden, weight, target, bias, reduction, ignore_index, by_index)
        c.forward(with_entropy, True)
        c.run()
        ctx.save_for_backward(hidden, weight, bias, target, c.stats)
        ctx.args = (reduction, ignore_index, by_index)
        if not with_entropy:
            return c.loss
        ctx.mark_non_differentiable(c.entropy)
        return c.loss, c.entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, dentropy=None):
        hidden, weight, bias, target, stats = ctx.saved_tensors
        c = _CeCall(hidden, weight, target, bias, *ctx.args)
        c.a.stats = stats.data_ptr()
        c.keep.append(stats)
        need = ctx.needs_input_grad
        c.backward(dloss.float(), 1.0, need[0], need[1], need[2] and bias is not None)
        c.run()
        return c.dx, c.dw, c.db, None, None, None, None, None


def linear_cross_entropy(hidden, weight, target, bias=None, *, reduction="mean", ignore_index=-100, return_entropy=False):
    """Softmax cross entropy of hidden @ weight.T + bias against target; what a call holds meanwhile: see the module.

    hidden    float32, bfloat16 or float16 [..., features]; weight [classes, features] and bias [classes] of its type.
    target    int64 [...]: class numbers; rows with ignore_index count for nothing.  Or float32 [..., classes]:
              probabilities (a search's visit shares), loss = -sum target log softmax.
    Returns the float32 loss (a scalar, or [...] with reduction='none'; the mean is over the rows that count, 0 when
    none does), with return_entropy also the entropy of the softmax, which takes no gradient."""
    by_index = _check_ce(hidden, weight, target, bias, reduction, ignore_index)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        _refuse_capture(hidden, weight, bias)
        return _LinearCrossEntropy.apply(hidden, weight, bias, target, reduction, ignore_index, by_index, bool(return_entropy))
    c = _CeCall(hidden.detach(), weight.detach(), target, None if bias is None else bias.detach(), reduction, ignore_index, by_index)
    c.forward(return_entropy, False)
    c.run()
    return (c.loss, c.entropy) if return_entropy else c.loss


def linear_cross_entropy_grad(hidden, weight, target, bias=None, *, reduction="mean", ignore_index=-100, return_entropy=False,
                              grad_loss=1.0):
    """linear_cross_entropy() and its gradients in one call: (loss, entropy, d_hidden, d_weight, d_bias); entropy is
    None unless asked for, d_bias without a bias.  grad_loss is the gradient at the loss: a number, or a float32 CUDA
    tensor of the loss's shape."""
    by_index = _check_ce(hidden, weight, target, bias, reduction, ignore_index)
    c = _CeCall(hidden.detach(), weight.detach(), target, None if bias is None else bias.detach(), reduction, ignore_index, by_index)
    c.forward(return_entropy, False)
    if torch.is_tensor(grad_loss):
        _check_tensor("grad_loss", grad_loss, torch.float32, hidden.device)
        if grad_loss.shape != c.loss.shape:
            raise ValueError("grad_loss has shape %s, the loss %s" % (tuple(grad_loss.shape), tuple(c.loss.shape)))
        c.backward(grad_loss.detach(), 1.0, True, True, bias is not None)
    else:
        c.backward(None, float(grad_loss), True, True, bias is not None)
    c.run()
    return LinearCrossEntropyGrad(c.loss, c.entropy, c.dx, c.dw, c.db)
