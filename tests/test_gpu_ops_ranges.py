"""The projection's softmax cross entropy where numbers are far apart: rows without a class, magnitudes and probabilities of
any size, rows that are certain.  Bounds are derived in each test; f = 2**-24, u = half a step of a type."""
import math

import pytest
import torch

from test_gpu_ops import DT, F, PATHS, half_step, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from alphazero_gomoku_amd import ops as o
    return o


def autograd(ops, x, w, t, b, **kw):
    """(loss, d_hidden, d_weight, d_bias): a forward pass and a backward pass by itself."""
    leaves = [q.clone().requires_grad_() for q in (x, w, b)]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], **kw)
    loss.sum().backward()
    return (loss.detach(),) + tuple(q.grad for q in leaves)


# ---------------------------------------------------------------- rows without a class
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["index", "probs"])
@pytest.mark.parametrize("n,h,v", PATHS)
def test_a_row_without_a_class_is_nan_everywhere(ops, dtype, kind, n, h, v):
    """Every class blocked: 0/0 in the softmax, so the loss and all that a counted row reaches is NaN -- the same in one call
    and in two, on every path; ignored rows stay zero."""
    x, w, b, t = make(n, h, v, dtype, kind, ignored=0.3 if kind == "index" else 0.0)
    used = (t != -100) if kind == "index" else torch.ones(n, dtype=torch.bool, device="cuda")
    b = torch.full_like(b, float("-inf"))
    one = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none", return_entropy=True)
    assert bool(torch.isnan(one.loss[used]).all()) and bool(torch.isnan(one.entropy[used]).all()) and not bool(one.loss[~used].any())
    for dx, dw, db in (one[2:], autograd(ops, x, w, t, b, reduction="none")[1:]):
        assert bool(torch.isnan(dx[used]).all()) and not bool(dx[~used].any())
        assert bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", PATHS)
def test_a_bad_target_reaches_blocked_classes_too(ops, dtype, n, h, v):
    """A row with a target outside the classes is NaN at every class, those without a finite logit among them."""
    x, w, b, t = make(n, h, v, dtype, "index")
    b[v // 2:] = float("-inf")
    t = t % (v // 2)
    t[5] = v
    one = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none")
    for dx, dw, db in (one[2:], autograd(ops, x, w, t, b, reduction="none")[1:]):
        assert bool(torch.isnan(dx[5]).all()) and bool(torch.isfinite(dx[:5]).all()) and bool(torch.isfinite(dx[6:]).all())
        assert bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())
