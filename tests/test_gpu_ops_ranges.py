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


# ---------------------------------------------------------------- the two halves of the autograd form
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", PATHS + [(7, 100, 5003), (31, 257, 9001), (300, 130, 2050), (2000, 64, 100), (700, 300, 3000)])
def test_a_backward_pass_by_itself_makes_the_same_logits(ops, dtype, n, h, v):
    """Logits of some 1e4 (half precision) to 1e7 with gaps of many times their rounding: a row has one class, so d_hidden is
    the difference of two classes' weights, off by two roundings of the type -- if the backward pass sees the logits that the
    forward pass took its maximum from."""
    x, w, b, t = make(n, h, v, dtype, "index", bias=False, seed=n + h + v)
    x *= 2.0 ** (12 if dtype == "f16" else 20)
    l = x.double() @ w.double().t()
    two = l.topk(2, 1)
    slack = 4 * ((h + 2) * F + 3 * 2.0 ** -22) * (x.double().abs() @ w.double().abs().t()).max(1).values
    clear = two.values[:, 0] - two.values[:, 1] > slack + 200       # (the other rows may fall on either side)
    assert int(clear.sum()) > n // 2
    want = w.double()[two.indices[:, 0]] - w.double()[t]
    bound = 2 * half_step(DT[dtype]) * want.abs() + 4 * F * (w.double()[two.indices[:, 0]].abs() + w.double()[t].abs())
    xl = x.clone().requires_grad_()
    ops.linear_cross_entropy(xl, w, t, reduction="sum").backward()
    one = ops.linear_cross_entropy_grad(x, w, t, reduction="sum")
    for got in (xl.grad, one.d_hidden):
        assert bool(((got.double() - want).abs() <= bound)[clear].all())


# ---------------------------------------------------------------- rows that are certain, logits with a common offset
def exact_logits(n, h, v, dtype, offset, peak, seed=3):
    """Rows of one 1 each, so that logits are weights and a bias: multiples of 1/8, at most 8 in magnitude, the same in every type
    and product.  Every bias is `offset`, and `peak` more at one class, which is the target of four rows of five."""
    gen = torch.Generator("cuda").manual_seed(seed)
    x = torch.zeros(n, h, device="cuda")
    at = torch.arange(n, device="cuda") % h
    x[torch.arange(n, device="cuda"), at] = 1.0
    w = torch.randint(-64, 65, (v, h), generator=gen, device="cuda").float() / 8
    b = torch.full((v,), float(offset), device="cuda")
    best = v // 3
    b[best] += peak
    t = torch.full((n,), best, dtype=torch.int64, device="cuda")
    t[::5] = torch.randint(0, v, (len(t[::5]),), generator=gen, device="cuda")
    dt = DT[dtype]
    l = w.double().t()[at] + b.to(dt).double()
    return x.to(dt), w.to(dt), b.to(dt), t, l


CERTAIN = PATHS + [(7, 104, 5003), (7, 100, 5003), (300, 64, 20000), (1000, 40, 16717), (1500, 96, 4300)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", CERTAIN)
@pytest.mark.parametrize("offset,peak", [(0, 0), (0, 16), (0, 32), (0, 96), (1024, 16), (-1024, 32)])
def test_loss_and_entropy_of_exact_logits(ops, dtype, n, h, v, offset, peak):
    """With d = l - max exact, an exponential is off by (|d| + 2) 2 f of itself (its argument, log2 e, the instruction) and a sum of
    positive numbers by 80 f (additions one after the other: at most 32 in a lane, 2 across lanes, 32 over spans, 6 across lanes),
    and by no more than the terms beside the maximum, twice, where these are less.  Nothing depends on an offset of all logits; a certain row's loss and entropy are at least 0."""
    x, w, b, t, l = exact_logits(n, h, v, dtype, offset, peak)
    d = l - l.max(1, keepdim=True).values
    e = torch.exp(d)
    s = e.sum(1)
    p = e / s[:, None]
    rel = (d.abs() + 2) * 2 * F
    rs = (p * rel).sum(1) + torch.clamp(2 * (1 - 1 / s), max=80 * F)
    for kind in ("index", "probs"):
        if kind == "index":
            target = t
            want = torch.log(s) - d.gather(1, t[:, None])[:, 0]
            bound = rs + 4 * F * want.abs()
        else:
            target = torch.zeros(n, v, device="cuda")
            target[torch.arange(n), t] = 0.75
            target[torch.arange(n), (t + 7) % v] += 0.25
            want = torch.log(s) - (target.double() * d).sum(1)
            bound = rs + 4 * F * torch.log(s) + 90 * F * (target.double() * d.abs()).sum(1)
        ent = torch.log(s) - (p * d).sum(1)
        b_ent = rs + (p * d.abs() * (rel + rs[:, None] + 90 * F)).sum(1) + 4 * F * ent
        outs = [ops.linear_cross_entropy(x, w, target, b, reduction="none", return_entropy=True)]
        one = ops.linear_cross_entropy_grad(x, w, target, b, reduction="none", return_entropy=True)
        outs.append(one[:2])
        for loss, entropy in outs:
            assert float(loss.min()) >= 0 and float(entropy.min()) >= 0
            assert bool(((loss.double() - want).abs() <= bound).all()), float(((loss.double() - want).abs() / bound.clamp_min(1e-300)).max())
            assert bool(((entropy.double() - ent).abs() <= b_ent).all()), float(((entropy.double() - ent).abs() / b_ent.clamp_min(1e-300)).max())
