"""The projection's softmax cross entropy where numbers are far apart: rows without a class, magnitudes and probabilities of
any size, rows that are certain.  Bounds are derived in each test; f = 2**-24, u = half a step of a type."""
import math

import pytest
import torch

from test_gpu_ops import DT, F, PATHS, half_step, make, philox

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from alphazero_gomoku_amd import ops as o
    return o


def autograd(ops, x, w, t, b, scale=1.0, **kw):
    """(loss, d_hidden, d_weight, d_bias): a forward pass and a backward pass by itself, of scale times the sum of the losses."""
    leaves = [q.clone().requires_grad_() for q in (x, w, b)]
    loss = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], **kw)
    (scale * loss.sum()).backward()
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


# ---------------------------------------------------------------- operands, probabilities and weights far apart
def elementwise(x, w, b, t, g, kept=False):
    """{name: (value in float64, bound)} of loss rows, d_hidden, d_weight and d_bias under sum g_i loss_i, every bound an
    element's own: products and sums of (H + 8) f sum|x w| in a logit (float32 leaves out 2 f of it); a probability by what its logit
    and the others' (weighted by their probabilities) may be off, by (2 |l - max| + 100) f of itself, and where one call keeps
    exponentials in 16 bits (`kept`) by 2^-11, or below 2^-39 of its neighbours' largest 2^-9, of itself; the gradient at the logits D by its rounding (bfloat16 half a step, half precision 2^-17); the products by what they
    leave out (float32 2 f, half precision 2^-16), (K + 40) f, and the result's rounding."""
    dt = x.dtype
    n, h = x.shape
    v = w.shape[0]
    by_index = t.dtype == torch.int64
    xd, wd = x.double(), w.double()
    l = xd @ wd.t() + (0 if b is None else b.double())
    dl = (h + 8) * F * (xd.abs() @ wd.abs().t()) + F * l.abs()
    q = torch.zeros_like(l) if by_index else t.double()
    if by_index:
        q[torch.arange(n), t] = 1.0
    m = l.max(1, keepdim=True).values
    lse = torch.logsumexp(l, 1, keepdim=True)
    p = torch.exp(l - lse)
    el = (p * dl).sum(1, keepdim=True)
    own = p * ((2 * (l - m).abs() + 100) * F + (torch.where(p < 2.0 ** -38 * p.max(1, keepdim=True).values, 2.0 ** -9, 2.0 ** -11) if kept else 0.0))
    up = torch.exp((l - lse + dl + el).clamp(max=0.0))               # a row with one class left: the others' bounds are what it may lose
    top = l == m
    low = torch.maximum(torch.exp(l - lse - dl - el), torch.where(top, 1 - torch.where(top, 0.0, up).sum(1, keepdim=True), 0.0))
    bp = torch.maximum(up - p, p - low) * (1 + 2.0 ** -10) + own
    qs = q.sum(1, keepdim=True)
    gd = g.double()[:, None]
    D = gd * (p * qs - q)
    bD0 = gd.abs() * (bp * qs.abs() + 4 * F * (p * qs.abs() + q.abs()))
    bD = bD0 + {torch.float32: F, torch.bfloat16: half_step(dt), torch.float16: 2.0 ** -17}[dt] * D.abs()
    out, u = (2.0 ** -25 if dt == torch.float16 else 0.0), half_step(dt)
    op = {torch.float32: 2 * F, torch.bfloat16: 0.0, torch.float16: 2.0 ** -16}[dt]

    def product(a, ba, c, k):
        r = a @ c
        return r, (ba @ c.abs() + ((k + 40) * F + op) * (a.abs() @ c.abs())) * (1 + 2 * u) + u * r.abs() * (1 + 1e-6) + out
    loss = ((m - l) * q).sum(1) + torch.log(torch.exp(l - m).sum(1)) * qs[:, 0]
    b_loss = (q.abs() * dl).sum(1) + qs.abs()[:, 0] * (el[:, 0] + 100 * F) + 8 * F * ((q.abs() * (m - l)).sum(1) + loss.abs())
    db = D.sum(0)
    return {"loss": (loss, b_loss), "d_hidden": product(D, bD, wd, v), "d_weight": product(D.t(), bD.t(), xd, n),
            "d_bias": (db, (bD0.sum(0) + (n + 40) * F * D.abs().sum(0)) * (1 + 2 * u) + u * db.abs() * (1 + 1e-6) + out)}


def within(name, got, want, bound, rows=slice(None)):
    err = (got.double() - want).abs()[rows]
    bad = ~(err <= bound[rows])
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g times its bound" % (name, int(bad.sum()), bad.numel(), float((err / bound[rows].clamp_min(1e-300)).max()))


FAR = PATHS + [(7, 100, 5003), (300, 130, 2050), (1500, 64, 6000), (300, 33, 34000)]


@pytest.mark.parametrize("n,h,v", FAR)
@pytest.mark.parametrize("size", [1e6, 1e8, 1e12])
@pytest.mark.parametrize("where", ["row", "class", "feature"])
def test_one_large_row_or_class_spoils_no_other(ops, n, h, v, size, where):
    """float32: a row, or a class, `size` times the others (a class that is so far below that no row has it), or one feature
    that is large in one row and that no class looks at.  All the other rows' and classes' results keep their own bounds."""
    x, w, b, t = make(n, h, v, "f32", "index", seed=n + h + v)
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    if where == "row":
        x[2] *= size
        rest[2] = False                                             # (whose logits are known to no better than size * f)
    elif where == "class":
        x[:, 0] = 1.0
        w[:, 0] = 0.0
        w[v // 2] = 0.0
        w[v // 2, 0] = -size
        t[t == v // 2] = 0
    else:
        w[:, 1] = 0.0
        x[2, 1] = size
    ref = elementwise(x, w, b, t, torch.ones(n, device="cuda"))
    for dx, dw, db, loss in ((lambda r: r[2:] + (r[0],))(ops.linear_cross_entropy_grad(x, w, t, b, reduction="none")),
                             (lambda r: r[1:] + (r[0],))(autograd(ops, x, w, t, b, reduction="none"))):
        within("loss", loss, *ref["loss"], rest)
        within("d_hidden", dx, *ref["d_hidden"], rest)
        within("d_weight", dw, *ref["d_weight"])
        within("d_bias", db, *ref["d_bias"])
    within("loss alone", ops.linear_cross_entropy(x, w, t, b, reduction="none"), *ref["loss"], rest)


@pytest.mark.parametrize("n,h,v", FAR)
def test_operands_of_every_magnitude(ops, n, h, v):
    """float32: rows of 2^-60 to 1 and classes of 2^-20 to 1 of the ordinary size, an empty row, and a row that holds the largest
    number, where no class looks at it, and 2^-100, which every class raises to 1 or -1."""
    x, w, b, t = make(n, h, v, "f32", "index", seed=n + h + v)
    x *= torch.exp2(torch.linspace(-60, 0, n, device="cuda").round())[:, None]
    w *= torch.exp2(torch.linspace(0, -20, v, device="cuda").round())[:, None]
    x[0], x[1], x[:, 1] = 0.0, 0.0, 0.0
    x[1, 0], x[1, 1], w[:, 0], w[:, 1] = 3.4028234e38, 2.0 ** -100, 0.0, 2.0 ** 100 * torch.sign(w[:, 1])
    ref = elementwise(x, w, b, t, torch.ones(n, device="cuda"))
    r = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none")
    for name, got in (("loss", r.loss), ("d_hidden", r.d_hidden), ("d_weight", r.d_weight), ("d_bias", r.d_bias)):
        within(name, got, *ref[name])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kind", ["index", "probs"])
@pytest.mark.parametrize("n,h,v", FAR)
def test_gradients_of_classes_that_are_hardly_ever_taken(ops, dtype, kind, n, h, v):
    """Classes of probability 1e-5 to 1e-25 in every row, next to ordinary ones: their rows of d_weight keep their digits, in one call
    and in two.  (Half precision with its gradients raised by 2^14; what falls below its own numbers counts as theirs.)"""
    x, w, b, t = make(n, h, v, dtype, kind, seed=n + h + v)
    rare = torch.arange(3, v, 7, device="cuda")
    b[rare] = -torch.linspace(5.0, 50.0 if dtype == "f32" else 24.0, len(rare), device="cuda").to(b.dtype)
    if kind == "index":
        t = torch.where(t % 7 == 3, t - 1, t)
    else:
        t[:, rare] = 0.0
    scale = 16384.0 if dtype == "f16" else 1.0
    ref = elementwise(x, w, b, t, torch.full((n,), scale, device="cuda"))
    for dw, db in (ops.linear_cross_entropy_grad(x, w, t, b, reduction="sum", grad_loss=scale)[3:],
                   autograd(ops, x, w, t, b, scale, reduction="sum")[2:]):
        within("d_weight", dw, *ref["d_weight"], rare)
        within("d_bias", db, *ref["d_bias"], rare)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kind", ["index", "probs"])
@pytest.mark.parametrize("n,h,v", PATHS + [(300, 130, 2050), (1500, 64, 6000), (9000, 24, 500)])
def test_rows_of_very_different_weight(ops, dtype, kind, n, h, v):
    """reduction='none' with weights from 1e-30 (half precision: 1e-6) to 1: every row of d_hidden against its own size."""
    x, w, b, t = make(n, h, v, dtype, kind, seed=n + h + v)
    g = torch.logspace(-30 if dtype != "f16" else -6, 0, n, device="cuda")
    g[::2] *= -1.0
    if kind == "probs":
        t = t * torch.logspace(0, -6, n, device="cuda")[:, None]
    if dtype == "f16":
        g *= 4096.0
    ref = elementwise(x, w, b, t, g)
    r = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none", grad_loss=g)
    for name, got in (("loss", r.loss), ("d_hidden", r.d_hidden), ("d_weight", r.d_weight), ("d_bias", r.d_bias)):
        within(name, got, *ref[name])


@pytest.mark.parametrize("kind", ["index", "probs"])
@pytest.mark.parametrize("n,h,v", FAR + [(64, 72, 4100)])
def test_bfloat16_gradients_of_classes_that_are_hardly_ever_taken(ops, kind, n, h, v):
    """As above in bfloat16, down to 1e-34: classes next to ordinary ones, and a run of 600 of them with one ordinary class in it."""
    x, w, b, t = make(n, h, v, "bf16", kind, seed=n + h + v)
    rare = torch.arange(3, v, 7, device="cuda")
    b[rare] = -torch.linspace(5.0, 70.0, len(rare), device="cuda").to(b.dtype)
    if v > 2000:
        b[1001:1600] = -30.0
        rare = torch.cat([rare, torch.arange(1001, 1600, device="cuda")])
    common = torch.ones(v, dtype=torch.bool, device="cuda")
    common[rare] = False
    if kind == "index":
        t = common.nonzero()[:, 0][t % int(common.sum())]
    else:
        t[:, rare] = 0.0
    g = torch.ones(n, device="cuda")
    for kept, (dw, db) in ((kind == "index", ops.linear_cross_entropy_grad(x, w, t, b, reduction="sum")[3:]), (False, autograd(ops, x, w, t, b, reduction="sum")[2:])):
        ref = elementwise(x, w, b, t, g, kept)
        within("d_weight", dw, *ref["d_weight"])
        within("d_bias", db, *ref["d_bias"])
        assert bool((dw[rare] != 0).any(1).all())


@pytest.mark.parametrize("kind", ["index", "probs"])
@pytest.mark.parametrize("n,h,v", PATHS + [(300, 130, 2050), (1500, 64, 6000), (9000, 24, 500)])
def test_bfloat16_rows_of_very_different_weight(ops, kind, n, h, v):
    x, w, b, t = make(n, h, v, "bf16", kind, seed=n + h + v)
    g = torch.logspace(-30, 0, n, device="cuda")
    g[::2] *= -1.0
    ref = elementwise(x, w, b, t, g, kind == "index")
    r = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none", grad_loss=g)
    for name, got in (("loss", r.loss), ("d_hidden", r.d_hidden), ("d_weight", r.d_weight), ("d_bias", r.d_bias)):
        within(name, got, *ref[name])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", [(1, 24, 5003), (2, 24, 65), (2, 24, 5003), (3, 8, 20000), (40, 24, 3000)])
@pytest.mark.parametrize("apart", [0.1, 0.01, 0.001])
def test_probabilities_that_are_nearly_met(ops, dtype, n, h, v, apart):
    """Target probabilities within `apart` of the softmax: the gradient at the logits is the small difference, rounded as such."""
    x, w, b, t = make(n, h, v, dtype, "index", seed=n + h + v)
    p = torch.softmax(x.double() @ w.double().t() + b.double(), 1)
    t = (p * (1 + apart * torch.randn(n, v, device="cuda"))).float()
    scale = 1024.0 if dtype == "f16" else 1.0
    ref = elementwise(x, w, b, t, torch.full((n,), scale, device="cuda"))
    one = ops.linear_cross_entropy_grad(x, w, t, b, reduction="sum", grad_loss=scale)
    for dx, dw, db in (one[2:], autograd(ops, x, w, t, b, scale, reduction="sum")[1:]):
        within("d_hidden", dx, *ref["d_hidden"])
        within("d_weight", dw, *ref["d_weight"])
        within("d_bias", db, *ref["d_bias"])


# ---------------------------------------------------------------- dropout's element numbers
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols,first,step", [(16, (1 << 60) - 2, 1), (7, ((1 << 64) - 2) // 7 - 1, 1), (13, (1 << 64) - 3, 1), (13, (1 << 64) - 3, 5),
                                             (100, (1 << 64) - 1, (1 << 64) - 1), (8, (1 << 61) - 1, 1)])
def test_dropout_numbers_elements_modulo_2_to_the_64(ops, dtype, cols, first, step):
    """Element (r, c) is number ((first + r step) cols + c) modulo 2^64, whatever the layout of the rows."""
    rows, seed, offset = 6, 77, 5
    x = (torch.rand(rows, cols, device="cuda") + 1).to(DT[dtype])
    keep = torch.empty(rows, cols, dtype=torch.bool)
    for r in range(rows):
        for c in range(cols):
            at = ((first + r * step) * cols + c) % (1 << 64)
            keep[r, c] = bool(philox(at - at % 8, 8, seed, offset)[at % 8] >= 32768)
    far = torch.zeros(rows, cols + 3, dtype=x.dtype, device="cuda")
    far[:, :cols] = x
    for view in (x, far[:, :cols]):
        y = ops.dropout(view, 0.5, seed, offset, first_row=first, row_step=step)
        assert torch.equal(y, torch.where(keep.cuda(), 2 * x, torch.zeros_like(x)))


# ---------------------------------------------------------------- derivatives that are not there
def test_forward_mode_and_second_derivatives_are_refused(ops):
    import torch.autograd.forward_ad as fw
    x, w, b, t = make(8, 16, 9, "f32")
    p = torch.rand(8, 9, device="cuda")
    g = torch.ones(8, device="cuda")
    with fw.dual_level():
        def dual(q):
            return fw.make_dual(q, torch.ones_like(q))
        for call in (lambda: ops.dropout(dual(x), 0.1, 1), lambda: ops.dropout(x, 0.1, 1, residual=dual(x)), lambda: ops.dropout_grad(dual(x), 0.1, 1),
                     lambda: ops.linear_cross_entropy(dual(x), w, t, b), lambda: ops.linear_cross_entropy(x, dual(w), t, b),
                     lambda: ops.linear_cross_entropy(x, w, t, dual(b)), lambda: ops.linear_cross_entropy(x, w, dual(p), b),
                     lambda: ops.linear_cross_entropy(x.clone().requires_grad_(), dual(w), t, b),
                     lambda: ops.linear_cross_entropy_grad(x, w, t, b, reduction="none", grad_loss=dual(g))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        ops.linear_cross_entropy(x, w, t, b)                        # without a tangent inside a dual level: as ever
    leaf = x.clone().requires_grad_()
    first, = torch.autograd.grad(ops.linear_cross_entropy(leaf, w, t, b), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()
