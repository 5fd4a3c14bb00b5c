"""The training heads' operators (alphazero_gomoku_amd.ops) against their definitions in 64 bits.

Tolerances are bounds, computed element by element from the inputs.  With u = half a step of a type
(torch.finfo(t).eps / 2), K the length of a sum and f = 2**-24:
  a float32 sum of K products is off by at most (K + 2) f sum|a b|; float32 operands are cut to two half-precision
  numbers, off by 2**-22 each, with one product of 2**-22 left out: 3 * 2**-22 sum|a b| more;
  so a logit is off by dl = ((H + 2) f + 3 * 2**-22 [float32]) sum|x w| + f |l|, a probability by p (2 max dl + 2**-20): the
  exponential, its argument (|l - m| <= 40 here: 40 f log2 e) and the reciprocal of the sum take less than 2**-20;
  the loss by 2 max dl + 8 f (|lse| + |l_t| + 2); the gradient at the logits D by its probability's part, its own rounding
  u |D| (float32: 2**-22; half precision holds D 2**14, so 2**-39 of D's scale below its smallest normal number); where
  loss and gradients come from one call, 16-bit types keep exp(l - m') of a run of classes with maximum m' in half precision
  meanwhile: 2**-11 of itself, or 2**-25 of exp(m' - lse) <= the row's largest probability, more; and the
  gradients by the two operands' errors, the float32 sum and the result's rounding (half precision: 2**-25 at least)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
F = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from alphazero_gomoku_amd import ops as o
    return o


def half_step(dt):
    return torch.finfo(dt).eps / 2


# ---------------------------------------------------------------- dropout
def philox(first, count, seed, offset):
    """uint16 of the element numbers first .. first + count - 1 (Philox4x32-10, numpy)."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    b0 = first >> 3
    blk = np.arange(0, ((first + count + 7) >> 3) - b0, dtype=np.uint64) + np.uint64(b0 & ((1 << 64) - 1))
    c = [blk & m, blk >> s, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    u = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=1).reshape(-1)
    return u[first - 8 * b0: first - 8 * b0 + count].astype(np.int64)


def keep_mask(rows, cols, p, seed, offset, first_row=0, row_step=1):
    t = int(math.floor(p * 65536 + 0.5))
    return torch.from_numpy(np.stack([philox((first_row + r * row_step) * cols, cols, seed, offset) >= t for r in range(rows)])).cuda(), t


def test_philox_known_answers():
    """The published known-answer vectors of Philox4x32-10 (all-zero and all-one counter and key)."""
    def words(ctr, key):
        c, k = [np.uint64(v) for v in ctr], list(key)
        m = np.uint64(0xFFFFFFFF)
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return [int(v) for v in c]
    assert words([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert words([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    z = philox(0, 8, 0, 0)
    assert [int(z[2 * i] | (z[2 * i + 1] << 16)) for i in range(4)] == words([0] * 4, [0] * 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols,p,first", [(1, 1, 0.5, 0), (1, 7, 0.3, 3), (3, 8, 0.5, 0), (5, 13, 0.25, 7), (64, 256, 0.1, 0),
                                               (17, 900, 0.3, 1 << 33), (2, 4099, 0.02, (1 << 61) + 5), (33, 65, 1.0, 0), (33, 65, 0.0, 2)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_against_definition(ops, dtype, rows, cols, p, first, residual):
    dt, seed, offset = DT[dtype], 0x9E3779B97F4A7C15, (1 << 40) + 12345
    gen = torch.Generator("cuda").manual_seed(rows * cols)
    x = torch.randn(rows, cols, generator=gen, device="cuda").to(dt)
    r = torch.randn(rows, cols, generator=gen, device="cuda").to(dt) if residual else None
    keep, t = keep_mask(rows, cols, p, seed, offset, first)
    y = ops.dropout(x, p, seed, offset, residual=r, first_row=first)
    want = torch.where(keep, x.double() * (65536.0 / (65536 - t) if t < 65536 else 0.0), 0.0)
    size = want.abs() + (r.double().abs() if residual else 0)
    if residual:
        want = want + r.double()
    assert y.dtype == dt and y.shape == x.shape
    assert bool(((y.double() - want).abs() <= half_step(dt) * want.abs() * (1 + 1e-6) + 3 * F * size + (2.0 ** -25 if dtype == "f16" else 0)).all())
    if not residual:
        assert bool(((y == 0) | keep).all())
        g = ops.dropout_grad(x, p, seed, offset, first_row=first)
        assert torch.equal(g, y)                                   # the gradient is the same map


def test_dropout_rows_of_ranks_make_one_mask(ops):
    x = torch.randn(96, 77, device="cuda")
    whole = ops.dropout(x, 0.4, 11, 3)
    for rank in range(3):
        assert torch.equal(ops.dropout(x[rank::3], 0.4, 11, 3, first_row=rank, row_step=3), whole[rank::3])
        assert torch.equal(ops.dropout(x[rank * 32:(rank + 1) * 32], 0.4, 11, 3, first_row=rank * 32), whole[rank * 32:(rank + 1) * 32])


def test_dropout_strides_shapes_and_empty(ops):
    base = torch.randn(40, 200, device="cuda").bfloat16()
    for view in (base[:, 3:150], base[::2, 1:], base[:, ::2], base.t(), base.view(4, 10, 200), base[5:6, 7:8], base.view(4, 10, 200).transpose(0, 1)):
        assert torch.equal(ops.dropout(view, 0.3, 5, 6), ops.dropout(view.contiguous(), 0.3, 5, 6))
        assert torch.equal(ops.dropout(view, 0.3, 5, 6, residual=view), ops.dropout(view.contiguous(), 0.3, 5, 6, residual=view.contiguous()))
    for shape in ((0, 5), (5, 0), (0,)):
        assert ops.dropout(torch.empty(shape, device="cuda"), 0.3, 1).shape == shape


def test_dropout_drops_infinities_and_nan_exactly(ops):
    x = torch.full((8, 100), float("inf"), device="cuda")
    x[::2] = float("nan")
    keep, _ = keep_mask(8, 100, 0.5, 1, 2)
    y = ops.dropout(x, 0.5, 1, 2)
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())


def test_dropout_autograd_and_device_offset(ops):
    x = torch.randn(10, 33, device="cuda", requires_grad=True)
    r = torch.randn(10, 33, device="cuda", requires_grad=True)
    off = torch.tensor([41], dtype=torch.int64, device="cuda")
    y = ops.dropout(x, 0.3, 9, off, residual=r)
    assert torch.equal(y, ops.dropout(x.detach(), 0.3, 9, 41, residual=r.detach()))
    off += 1                                                       # the next step's: the backward pass keeps this call's
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(x.grad, ops.dropout_grad(dy, 0.3, 9, 41)) and torch.equal(r.grad, dy)
    xd = torch.randn(4, 9, device="cuda", dtype=torch.float32)
    e = 2.0 ** -10                                                 # a linear map: differences are exact up to rounding
    d = torch.randn_like(xd)
    num = (ops.dropout(xd + e * d, 0.3, 9, 1).double() - ops.dropout(xd - e * d, 0.3, 9, 1).double()) / (2 * e)
    assert float((num - ops.dropout_grad(d, 0.3, 9, 1).double()).abs().max()) <= 8 * F * float(xd.abs().max() + 1) / e * 1.5


def test_dropout_in_a_replayed_graph_draws_new_masks(ops):
    x = torch.randn(64, 130, device="cuda").half()
    off = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.dropout(x, 0.2, 3, off)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.dropout(x, 0.2, 3, off)
        off += 1
    for i in range(4):
        x.copy_(torch.randn(64, 130, device="cuda"))
        want = ops.dropout(x, 0.2, 3, i)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i


# ---------------------------------------------------------------- projection + softmax cross entropy
def reference(x, w, b, t, g, ignore=-100):
    """Everything in float64: per-row loss and entropy, gradients of sum g_i loss_i, and the bounds of the docstring."""
    dt = x.dtype
    f32 = dt == torch.float32
    by_index = t.dtype == torch.int64
    n, h = x.shape
    v = w.shape[0]
    used = (t != ignore) if by_index else torch.ones(n, dtype=torch.bool, device=x.device)
    xd, wd = torch.where(used[:, None], x, torch.zeros_like(x)).double(), w.double()
    bd = torch.zeros(v, dtype=torch.float64, device=x.device) if b is None else b.double()
    l = xd @ wd.t() + bd
    q = torch.zeros_like(l) if by_index else t.double()
    if by_index:
        q[torch.arange(n, device=x.device)[used], t[used]] = 1.0
    lse = torch.logsumexp(l, 1)
    p = torch.softmax(l, 1)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    loss = torch.where(used, lse * q.sum(1) - torch.where(q != 0, q * l, zero).sum(1), zero)
    ent = torch.where(used, lse - torch.where(p > 0, p * l, zero).sum(1), zero)
    gd = torch.where(used, g.double(), zero)
    D = gd[:, None] * (p * q.sum(1, keepdim=True) - q)
    op = 3 * 2.0 ** -22 if f32 else 0.0
    dl = ((h + 2) * F + op) * (xd.abs() @ wd.abs().t()) + F * torch.where(torch.isfinite(l), l.abs(), zero)
    dl = torch.where(torch.isfinite(l), dl, zero)
    dlm = dl.max(1).values
    qs, qa = q.sum(1), q.abs().sum(1)
    fin = torch.where(torch.isfinite(l), l.abs(), zero)
    big = lse.abs() + (q.abs() * fin).sum(1) / qa.clamp_min(1e-30) + 2
    b_loss = torch.where(used, qa * (2 * dlm + (8 + math.log2(v) + 40) * F * big), zero)
    b_ent = torch.where(used, 2 * dlm * (1 + (p * fin).sum(1)) + 2.0 ** -19 * ((p * fin).sum(1) + lse.abs() + 1), zero)
    rel_p = 2 * dlm[:, None] + 2.0 ** -20
    uD = 2.0 ** -22 if f32 else half_step(dt)
    top = float((gd.abs() * qa).max()) * 2                          # the images' scale
    if not f32:
        rel_p = rel_p + 2.0 ** -11
    kept = 0.0 if f32 else 2.0 ** -25 * p.max(1, keepdim=True).values
    bD0 = gd.abs()[:, None] * ((p * rel_p + kept) * qs.abs()[:, None] + 4 * F * (p * qs.abs()[:, None] + q.abs()))
    bD = bD0 + uD * D.abs() + (2.0 ** -39 * top if dt != torch.bfloat16 else 0)
    out_abs = 2.0 ** -25 if dt == torch.float16 else 0.0
    u = half_step(dt)

    def product(a, ba, c, k):
        r = a @ c
        mag = a.abs() @ c.abs()
        e = ba @ c.abs() + ((k + 40) * F + (3 * 2.0 ** -22 if f32 else 0)) * mag
        return r, e * (1 + 2 * u) + u * r.abs() * (1 + 1e-6) + out_abs
    dx, b_dx = product(D, bD, wd, v)
    dw, b_dw = product(D.t(), bD.t(), xd, n)
    db = D.sum(0)
    b_db = (bD0.sum(0) + (n + 40) * F * D.abs().sum(0)) * (1 + 2 * u) + u * db.abs() * (1 + 1e-6) + out_abs
    return dict(loss=(loss, b_loss), ent=(ent, b_ent), dx=(dx, b_dx), dw=(dw, b_dw), db=(db, b_db), count=int(used.sum()))


def close(name, got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g times its bound (%.3g of %.3g)" % (
        name, int(bad.sum()), bad.numel(), float((err / bound.clamp_min(1e-300)).max()), float(err.max()), float(want.abs().max()))


def make(n, h, v, dtype, kind="index", bias=True, ignored=0.0, seed=1, spread=2.0):
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = DT[dtype]
    x = torch.randn(n, h, generator=gen, device="cuda").to(dt)
    w = (torch.randn(v, h, generator=gen, device="cuda") * spread / math.sqrt(h)).to(dt)
    b = torch.randn(v, generator=gen, device="cuda").to(dt) if bias else None
    if kind == "index":
        t = torch.randint(0, v, (n,), generator=gen, device="cuda")
        if ignored:
            t[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    else:
        t = torch.rand(n, v, generator=gen, device="cuda") ** 4
        t = torch.where(t > 0.2, t, torch.zeros_like(t))
        t[:, 0] += 1e-2
        t = t / t.sum(1, keepdim=True)
    return x, w, b, t


def check_all(ops, x, w, b, t, ignore=-100, scale=1.0):
    n = x.shape[0]
    by_index = t.dtype == torch.int64
    count = int((t != ignore).sum()) if by_index else n
    g = torch.full((n,), scale / max(count, 1), device="cuda")
    ref = reference(x, w, b, t, g, ignore)
    close("loss rows", *((ops.linear_cross_entropy(x, w, t, b, reduction="none", ignore_index=ignore),) + ref["loss"]))
    r = ops.linear_cross_entropy_grad(x, w, t, b, ignore_index=ignore, grad_loss=scale, return_entropy=True)
    c = max(count, 1)
    close("loss", r.loss, ref["loss"][0].sum() / c, ref["loss"][1].sum() / c + F * ref["loss"][0].sum().abs() / c)
    close("entropy", r.entropy, ref["ent"][0].sum() / c, ref["ent"][1].sum() / c + F * ref["ent"][0].sum().abs() / c)
    close("d_hidden", r.d_hidden, *ref["dx"])
    close("d_weight", r.d_weight, *ref["dw"])
    if b is not None:
        close("d_bias", r.d_bias, *ref["db"])
    return r


SIZES = [(1, 1, 1), (1, 64, 64), (2, 8, 3), (7, 40, 65), (16, 64, 129), (17, 72, 300), (33, 100, 257), (64, 256, 64), (100, 900, 225),
         (130, 520, 1000), (257, 33, 513), (300, 128, 2050)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", SIZES)
def test_cross_entropy_index(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.3 if n > 8 else 0.0, seed=n + h + v)
    check_all(ops, x, w, b, t, scale=1024.0 if dtype == "f16" else 1.0)
    check_all(ops, x, w, None, t, scale=1024.0 if dtype == "f16" else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", [(1, 1, 1), (2, 8, 3), (17, 72, 300), (64, 256, 64), (100, 900, 225), (257, 33, 513)])
def test_cross_entropy_probabilities(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "probs", seed=n + h + v)
    check_all(ops, x, w, b, t, scale=1024.0 if dtype == "f16" else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", [(1024, 512, 4096), (2100, 200, 6000), (1, 4096, 20011), (40, 2048, 33000)])
def test_cross_entropy_larger(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.1 if n > 8 else 0.0, seed=5)
    check_all(ops, x, w, b, t, scale=1024.0 if dtype == "f16" else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,n,h,v", [("index", 7, 40, 4100), ("index", 33, 100, 5003), ("index", 130, 520, 4097), ("index", 300, 33, 9001),
                                        ("index", 2100, 1030, 7001), ("index", 65, 64, 70001), ("probs", 64, 72, 4100), ("probs", 257, 33, 6001),
                                        ("probs", 1, 1, 5000), ("probs", 700, 256, 4352)])
def test_cross_entropy_many_classes(ops, dtype, kind, n, h, v):
    x, w, b, t = make(n, h, v, dtype, kind, ignored=0.3 if n > 8 and kind == "index" else 0.0, seed=n + h + v)
    check_all(ops, x, w, b, t, scale=1024.0 if dtype == "f16" else 1.0)


# two lists of sizes for what does not depend on a size: one that the path for small problems takes, one that it does not
PATHS = [(37, 100, 65), (37, 100, 4501)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", PATHS + [(5000, 24, 150)])
@pytest.mark.parametrize("kind", ["index", "probs"])
def test_cross_entropy_rows_with_their_own_gradient(ops, dtype, n, h, v, kind):
    x, w, b, t = make(n, h, v, dtype, kind, ignored=0.2 if kind == "index" else 0.0)
    if kind == "probs":
        t = t * torch.linspace(0.0, 3.0, n, device="cuda")[:, None]             # any real weights, a row of zeros among them
        t[1, ::7] *= -1.0
    g = torch.linspace(-1.0, 2.0, n, device="cuda") * (256.0 if dtype == "f16" else 1.0)
    g[3] = 0.0
    ref = reference(x, w, b, t, g)
    r = ops.linear_cross_entropy_grad(x, w, t, b, reduction="none", grad_loss=g, return_entropy=True)
    close("loss", r.loss, *ref["loss"])
    close("entropy", r.entropy, *ref["ent"])
    close("d_hidden", r.d_hidden, *ref["dx"])
    close("d_weight", r.d_weight, *ref["dw"])
    close("d_bias", r.d_bias, *ref["db"])
    s = ops.linear_cross_entropy(x, w, t, b, reduction="sum")
    close("sum", s, ref["loss"][0].sum(), ref["loss"][1].sum() + F * ref["loss"][0].sum().abs())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", PATHS + [(1500, 300, 6000), (1100, 64, 300), (40, 33, 1500)])
def test_cross_entropy_autograd(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.2)
    leaves = [q.clone().requires_grad_() for q in (x, w, b)]
    scale = 3.0
    loss, ent = ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], return_entropy=True)
    assert not ent.requires_grad
    (loss * scale).backward()
    count = int((t != -100).sum())
    ref = reference(x, w, b, t, torch.full((n,), scale / count, device="cuda"))
    for name, leaf, key in (("d_hidden", leaves[0], "dx"), ("d_weight", leaves[1], "dw"), ("d_bias", leaves[2], "db")):
        close(name, leaf.grad, *ref[key])
    only = w.clone().requires_grad_()                              # one gradient alone, no bias
    ops.linear_cross_entropy(x, only, t, reduction="sum").backward()
    close("d_weight alone", only.grad, *reference(x, w, None, t, torch.ones(n, device="cuda"))["dw"])


@pytest.mark.parametrize("n,h,v", PATHS)
def test_cross_entropy_gradient_against_differences(ops, n, h, v):
    """Central differences: off by e^2 / 6 times the third derivative along the direction -- at most R^3 a row, R the range of
    the logits' change -- and by the losses' own bounds over e."""
    x, w, b, t = make(n, h, v, "f32", "index", ignored=0.2, spread=1.0)
    r = ops.linear_cross_entropy_grad(x, w, t, b, reduction="sum")
    ref = reference(x, w, b, t, torch.ones(n, device="cuda"))
    used = t != -100
    e = 2.0 ** -6
    dx, dw, db = torch.randn_like(x) / math.sqrt(h), torch.randn_like(w) / math.sqrt(h), torch.randn_like(b)
    for d in ((dx, 0 * dw, 0 * db), (0 * dx, dw, 0 * db), (0 * dx, 0 * dw, db)):
        f = [ops.linear_cross_entropy(x + s * e * d[0], w + s * e * d[1], t, b + s * e * d[2], reduction="sum").double() for s in (1, -1)]
        want = sum(float((g.double() * q.double()).sum()) for g, q in zip((r.d_hidden, r.d_weight, r.d_bias), d))
        u = d[0].double() @ w.double().t() + x.double() @ d[1].double().t() + d[2].double()
        big = (u.max(1).values - u.min(1).values)[used]
        # (x + e d is itself rounded: 2^-24 of every operand, on both sides)
        slack = e * e / 6 * float((big ** 3).sum()) * 1.1 + (float(ref["loss"][1].sum()) * 2 + 4 * F * float(ref["loss"][0].sum())) / e
        slack += 4 * F * float(((x.double().abs() @ w.double().abs().t()) + b.double().abs()).max(1).values.sum()) / e
        slack += sum(float((bd * q.double().abs()).sum()) for bd, q in zip((ref["dx"][1], ref["dw"][1], ref["db"][1]), d))
        assert abs(float((f[0] - f[1]) / (2 * e)) - want) <= slack


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,v", PATHS)
def test_cross_entropy_ignored_rows_may_hold_anything(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.3)
    t[2], t[9] = -100, -100
    clean = x.clone()
    clean[t == -100] = 0
    dirty = x.clone()
    dirty[2], dirty[9] = float("nan"), float("inf")
    dirty[t == -100, ::3] = torch.finfo(DT[dtype]).max
    a = ops.linear_cross_entropy_grad(clean, w, t, b, return_entropy=True)
    c = ops.linear_cross_entropy_grad(dirty, w, t, b, return_entropy=True)
    for p, q in zip(a, c):
        assert torch.equal(p, q)
    leaf = dirty.clone().requires_grad_()
    wl = w.clone().requires_grad_()
    ops.linear_cross_entropy(leaf, wl, t, b).backward()
    assert bool(torch.isfinite(wl.grad).all()) and not bool(leaf.grad[t == -100].any())
    # every row ignored; an ignore_index that is a class
    t[:] = -100
    r = ops.linear_cross_entropy_grad(dirty, w, t, b, return_entropy=True)
    assert float(r.loss) == 0 and float(r.entropy) == 0 and not any(bool(q.any()) for q in r[2:])
    t = torch.randint(0, 3, (n,), device="cuda")
    check_all(ops, x, w, b, t, ignore=1)


@pytest.mark.parametrize("n,h,v", PATHS)
def test_cross_entropy_blocked_classes_and_bad_targets(ops, n, h, v):
    x, w, b, t = make(n, h, v, "f32", "index")
    b[::3] = float("-inf")                                          # classes nobody may take
    t = t // 3 * 3 + 1
    t.clamp_(max=v - 1 - (v - 1) % 3 - 1)
    check_all(ops, x, w, b, t)
    b[::3] = torch.finfo(torch.float32).min
    check_all(ops, x, w, b, t)
    t[4] = 0                                                        # a blocked target: no finite loss
    b[::3] = float("-inf")
    assert float(ops.linear_cross_entropy(x, w, t, b, reduction="none")[4]) == float("inf")
    every = ops.linear_cross_entropy(x, w, t, torch.full_like(b, float("-inf")), reduction="none")
    assert not bool(torch.isfinite(every).any())
    good = ops.linear_cross_entropy(x, w, t, reduction="none")
    for bad in (v, -1, 1 << 40, -(1 << 62)):
        u = t.clone()
        u[5] = bad
        r = ops.linear_cross_entropy(x, w, u, reduction="none")
        assert math.isnan(float(r[5]))
        r[5] = good[5]
        assert torch.equal(r, good)
        g = ops.linear_cross_entropy_grad(x, w, u, reduction="none")
        assert bool(torch.isnan(g.d_hidden[5]).all()) and bool(torch.isfinite(g.d_hidden[:5]).all())
        assert bool(torch.isnan(g.d_weight).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", PATHS + [(40, 128, 4608)])
def test_cross_entropy_strides_and_alignments(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.2)
    want = ops.linear_cross_entropy_grad(x, w, t, b)

    def inside(q, pad, at):                                         # q as a view of a larger tensor
        big = torch.full((q.shape[0] + 2, q.shape[1] + pad), float("nan"), dtype=q.dtype, device="cuda")
        big[1:-1, at:at + q.shape[1]] = q
        return big[1:-1, at:at + q.shape[1]]
    for pad, at in ((1, 1), (3, 0), (8, 8), (64, 24)):
        for xv, wv in ((inside(x, pad, at), w), (x, inside(w, pad, at)), (inside(x, pad, at), inside(w, pad, at)),
                       (x.t().contiguous().t(), w.t().contiguous().t())):
            got = ops.linear_cross_entropy_grad(xv, wv, t, b)
            for p, q in zip(want, got):
                assert p is None and q is None or torch.equal(p, q)
    both = torch.stack([t, t], 1)
    assert torch.equal(ops.linear_cross_entropy(x, w, both[:, 1], torch.stack([b, b], 1)[:, 0]), ops.linear_cross_entropy(x, w, t, b))
    p = torch.rand(n, v + 3, device="cuda")
    assert torch.equal(ops.linear_cross_entropy(x, w, p[:, 2:v + 2], b), ops.linear_cross_entropy(x, w, p[:, 2:v + 2].contiguous(), b))
    cube = ops.linear_cross_entropy(x[:36].view(4, 9, h), w, t[:36].view(4, 9), b, reduction="none")
    assert cube.shape == (4, 9) and torch.equal(cube.view(-1), ops.linear_cross_entropy(x[:36], w, t[:36], b, reduction="none"))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cross_entropy_empty_batch(ops, dtype):
    w, b = torch.randn(70, 24, device="cuda").to(DT[dtype]), torch.randn(70, device="cuda").to(DT[dtype])
    x, t = torch.empty(0, 24, dtype=DT[dtype], device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    r = ops.linear_cross_entropy_grad(x, w, t, b, return_entropy=True)
    assert float(r.loss) == 0 and float(r.entropy) == 0 and r.d_hidden.shape == (0, 24)
    assert not bool(r.d_weight.any()) and not bool(r.d_bias.any())
    assert ops.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    wl, xl = w.clone().requires_grad_(), x.clone().requires_grad_()
    ops.linear_cross_entropy(xl, wl, t).backward()
    assert not bool(wl.grad.any()) and xl.grad.shape == (0, 24)


@pytest.mark.parametrize("dtype,n,h,v", [("bf16", 70000, 24, 8200), ("f32", 36000, 17, 8200)])
def test_cross_entropy_in_pieces_of_the_classes(ops, dtype, n, h, v):
    """More than a gigabyte of images: the classes are cut and their products made twice."""
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.1)
    check_all(ops, x, w, b, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", [(40, 64, 4096), (40, 64, 4097), (1024, 24, 4096), (1025, 24, 4096), (512, 256, 1024), (513, 256, 1024), (40000, 3, 100),
                                   (1024, 40, 300), (1025, 40, 300), (256, 128, 1024), (257, 128, 1024), (256, 128, 1025), (20000, 48, 60)])
def test_cross_entropy_around_the_ends_of_the_small_path(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.2, seed=n + h + v)
    check_all(ops, x, w, b, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,n,h,v", [("index", 1, 77, 5000), ("index", 32, 900, 4097), ("probs", 17, 33, 6001), ("probs", 1, 1, 5001), ("index", 4, 1892, 50047),
                                        ("index", 31, 2049, 20000)])
def test_cross_entropy_scores_of_few_rows(ops, dtype, kind, n, h, v):
    """Few rows of odd lengths against many classes, alone and before a backward pass by itself."""
    x, w, b, t = make(n, h, v, dtype, kind, ignored=0.2 if kind == "index" and n > 8 else 0.0, seed=n + h + v)
    if kind == "index":
        t[0] = v - 1
    ref = reference(x, w, b, t, torch.ones(n, device="cuda"))
    for bias in (b, None):
        if bias is None:
            ref = reference(x, w, None, t, torch.ones(n, device="cuda"))
        loss, ent = ops.linear_cross_entropy(x, w, t, bias, reduction="none", return_entropy=True)
        close("loss", loss, *ref["loss"])
        close("entropy", ent, *ref["ent"])
    leaves = [q.clone().requires_grad_() for q in (x, w)]
    ops.linear_cross_entropy(leaves[0], leaves[1], t, reduction="sum").backward()
    for leaf, key in zip(leaves, ("dx", "dw")):
        close(key, leaf.grad, *ref[key])
    with torch.no_grad():
        blocked = torch.zeros(v, device="cuda").to(x.dtype)
        blocked[1:v - 1] = float("-inf")                            # spans of which nothing is left
        tb = torch.zeros(n, dtype=torch.int64, device="cuda")
        close("blocked", ops.linear_cross_entropy(x, w, tb, blocked, reduction="none"), *reference(x, w, blocked, tb, torch.ones(n, device="cuda"))["loss"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind,n,h,v", [("index", 1000, 40, 16717), ("probs", 300, 33, 33029), ("index", 256, 64, 65537), ("index", 2048, 72, 8300), ("probs", 1030, 8, 14000)])
def test_cross_entropy_scores_of_mixed_tiles(ops, dtype, kind, n, h, v):
    """More tiles than one round of the compute units, and a few: large and small ones in one launch.  Then a backward pass by itself."""
    x, w, b, t = make(n, h, v, dtype, kind, ignored=0.2 if kind == "index" else 0.0, seed=n + h + v)
    ref = reference(x, w, b, t, torch.full((n,), 0.5, device="cuda"))
    loss, ent = ops.linear_cross_entropy(x, w, t, b, reduction="none", return_entropy=True)
    close("loss", loss, *ref["loss"])
    close("entropy", ent, *ref["ent"])
    leaves = [q.clone().requires_grad_() for q in (x, w, b)]
    (0.5 * ops.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="sum")).backward()
    for leaf, key in zip(leaves, ("dx", "dw", "db")):
        close(key, leaf.grad, *ref[key])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", [(128, 16392, 128), (60, 40001, 64), (1, 1 << 20, 129)])
def test_cross_entropy_of_very_many_features(ops, dtype, n, h, v):
    x, w, b, t = make(n, h, v, dtype, "index", seed=n + h + v)
    check_all(ops, x, w, b, t)


@pytest.mark.parametrize("dtype,n", [("bf16", 4300000), ("f32", 300001)])
def test_cross_entropy_of_very_many_rows(ops, dtype, n):
    x, w, b, t = make(n, 8, 5, dtype, "index", ignored=0.2)
    check_all(ops, x, w, b, t)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", PATHS)
def test_cross_entropy_of_single_rows_with_any_stride(ops, dtype, n, h, v):
    """One row (or one class) of a matrix whose row stride says nothing; rows further apart than the kernels take."""
    x, w, b, t = make(n, h, v, dtype, "index")
    far = torch.empty(2, 5 << 20, dtype=x.dtype, device="cuda")
    far[:, :h] = x[:2]
    want = ops.linear_cross_entropy_grad(x[:2], w, t[:2], b)
    got = ops.linear_cross_entropy_grad(far[:, :h], w, t[:2], b)
    assert all(torch.equal(p, q) for p, q in zip(want, got) if p is not None)
    want = ops.linear_cross_entropy_grad(x[:1], w, t[:1], b)
    got = ops.linear_cross_entropy_grad(far[:1, :h], w, t[:1], b)
    assert all(torch.equal(p, q) for p, q in zip(want, got) if p is not None)
    far[0, :h] = w[0]
    t1 = torch.zeros_like(t)
    want, got = ops.linear_cross_entropy_grad(x, w[:1], t1), ops.linear_cross_entropy_grad(x, far[:1, :h], t1)
    assert torch.equal(want.loss, got.loss) and torch.equal(want.d_weight, got.d_weight)
    assert torch.equal(ops.dropout(far[:1, :h], 0.5, 1), ops.dropout(w[:1], 0.5, 1))


def test_cross_entropy_weights_beyond_32_bits(ops):
    n, h, v = 5, 16384, 140001                                      # 4.6 GB of weights
    w = torch.empty(v, h, dtype=torch.bfloat16, device="cuda")
    for q in w.split(8192):
        q.copy_(torch.randn(q.shape, device="cuda") / 128)
    x = torch.randn(n, h, device="cuda").bfloat16()
    t = torch.tensor([v - 1, 0, 131072, v - 2, 7], device="cuda")
    l = torch.cat([x.double() @ q.double().t() for q in w.split(8192)], 1)
    mag = torch.cat([x.double().abs() @ q.double().abs().t() for q in w.split(8192)], 1)
    dl = ((h + 2) * F * mag + F * l.abs()).max(1).values
    want = torch.logsumexp(l, 1) - l.gather(1, t[:, None])[:, 0]
    r = ops.linear_cross_entropy_grad(x, w, t, reduction="sum")
    err = (ops.linear_cross_entropy(x, w, t, reduction="none").double() - want).abs()
    assert bool((err <= 2 * dl + 80 * F * (want.abs() + l.abs().max(1).values + 2)).all())
    p = torch.softmax(l, 1)
    d = p.clone()
    d[torch.arange(n), t] -= 1
    for c in (0, 7, 131071, 131072, 131073, v - 2, v - 1):
        got, ref = r.d_weight[c].double(), d[:, c] @ x.double()
        rel = 2 * dl[:, None] + 2.0 ** -20 + 2.0 ** -11 + 2.0 ** -8
        bound = ((p * rel).max() + d[:, c].abs() @ (torch.full((n, 1), 2.0 ** -8, device="cuda", dtype=torch.float64) * x.double().abs())
                 + (p[:, c, None] * rel).t() @ x.double().abs())
        assert bool(((got - ref).abs() <= bound + 2.0 ** -8 * ref.abs() + 50 * F * (d[:, c].abs() @ x.double().abs())).all()), c


def test_dropout_beyond_32_bits_of_elements(ops):
    n = (1 << 32) + 12345
    x = torch.ones(1, n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.25, 77, 5, residual=x)
    for at in (0, (1 << 31) - 50, (1 << 32) - 50, n - 100):
        keep = torch.from_numpy(philox(at, 100, 77, 5) >= 16384).cuda()
        assert torch.equal(y[0, at:at + 100], torch.where(keep, 1 + 65536 / 49152, 1.0).bfloat16()), at
    del y
    assert 0.7499 < float(ops.dropout(x, 0.25, 77, 6).gt(0).sum(dtype=torch.int64)) / n < 0.7501


# ---------------------------------------------------------------- streams, graphs, threads, a whole step
@pytest.mark.parametrize("n,h,v", PATHS + [(600, 256, 5000)])
def test_cross_entropy_repeats_its_bits_on_any_stream_and_in_threads(ops, n, h, v):
    import threading
    x, w, b, t = make(n, h, v, "bf16", "index", ignored=0.2)
    want = ops.linear_cross_entropy_grad(x, w, t, b, return_entropy=True)
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                got = ops.linear_cross_entropy_grad(x, w, t, b, return_entropy=True)
                s.synchronize()
                bad.extend(1 for p, q in zip(want, got) if not torch.equal(p, q))
    work()
    threads = [threading.Thread(target=work) for _ in range(3)]
    for q in threads:
        q.start()
    for q in threads:
        q.join()
    assert not bad


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,v", PATHS + [(2100, 200, 6000)])
def test_training_head_in_replayed_graphs(ops, dtype, n, h, v):
    """features -> dropout -> projection's loss and gradients -> dropout's gradient, captured twice, replayed in turn with
    other inputs and eager work between: every replay gives the eager results' bits."""
    x, w, b, t = make(n, h, v, dtype, "index", ignored=0.2)
    off = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step(offset):
        y = ops.dropout(x, 0.3, 9, offset)
        r = ops.linear_cross_entropy_grad(y, w, t, b, return_entropy=True)
        return [r.loss, r.entropy, ops.dropout_grad(r.d_hidden, 0.3, 9, offset), r.d_weight, r.d_bias]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(off)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(off)
        graphs.append((g, out))
    for i in range(6):
        x.copy_(torch.randn(n, h, device="cuda"))
        t.copy_(torch.where(torch.rand(n, device="cuda") < 0.3, -100, torch.randint(0, v, (n,), device="cuda")))
        off.fill_(i)
        want = step(i)
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        for o in out:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        for p, q in zip(want, out):
            assert torch.equal(p, q), i


def test_autograd_forms_refuse_to_be_captured(ops):
    x, w, b, t = make(8, 16, 9, "f32")
    xl = x.clone().requires_grad_()
    eager = ops.linear_cross_entropy(ops.dropout(xl, 0.2, 1), w, t, b)           # (a live eager graph of the same leaf)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.graph(g):
        for call in (lambda: ops.linear_cross_entropy(xl, w, t, b), lambda: ops.dropout(xl, 0.2, 1), lambda: ops.dropout(x, 0.2, 1, residual=xl)):
            try:
                call()
            except RuntimeError as err:
                refused.append(str(err))
        with torch.no_grad():
            out = ops.linear_cross_entropy(xl, w, t, b)
    assert len(refused) == 3 and all("captured" in r for r in refused)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.linear_cross_entropy(x, w, t, b))
    eager.backward()
    assert bool(torch.isfinite(xl.grad).all())


@pytest.mark.parametrize("n,h,v", PATHS)
def test_head_step_against_autograd_of_its_definition(ops, n, h, v):
    """The run of the operators against float64 autograd of the formulas under the same mask."""
    x, w, b, t = make(n, h, v, "f32", "probs")
    res = torch.randn_like(x)
    leaves = [q.clone().requires_grad_() for q in (x, res, w, b)]
    y = ops.dropout(leaves[0], 0.4, 123, 7, residual=leaves[1], first_row=11)
    loss = ops.linear_cross_entropy(y, leaves[2], t, leaves[3])
    loss.backward()
    keep, thr = keep_mask(n, h, 0.4, 123, 7, 11)
    d = [q.double().requires_grad_() for q in (x, res, w, b)]
    yd = d[1] + torch.where(keep, d[0] * (65536.0 / (65536 - thr)), 0.0)
    logits = yd @ d[2].t() + d[3]
    ld = -(t.double() * torch.log_softmax(logits, 1)).sum(1).mean()
    ld.backward()
    ref = reference(yd.detach().float(), w, b, t, torch.full((n,), 1.0 / n, device="cuda"))
    scale = 65536.0 / (65536 - thr)
    # (y is rounded once in float32: 2 * 2^-24 of it, another input error of that size in every bound)
    near = 4 * F * float((yd.detach().abs() @ w.double().abs().t()).max())
    for name, leaf, exact, key, k in (("x", leaves[0], d[0], "dx", scale), ("residual", leaves[1], d[1], "dx", 1.0), ("w", leaves[2], d[2], "dw", 1.0),
                                      ("b", leaves[3], d[3], "db", 1.0)):
        bound = ref[key][1] * k + 2 * near * float(exact.grad.abs().max()) + 4 * F * exact.grad.abs()
        assert bool(((leaf.grad.double() - exact.grad).abs() <= bound).all()), name
    assert abs(float(loss.detach()) - float(ld.detach())) <= float(ref["loss"][1].mean()) + 2 * near + 4 * F * float(ld.detach())


def test_refusals(ops):
    x, w, b, t = make(8, 16, 9, "f32")
    p = torch.rand(8, 9, device="cuda")
    ce, grad, drop = ops.linear_cross_entropy, ops.linear_cross_entropy_grad, ops.dropout
    for call, what in ((lambda: ce(x.cpu(), w, t), "CUDA"), (lambda: ce(x, w.cpu(), t), "CUDA"), (lambda: ce(x, w, t.cpu()), "CUDA"),
                       (lambda: ce(x.double(), w, t), "float32"), (lambda: ce(x, w.half(), t), "float32"), (lambda: ce(x, w, t, b.bfloat16()), "float32"),
                       (lambda: ce(x, w[:, :5], t), "features"), (lambda: ce(x, w, t[:5]), "shape"), (lambda: ce(x, w, t.int()), "int64"),
                       (lambda: ce(x, w, p.half()), "float32"), (lambda: ce(x, w, p[:, :5]), "classes"), (lambda: ce(x, w, t, b[:5]), "classes"),
                       (lambda: ce(x, w, t, reduction="max"), "reduction"), (lambda: ce(x, w, t, ignore_index=1.5), "ignore_index"),
                       (lambda: ce(x, w, t, ignore_index=1 << 63), "ignore_index"), (lambda: ce(x, w[:0], t), "class"),
                       (lambda: ce(x, w, p.clone().requires_grad_()), "gradient"), (lambda: grad(x, w, t, grad_loss=torch.ones(8, device="cuda")), "shape"),
                       (lambda: grad(x, w, t, grad_loss=torch.ones((), device="cuda").half()), "float32"), (lambda: ce(x[0, 0], w, t), "features"),
                       (lambda: drop(x.cpu(), 0.1, 1), "CUDA"), (lambda: drop(x.double(), 0.1, 1), "float32"), (lambda: drop(x, 1.1, 1), "p must"),
                       (lambda: drop(x, -0.1, 1), "p must"), (lambda: drop(x, float("nan"), 1), "p must"), (lambda: drop(x, 0.1, -1), "seed"),
                       (lambda: drop(x, 0.1, 1 << 64), "seed"), (lambda: drop(x, 0.1, 1, -1), "offset"), (lambda: drop(x, 0.1, 1, residual=x[:4]), "shape"),
                       (lambda: drop(x, 0.1, 1, residual=x.half()), "residual"), (lambda: drop(x, 0.1, 1, torch.zeros(2, dtype=torch.int64, device="cuda")), "offset"),
                       (lambda: drop(x, 0.1, 1, torch.zeros(1, device="cuda")), "offset"), (lambda: drop(x[0, 0], 0.1, 1), "dimension"),
                       (lambda: drop(x, 0.1, 1, first_row=-1), "first_row")):
        with pytest.raises((ValueError, TypeError), match=what):
            call()
    with pytest.raises(TypeError):
        ce([1.0], w, t)
