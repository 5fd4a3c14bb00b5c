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
