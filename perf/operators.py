"""Cases, inputs and plain forms of the training-head operators: counter-based dropout and the softmax
cross entropy of a projection.  `own` selects whether run() calls the framework's operators or their plain
forms."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100


# ---------------------------------------------------------------- cases
def _drop(name, rows, cols, dtype, mode, p, first_row=0):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "mode": mode, "p": p, "first_row": first_row}


def _ce(name, n, hidden, classes, dtype, target, grad, bias=True, ignored=0.0, entropy=False):
    return {"name": name, "op": "cross_entropy", "n": n, "hidden": hidden, "classes": classes, "dtype": dtype, "target": target,
            "grad": grad, "bias": bias, "ignored": ignored, "entropy": entropy}


def listed():
    return [
        # the policy head's features of a mini-batch of 512 positions on 8x8 (4 channels x 64 cells): latency
        _drop("dropout_head_8x8", 512, 256, "f32", "forward", 0.3),
        # the gradient at the same features on 15x15
        _drop("dropout_head_15x15_grad", 512, 900, "f32", "backward", 0.3),
        # rows of an odd length, the shard of a data-parallel batch whose element numbers lie beyond 32 bits
        _drop("dropout_odd_shard", 4099, 1111, "f16", "forward", 0.1, first_row=4500001),
        # a block's output added to its residual stream: bandwidth
        _drop("dropout_residual", 16384, 4096, "bf16", "residual", 0.1),
        # the policy heads' loss, entropy and gradients against visit distributions, 512 positions on 8x8 and 15x15
        _ce("policy_8x8", 512, 256, 64, "f32", "probs", True, entropy=True),
        _ce("policy_15x15", 512, 900, 225, "f32", "probs", True, entropy=True),
        # the loss of one row over a large set of classes: reads the weights once
        _ce("score_one_row", 1, 4096, 65536, "bf16", "index", False, bias=False),
        # the loss of a held-out batch, odd number of classes
        _ce("score_batch", 2048, 1024, 50001, "f16", "index", False),
        # odd sizes throughout, a third of the rows padded
        _ce("train_odd", 777, 513, 4099, "bf16", "index", True, ignored=0.33),
        # ordinary training steps over a large set of classes, in float32 and in bfloat16
        _ce("train_f32", 2048, 1024, 32000, "f32", "index", True),
        _ce("train_bf16", 4096, 2048, 32000, "bf16", "index", True, bias=False, ignored=0.1),
        # the largest
        _ce("train_large", 8192, 4096, 65536, "bf16", "index", True, bias=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.4:
        mode = rng.choice(["forward", "residual", "backward"])
        cols = _log_int(rng, 8, 16384)
        rows = _log_int(rng, 1, min(1 << 17, (16384 * 4096) // (cols * (2 if dtype == "f32" else 1))))
        first = rng.choice([0, rng.randrange(1, 1 << 24)])
        return _drop("", rows, cols, dtype, mode, round(rng.uniform(0.02, 0.6), 3), first)
    n, hidden, classes = _log_int(rng, 1, 8192), _log_int(rng, 16, 4096), _log_int(rng, 32, 65536)
    target = "probs" if classes <= 4096 and rng.random() < 0.5 else "index"
    return _ce("", n, hidden, classes, dtype, target, rng.random() < 0.7, bias=rng.random() < 0.5,
               ignored=rng.choice([0.0, 0.25]) if target == "index" and n > 8 else 0.0, entropy=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        st = {"case": case, "seed": seed * 0x9E3779B97F4A7C15 % (1 << 64), "offset": (1 << 33) + seed,
              "x": randn(rows, cols).to(dt), "residual": None}
        if case["mode"] == "residual":
            st["residual"] = randn(rows, cols).to(dt)
        return st
    n, hidden, classes = case["n"], case["hidden"], case["classes"]
    # normalised features; weights that spread the logits by about two
    st = {"case": case, "hidden": randn(n, hidden).to(dt), "weight": (randn(classes, hidden) * (2.0 / math.sqrt(hidden))).to(dt),
          "bias": randn(classes).to(dt) if case["bias"] else None,
          # half-precision training scales its loss so that gradients stay above the type's smallest number
          "grad_loss": 1024.0 if case["dtype"] == "f16" else 1.0}
    if case["target"] == "index":
        target = torch.randint(0, classes, (n,), generator=gen, device="cuda")
        if case["ignored"]:
            target[torch.rand(n, generator=gen, device="cuda") < case["ignored"]] = IGNORE
            target[0] = 0                                         # one row at least counts
        st["target"] = target
    else:                                                         # visit shares: most classes unvisited
        w = torch.rand((n, classes), generator=gen, device="cuda")
        w = torch.where(w > 0.7, (w - 0.7) ** 3, torch.zeros((), device="cuda"))
        w[:, 0] += 1e-3
        st["target"] = w / w.sum(1, keepdim=True)
    return st


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    return _own_ce(state) if own else _plain_ce(state)


def _own_dropout(st):
    from alphazero_gomoku_amd import ops
    c = st["case"]
    if c["mode"] == "backward":
        return ops.dropout_grad(st["x"], c["p"], st["seed"], st["offset"], first_row=c["first_row"])
    return ops.dropout(st["x"], c["p"], st["seed"], st["offset"], residual=st["residual"], first_row=c["first_row"])


def _own_ce(st):
    from alphazero_gomoku_amd import ops
    c = st["case"]
    if not c["grad"]:
        r = ops.linear_cross_entropy(st["hidden"], st["weight"], st["target"], st["bias"], reduction="none", ignore_index=IGNORE,
                                     return_entropy=c["entropy"])
        return {"loss": r[0], "entropy": r[1]} if c["entropy"] else {"loss": r}
    g = ops.linear_cross_entropy_grad(st["hidden"], st["weight"], st["target"], st["bias"], reduction="mean", ignore_index=IGNORE,
                                      grad_loss=st["grad_loss"], return_entropy=c["entropy"])
    out = {"loss": g.loss, "d_hidden": g.d_hidden, "d_weight": g.d_weight}
    if c["bias"]:
        out["d_bias"] = g.d_bias
    if c["entropy"]:
        out["entropy"] = g.entropy
    return out


# ---------------------------------------------------------------- plain forms
def _mul_32x32(a, m):
    """(high, low) 32 bits of a * m for an int64 tensor a of 32-bit values and a 32-bit constant m."""
    lo = a * (m & 0xFFFF)                                         # < 2^48
    hi = a * (m >> 16) + (lo >> 16)
    return (hi >> 16) & 0xFFFFFFFF, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def _plain_keep(rows, cols, first_row, p, seed, offset):
    """keep [rows, cols]: Philox4x32-10 on the element number's block of eight, 16 bits an element."""
    first = first_row * cols
    b0 = first // 8
    blocks = torch.arange(b0, (first + rows * cols + 7) // 8, dtype=torch.int64, device="cuda")
    c0, c1 = blocks & 0xFFFFFFFF, blocks >> 32
    c2 = torch.full_like(c0, offset & 0xFFFFFFFF)
    c3 = torch.full_like(c0, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _mul_32x32(c0, 0xD2511F53)
        h1, l1 = _mul_32x32(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], dim=1)
    half = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)
    u = half[first - 8 * b0: first - 8 * b0 + rows * cols].reshape(rows, cols)
    return u >= int(round(p * 65536))


def _plain_dropout(st):
    c, x = st["case"], st["x"]
    keep = _plain_keep(c["rows"], c["cols"], c["first_row"], c["p"], st["seed"], st["offset"])
    scale = 65536.0 / (65536 - int(round(c["p"] * 65536)))
    y = torch.where(keep, x.float() * scale, torch.zeros((), device="cuda"))
    if st["residual"] is not None:
        y = st["residual"].float() + y
    return y.to(x.dtype)


def _plain_ce(st):
    c, target = st["case"], st["target"]
    dt = DTYPES[c["dtype"]]
    x, w = st["hidden"].float(), st["weight"].float()
    rows = torch.arange(x.shape[0], device="cuda")
    if c["target"] == "index":
        valid = target != IGNORE
        safe = torch.where(valid, target, torch.zeros_like(target))
        x = torch.where(valid[:, None], x, torch.zeros((), device="cuda"))
    else:
        valid = None
    logits = x @ w.t()
    if st["bias"] is not None:
        logits += st["bias"].float()
    m = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - m)
    s = e.sum(1, keepdim=True)
    lse = (m + torch.log(s))[:, 0]
    p = e.div_(s)
    if valid is not None:
        loss = torch.where(valid, lse - logits[rows, safe], torch.zeros((), device="cuda"))
        count = valid.sum()
    else:
        loss = lse * target.sum(1) - (target * logits).sum(1)
        count = x.shape[0]
    entropy = None
    if c["entropy"]:
        entropy = lse - (p * logits).sum(1)
        if valid is not None:
            entropy = torch.where(valid, entropy, torch.zeros((), device="cuda"))
    del logits
    if not c["grad"]:
        return {"loss": loss, "entropy": entropy} if c["entropy"] else {"loss": loss}
    if valid is not None:
        p[rows, safe] -= 1.0
        p = torch.where(valid[:, None], p, torch.zeros((), device="cuda"))
    else:
        p = p * target.sum(1, keepdim=True) - target
    g = st["grad_loss"] / count
    out = {"loss": loss.sum() / count, "d_hidden": (p @ w * g).to(dt), "d_weight": (p.t() @ x * g).to(dt)}
    if st["bias"] is not None:
        out["d_bias"] = (p.sum(0) * g).to(dt)
    if c["entropy"]:
        out["entropy"] = entropy.sum() / count
    return out


# ---------------------------------------------------------------- what is done, and what is right
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size * (3 if case["mode"] == "residual" else 2), "flops": 2 * n}
    n, hidden, classes = case["n"], case["hidden"], case["classes"]
    params = n * hidden + classes * hidden + (classes if case["bias"] else 0)
    target = n * 8 if case["target"] == "index" else n * classes * 4
    if not case["grad"]:
        return {"bytes": params * size + target + 4 * n * (2 if case["entropy"] else 1), "flops": 2 * n * hidden * classes}
    return {"bytes": 2 * params * size + target + (8 if case["entropy"] else 4), "flops": 6 * n * hidden * classes}


def _philox_halfwords(first, count, seed, offset):
    """The same generator over numpy's unsigned 64-bit integers: uint16 [count]."""
    b0, b1 = first >> 3, (first + count + 7) >> 3
    out = np.empty((b1 - b0, 8), dtype=np.uint16)
    mask, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for at in range(b0, b1, 1 << 18):
        blk = np.arange(at, min(b1, at + (1 << 18)), dtype=np.uint64)
        x = [blk & mask, blk >> sh, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, offset >> 32)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = [(b >> sh) ^ x[1] ^ np.uint64(key[0]), b & mask, (a >> sh) ^ x[3] ^ np.uint64(key[1]), a & mask]
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        o = out[at - b0: at - b0 + blk.size]
        for q in range(4):
            o[:, 2 * q] = x[q] & np.uint64(0xFFFF)
            o[:, 2 * q + 1] = x[q] >> np.uint64(16)
    return out.reshape(-1)[first - 8 * b0: first - 8 * b0 + count]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        t = int(round(case["p"] * 65536))
        u = _philox_halfwords(case["first_row"] * cols, rows * cols, st["seed"], st["offset"])
        kept = torch.from_numpy(u >= t).to("cuda").reshape(rows, cols)
        y = st["x"].double() * 65536 / (65536 - t)
        y[~kept] = 0.0
        return y if st["residual"] is None else y + st["residual"].double()
    x, w, t = st["hidden"].double(), st["weight"].double(), st["target"]
    b = st["bias"].double() if st["bias"] is not None else None
    n, classes, by_index = case["n"], case["classes"], case["target"] == "index"
    used = (t != IGNORE) if by_index else torch.ones(n, dtype=torch.bool, device="cuda")
    total = int(used.sum())
    loss, ent = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(classes, dtype=torch.float64, device="cuda")
    which = used.nonzero()[:, 0]
    for ids in which.split(1024):                                 # a thousand rows at a time
        xi = x[ids]
        z = torch.mm(xi, w.t())
        if b is not None:
            z = z + b
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        del z
        q = torch.zeros_like(logp).scatter_(1, t[ids][:, None], 1.0) if by_index else t[ids].double()
        loss[ids] = -(q * logp).sum(1)
        prob = logp.exp()
        ent[ids] = -(prob * logp).sum(1)
        if case["grad"]:
            d = (prob * q.sum(1, keepdim=True) - q) * (st["grad_loss"] / total)
            dx[ids] = torch.mm(d, w)
            dw += torch.mm(d.t(), xi)
            db += d.sum(0)
    if not case["grad"]:
        return {"loss": loss, "entropy": ent} if case["entropy"] else {"loss": loss}
    out = {"loss": loss.sum() / total, "d_hidden": dx, "d_weight": dw}
    if b is not None:
        out["d_bias"] = db
    if case["entropy"]:
        out["entropy"] = ent.sum() / total
    return out
