"""Dropout in the training step: azg_train_set_dropout, PolicyValueNet(dropout=...), TrainPipeline(dropout=...)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from test_gpu_ops import keep_mask

pytestmark = pytest.mark.gpu


def batch(n, size, seed=0):
    rng = np.random.RandomState(seed)
    s = (rng.rand(n, 4, size, size) < 0.2).astype(np.float32)
    p = rng.dirichlet([0.3] * size * size, n).astype(np.float32)
    z = rng.choice([-1.0, 0.0, 1.0], n).astype(np.float32)
    return [torch.from_numpy(a).cuda() for a in (s, p, z)]


def net(size, **kw):
    from alphazero_gomoku_amd import PolicyValueNet
    torch.manual_seed(3)
    return PolicyValueNet(size, size, **kw)


def definition(module, s, p, z, rate, seed, offset, dtype):
    """Loss, entropy and flat gradient of the step's definition by autograd in dtype, masks from the generator's definition."""
    import copy
    m = copy.deepcopy(module).to(dtype)
    s, p, z = s.to(dtype), p.to(dtype), z.to(dtype)
    a, v = m.features(s)
    ka, t = keep_mask(a.shape[0], a.shape[1], rate, seed, 2 * offset)
    kv, _ = keep_mask(v.shape[0], v.shape[1], rate, seed, 2 * offset + 1)
    scale = 65536.0 / (65536 - t)
    logp = F.log_softmax(m.act_fc1(torch.where(ka, a * scale, torch.zeros_like(a))), 1)
    val = m.value(torch.where(kv, v * scale, torch.zeros_like(v)))
    loss = F.mse_loss(val.view(-1), z) - (p * logp).sum(1).mean()
    loss.backward()
    ent = -(logp.exp() * logp).sum(1).mean()
    return float(loss), float(ent), [dict(m.named_parameters())[k].grad.double().reshape(-1) for k in order()]


def order():
    from alphazero_gomoku_amd.net import PARAM_ORDER
    return PARAM_ORDER


@pytest.mark.parametrize("size,n", [(6, 33), (8, 64), (8, 512), (15, 40), (16, 24)])
@pytest.mark.parametrize("rate", [0.3, 0.75])
def test_gradients_against_definition(size, n, rate):
    """Every parameter's gradient within three times the error that PyTorch's own float32 autograd of the same masked step has
    against float64 (and 2**-20 of its norm, for tensors that float32 happens to get exactly)."""
    s, p, z = batch(n, size)
    q = net(size, dropout=rate, dropout_seed=0x123456789ABCDEF)
    grad, loss, ent = q.native_gradients(s, p, z)
    l64, e64, g64 = definition(q.policy_value_net, s, p, z, rate, 0x123456789ABCDEF, 1, torch.float64)
    l32, e32, g32 = definition(q.policy_value_net, s, p, z, rate, 0x123456789ABCDEF, 1, torch.float32)
    assert abs(loss - l64) <= 3 * abs(l32 - l64) + 2.0 ** -20 * abs(l64) and abs(ent - e64) <= 3 * abs(e32 - e64) + 2.0 ** -20 * abs(e64)
    at = 0
    for name, want, other in zip(order(), g64, g32):
        got = grad[at:at + want.numel()].double()
        at += want.numel()
        assert float((got - want).norm()) <= 3 * float((other - want).norm()) + 2.0 ** -20 * float(want.norm()), name
    assert at == grad.numel()


@pytest.mark.parametrize("world", [2, 4])
def test_ranks_average_to_the_whole_batch(world):
    """Every rank's gradient of its rows, under the masks of its rows, averaged: the gradient of the whole batch (bounds as above)."""
    s, p, z = batch(64, 8)
    q = net(8, dropout=0.4, dropout_seed=9)
    total, losses = None, []
    for rank in range(world):
        q._dropout_args = lambda step: (0.4, 9, step, rank, world)
        g, loss, _ = q.native_gradients(s[rank::world], p[rank::world], z[rank::world])
        total = g.double() if total is None else total + g.double()
        losses.append(loss)
    del q._dropout_args
    l64, _, g64 = definition(q.policy_value_net, s, p, z, 0.4, 9, 1, torch.float64)
    _, _, g32 = definition(q.policy_value_net, s, p, z, 0.4, 9, 1, torch.float32)
    assert abs(sum(losses) / world - l64) <= 2.0 ** -18 * abs(l64)
    at = 0
    for name, want, other in zip(order(), g64, g32):
        got = total[at:at + want.numel()] / world
        at += want.numel()
        assert float((got - want).norm()) <= 3 * float((other - want).norm()) + 2.0 ** -20 * float(want.norm()), name


def test_autograd_steps_leave_the_native_optimiser_alone():
    """A step through autograd counts for the masks and not for the library's Adam."""
    s, p, z = batch(64, 8)
    q = net(8, dropout=0.3, dropout_seed=5)
    q.train_step(s, p, z, 1e-3)
    q.native_train = False
    q.train_step(s, p, z, 1e-3)
    assert (q._adam_step, q._dropout_step) == (1, 2)


def test_step_takes_the_mask_of_its_number_and_repeats():
    s, p, z = batch(128, 8)
    a, b = net(8, dropout=0.3, dropout_seed=5), net(8, dropout=0.3, dropout_seed=5)
    masks = []
    for _ in range(3):
        g, _, _ = a.native_gradients(s, p, z)
        masks.append(g)
        la = a.train_step(s, p, z, 1e-3)
        lb = b.train_step(s, p, z, 1e-3)
        assert la == lb
        for u, v in zip(a.param_tensors(), b.param_tensors()):
            assert torch.equal(u, v)
    c = net(8, dropout=0.3, dropout_seed=6)
    assert not torch.equal(c.native_gradients(s, p, z)[0], masks[0])


def test_autograd_step_is_the_same_step():
    """native_train=False: ops.dropout and ops.linear_cross_entropy under PyTorch's autograd and Adam."""
    s, p, z = batch(128, 8)
    a, b = net(8, dropout=0.3, dropout_seed=5), net(8, dropout=0.3, dropout_seed=5, native_train=False)
    for i in range(3):
        la, ea = a.train_step(s, p, z, 1e-3)
        lb, eb = b.train_step(s, p, z, 1e-3)
        # (the same float32 formulas in another order of sums; Adam's first steps divide by |g|, so a parameter may differ by
        #  the rounding of tiny gradients times the learning rate)
        assert abs(la - lb) <= 1e-4 * abs(lb) and abs(ea - eb) <= 1e-4 * abs(eb), i
    for u, v in zip(a.param_tensors(), b.param_tensors()):
        assert float((u - v).abs().max()) <= 2 * 3 * 1e-3


def test_off_is_off_bit_for_bit():
    s, p, z = batch(96, 8)
    q = net(8)
    eng = q._engine_handle()
    before = q.native_gradients(s, p, z)
    eng._chk(eng.L.azg_train_set_dropout(eng.h, 0.5, 1, 2, 0, 1))
    other = torch.zeros_like(before[0])
    q.dropout = 0.5
    dropped = q.native_gradients(s, p, z)
    q.dropout = 0.0
    after = q.native_gradients(s, p, z)
    assert torch.equal(before[0], after[0]) and before[1:] == after[1:]
    assert not torch.equal(before[0], dropped[0]) and other is not None


def test_forward_passes_never_drop():
    s, _, _ = batch(64, 8)
    a, b = net(8, dropout=0.6, dropout_seed=1), net(8)
    a._set_dropout(a._engine_handle(), 1)
    for u, v in zip(a.policy_value_in_training(s), b.policy_value_in_training(s)):
        assert torch.equal(u, v)


def test_epoch_is_step_then_forward():
    s, p, z = batch(128, 8)
    a, b = net(8, dropout=0.3, dropout_seed=5), net(8, dropout=0.3, dropout_seed=5)
    old, _ = a.policy_value_in_training(s)
    r = a.train_epoch(s, p, z, 1e-3, s, old)
    assert r[:2] == b.train_step(s, p, z, 1e-3)
    probs, vals, kl = b.policy_value_in_training(s, old)
    assert torch.equal(r[2], probs) and torch.equal(r[3], vals) and r[4] == kl


def test_refusals():
    from alphazero_gomoku_amd import PolicyValueNet, _lib
    for bad in (1.0, -0.1, float("nan")):
        with pytest.raises(ValueError):
            PolicyValueNet(8, 8, dropout=bad)
    with pytest.raises(ValueError):
        PolicyValueNet(8, 8, dropout_seed=-1)
    q = net(8)
    eng = q._engine_handle()
    for bad in (1.0, -0.5, float("nan")):
        assert eng.L.azg_train_set_dropout(eng.h, bad, 0, 0, 0, 1) == -1
    from alphazero_gomoku_amd.train import TrainPipeline
    with pytest.raises(ValueError):
        TrainPipeline(policy_value_net=q, dropout=0.1)
    assert _lib is not None


def test_pipeline_trains_with_dropout():
    from alphazero_gomoku_amd.train import TrainPipeline
    tp = TrainPipeline(board_width=6, board_height=6, n_in_row=4, n_playout=20, play_batch_size=16, n_parallel=16, game_batch_num=1,
                       batch_size=64, buffer_size=4096, epochs=2, dropout=0.25)
    tp.collect_selfplay_data(16)
    before = [q.clone() for q in tp.policy_value_net.param_tensors()]
    loss, entropy = tp.policy_update()
    assert np.isfinite(loss) and np.isfinite(entropy) and tp.policy_value_net.dropout == 0.25
    assert all(bool(torch.isfinite(q).all()) for q in tp.policy_value_net.param_tensors())
    assert any(not torch.equal(u, v) for u, v in zip(before, tp.policy_value_net.param_tensors()))
