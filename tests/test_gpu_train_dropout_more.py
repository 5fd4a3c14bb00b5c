"""Dropout in the training step: going on from saved weights, both paths' gradients, the switch of the C entry point."""
import pytest
import torch

from test_gpu_train_dropout import batch, definition, net, order

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_a_run_that_goes_on_draws_new_masks(tmp_path, native):
    """Weights saved after three steps and read by another net: with the step number the next masks are the ones the first
    run would have drawn (bit-equal gradients of the next step), without it they are the first step's again."""
    s, p, z = batch(64, 8)
    a = net(8, dropout=0.3, dropout_seed=5, native_train=native)
    for _ in range(3):
        a.train_step(s, p, z, 1e-3)
    assert a.dropout_step == 3
    path = str(tmp_path / "weights.pt")
    a.save_model(path)
    want = a.native_gradients(s, p, z)
    b = net(8, model_file=path, dropout=0.3, dropout_seed=5, dropout_step=a.dropout_step, native_train=native)
    assert b.dropout_step == 3
    got = b.native_gradients(s, p, z)
    assert torch.equal(want[0], got[0]) and want[1:] == got[1:]
    b.train_step(s, p, z, 1e-3)
    assert b.dropout_step == 4
    again = net(8, model_file=path, dropout=0.3, dropout_seed=5, native_train=native)
    assert not torch.equal(again.native_gradients(s, p, z)[0], want[0])


def test_pipeline_goes_on_from_a_step(tmp_path):
    from alphazero_gomoku_amd.train import TrainPipeline
    a = net(6)
    path = str(tmp_path / "weights.pt")
    a.save_model(path)
    tp = TrainPipeline(board_width=6, board_height=6, n_in_row=4, init_model=path, dropout=0.25, dropout_step=70)
    assert tp.policy_value_net.dropout_step == 70
    with pytest.raises(ValueError):
        TrainPipeline(policy_value_net=a, dropout_step=70)
    for bad in (-1, 1 << 62):
        with pytest.raises(ValueError):
            net(8, dropout_step=bad)


def parts(flat, like):
    at = 0
    for q in like:
        yield flat[at:at + q.numel()].double()
        at += q.numel()
    assert at == flat.numel()


@pytest.mark.parametrize("size,n", [(6, 33), (8, 128)])
def test_both_paths_make_the_gradient_of_the_definition(size, n):
    """The first step's gradients of the library and of PyTorch's autograd over the operators, every tensor within three times the
    error that PyTorch's own float32 autograd of the masked step has against float64 (and 2**-20 of its norm)."""
    s, p, z = batch(n, size)
    a, b = net(size, dropout=0.3, dropout_seed=5), net(size, dropout=0.3, dropout_seed=5, native_train=False)
    g64 = definition(a.policy_value_net, s, p, z, 0.3, 5, 1, torch.float64)[2]
    g32 = definition(a.policy_value_net, s, p, z, 0.3, 5, 1, torch.float32)[2]
    native = a.native_gradients(s, p, z)[0]
    b.train_step(s, p, z, 1e-3)
    named = dict(b.policy_value_net.named_parameters())
    for name, want, other, u, v in zip(order(), g64, g32, parts(native, g64), (named[k].grad.double().reshape(-1) for k in order())):
        bound = 3 * float((other - want).norm()) + 2.0 ** -20 * float(want.norm())
        assert float(want.norm()) > 0 and float((u - want).norm()) <= bound and float((v - want).norm()) <= bound, name


def test_the_entry_point_switches_dropout_on_and_off():
    """azg_train_set_dropout by itself, the net's own calls of it held back: on, the next backward pass is the masked step's; off
    again, it is bit for bit the one before."""
    s, p, z = batch(96, 8)
    q = net(8)
    eng = q._engine_handle()
    q._set_dropout = lambda *_: None
    before = q.native_gradients(s, p, z)
    eng._chk(eng.L.azg_train_set_dropout(eng.h, 0.5, 1, 2, 0, 1))
    on = q.native_gradients(s, p, z)
    eng._chk(eng.L.azg_train_set_dropout(eng.h, 0.0, 1, 2, 0, 1))
    off = q.native_gradients(s, p, z)
    assert torch.equal(before[0], off[0]) and before[1:] == off[1:] and not torch.equal(before[0], on[0])
    g64 = definition(q.policy_value_net, s, p, z, 0.5, 1, 2, torch.float64)
    g32 = definition(q.policy_value_net, s, p, z, 0.5, 1, 2, torch.float32)
    assert abs(on[1] - g64[0]) <= 3 * abs(g32[0] - g64[0]) + 2.0 ** -20 * abs(g64[0])
    for name, want, other, got in zip(order(), g64[2], g32[2], parts(on[0], g64[2])):
        assert float((got - want).norm()) <= 3 * float((other - want).norm()) + 2.0 ** -20 * float(want.norm()), name
