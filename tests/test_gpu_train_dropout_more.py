"""Dropout in the training step: going on from saved weights, both paths' gradients, the switch of the C entry point."""
import ctypes as C

import pytest
import torch

from test_gpu_train_dropout import batch, net

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
