"""Fused layers, distillation and evaluation in the trainer on the GPU."""

import pytest
import torch

from atomo_amd.codings import make_codec
from atomo_amd.data import make_loaders
from atomo_amd.models import build_model
from atomo_amd.parallel import Comm, PSTrainer

pytestmark = pytest.mark.gpu


def _trainer(dev, **kw):
    return PSTrainer(
        model_name=kw.pop("model", "FC"), codec=make_codec(kw.pop("code", "sgd"), rank=3),
        comm=Comm(device=dev), lr=0.05, num_classes=10, in_channels=1, seed=7,
        device=dev, **kw)


@pytest.fixture
def dev():
    return torch.device("cuda:0")


@pytest.fixture
def teacher(dev, tmp_path):
    return _trainer(dev, train_dir=str(tmp_path)).save_checkpoint()


def test_fused_model_answers_and_learns_alike(dev):
    torch.manual_seed(0)
    plain = build_model("FC", 10, 1).to(dev)
    fused = build_model("FC", 10, 1, fused_linear=True).to(dev)
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(64, 1, 28, 28, device=dev)
    up = torch.randn(64, 10, device=dev)
    a, b = fused(x), plain(x)
    # fp32 sums of at most 800 terms on both sides, over three layers
    tol = 2 * 3 * 800 * 2.0 ** -24
    assert (a - b).abs().max() <= tol * float(b.detach().abs().max())
    a.backward(up)
    b.backward(up)
    for p, q in zip(fused.parameters(), plain.parameters()):
        assert (p.grad - q.grad).abs().max() <= 2 * tol * float(q.grad.abs().max())


@pytest.mark.parametrize("amp", [False, True])
def test_distilling_steps_run(dev, teacher, amp):
    trainer = _trainer(dev, code="svd", distill_from=teacher, distill_top=4,
                       fused_linear=True, amp=amp)
    train, test = make_loaders("mnist", 32, 32, dev, seed=1)
    start = trainer.flat.clone()
    for i, (x, y) in enumerate(train):
        loss = trainer.train_step(x, y)
        assert loss == loss
        if i == 2:
            break
    assert not torch.equal(trainer.flat, start)
    test = [test.next_batch() for _ in range(2)]  # the loader goes on otherwise
    plain = trainer.evaluate(test, max_batches=2)
    full = trainer.evaluate(test, max_batches=2, entropy=True)
    assert full["loss"] == pytest.approx(plain["loss"], rel=64 * 2.0 ** -24)
    assert full["prec1"] == pytest.approx(plain["prec1"], rel=2.0 ** -22)
    assert 0 < full["entropy"] <= 2.302586


def test_graphed_steps_equal_eager_ones(dev, teacher):
    kw = dict(distill_from=teacher, distill_top=5, distill_weight=0.6, fused_linear=True)
    eager, graphed = _trainer(dev, **kw), _trainer(dev, use_graph=True, **kw)
    assert graphed.graph_whole
    graphed.flat.copy_(eager.flat)
    graphed_start = eager.flat.clone()
    train, _ = make_loaders("mnist", 32, 32, dev, seed=1)
    batches = [b for _, b in zip(range(4), train)]
    # capturing warms up with steps of its own: begin again from the start
    graphed.train_step(*batches[0])
    assert graphed.graph_whole
    graphed.flat.copy_(graphed_start)
    graphed.opt.buf.zero_()
    for x, y in batches:
        a = graphed.train_step(x, y)
        b = eager.train_step(x, y)
        torch.cuda.synchronize()
        assert a == b
    assert torch.equal(graphed.flat, eager.flat)
