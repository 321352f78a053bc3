"""The head-to-loss operators where the framework calls them: models, trainer,
evaluation, commands (CPU)."""

import json
import os
import sys

import pytest
import torch
import torch.nn.functional as F

from atomo_amd.codings import make_codec
from atomo_amd.data import make_loaders
from atomo_amd.models import build_model, fuse_linears
from atomo_amd.ops.linear_ops import FusedLinear
from atomo_amd.ops.logit_ops import label_logprobs
from atomo_amd.parallel import Comm, PSTrainer
from atomo_amd.utils import accuracy, answers

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPU = torch.device("cpu")


def _trainer(**kw):
    return PSTrainer(
        model_name=kw.pop("model", "LeNet"), codec=make_codec("sgd"),
        comm=Comm(device=CPU), lr=0.05, num_classes=10, in_channels=1, seed=7,
        device=CPU, **kw)


@pytest.mark.parametrize("name,shape,relus", [
    ("LeNet", (1, 28, 28), 1), ("FC", (1, 28, 28), 2), ("VGG11", (3, 32, 32), 2),
    ("AlexNet", (3, 64, 64), 2), ("ResNet18", (3, 32, 32), 0)])
def test_fused_models_answer_alike(name, shape, relus):
    torch.manual_seed(0)
    plain = build_model(name, 10, shape[0]).eval()
    fused = build_model(name, 10, shape[0], fused_linear=True).eval()
    layers = [m for m in fused.modules() if isinstance(m, FusedLinear)]
    assert sum(m.activation == "relu" for m in layers) == relus
    assert not any(type(m) is torch.nn.Linear for m in fused.modules())
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(2, *shape)
    with torch.no_grad():
        a, b = fused(x), plain(x)
    # the plain side's fp32 sums of at most 9216 terms, over three layers
    assert (a - b).abs().max() <= 3 * 9216 * 2.0 ** -24 * max(1.0, float(b.abs().max()))


def test_fuse_takes_over_parameters():
    model = build_model("VGG11", 10, 3)
    before = dict(model.named_parameters())
    after = dict(fuse_linears(model).named_parameters())
    assert list(before) == list(after) and all(before[n] is after[n] for n in before)


def test_fused_linears_of_modules_that_are_shared_hooked_or_their_own():
    nn = torch.nn

    class Backwards(nn.Sequential):
        def forward(self, x):
            for layer in reversed(self):
                x = layer(x)
            return x

    torch.manual_seed(0)
    act, norm = nn.ReLU(), nn.Hardtanh(-4.0, -1.0)
    shared = nn.Linear(6, 6)
    hooked = nn.Linear(6, 6)
    hooked.register_forward_hook(lambda layer, args, out: out + 1)
    watched = nn.ReLU()
    watched.register_forward_hook(lambda layer, args, out: out - 1)
    model = nn.Sequential(
        nn.Linear(6, 6), norm, nn.Linear(6, 6), norm, act, shared, act, shared,
        hooked, nn.ReLU(), nn.Linear(6, 6), watched,
        Backwards(nn.Linear(6, 6), nn.ReLU(), nn.Linear(6, 6)))
    for p in model.parameters():
        p.data = torch.randint(-1, 2, p.shape).float()  # whole numbers: exact sums
    x = torch.randint(-1, 2, (50, 6)).float()
    want = model(x)
    keys = list(model.state_dict())
    got = fuse_linears(model)(x)
    assert want.abs().max() < 2 ** 20 and torch.equal(got, want)
    assert list(model.state_dict()) == keys and model[8] is hooked
    assert [m.activation for m in model if isinstance(m, FusedLinear)] == [
        "none", "none", "relu", "none", "none"]


def test_answers_are_loss_accuracy_and_entropy():
    g = torch.Generator().manual_seed(0)
    z, y = torch.randn(50, 10, generator=g), torch.randint(0, 10, (50,), generator=g)
    loss, precs, entropy = answers(z, y, topk=(1, 5))
    # fp32 log probabilities, below 16: half a step is 2^-21
    assert loss == pytest.approx(float(F.cross_entropy(z.double(), y)), abs=2.0 ** -21)
    # percentages: accuracy() counts in fp32
    assert precs == pytest.approx(accuracy(z, y, topk=(1, 5)), rel=2.0 ** -22)
    p = z.double().softmax(1)
    assert entropy == pytest.approx(float(-(p * p.log()).sum(1).mean()), abs=2.0 ** -21)


def test_evaluate_with_entropy():
    trainer = _trainer()
    _, test = make_loaders("mnist", 16, 16, CPU, seed=1)
    test = [test.next_batch() for _ in range(2)]  # the loader goes on otherwise
    plain = trainer.evaluate(test, max_batches=2)
    assert set(plain) == {"loss", "prec1", "prec5"}
    full = trainer.evaluate(test, max_batches=2, entropy=True)
    assert full["prec1"] == pytest.approx(plain["prec1"], rel=2.0 ** -22)
    assert full["prec5"] == pytest.approx(plain["prec5"], rel=2.0 ** -22)
    # cross_entropy's fp32 sums over ten classes and sixteen rows
    assert full["loss"] == pytest.approx(plain["loss"], rel=64 * 2.0 ** -24)
    assert 0.0 < full["entropy"] <= 2.302586


@pytest.mark.parametrize("fused", [False, True])
def test_trainer_distills(tmp_path, fused):
    teacher = _trainer(train_dir=str(tmp_path), model="FC")
    path = teacher.save_checkpoint()
    trainer = _trainer(distill_from=path, distill_network="FC", distill_top=3,
                       distill_temperature=2.0, distill_weight=0.75,
                       fused_linear=fused)
    start = trainer.flat.clone()
    train, _ = make_loaders("mnist", 16, 16, CPU, seed=1)
    x, y = next(iter(train))
    loss = trainer.train_step(x, y)
    assert not torch.equal(trainer.flat, start)
    # the same step by hand, in 64 bits from the fp32 logits on
    student = build_model("LeNet", 10, 1)
    with torch.no_grad():
        for p, q in zip(student.parameters(), trainer.model.parameters()):
            n = p.numel()
            p.copy_(start[:n].view_as(p))
            start = start[n:]
    out = student(x)
    top = teacher.model(x).detach().double().topk(3, dim=1)
    q = torch.zeros(16, 10, dtype=torch.float64).scatter_(
        1, top.indices, torch.softmax(top.values / 2, 1))
    log_p = F.log_softmax(out.double() / 2, 1)
    want = 0.75 * 4 * (torch.special.xlogy(q, q) - q * log_p).sum(1).mean() + \
        0.25 * F.cross_entropy(out.double(), y)
    # two fp32 networks, sums of at most 800 terms each way
    assert loss == pytest.approx(float(want.detach()), rel=2 * 800 * 2.0 ** -24)
    want.backward()
    got = trainer.flat_grad
    ref = torch.cat([p.grad.reshape(-1) for p in student.parameters()])
    assert (got - ref).abs().max() <= 4 * 800 * 2.0 ** -24 * float(ref.abs().max())
    assert all(p.grad is None for p in trainer.teacher.parameters())


def test_commands(tmp_path, capsys):
    sys.path.insert(0, REPO)
    import distributed_evaluator
    import single_machine

    base = ["--network", "FC", "--dataset", "mnist", "--code", "svd",
            "--batch-size", "8", "--test-batch-size", "16", "--log-interval", "1",
            "--no-cuda", "--train-dir", str(tmp_path)]
    assert single_machine.main(base + ["--max-steps", "2", "--checkpoint-freq", "2"]) == 0
    path = os.path.join(str(tmp_path), "model_step_2")
    assert single_machine.main(
        base + ["--max-steps", "2", "--fused-linear", "--distill-from", path,
                "--distill-top", "4", "--eval-entropy"]) == 0
    out = capsys.readouterr().out
    recs = [json.loads(line) for line in out.splitlines() if line.startswith("{")]
    evals = [r for r in recs if r.get("log") == "eval"]
    assert "entropy" not in evals[0] and evals[1]["entropy"] > 0
    plain = distributed_evaluator.evaluate_checkpoint(path, "FC", "mnist", 16, CPU)
    full = distributed_evaluator.evaluate_checkpoint(path, "FC", "mnist", 16, CPU, entropy=True)
    assert set(full) - set(plain) == {"entropy"}
    assert full["loss"] == pytest.approx(plain["loss"], rel=64 * 2.0 ** -24)


def test_teacher_of_another_network_is_refused(tmp_path):
    path = _trainer(train_dir=str(tmp_path), model="FC").save_checkpoint()
    with pytest.raises(RuntimeError):
        _trainer(distill_from=path)


@pytest.mark.parametrize("wrong", [
    dict(distill_top=0), dict(distill_top=129), dict(distill_weight=1.5),
    dict(distill_temperature=0.0)])
def test_wrong_distillation_is_refused(tmp_path, wrong):
    path = _trainer(train_dir=str(tmp_path)).save_checkpoint()
    with pytest.raises(ValueError):
        _trainer(distill_from=path, **wrong)


def test_many_classes_keep_the_top():
    z = torch.randn(3, 300)
    assert label_logprobs(z, top=128).top_index.shape == (3, 128)


def test_fused_models_take_double_precision():
    plain, fused = (build_model("FC", 10, 1, fused_linear=f).double() for f in (False, True))
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(2, 1, 28, 28, dtype=torch.float64)
    assert torch.equal(fused(x), plain(x))
