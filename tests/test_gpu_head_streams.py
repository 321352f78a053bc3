"""The head-to-loss operators on several streams, in several graphs and from
several threads at once."""

import threading

import pytest
import torch

from side_by_side import run_threads

from atomo_amd.ops.linear_ops import linear_act
from atomo_amd.ops.logit_ops import distill_loss, label_logprobs

pytestmark = pytest.mark.gpu


def _job(seed):
    """Inputs, and a pass over all three operators, each with a workspace: a
    split product and a split row."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(40, 3000, generator=g, device="cuda").requires_grad_()
    w = torch.randn(700, 3000, generator=g, device="cuda").div_(50).requires_grad_()
    teacher = torch.randn(40, 20000, generator=g, device="cuda")
    head = torch.randn(20000, 700, generator=g, device="cuda").div_(20).requires_grad_()
    y = torch.randint(0, 20000, (40,), generator=g, device="cuda")

    def run():
        h = linear_act(x, w, None, "silu")
        z = linear_act(h, head)
        top = label_logprobs(teacher, y, top=32)
        loss = distill_loss(z, top.top_logprob, top.top_index, y,
                            temperature=2.0, weight=0.5)
        grads = torch.autograd.grad(loss, (x, w, head))
        return (loss.detach(), top.logprob, top.top_index, *grads)

    return run


def _equal(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_repeated_calls_are_equal_to_the_bit():
    run = _job(0)
    want = run()
    for _ in range(5):
        assert _equal(run(), want)


def test_streams_side_by_side():
    jobs = [_job(i) for i in range(4)]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(5):
        for i, run in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i].append(run())
    torch.cuda.synchronize()
    for i in range(4):
        assert all(_equal(out, want[i]) for out in got[i])


def test_threads_side_by_side():
    jobs = [_job(i) for i in range(3)]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                out = jobs[i]()
                torch.cuda.current_stream().synchronize()
                if not _equal(out, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and not any(t.is_alive() for t in threads)


def test_two_graphs_in_turn():
    jobs = [_job(i) for i in range(2)]
    want = [run() for run in jobs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for run in jobs:
            run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for run in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            eager = jobs[1 - i]()
            torch.cuda.synchronize()
            assert _equal(outs[i], want[i]) and _equal(eager, want[1 - i])


def test_threads_side_by_side_make_all_of_their_passes():
    """The same with what a thread raises, and passes that are counted."""
    jobs = [_job(i) for i in range(3)]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]

    def work(i):
        with torch.cuda.stream(streams[i]):
            out = jobs[i]()
            streams[i].synchronize()
        assert _equal(out, want[i])

    run_threads([lambda i=i: work(i) for i in range(3)], 5)
