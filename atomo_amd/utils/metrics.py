"""Top-k accuracy (the helper the reference duplicates in four files —
nn_ops.py:86-99, distributed_worker.py:42-55, sync_replicas_master_nn.py:41-54,
distributed_evaluator.py:25-37 — defined once here)."""

import torch

from ..ops.logit_ops import label_logprobs


@torch.no_grad()
def accuracy(output: torch.Tensor, target: torch.Tensor, topk=(1,)):
    maxk = max(topk)
    _, pred = output.topk(maxk, dim=1, largest=True, sorted=True)
    pred = pred.t()
    correct = pred.eq(target.view(1, -1).expand_as(pred))
    res = []
    batch = target.size(0)
    for k in topk:
        correct_k = correct[:k].reshape(-1).float().sum(0)
        res.append(float(correct_k.mul_(100.0 / batch)))
    return res


@torch.no_grad()
def answers(output: torch.Tensor, target: torch.Tensor, topk=(1,)):
    """Mean cross entropy, top-k accuracies (percent) and mean entropy of a
    batch, from one pass over the logits (ops.logit_ops.label_logprobs).
    Equal logits count in the order of their classes."""
    top = label_logprobs(output, target, top=max(topk))
    correct = top.top_index == target.view(-1, 1)
    hits = torch.stack([correct[:, :k].sum() for k in topk]) * (100.0 / target.size(0))
    both = torch.stack([-top.logprob.double().mean(), top.entropy.double().mean()])
    values = torch.cat([both, hits.double()]).tolist()
    return values[0], values[2:], values[1]
