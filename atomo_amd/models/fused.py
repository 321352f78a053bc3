"""The model zoo's fully connected layers on the fused kernel."""

import torch.nn as nn

from ..ops.linear_ops import FusedLinear


def fuse_linears(model: nn.Module) -> nn.Module:
    """Puts ``FusedLinear`` in the place of every ``nn.Linear``, with the ReLU
    that follows it: the next module of a ``Sequential``, or, for modules
    whose ``forward`` calls ``linear_relu``, the names in ``linear_relus``.
    Parameters and their names stay (checkpoints fit either form)."""
    for module in model.modules():
        named = getattr(module, "linear_relus", ())
        children = list(module.named_children())
        for at, (name, child) in enumerate(children):
            if type(child) is not nn.Linear:
                continue
            activation = "relu" if name in named else "none"
            if isinstance(module, nn.Sequential) and at + 1 < len(children):
                after, follower = children[at + 1]
                if type(follower) is nn.ReLU:
                    activation = "relu"
                    setattr(module, after, nn.Identity())
            setattr(module, name, FusedLinear.of(child, activation))
    return model
