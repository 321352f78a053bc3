"""The model zoo's fully connected layers on the fused kernel."""

import torch.nn as nn

from ..ops.linear_ops import FusedLinear


def _plain(module: nn.Module, kind: type) -> bool:
    """A module of that very type, without hooks."""
    return type(module) is kind and not any(
        hooks for name, hooks in vars(module).items() if name.endswith("_hooks"))


def fuse_linears(model: nn.Module) -> nn.Module:
    """Puts ``FusedLinear`` in the place of every ``nn.Linear``, with the ReLU
    that follows it: the next module of a ``Sequential``, or, for modules
    whose ``forward`` calls ``linear_relu``, the names in ``linear_relus``.
    Parameters and their names stay (checkpoints fit either form).  Layers with
    hooks stay as they are."""
    for module in model.modules():
        named = getattr(module, "linear_relus", ())
        in_order = (isinstance(module, nn.Sequential)
                    and type(module).forward is nn.Sequential.forward)
        # named_children() would leave out what is there twice
        children = list(module._modules.items())
        for at, (name, child) in enumerate(children):
            if not _plain(child, nn.Linear):
                continue
            activation = "relu" if name in named else "none"
            if in_order and at + 1 < len(children):
                after, follower = children[at + 1]
                if _plain(follower, nn.ReLU):
                    activation = "relu"
                    setattr(module, after, nn.Identity())
            setattr(module, name, FusedLinear.of(child, activation))
    return model
