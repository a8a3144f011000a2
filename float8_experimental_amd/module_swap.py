"""Layers of one kind swapped throughout a model."""
from typing import Callable

import torch.nn as nn


def swap_modules(module: nn.Module, kind: type, from_float: Callable[[nn.Module], nn.Module]) -> nn.Module:
    """Every ``kind`` of ``module`` (itself, no subclass) replaced by ``from_float`` of it, one that is held under several names or by several modules by the same one; a root-level one is
    returned converted."""
    if type(module) is kind:
        return from_float(module)
    made = {}

    def visit(mod: nn.Module) -> None:
        for name, child in mod._modules.items():  # (named_children() has each module under one of its names)
            if type(child) is kind:
                if child not in made:
                    made[child] = from_float(child)
                setattr(mod, name, made[child])
            elif child is not None:
                visit(child)

    visit(module)
    return module
