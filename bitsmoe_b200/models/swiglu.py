"""Whether a module computes down_proj(silu(gate_proj(x)) * up_proj(x)) and nothing else.

The blocks hand MLPs of that kind to the library's kernels, which read the three weights and never call the module.  Names and shapes do
not tell: a module of three bias-free Linears may have another activation, a forward of its own, hooks, or Linears that do more.  So the
module's own ``forward`` is run once on a symbol in place of its input, with symbols in place of the three Linears, and the
formula that comes out is compared.  Whatever the symbols do not support (shapes, other functions, branches on values, writes to the
module) makes it another kind of module, which the block then calls as it is.
"""
from __future__ import annotations

import operator
import weakref

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules import module as _module

from bitsmoe_b200.quant.linear4 import Linear4

_NAMES = ("gate_proj", "up_proj", "down_proj")
_SILU = (F.silu, torch._C._nn.silu)
_TRACED = weakref.WeakKeyDictionary()       # module -> (what its forward was traced with, whether it was the formula)
_MUL = (torch.mul, torch.multiply, torch.Tensor.mul, torch.Tensor.multiply, torch.Tensor.__mul__)


class _Symbol:
    """A value known by the formula it came from."""

    def __init__(self, *formula):
        self.formula = formula

    def __mul__(self, other):
        return _Symbol("mul", self, other) if isinstance(other, _Symbol) else NotImplemented

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        if func in _SILU and len(args) == 1 and isinstance(args[0], _Symbol):
            return cls("silu", args[0])
        if func in _MUL and len(args) == 2 and all(isinstance(a, _Symbol) for a in args) and not kwargs:
            return cls("mul", *args)
        return NotImplemented

    def same(self, other) -> bool:
        if len(self.formula) != len(other.formula) or self.formula[0] != other.formula[0]:
            return False
        mine, theirs = self.formula[1:], other.formula[1:]
        return (all(a.same(b) for a, b in zip(mine, theirs)) or
                (self.formula[0] == "mul" and mine[0].same(theirs[1]) and mine[1].same(theirs[0])))


class _StandIn:
    """``self`` of the traced forward: the module with its Linears replaced by symbols.  It hands out plain values, a configuration and
    activations without state of their own, so that a forward that keeps a record of its calls neither runs nor passes."""

    def __init__(self, module):
        object.__setattr__(self, "_module", module)

    def __getattr__(self, name):
        if name in _NAMES:
            return lambda x: _Symbol(name, x) if isinstance(x, _Symbol) else NotImplemented
        value = getattr(self._module, name)
        if name == "config" or value is None or type(value) in (bool, int, float, str) or any(value is f for f in _SILU) or (
                isinstance(value, nn.Module) and (type(value) is nn.SiLU or type(value).__module__ == "transformers.activations")):
            return value
        raise AttributeError(name)

    def __setattr__(self, name, value):
        raise AttributeError(name)


def _hooked(m) -> bool:
    return bool(m._forward_hooks or m._forward_pre_hooks or "forward" in m.__dict__)


def _traces_as_swiglu(module) -> bool:
    x = _Symbol("x")
    try:
        got = type(module).forward(_StandIn(module), x)
    except Exception:
        return False
    want = _Symbol("down_proj", _Symbol("mul", _Symbol("silu", _Symbol("gate_proj", x)), _Symbol("up_proj", x)))
    return isinstance(got, _Symbol) and got.same(want)


def runs_as_swiglu(module) -> bool:
    """True for an unhooked module whose gate_proj, up_proj and down_proj are bias-free Linears (of nn.Linear itself or Linear4) and whose
    forward is down_proj(silu(gate_proj(x)) * up_proj(x)).  What can change without the module being another object is looked at in
    every call; the forward is traced again when its class, its children or one of its attributes has changed."""
    if not isinstance(module, nn.Module) or type(module).__call__ is not nn.Module.__call__ or _hooked(module):
        return False
    if _module._global_forward_hooks or _module._global_forward_pre_hooks:
        return False
    children = module._modules
    for n in _NAMES:
        m = children.get(n)
        if type(m) is nn.Linear:
            if m._parameters.get("bias") is not None:
                return False
        elif type(m) is not Linear4:
            return False
    attributes = module.__dict__
    state = [type(module).forward, *children.values(), *[attributes[k] for k in attributes if k[0] != "_"]]
    known = _TRACED.get(module)
    if known is None or len(known[0]) != len(state) or not all(map(operator.is_, known[0], state)):
        known = (state, _traces_as_swiglu(module))
        _TRACED[module] = known
    if not known[1]:
        return False
    for m in children.values():
        if m is not None and (m._forward_hooks or m._forward_pre_hooks or "forward" in m.__dict__):
            return False
    return True
