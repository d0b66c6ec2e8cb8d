"""What the differentiable operators share."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

_EAGER = "keep_amd: eager graph"
_NODES = 12  # steps looked at between a call's argument and its leaves: views, casts, a merge of weights


def wanted(*tensors) -> bool:
    """Whether autograd records a call on these tensors. A forward-mode tangent counts too: the operators' functions
    have no rule for one, and refuse it."""

    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:  # inside a dual_level
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _leaf_nodes(node) -> list:
    """The gradient nodes of the leaves near ``node`` (parameters, their views, casts and sums)."""

    leaves, todo = [], [node]
    for node in todo:
        if hasattr(node, "variable"):
            leaves.append(node)
        elif len(todo) < _NODES:
            todo.extend(f for f, _ in node.next_functions if f is not None)
    return leaves


def check_capture(*tensors) -> None:
    """Refuse to record a graph capture of a call on leaves that a live eager graph of these operators holds.

    A leaf has one gradient node at a time, bound to the stream that made it. While an eager graph is alive, a
    backward pass under capture would make that other stream wait on the capturing one, which ends the process. Eager
    calls leave a mark on the node (``mark``), which lives as long as something holds it: a graph, or what keeps the
    node itself (a data-parallel wrapper, a stored gradient edge), where the node stays bound to its stream too."""

    if not torch.cuda.is_current_stream_capturing():
        return
    for t in tensors:
        if t is not None and t.requires_grad:
            for node in _leaf_nodes(torch.autograd.graph.get_gradient_edge(t).node):
                if _EAGER in node.metadata:
                    raise RuntimeError("graph capture of a differentiable call on a leaf whose gradient node an eager "
                                       "graph made and something still holds: drop that graph's outputs (and what else "
                                       "holds the node) first, or capture on leaves of its own, as t.detach()"
                                       ".requires_grad_()")


def mark(out: torch.Tensor) -> torch.Tensor:
    """``out`` of an eager call, its leaves' gradient nodes marked."""

    if not torch.cuda.is_current_stream_capturing():
        for first, _ in out.grad_fn.next_functions:
            if first is not None:
                for node in _leaf_nodes(first):
                    node.metadata[_EAGER] = True
    return out


def saved(ctx) -> list:
    """The tensors that the forward pass saved, dense: a saved-tensor hook (offloading, compression) may give them back
    with other strides than it took them."""

    return [None if t is None else t.contiguous() for t in ctx.saved_tensors]


class _Partial(torch.autograd.Function):
    @staticmethod
    def forward(ctx, out, x):
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("a product with codes has no gradient, and this layer's input requires one: detach the input "
                           "to train what does not pass the codes")


def partial(out: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """``out`` of a layer on codes, with a graph from its other paths. Where ``x`` requires a gradient too, the backward
    pass would give it the share of those paths alone, and raises instead."""

    return _Partial.apply(out, x) if wanted(x) else out
