"""What the differentiable operators share."""

from __future__ import annotations

import torch

_EAGER = "keep_amd: eager graph"
_VIEWS = {n + "Backward0" for n in ("View", "UnsafeView", "ReshapeAlias", "Transpose", "Permute", "Select", "Slice")}


def wanted(*tensors) -> bool:
    """Whether autograd records a call on these tensors."""

    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def check_capture(*tensors) -> None:
    """Refuse to record a graph capture of a call on leaves that a live eager graph of these operators holds.

    A leaf has one gradient node at a time, bound to the stream that made it. While an eager graph is alive, a
    backward pass under capture would make that other stream wait on the capturing one, which ends the process. Eager
    calls leave a mark on the node (``mark``), which lives as long as some graph holds it."""

    if not torch.cuda.is_current_stream_capturing():
        return
    for t in tensors:
        if t is not None and t.requires_grad and not t.is_leaf and t._is_view():
            t = t._base
        if t is not None and t.requires_grad and t.is_leaf:
            if _EAGER in torch.autograd.graph.get_gradient_edge(t).node.metadata:
                raise RuntimeError("graph capture of a differentiable call on a leaf that an eager graph still holds: "
                                   "drop that graph's outputs first, or capture on leaves of its own")


def mark(out: torch.Tensor) -> torch.Tensor:
    """``out`` of an eager call, its leaves' gradient nodes marked."""

    if not torch.cuda.is_current_stream_capturing():
        for node, _ in out.grad_fn.next_functions:
            while node is not None and node.name() in _VIEWS:
                node = node.next_functions[0][0]
            if node is not None and hasattr(node, "variable"):  # a leaf's
                node.metadata[_EAGER] = True
    return out
