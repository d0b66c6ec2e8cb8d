"""What the differentiable operators share."""

from __future__ import annotations

import torch


def wanted(*tensors) -> bool:
    """Whether autograd records a call on these tensors."""

    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


_EAGER = "keep_amd: eager graph"


def check_capture(*tensors) -> list:
    """The gradient nodes of the leaves among ``tensors``, marked, to be held until the call is recorded; raises where
    a graph capture would record a call on leaves that a live eager graph of these operators holds.

    A leaf has one gradient node at a time, bound to the stream that made it. While an eager graph is alive, a
    backward pass under capture would make that other stream wait on the capturing one, which ends the process. Eager
    calls leave a mark on the node, which lives as long as some graph holds it."""

    nodes = []
    capturing = torch.cuda.is_current_stream_capturing()
    for t in tensors:
        if t is None or not t.requires_grad or not t.is_leaf:
            continue
        nodes.append(torch.autograd.graph.get_gradient_edge(t).node)
        notes = nodes[-1].metadata
        if not capturing:
            notes[_EAGER] = True
        elif _EAGER in notes:
            raise RuntimeError("graph capture of a differentiable call on a leaf that an eager graph still holds: drop "
                               "that graph's outputs first, or capture on leaves of its own")
    return nodes
