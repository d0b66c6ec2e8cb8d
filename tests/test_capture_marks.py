"""Which leaves an eager graph marks, so that a capture on them is refused: the process would end in its backward pass."""

import pytest
import torch

from keep_amd import _grad


@pytest.fixture
def capturing(monkeypatch):
    state = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state[0])

    def switch(on):
        state[0] = on
    return switch


@pytest.mark.parametrize("argument", [
    lambda w, a, b: w + 0.5 * (b @ a),                      # a merged low-rank update
    lambda w, a, b: (w + 0.5 * (b @ a)).to(torch.bfloat16).transpose(0, 1),
    lambda w, a, b: torch.cat([w, b @ a]),
    lambda w, a, b: w * b.sum() + a.mean(),
])
def test_leaves_behind_steps_of_several_inputs(capturing, argument):
    leaves = [torch.randn(4, 4, requires_grad=True) for _ in range(3)]
    held = _grad.mark(argument(*leaves) * 2)
    capturing(True)
    for i in range(3):  # each of the three alone
        others = [t if j == i else t.detach().requires_grad_() for j, t in enumerate(leaves)]
        with pytest.raises(RuntimeError, match="eager graph"):
            _grad.check_capture(argument(*others))
    _grad.check_capture(argument(*(t.detach().requires_grad_() for t in leaves)))
    del held
    _grad.check_capture(argument(*leaves))


def test_the_error_names_what_else_holds_the_node(capturing):
    """A held node keeps its stream after the graph is gone, so the capture stays refused, and leaves of its own pass."""
    w = torch.randn(3, requires_grad=True)
    edge = torch.autograd.graph.get_gradient_edge(w)
    held = _grad.mark(w * 2)
    del held
    capturing(True)
    with pytest.raises(RuntimeError, match="what else holds the node"):
        _grad.check_capture(w)
    _grad.check_capture(w.detach().requires_grad_())
    del edge
    _grad.check_capture(w)


def test_a_long_history_is_not_walked():
    h = torch.randn(3, requires_grad=True)
    for _ in range(1000):
        h = h * 1.01 + h
    assert _grad._leaf_nodes(h.grad_fn) == []
