"""What the C++ nodes refuse before they look for a GPU, and the options of modules and attached criteria (CPU)."""
import pickle

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from detr_amd import _lib, criterion, losses
from detr_amd._lib import lib


def node_calls():
    nodes = losses._loss_nodes()
    cls, status = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    return {"focal": lambda x: nodes.focal_losses([x], [cls], 0.25, 2.0, [1.0], None, True, status),
            "ce": lambda x: nodes.cross_entropies([x], [cls], None, -100, True, status),
            "balance": lambda x: nodes.balance_losses([x], 1, [None], [None], None, False, False, status)[0]}


@pytest.mark.parametrize("name", ["focal", "ce", "balance"])
def test_forward_mode_and_tracing_are_refused(name):
    call = node_calls()[name]
    x = torch.zeros(2, 3, 4)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(x, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match="trace"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(NotImplementedError, match="trace"):
        make_fx(call)(x)
    with pytest.raises(RuntimeError, match="GPU"):          # (neither: what the call says of its tensors)
        call(x)


def test_forward_mode_of_the_weight_is_refused():
    nodes = losses._loss_nodes()
    x, cls, status = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nodes.cross_entropies([x], [cls], fw.make_dual(torch.ones(4), torch.ones(4)), -100, True, status)


def test_tracing_the_counts_is_refused():
    status = torch.zeros(1, dtype=torch.int32)
    call = lambda x: losses._loss_nodes().expert_counts([x], 1, [None], False, status)
    for trace in (lambda: torch.jit.trace(call, (torch.zeros(2, 3, 4),), check_trace=False), lambda: make_fx(call)(torch.zeros(2, 3, 4))):
        with pytest.raises(NotImplementedError, match="trace"):
            trace()
