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


def test_a_gamma_below_zero_is_refused():
    # (a call of no rows ends on the host)
    assert lib.dm_focal_loss_from_saved(None, None, 0, None, 0, 4, 0.25, -0.5, 1.0, 0, 0, None, None, None) == _lib.E_INVALID_ARG
    assert lib.dm_focal_loss_from_saved(None, None, 0, None, 0, 4, 0.25, 0.5, 1.0, 0, 0, None, None, None) == 0
    with pytest.raises(ValueError, match="gamma"):
        losses._loss_nodes().focal_losses([torch.zeros(1, 2)], [torch.zeros(1, dtype=torch.int64)], 0.25, -0.5, [1.0], None, True,
                                          torch.zeros(1, dtype=torch.int32))


class FocalLoss(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.alpha, self.gamma, self.n_cls = 0.25, 2.0, 6

    def forward(self, inputs, targets, num_boxes):
        return "own"


class Criterion(torch.nn.Module):
    def __init__(self):
        super().__init__()
        import detr_amd

        self.matcher = detr_amd.HungarianMatcher()
        self.cls_criterion = FocalLoss()
        self.n_cls = 6

    def calc_cls_loss_with_ignore(self, outputs, targets, pos_indices, neg_indices):
        return "own"

    def forward(self, outputs, targets):
        return None


def bits_of(monkeypatch, c):
    """The saved_bits that the two classification losses of an attached criterion are called with."""
    got = []
    monkeypatch.setattr(losses, "_takes", lambda *a, **k: True)
    monkeypatch.setattr(losses, "focal_loss", lambda *a, saved_bits=32, **k: got.append(saved_bits))
    c.cls_criterion(torch.zeros(2, 3, 6), torch.zeros(2, 3, dtype=torch.int64), 1)
    none = [(torch.zeros(0, dtype=torch.int64),) * 2] * 2
    c.calc_cls_loss_with_ignore({"pred_logits": torch.zeros(2, 3, 6)}, [], none, [torch.zeros(0, dtype=torch.int64)] * 2)
    monkeypatch.undo()
    return got


def test_a_second_attach_with_other_bits(monkeypatch):
    for first, second in ((32, 8), (8, 32), (8, 8)):
        c = Criterion()
        criterion.attach(c, fused_consumers=True, saved_bits=first)
        assert bits_of(monkeypatch, c) == [first, first]
        criterion.attach(c, fused_consumers=True, saved_bits=second)
        assert bits_of(monkeypatch, c) == [second, second]
        criterion.attach(c)                                # (asks for nothing: nothing changes)
        assert bits_of(monkeypatch, c) == [second, second]
        criterion.detach(c)
        assert c.cls_criterion(None, None, None) == "own" and c.calc_cls_loss_with_ignore(None, None, None, None) == "own"


def test_bits_without_the_fused_consumers_are_refused():
    c = Criterion()
    criterion.attach(c)
    with pytest.raises(ValueError, match="detach"):
        criterion.attach(c, fused_consumers=True, saved_bits=8)
    criterion.attach(c, fused_consumers=True)              # (as before: harmless)
    criterion.detach(c)
    criterion.attach(c, fused_consumers=True, saved_bits=8)
    assert "forward" in c.cls_criterion.__dict__


def test_fusing_a_module_again(monkeypatch):
    got = []
    module = FocalLoss()
    for bits in (32, 8, 32):
        assert criterion.fuse_cls_criterion(module, saved_bits=bits)
        monkeypatch.setattr(losses, "_takes", lambda *a, **k: True)
        monkeypatch.setattr(losses, "focal_loss", lambda *a, saved_bits=32, **k: got.append(saved_bits))
        module(torch.zeros(2, 3, 6), torch.zeros(2, 3, dtype=torch.int64), 1)
        monkeypatch.undo()
    assert got == [32, 8, 32]
    other = FocalLoss()
    other.forward = lambda *a: "somebody else's"
    assert criterion.fuse_cls_criterion(other)
    assert not criterion.fuse_cls_criterion(other, saved_bits=8) and other() == "somebody else's"


def test_a_gamma_below_zero_stays_with_the_module():
    module = FocalLoss()
    module.gamma = -0.5
    criterion.fuse_cls_criterion(module, saved_bits=8)
    assert not losses._takes(torch.zeros(2, 3, 6), torch.zeros(2, 3, dtype=torch.int64), 8, gamma=-0.5)
    assert module(torch.zeros(2, 3, 6), torch.zeros(2, 3, dtype=torch.int64), 1) == "own"


def test_modules_saved_before_there_was_a_choice():
    for module in (losses.FocalLoss(0.25, 2.0, 6, fallback=print), losses.CrossEntropy(torch.ones(6), fallback=print)):
        del module.__dict__["saved_bits"]
        again = pickle.loads(pickle.dumps(module))
        assert again.saved_bits == 32
        again(torch.zeros(2, 3, 6), torch.zeros(2, 3, dtype=torch.int64), 1)          # (CPU: the fallback)
