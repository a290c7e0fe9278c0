"""The calls that keep 8 bits per logit check their arguments on the host, before any HIP call (CPU)."""
import pytest
import torch

from detr_amd import _lib, criterion, losses
from detr_amd._lib import lib

P = 0x1000          # an address that is checked and never followed
BAD, BIG = _lib.E_INVALID_ARG, _lib.E_UNSUPPORTED


def focal(logits=P, dtype=0, cls=P, rows=5, C=4, out=P, codes=P, heads=P, partials=P, status=P):
    return lib.dm_focal_loss_saved(logits, dtype, cls, rows, C, 0.25, 2.0, 1.0, 0, 0, out, codes, heads, partials, status, None)


def ce(logits=P, dtype=0, cls=P, rows=5, C=4, out=P, codes=P, steps=P, partials=P, status=P):
    return lib.dm_cross_entropy_saved(logits, dtype, cls, None, rows, C, -100, out, codes, steps, partials, status, None)


@pytest.mark.parametrize("call", [focal, ce])
def test_forward_arguments_are_refused(call):
    marks = "heads" if call is focal else "steps"
    for wrong in (dict(rows=-1), dict(C=0), dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(cls=None), dict(out=None),
                  dict(partials=None), dict(status=None), dict(codes=None), {marks: None}):
        assert call(**wrong) == BAD, wrong
    assert call(rows=1 << 20, C=1 << 11) == BIG
    if call is focal:
        assert focal(codes=P + 1) == BAD and focal(heads=P + 2) == BAD


def test_backward_arguments_are_refused():
    def focal_back(codes=P, heads=P, dtype=0, cls=P, rows=5, C=4, g=P, out=P):
        return lib.dm_focal_loss_from_saved(codes, heads, dtype, cls, rows, C, 0.25, 2.0, 1.0, 0, 0, g, out, None)

    def ce_back(codes=P, heads=P, dtype=0, cls=P, rows=5, C=4, g=P, out=P, inv=P):
        return lib.dm_cross_entropy_from_saved(codes, heads, dtype, cls, None, rows, C, -100, inv, g, out, None)

    for call in (focal_back, ce_back):
        for wrong in (dict(codes=None), dict(heads=None), dict(dtype=9), dict(cls=None), dict(rows=-1), dict(C=0), dict(g=None),
                      dict(out=None)):
            assert call(**wrong) == BAD, wrong
        assert call(rows=1 << 20, C=1 << 11) == BIG
        assert call(rows=0, codes=None, heads=None, cls=None, out=None, g=None) == 0
    assert ce_back(inv=None) == BAD and focal_back(codes=P + 2) == BAD


def test_python_refusals():
    x, cls = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda b: losses.focal_loss(x, cls, 1, saved_bits=b), lambda b: losses.cross_entropy(x, cls, saved_bits=b)):
        with pytest.raises(ValueError, match="saved_bits"):
            call(4)
        with pytest.raises(RuntimeError, match="GPU"):
            call(8)

    class Criterion(torch.nn.Module):
        pass

    for kwargs in (dict(saved_bits=8), dict(saved_bits=16, fused_consumers=True)):
        with pytest.raises(ValueError, match="saved_bits"):
            criterion.attach(Criterion(), **kwargs)
