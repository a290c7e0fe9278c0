"""How the nodes of the 8-bit classification losses and of the balance loss stand in torch's machinery: hooks on saved tensors,
checkpointing, forward mode, tracing, a first call inside a capture, inputs that need no gradient."""
import pytest
import torch

from detr_amd import losses

pytestmark = pytest.mark.gpu


def data(seed=0, B=4, Q=60, C=21):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(B, Q, C, generator=gen).cuda(), torch.randint(0, C, (B, Q), generator=gen).cuda()


def calls(cls, mask=None):
    """name -> (loss of logits, least bytes that it keeps for the backward pass beside its inputs)"""
    weight = torch.rand(21, generator=torch.Generator().manual_seed(9)).cuda() + 0.5
    n = cls.numel() * 21

    def balance(scores):
        def loss(x):
            out = losses.balance_losses([x, 2 * x], 3, mask=mask, scores=scores)
            return out.balance.sum() if out.z is None else out.balance.sum() + out.z.sum()
        return loss

    return {"focal": (lambda x: losses.focal_loss(x, cls, 3.0, saved_bits=8), n),
            "ce": (lambda x: losses.cross_entropy(x, cls, weight, saved_bits=8), n),
            "balance": (balance("softmax"), 4 * 2 * 22), "sigmoid": (balance("sigmoid"), 4 * 2 * 22)}


NAMES = ["focal", "ce", "balance", "sigmoid"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_and_tracing_are_refused(name):
    import torch.autograd.forward_ad as fw

    x, cls = data()
    loss, _ = calls(cls)[name]
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            loss(fw.make_dual(x, torch.ones_like(x)))
    loss(x)
    with pytest.raises(RuntimeError):
        torch.jit.trace(loss, (x,), check_trace=False)
    counts = lambda t: losses.expert_counts(t, 2)
    with pytest.raises(RuntimeError):
        torch.jit.trace(counts, (x,), check_trace=False)
    with fw.dual_level():                # (whole numbers have no tangent)
        assert torch.equal(counts(fw.make_dual(x, torch.ones_like(x))), counts(x))
