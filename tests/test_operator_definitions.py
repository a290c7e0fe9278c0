"""The plain and the 64-bit forms of perf/operators.py state the same operators as the oracles that the tests hold the kernels to,
rows that do not count among them (CPU)."""
import math

import numpy as np
import pytest
import torch

from oracle import balance_loss, saved_logits
from perf import operators

U = 2.0 ** -24


def cls_inputs(dtype, shape, seed, ignored):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=gen) * 2 - 1).to(operators.DTYPES[dtype])
    cls = torch.where(torch.rand(shape[:-1], generator=gen) < 0.2, torch.randint(0, C, shape[:-1], generator=gen), C)
    return x, torch.where(torch.rand(shape[:-1], generator=gen) < ignored, -1, cls)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("C", [2, 3, 11, 91, 130, 300])
@pytest.mark.parametrize("ignored", [0.0, 0.2, 0.9])
def test_focal(dtype, C, ignored):
    x, cls = cls_inputs(dtype, (3, 41, C), C, ignored)
    case = operators._focal("", 3, 41, C, dtype, 1.5, ignored)
    state = {"case": case, "logits": x, "cls": cls, "boxes": 7.0, "grad": torch.tensor(1.0), "weight": None}
    loss, grad, _ = saved_logits.focal(x.double().numpy(), cls.numpy(), 7.0, 0.25, 1.5, -1)
    exact, plain = operators._exact_focal(case, state), operators._plain_focal(case, state)
    # (two ways to write the same in 64 bits; the plain form in 32, rounded to the type)
    np.testing.assert_allclose(exact["loss"], loss, rtol=1e-12, atol=1e-300)
    np.testing.assert_allclose(exact["grad"], grad, rtol=1e-10, atol=1e-15)
    np.testing.assert_allclose(plain["grad"].double().numpy(), grad, rtol=500 * U + torch.finfo(x.dtype).eps / 2, atol=1e-12)


@pytest.mark.parametrize("C", [2, 5, 92, 300])
@pytest.mark.parametrize("ignored", [0.0, 0.3])
def test_cross_entropy(C, ignored):
    x, cls = cls_inputs("float32", (3, 41, C), C, ignored)
    cls = cls.clamp(max=C - 1)
    weight = torch.rand(C, generator=torch.Generator().manual_seed(C)) + 0.1
    case = operators._ce("", 3, 41, C, ignored=ignored)
    state = {"case": case, "logits": x, "cls": cls, "grad": torch.tensor(1.0), "weight": weight}
    loss, grad, p = saved_logits.cross_entropy(x.double().numpy(), cls.numpy(), weight.double().numpy(), -1)
    exact = operators._exact_ce(case, state)
    np.testing.assert_allclose(exact["loss"], loss, rtol=1e-12)
    np.testing.assert_allclose(exact["grad"], grad, rtol=1e-10, atol=1e-14)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("per_image", [False, True])
@pytest.mark.parametrize("given", [False, True])
def test_balance(scores, per_image, given):
    gen = torch.Generator().manual_seed(5)
    B, Q, E, k = 3, 17, 9, 2
    x = torch.randn(B, Q, E, generator=gen)
    x[..., 4] = -math.inf
    mask = torch.rand(B, Q, generator=gen) < 0.7
    experts = torch.randint(-1, E, (B, Q, k), generator=gen) if given else None
    groups = (1, B) if per_image else (1,)
    case = operators._balance("", 1, B, Q, E, k, scores=scores, per_image=per_image, padded=0.3, given=given)
    state = {"case": case, "logits": [x], "mask": mask, "given": [experts] if given else None,
             "grad_balance": torch.rand(groups, generator=gen), "grad_z": torch.rand(groups, generator=gen)}
    want = balance_loss.balance_losses(x.double().numpy(), k, mask.numpy(), experts.numpy() if given else None, None, scores, per_image,
                                       state["grad_balance"][0].double().numpy(),
                                       None if scores == "sigmoid" else state["grad_z"][0].double().numpy())
    exact = operators._exact_balance(case, state)
    np.testing.assert_allclose(exact["balance"].reshape(-1), want["balance"], rtol=1e-12)
    np.testing.assert_allclose(exact["grads"][0], want["grad"], rtol=1e-9, atol=1e-13)
    if scores == "softmax":
        np.testing.assert_allclose(exact["z"].reshape(-1), want["z"], rtol=1e-12)
    assert np.array_equal(operators._plain_balance(case, state)["counts"].numpy().reshape(want["counts"].shape), want["counts"])
