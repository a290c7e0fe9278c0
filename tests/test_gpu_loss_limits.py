"""The 8-bit classification losses and the balance loss at the ends of what they take: infinite logits of sigmoid routers, sums of
very many equal terms, a row of more than 2^30 classes, gammas below zero."""
import math

import numpy as np
import pytest
import torch

from detr_amd import _lib, losses
from detr_amd._lib import lib
from oracle import balance_loss as oracle
from test_gpu_balance_loss import check_set
from test_gpu_saved_logits import check_focal

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("E", [3, 8, 13, 40, 160, 700])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per_image", [False, True])
def test_gradient_of_infinite_logits_with_sigmoid_scores(E, dtype, per_image):
    """sigmoid(+inf) = 1: the loss is finite, and so is its gradient (0 at the infinite logit, whose score no longer moves).
    The bound of tests/test_gpu_balance_loss.py: scores off by (5 D + 40) u with D the largest finite |x|, below 8 here."""
    gen = torch.Generator().manual_seed(E)
    x = torch.randn(3, 21, E, generator=gen).clamp(-7, 7).to(DTYPES[dtype])
    x[0, 3, 1] = x[1, 4, E - 1] = x[1, 20, 0] = math.inf
    x[2, 7, :2] = math.inf
    x[2, 8] = math.inf                                     # even scores
    x[0, 5, 0], x[0, 5, 2] = -math.inf, math.inf
    leaf = x.cuda().requires_grad_(True)
    out = losses.balance_losses(leaf, 2, scores="sigmoid", per_image=per_image)
    (grad,) = torch.autograd.grad(out.balance.sum(), leaf)
    want = oracle.balance_losses(x.double().numpy(), 2, scores="sigmoid", per_image=per_image,
                                 grad_balance=np.ones(3 if per_image else 1))
    assert np.isfinite(want["grad"]).all() and bool(grad.isfinite().all())
    assert bool((grad[leaf.isinf()] == 0).all())
    t = (5 * 8 + 40) * U
    np.testing.assert_allclose(out.balance.detach().double().cpu().numpy().reshape(-1), want["balance"], rtol=t + 314 * U, atol=0)
    fi = torch.finfo(grad.dtype)
    p, f = want["p"], np.abs(want["f"])[:, None]
    scale = np.abs(want["gb"])[:, None, None] * (f + (p * f).sum(-1, keepdims=True))
    bound = t * p * scale + (fi.eps / 2 + 4 * U) * np.abs(want["grad"]) + fi.smallest_normal * fi.eps + 2.0 ** -126 * (1 + scale)
    off = np.abs(grad.double().cpu().numpy() - want["grad"])
    assert (off <= bound).all(), float((off / bound).max())


def test_sums_of_very_many_equal_rows_cross_entropy():
    """2730 rows a lane, all of weight 0.1: added up in float32 they would be off by 450 u, each rounding to the same side.
    A row's loss is log 2: the constant, the product with the weight and three roundings of the sums' ends, and the hardware's
    logarithm to a step: 16 u; the sum of the weights three roundings."""
    rows = 1536 * 256 * 2730
    assert 2 * rows < 1 << 31
    x = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda")
    cls = torch.zeros(rows, dtype=torch.int64, device="cuda")
    weight = torch.full((2,), 0.1, device="cuda")
    out = torch.zeros(2, device="cuda")
    partials = torch.empty(_lib.CLS_LOSS_PARTIALS, dtype=torch.float64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = lib.dm_cross_entropy_saved(x.data_ptr(), 1, cls.data_ptr(), weight.data_ptr(), rows, 2, -100, out.data_ptr(), None, None,
                                    partials.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    loss, inverse = out.tolist()
    assert abs(inverse * rows * float(np.float32(0.1)) - 1) <= 4 * U
    assert abs(loss / math.log(2) - 1) <= 16 * U


def test_sums_of_very_many_equal_logits_focal():
    """341 times 16 logits a lane, all 0: each is 0.75 log 2 / 4 (1/x and the logarithm to a step, six products), a lane's 16 are
    added in float32 (at most six roundings), the rest in 64 bits: 16 u, where a float32 sum would be off by 43 u."""
    n = 1534 * 4096 * 341
    assert n < 1 << 31
    x = torch.zeros(n // 2, 2, dtype=torch.bfloat16, device="cuda")
    cls = torch.full((n // 2,), 2, dtype=torch.int64, device="cuda")
    loss = losses.focal_loss(x, cls, float(n), saved_bits=8).item()
    assert abs(loss / (0.75 * math.log(2) / 4) - 1) <= 20 * U


def test_sums_of_very_many_equal_rows_balance():
    """2731 rows a lane, the same row: a lane's float32 runs are 64 rows long, beyond that sums are of 64 bits.  A score 1/10 is
    good to a step and the product's rounding, so balance = 1 to (64 + 8) u; log 10 to 5 u (its logarithm to a step, constant,
    product, sum), twice in the square: 12 u.  In float32 throughout both were off by 450 u."""
    B, Q, E = 48, 256 * 2731, 10
    long = torch.zeros(B, Q, E, dtype=torch.bfloat16, device="cuda")
    short = torch.zeros(B, 1, E, dtype=torch.bfloat16, device="cuda")
    out = losses.balance_losses([short] * 7 + [long] + [short] * 8, 2, per_image=True)
    for s in (7, 0):
        assert float((out.balance[s].double() - 1).abs().max()) <= 72 * U
        assert float((out.z[s].double() / math.log(10) ** 2 - 1).abs().max()) <= 14 * U
    assert out.counts[7].unique().tolist() == [0, Q] and out.counts[7].sum().item() == 2 * B * Q


@pytest.mark.parametrize("E", [9, 30, 100, 300, 600])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_runs_of_rows_in_a_lane(E, dtype):
    """Rows beyond one float32 run of a lane (64), and a run that ends with the rows: with so many images a workgroup each."""
    lanes = 1 if E <= 16 else 2 if E <= 32 else 8 if E <= 128 else 32 if E <= 512 else 64
    trip = 256 // lanes
    for Q in (64 * trip, 64 * trip + 1, 131 * trip - 1):
        gen = torch.Generator().manual_seed(E + Q)
        x = torch.randn(1, Q, E, generator=gen).to(DTYPES[dtype])
        long = torch.zeros(48, Q, E, dtype=x.dtype, device="cuda")
        long[5] = x[0].cuda()
        short = torch.zeros(48, 1, E, dtype=x.dtype, device="cuda")
        out = losses.balance_losses([long] + [short] * 15, 2, per_image=True)
        want = oracle.balance_losses(x.double().numpy(), 2, per_image=True)
        check_set(x, want, out.balance[0, 5:6], out.z[0, 5:6], out.counts[0, 5:6], None)


def test_a_row_of_more_than_2_30_classes():
    """No class is the row's: every logit is a negative one, its gradient positive."""
    C = (1 << 30) + 1000
    x = torch.zeros(1, C, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    for label, hot in ((C, None), (C - 1, C - 1), (5, 5)):
        cls = torch.full((1,), label, dtype=torch.int64, device="cuda")
        (grad,) = torch.autograd.grad(losses.focal_loss(x, cls, 1.0, saved_bits=8), x)
        negative = (grad[0] <= 0).nonzero().flatten().tolist()
        assert negative == ([] if hot is None else [hot])
        del grad


@pytest.mark.parametrize("C", [1, 2, 3, 11, 91, 128, 130, 300, 1203])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rows_that_do_not_count_are_part_of_the_ranges(C, dtype):
    """They widen a block's step with what they hold within +-20; what lies beyond, infinities and NaN count as 0."""
    gen = torch.Generator().manual_seed(C)
    Q = 37 if C < 1000 else 5
    x = torch.randn(5, Q, C, generator=gen)
    cls = torch.where(torch.rand(5, Q, generator=gen) < 0.2, torch.randint(0, C, (5, Q), generator=gen), C)
    ignored = torch.rand(5, Q, generator=gen) < 0.4
    ignored[1] = True
    ignored[4, Q - 1] = C % 2 == 0
    cls[ignored] = -1
    x[ignored] *= 8
    x = x.clamp(-20, 20).to(DTYPES[dtype])
    check_focal(x, cls, ignore_index=-1)
    held = torch.rand(x.shape, generator=gen)
    for value, low in ((20.0, 0.9), (-20.0, 0.8), (math.inf, 0.7), (-math.inf, 0.6), (math.nan, 0.5), (25.0, 0.4), (-30000.0, 0.3)):
        x[ignored[..., None] & (held > low) & (held < low + 0.1)] = value
    dev = x.cuda().requires_grad_(True)
    loss = losses.focal_loss(dev, cls.cuda(), 3.0, ignore_index=-1, saved_bits=8)
    (grad,) = torch.autograd.grad(loss, dev)
    y = torch.where(ignored[..., None] & ~(x.abs() <= 20), torch.zeros_like(x), x)
    dev = y.cuda().requires_grad_(True)
    same = losses.focal_loss(dev, cls.cuda(), 3.0, ignore_index=-1, saved_bits=8)
    assert torch.equal(loss, same) and torch.equal(grad, torch.autograd.grad(same, dev)[0])
    check_focal(y, cls, ignore_index=-1)
    # (the last logit is a live one beyond the clamp: what is behind it in the block adds nothing)
    cls[4, Q - 1], y[4, Q - 1] = C, 40.0
    check_focal(y, cls, ignore_index=-1)


def test_a_gamma_below_zero_is_refused():
    x = torch.randn(3, 7, 5, device="cuda")
    cls = torch.zeros(3, 7, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="gamma"):
        losses.focal_loss(x, cls, 1.0, gamma=-0.5, saved_bits=8)
    seen = []
    module = losses.FocalLoss(0.25, -0.5, 5, fallback=lambda *a: seen.append(a) or "own", saved_bits=8)
    assert module(x, cls, 1.0) == "own" and len(seen) == 1
    with pytest.raises(ValueError, match="gamma"):
        losses.FocalLoss(0.25, -0.5, 5, saved_bits=8)(x, cls, 1.0)
    # (the 32-bit form has it)
    assert losses.focal_loss(x, cls, 1.0, gamma=-0.5).isfinite()
    assert losses.FocalLoss(0.25, -0.5, 5)(x, cls, 1.0).isfinite()
