"""losses.balance_losses / expert_counts / balance_loss_total (dm_balance_loss, dm_balance_backward, dm_expert_counts)
against the 64-bit restatement in oracle/balance_loss.py.

Tolerances, in units u = 2^-24 (half a step of float32, relative).  With D the largest distance of a logit from its row's
largest: x - max rounds once, its product with log2 e twice (the constant, the product) -> 2.5 D u in the exponent, and as much
again from the sum that p is divided by; exp2 and 1/x are good to a step (2 u each, exp2 twice); a sum has up to 16 terms in a
lane and 6 steps over lanes (22 u); three products (3 u).  With sigmoid scores there are two more products, a sum and a 1/x:
    p(1 +- t),  t = (5 D + 40) u.
P and z add up to 300 rows in a lane and 12 partial sums in float32: 312 u more.  A gradient p (gb (f - dot) + gz 2 lse) is
off by t p (|gb| (|f| + sum p |f|) + 2 |gz| (|lse| + 1 + |max|)), the +1 for the relative error of the sum inside the log, and
is rounded once to the logits' type (half a step, and half the smallest subnormal); scores below 2^-126 are zero."""
import numpy as np
import pytest
import torch

from oracle import balance_loss as oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def make(shape, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * spread).to(DTYPES[dtype])


def check_set(x, want, balance, z, counts, grad, sigmoid=False):
    """One set's results (tensors) against the oracle's."""
    xf = x.double().numpy()
    finite = np.where(np.isfinite(xf), xf, np.nan)
    assert np.array_equal(counts.cpu().numpy().reshape(want["counts"].shape), want["counts"])
    if xf.size == 0 or not want["counted"].any():
        spans, tops = 0.0, 0.0
    else:
        rows = finite[want["counted"]]
        spans = float(np.nanmax(np.nanmax(rows, -1) - np.nanmin(rows, -1)))
        tops = float(np.nanmax(np.abs(np.nanmax(rows, -1))))
        if sigmoid:
            spans = max(spans, float(np.nanmax(np.abs(rows))))
    t = (5 * min(spans, 200.0) + 40) * U
    np.testing.assert_allclose(balance.detach().double().cpu().numpy().reshape(-1), want["balance"], rtol=t + 314 * U, atol=0)
    if z is not None:
        lse = np.abs(want["lse"])
        top = float(lse.max()) if lse.size else 0.0
        with np.errstate(over="ignore"):
            square = want["z"].astype(np.float32).astype(np.float64)        # (the lowest value's square is beyond float32)
        np.testing.assert_allclose(z.detach().double().cpu().numpy().reshape(-1), square, rtol=316 * U,
                                   atol=2 * min(top, 1e18) * (t + 4 * U * (min(tops + top, 1e18) + 1)))
    if grad is None:
        return
    fi = torch.finfo(grad.dtype)
    p, f = want["p"], np.abs(want["f"])[:, None]
    scale = np.abs(want["gb"])[:, None, None] * (f + (p * f).sum(-1, keepdims=True)) + \
        2 * np.abs(want["gz"])[:, None, None] * (np.abs(want["lse"])[..., None] + 1 + tops)
    bound = t * p * scale + (fi.eps / 2 + 4 * U) * np.abs(want["grad"]) + fi.smallest_normal * fi.eps + 2.0 ** -126 * (1 + scale)
    off = np.abs(grad.detach().double().cpu().numpy() - want["grad"])
    assert (off <= bound).all(), (float((off / bound).max()), float(np.abs(want["grad"]).max()))


def run_and_check(xs, top_k, masks=None, experts=None, counts=None, scores="softmax", per_image=False, device_xs=None):
    from detr_amd import losses

    S, B = len(xs), xs[0].shape[0]
    dev = device_xs if device_xs is not None else [x.cuda().requires_grad_(True) for x in xs]
    groups = (S, B) if per_image else (S,)
    gen = torch.Generator().manual_seed(7)
    gb, gz = torch.rand(groups, generator=gen) + 0.25, torch.rand(groups, generator=gen) * 0.1 - 0.05
    put = lambda v: None if v is None else [None if t is None else t.cuda() for t in v]
    out = losses.balance_losses(dev, top_k, mask=put(masks), experts=put(experts), counts=None if counts is None else counts.cuda(),
                                scores=scores, per_image=per_image)
    assert out.balance.shape == groups and out.counts.shape == groups + (xs[0].shape[2],) and out.counts.dtype == torch.int64
    sigmoid = scores == "sigmoid"
    if sigmoid:
        assert out.z is None
        grads = torch.autograd.grad(out.balance, dev, gb.cuda())
    else:
        grads = torch.autograd.grad([out.balance, out.z], dev, [gb.cuda(), gz.cuda()])
    for s, x in enumerate(xs):
        want = oracle.balance_losses(x.double().numpy(), top_k, None if masks is None or masks[s] is None else masks[s].numpy(),
                                     None if experts is None else experts[s].numpy(),
                                     None if counts is None else counts[s].numpy(), scores, per_image,
                                     gb[s].numpy(), None if sigmoid else gz[s].numpy())
        assert grads[s].dtype == x.dtype and grads[s].shape == x.shape
        check_set(x, want, out.balance[s], None if sigmoid else out.z[s], out.counts[s], grads[s], sigmoid)
    if experts is None:
        again = losses.expert_counts([d.detach() for d in dev], top_k, mask=put(masks), per_image=per_image)
        assert torch.equal(again, out.counts)
    return out, grads


# (every width of a row's group of lanes and of a lane's share, odd ends, one expert, the largest number)
@pytest.mark.parametrize("E", [1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 16, 17, 24, 31, 32, 33, 48, 49, 64, 65, 96, 97, 100, 128, 129, 160, 192, 193,
                               255, 256, 257, 384, 385, 512, 513, 768, 769, 1000, 1023, 1024])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_number_of_experts(E, dtype):
    xs = [make((2, q, E), dtype, 100 * E + q) for q in (5, 1)]
    run_and_check(xs, min(E, 3))
    run_and_check(xs, 1, scores="sigmoid", per_image=True)


# (the same with rows for several workgroups per set, and per image)
@pytest.mark.parametrize("E", [1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 16, 17, 24, 31, 32, 33, 48, 49, 64, 65, 96, 97, 100, 128, 129, 160, 192, 193,
                               255, 256, 257, 384, 385, 512, 513, 768, 769, 1000, 1023, 1024])
@pytest.mark.parametrize("per_image", [False, True])
def test_more_rows_than_one_workgroup_takes(E, per_image):
    Q = 1300 * 16 // max(E, 16) + 3
    xs = [make((2, q, E), "f32", 100 * E + q) for q in (Q, 7)]
    run_and_check(xs, min(E, 2), per_image=per_image)
    run_and_check([make((1, Q, E), "bf16", E)], min(E, 5), scores="sigmoid", per_image=per_image)


@pytest.mark.parametrize("k", [1, 2, 4, 7, 8, 16, 33, 40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_number_of_choices(k, dtype):
    run_and_check([make((3, 11, 40), dtype, k)], k)


@pytest.mark.parametrize("E,k", [(20, 17), (24, 24), (33, 9), (90, 15), (96, 96), (100, 17), (256, 16), (256, 20), (300, 64), (1000, 31), (1024, 1024)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_many_choices(E, k, dtype):
    x = make((2, 23, E), dtype, E + k)
    run_and_check([x], k)
    x[:, ::2] = (x[:, ::2].float() * 4).round().div(4).to(x.dtype)          # (equal ones, across lanes and in one lane's share)
    x[:, 5, ::2] = -float("inf")
    x[0, 7] = x[0, 7, 0]
    run_and_check([x], k)


@pytest.mark.parametrize("S,B,Q,E,k", [(1, 1, 1, 8, 2), (1, 1, 2000, 8, 1), (6, 4, 150, 16, 2), (2, 7, 301, 24, 3), (18, 2, 9, 6, 2),
                                       (1, 300, 3, 10, 2), (3, 33, 65, 64, 4)])
@pytest.mark.parametrize("per_image", [False, True])
def test_sizes(S, B, Q, E, k, per_image):
    xs = [make((B, Q + 3 * (s % 2), E), "f32", S * B + s) for s in range(S)]
    run_and_check(xs, k, per_image=per_image)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per_image", [False, True])
def test_masks_and_disabled_experts(scores, dtype, per_image):
    B, Q, E, k = 4, 37, 20, 3
    gen = torch.Generator().manual_seed(5)
    xs, masks = [], []
    for s in range(3):
        x = make((B, Q, E), dtype, 40 + s)
        x[..., 3] = -float("inf")                      # an expert that is switched off
        x[0, 4] = -float("inf")                        # a row that is left with nothing
        x[1, 5, 2:] = -float("inf")                    # fewer experts left than are to be chosen
        x[1, 6] = torch.finfo(x.dtype).min             # the type's lowest value everywhere
        x[2, 7, :10] = torch.finfo(x.dtype).min        # ... and in half of a row
        m = torch.rand(B, Q, generator=gen) < 0.7
        if s == 1:
            m[2] = False                               # an image none of whose rows count
        if s == 2:
            m[:] = False                               # a set none of whose rows count
        hidden = ~m
        x[hidden] = torch.where(torch.rand(int(hidden.sum()), E, generator=gen) < 0.2, float("nan"), x[hidden].float()).to(x.dtype)
        x[:, 9][~m[:, 9]] = float("inf")
        xs.append(x)
        masks.append(m)
    out, grads = run_and_check(xs, k, masks=masks, scores=scores, per_image=per_image)
    assert float(out.balance[2].abs().max()) == 0.0 and float(grads[2].float().abs().max()) == 0.0
    for g, m in zip(grads, masks):
        assert torch.equal(g[~m.cuda()], torch.zeros_like(g[~m.cuda()]))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E", [6, 20, 64, 100, 300])
def test_equal_logits_go_to_the_lowest_index(dtype, E):
    gen = torch.Generator().manual_seed(E)
    x = torch.randint(-2, 3, (3, 50, E), generator=gen).to(DTYPES[dtype])
    x[0, :10] = 0.0                                    # a router before its first step
    x[0, 3, 1::2] = -0.0                               # (the two zeros are equal)
    x[1, 5] = torch.finfo(x.dtype).min
    x[1, 6, 4:] = -float("inf")
    for k in (1, 2, min(5, E), E):
        out, _ = run_and_check([x], k)
    zero = torch.zeros(1, 9, E, dtype=x.dtype)
    out, _ = run_and_check([zero], 2)
    assert out.counts[0].tolist() == [9, 9] + [0] * (E - 2)


@pytest.mark.parametrize("per_image", [False, True])
def test_empty_sets_and_batches(per_image):
    from detr_amd import losses

    out, _ = run_and_check([make((3, 0, 7), "f32", 1), make((3, 5, 7), "f32", 2)], 2, per_image=per_image)
    assert out.counts[0].sum() == 0 and float(out.balance[0].abs().sum()) == 0.0
    x = torch.zeros(0, 4, 7, device="cuda", requires_grad=True)
    out = losses.balance_losses(x, 2, per_image=per_image)
    assert out.balance.shape == ((1, 0) if per_image else (1,))
    (out.balance.sum() + out.z.sum()).backward()
    assert x.grad.shape == x.shape
    assert losses.expert_counts(x, 2).tolist() == [[0] * 7]


@pytest.mark.parametrize("per_image", [False, True])
def test_given_experts(per_image):
    from detr_amd import losses

    losses.check_cls_status()
    B, Q, E, k = 3, 41, 13, 4
    gen = torch.Generator().manual_seed(2)
    xs = [make((B, Q, E), "f32", 60 + s) for s in range(2)]
    experts = [torch.randint(-1, E, (B, Q, k), generator=gen) for _ in xs]      # the same index may stand twice in a row
    experts[0][0, 0] = 5
    masks = [torch.rand(B, Q, generator=gen) < 0.8, None]
    run_and_check(xs, k, masks=masks, experts=experts, per_image=per_image)
    # more choices than experts, when they are given
    run_and_check([make((2, 5, 3), "bf16", 9)], 8, experts=[torch.randint(-1, 3, (2, 5, 8), generator=gen)], per_image=per_image)
    losses.check_cls_status()
    # an index that names no expert counts as -1 and is reported
    bad = [e.clone() for e in experts]
    bad[1][1, 2, 0], bad[1][1, 2, 1] = E, -2
    experts[1][1, 2, :2] = -1
    a = losses.balance_losses([x.cuda() for x in xs], k, experts=[e.cuda() for e in bad], per_image=per_image)
    with pytest.raises(RuntimeError):
        losses.check_cls_status()
    b = losses.balance_losses([x.cuda() for x in xs], k, experts=[e.cuda() for e in experts], per_image=per_image)
    losses.check_cls_status()
    assert torch.equal(a.counts, b.counts) and torch.equal(a.balance, b.balance)


@pytest.mark.parametrize("E", [10, 40, 300])
@pytest.mark.parametrize("per_image", [False, True])
def test_many_rows_with_masks_indices_and_counts(E, per_image):
    B, Q, k = 6, 700, 3
    gen = torch.Generator().manual_seed(E)
    xs = [make((B, Q, E), "f16", 70 + s) for s in range(2)]
    masks = [torch.rand(B, Q, generator=gen) < 0.7, torch.rand(B, Q, generator=gen) < 0.5]
    masks[1][2] = False
    experts = [torch.randint(-1, E, (B, Q, k), generator=gen) for _ in xs]
    counts = torch.randint(0, 400, (2, B, E) if per_image else (2, E), generator=gen)
    run_and_check(xs, k, masks=masks, per_image=per_image)
    run_and_check(xs, k, masks=masks, experts=experts, per_image=per_image)
    run_and_check(xs, k, masks=masks, counts=counts, per_image=per_image)
    run_and_check(xs, k, masks=masks, experts=experts, counts=counts, scores="sigmoid", per_image=per_image)
    # images apart in memory, the rows of each dense
    whole = torch.zeros(B, Q + 5, E, dtype=torch.float16, device="cuda")
    views = []
    for x in xs:
        whole[:, 3:Q + 3].copy_(x)
        views.append(whole[:, 3:Q + 3].detach().requires_grad_(True))
        whole = torch.zeros_like(whole)
    run_and_check(xs, k, masks=masks, per_image=per_image, device_xs=views)


@pytest.mark.parametrize("per_image", [False, True])
def test_counts_of_all_ranks(per_image):
    """Two halves of a batch with the counts of both: the mean of their losses is the loss of the whole batch."""
    from detr_amd import dist, losses

    x = make((6, 50, 12), "f32", 3)
    counts = torch.randint(0, 40, (1, 6, 12) if per_image else (1, 12))
    run_and_check([x], 2, counts=counts, per_image=per_image)
    run_and_check([x], 2, counts=torch.zeros_like(counts), per_image=per_image)          # nothing was chosen anywhere
    if not per_image:
        halves = [x[:3].cuda(), x[3:].cuda()]
        both = sum(losses.expert_counts(h, 2) for h in halves)
        whole = losses.balance_losses(x.cuda(), 2)
        assert torch.equal(both, whole.counts)
        mean = sum(losses.balance_losses(h, 2, counts=both).balance for h in halves) / 2
        torch.testing.assert_close(mean, whole.balance, rtol=700 * U, atol=0)
        assert torch.equal(dist.all_reduce_expert_counts(both), both)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per_image", [False, True])
def test_views(dtype, per_image):
    """The tail of every image's rows is read in place; anything else is copied.  Rows of odd length, odd addresses."""
    B, Q, E = 3, 29, 11
    whole = make((B, Q + 8, E), dtype, 77)
    base = whole.cuda()
    tail = base.split([8, Q], dim=1)[1].detach().requires_grad_(True)
    assert not tail.is_contiguous()
    run_and_check([whole[:, 8:]], 3, per_image=per_image, device_xs=[tail])
    wide = make((B, Q, E + 5), dtype, 78)
    part = wide.cuda()[..., 2:2 + E].detach().requires_grad_(True)
    run_and_check([wide[..., 2:2 + E]], 3, per_image=per_image, device_xs=[part])
    turned = make((Q, B, E), dtype, 79)
    run_and_check([turned.transpose(0, 1)], 3, per_image=per_image, device_xs=[turned.cuda().transpose(0, 1).detach().requires_grad_(True)])
    flat = torch.zeros(1 + B * Q * E, dtype=DTYPES[dtype], device="cuda")
    odd = flat[1:].view(B, Q, E)
    odd.copy_(whole[:, :Q])
    run_and_check([whole[:, :Q]], 2, per_image=per_image, device_xs=[odd.detach().requires_grad_(True)])


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [5, 40])
def test_large_and_infinite_logits(scores, E):
    from detr_amd import losses

    # far from zero (a plain sigmoid underflows to 0 / 0), far apart
    for shift, spread in ((-200.0, 3.0), (90.0, 2.0), (0.0, 40.0), (1e4, 1.0)):
        run_and_check([make((2, 19, E), "f32", 11, spread) + shift], 2, scores=scores)
    # a NaN or (softmax) an infinity in a row that counts makes its own group NaN, no other
    x = make((3, 9, E), "f32", 12).cuda()
    x[1, 4, 2] = float("nan")
    out = losses.balance_losses(x, 2, scores=scores, per_image=True)
    assert out.balance[0].isnan().tolist() == [False, True, False]
    assert int(out.counts.sum()) == 3 * 9 * 2                # the NaN was not chosen, the next best was
    x[1, 4] = float("nan")
    assert int(losses.balance_losses(x, 2, scores=scores).counts.sum()) == (3 * 9 - 1) * 2
    x[1, 4] = 0.0
    x[2, 3, 1] = float("inf")
    out = losses.balance_losses(x, 1, scores=scores, per_image=True)
    assert out.balance[0].isnan().tolist() == [False, False, scores == "softmax"]
    assert int(out.counts[0, 2, 1]) >= 1


@pytest.mark.parametrize("E", [4, 8, 40, 200, 700])
def test_a_signalling_nan_is_not_chosen(E):
    from detr_amd import losses

    x = make((2, 67, E), "f32", E)
    quiet, signalling = x.clone(), x.clone()
    quiet[:, ::3, 1::2] = float("nan")
    signalling.view(torch.int32)[:, ::3, 1::2] = 0x7F800001
    for k in (1, 2):
        assert torch.equal(losses.expert_counts(signalling.cuda(), k), losses.expert_counts(quiet.cuda(), k))
        assert losses.balance_losses(signalling.cuda(), k).balance.isnan().all()


def test_offsets_beyond_32_bits():
    """More than 2^32 logits: the rows of a short pattern over and over.  A lane adds Q / (768 x 256) = 2731 rows."""
    from detr_amd import losses

    pattern = make((1, 4096, 8), "bf16", 5)
    times = 131073
    x = pattern[0].cuda().expand(times, 4096, 8).reshape(1, -1, 8).requires_grad_(True)
    assert x.numel() > 1 << 32
    out = losses.balance_losses(x, 2)
    want = losses.balance_losses(pattern.cuda().requires_grad_(True), 2)
    assert torch.equal(out.counts, want.counts * times)
    assert torch.equal(losses.expert_counts(x, 2), out.counts)
    assert abs(out.balance.item() - want.balance.item()) <= (2731 + 700) * U * want.balance.item()
    assert abs(out.z.item() - want.z.item()) <= (2731 + 700) * U * want.z.item()
    (grad,) = torch.autograd.grad(out.balance.sum() + out.z.sum(), x, retain_graph=False, grad_outputs=torch.tensor(1e6).cuda())
    tiles = grad.view(times, 4096, 8)
    assert bool(tiles[0].ne(0).any()) and bool((tiles == tiles[:1]).all())


def test_gradient_against_differences():
    """Central differences of the loss itself, in the kernel's own arithmetic.  The loss is a smooth function of the logits
    while no choice changes (steps of 2^-6 between logits that lie at least 2^-4 apart): the difference quotient is off by
    h^2 / 6 times the third derivative (of balance: p has derivatives below 1, 40 rows: below 6 max f / n) and by the
    rounding of the two losses over 2 h."""
    from detr_amd import losses

    gen = torch.Generator().manual_seed(8)
    B, Q, E, k = 1, 4, 6, 2
    x = (torch.stack([torch.randperm(E, generator=gen) for _ in range(B * Q)]).view(B, Q, E).float() - 2.5) * 0.5
    h = 2.0 ** -6
    for scores in ("softmax", "sigmoid"):
        dev = x.cuda().requires_grad_(True)
        out = losses.balance_losses(dev, k, scores=scores)
        value = (lambda o: o.balance + 0.5 * o.z) if scores == "softmax" else (lambda o: o.balance)
        (grad,) = torch.autograd.grad(value(out), dev)
        f = float((out.counts.double() * E / out.counts.sum()).max())
        size = float(value(out))
        bound = h * h / 6 * 6 * (f + 0.5 * 12) / (B * Q) + 2 * 60 * U * size / (2 * h)
        for q in range(Q):
            for e in range(E):
                up, down = x.clone(), x.clone()
                up[0, q, e] += h
                down[0, q, e] -= h
                d = (value(losses.balance_losses(up.cuda(), k, scores=scores)) -
                     value(losses.balance_losses(down.cuda(), k, scores=scores))).item() / (2 * h)
                assert abs(d - grad[0, q, e].item()) <= bound, (scores, q, e, d, grad[0, q, e].item(), bound)


def test_same_bits_every_time_and_on_another_stream():
    from detr_amd import losses

    xs = [make((16, 300, 24), "f32", 31).cuda().requires_grad_(True)]

    def step():
        out = losses.balance_losses(xs, 2)
        return [out.balance, out.z, out.counts, *torch.autograd.grad((out.balance + out.z).sum(), xs)]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, other, again))


def test_only_one_of_the_losses_is_differentiated():
    from detr_amd import losses

    x = make((2, 30, 9), "f32", 4)
    for which in (0, 1):
        dev = x.cuda().requires_grad_(True)
        out = losses.balance_losses(dev, 2)
        (grad,) = torch.autograd.grad(out[which].sum(), dev)
        want = oracle.balance_losses(x.double().numpy(), 2, grad_balance=[1.0 - which], grad_z=[float(which)])
        check_set(x, want, out.balance[0], out.z[0], out.counts[0], grad)
    # one of two sets needs a gradient; none does
    a, b = x.cuda().requires_grad_(True), x.cuda()
    losses.balance_losses([a, b], 2).balance.sum().backward()
    assert a.grad is not None and b.grad is None
    assert not losses.balance_losses([b], 2).balance.requires_grad
    # (a gradient of the gradient is refused)
    (grad,) = torch.autograd.grad(losses.balance_losses(a, 2).balance.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_the_graph_is_kept_or_not():
    from detr_amd import losses

    a = make((2, 30, 9), "f32", 4).cuda().requires_grad_(True)
    out = losses.balance_losses(a, 2)
    (first,) = torch.autograd.grad(out.balance.sum(), a, retain_graph=True)
    (second,) = torch.autograd.grad(out.balance.sum(), a)
    assert torch.equal(first, second)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out.z.sum(), a)
    # logits that were changed in place since are noticed
    b = a.detach().clone().requires_grad_(True)
    out = losses.balance_losses(b, 2)
    with torch.no_grad():
        b.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace|in-place"):
        out.balance.sum().backward()


def test_one_tensor_for_two_sets_and_broadcast_logits():
    from detr_amd import losses

    x = make((2, 30, 9), "f32", 4)
    dev = x.cuda().requires_grad_(True)
    out = losses.balance_losses([dev, dev], 2)
    weight = torch.tensor([1.0, 3.0]).cuda()
    (twice,) = torch.autograd.grad(out.balance, dev, weight)
    (once,) = torch.autograd.grad(losses.balance_losses(dev, 2).balance, dev, weight[:1])
    torch.testing.assert_close(twice, 4 * once, rtol=8 * U, atol=2.0 ** -126)
    # a row of logits for all queries, images that share their logits
    row = make((1, 1, 9), "f32", 5).cuda().requires_grad_(True)
    wide = row.expand(2, 30, 9)
    out = losses.balance_losses(wide, 2)
    want = oracle.balance_losses(row.detach().cpu().double().numpy(), 2, grad_balance=[1.0])
    (grad,) = torch.autograd.grad(out.balance.sum(), row)
    assert out.counts.tolist()[0] == (60 * want["counts"][0]).tolist()
    # (60 gradients of 1 / 60 of the row's, added up in float32)
    scale = np.abs(want["p"]) * (np.abs(want["f"]).max() * 2)
    assert (np.abs(grad.cpu().numpy() - want["grad"]) <= (5 * 10 + 40 + 64) * U * (scale + np.abs(want["grad"])) + 2.0 ** -126).all()
    shared = make((1, 30, 9), "f32", 6).cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(losses.balance_losses(shared.expand(3, 30, 9), 2).balance.sum(), shared)
    (want,) = torch.autograd.grad(losses.balance_losses(shared, 2).balance.sum(), shared)
    torch.testing.assert_close(grad, want, rtol=0, atol=float(300 * U * want.abs().max()))


def test_total():
    from detr_amd import losses

    xs = [make((2, 20, 6), "f32", s).cuda().requires_grad_(True) for s in range(3)]
    for per_image in (False, True):
        out = losses.balance_losses(xs, 2, per_image=per_image)
        mean = losses.balance_loss_total(xs, 2, 0.02, 0.003, per_image=per_image)
        torch.testing.assert_close(mean, 0.02 * out.balance.mean() + 0.003 * out.z.mean(), rtol=16 * U, atol=0)
        total = losses.balance_loss_total(xs, 2, 0.02, 0.003, per_image=per_image, reduction="sum")
        torch.testing.assert_close(total, 3 * mean, rtol=16 * U, atol=0)
    mean.backward()
    assert all(x.grad is not None for x in xs)


@pytest.mark.parametrize("per_image", [False, True])
def test_two_captured_steps_side_by_side(per_image):
    """Two graphs of forward and backward over their own inputs, replayed in turn and at the same time on two streams, with
    eager steps between the replays: every replay gives the eager result."""
    from detr_amd import losses

    def step(xs):
        out = losses.balance_losses(xs, 2, per_image=per_image)
        return [out.balance, out.z, out.counts, *torch.autograd.grad([out.balance, out.z], xs, [torch.ones_like(out.balance),
                                                                                               torch.ones_like(out.z)])]

    inputs = [[torch.zeros(8, 400, 16, device="cuda", requires_grad=True) for _ in range(2)] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for xs in inputs:
            step(xs)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for xs in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(xs))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        with torch.no_grad():
            for i, xs in enumerate(inputs):
                for j, x in enumerate(xs):
                    x.copy_(make((8, 400, 16), "f32", 1000 * turn + 10 * i + j))
        torch.cuda.synchronize()
        if turn % 2:
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        else:
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for xs, result in zip(inputs, results):
            for got, want in zip(result, step(xs)):
                assert torch.equal(got, want)


def test_refusals():
    from detr_amd import losses

    x = torch.zeros(2, 5, 6, device="cuda")
    with pytest.raises(RuntimeError):
        losses.balance_losses(x.cpu(), 2)
    for dtype in (torch.float64, torch.int32):
        with pytest.raises(TypeError):
            losses.balance_losses(x.to(dtype), 2)
    for k in (0, 7, -1, 2.0):
        with pytest.raises(ValueError):
            losses.balance_losses(x, k)
    with pytest.raises(ValueError):
        losses.balance_losses([], 2)
    with pytest.raises(ValueError):
        losses.balance_losses(x[0], 2)
    with pytest.raises(ValueError):
        losses.balance_losses([x, x[:1]], 2)
    with pytest.raises(ValueError):
        losses.balance_losses([x, x[..., :5]], 2)
    with pytest.raises(ValueError):
        losses.balance_losses(x[..., :0], 1)
    with pytest.raises(TypeError):
        losses.balance_losses([x, x.half()], 2)
    with pytest.raises(TypeError):
        losses.balance_losses(x, 2, mask=torch.ones(2, 5, device="cuda"))
    with pytest.raises(ValueError):
        losses.balance_losses(x, 2, mask=torch.ones(2, 4, dtype=torch.bool, device="cuda"))
    with pytest.raises(TypeError):
        losses.balance_losses(x, 2, mask=torch.ones(2, 5, dtype=torch.bool))
    with pytest.raises(TypeError):
        losses.balance_losses(x, 2, experts=torch.zeros(2, 5, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        losses.balance_losses(x, 2, experts=torch.zeros(2, 5, 3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        losses.balance_losses([x, x], 2, experts=[torch.zeros(2, 5, 2, dtype=torch.int64, device="cuda"), None])
    with pytest.raises(ValueError):
        losses.balance_losses([x, x], 2, experts=[None, torch.zeros(2, 5, 2, dtype=torch.int64, device="cuda")])
    with pytest.raises(TypeError):
        losses.balance_losses(x, 2, counts=torch.zeros(1, 6, device="cuda"))
    with pytest.raises(ValueError):
        losses.balance_losses(x, 2, counts=torch.zeros(6, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        losses.balance_losses(x, 2, scores="relu")
    with pytest.raises(ValueError):
        losses.balance_loss_total(x, 2, z_weight=0.1, scores="sigmoid")
    with pytest.raises(ValueError):
        losses.balance_loss_total(x, 2, reduction="max")
    with pytest.raises(NotImplementedError):
        losses.balance_losses(torch.zeros(1, 1, 1025, device="cuda"), 1)
