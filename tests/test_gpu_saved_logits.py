"""focal_loss / cross_entropy with saved_bits=8 (dm_focal_loss_saved and the three calls beside it) against the 64-bit
restatement in oracle/saved_logits.py: the bytes exactly, losses and gradients within what float32 arithmetic may cost.

Tolerances, in units u = 2^-24 (half a step of float32, relative), with the hardware's exp2, log2 and 1/x good to a step (2 u):
  focal   e = exp(-|z|) is off by (2.5 |z| + 2) u (the product with log2 e rounds, its constant too); sigmoid, 1 - sigmoid and
          log1p(e) inherit that and add at most 8 u.  The loss of a logit and its slope are sums of products of positive
          terms, sigmoid twice and one of the others: (10 |z| + 30) u.  With a gamma that is not 2, sigmoid^gamma comes from
          exp(-gamma s), s = softplus(-z) <= |z| + 0.7, off by gamma times the error of s and of its two products:
          4 gamma (|z| + 10) u more.
  cross   p = exp(x - max) / sum: (5 D + 40) u with D the row's range (33 at most in what the bytes stand for), the
  entropy gradient (p - 1 or p) w g three roundings more; a row's loss is off by that and by 4 u (|max| + |lse| + |x_y|).
  sums    float32 in a thread (at most 40 terms here), 64 bits beyond: 40 u.
  A gradient is rounded once to the logits' type: half a step, and half the smallest subnormal."""
import ctypes

import numpy as np
import pytest
import torch

import golden_io
from oracle import saved_logits as oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def inputs(shape, dtype, seed, spread=2.0, shift=0.0, objects=0.1, none=None):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=gen) * spread + shift).to(DTYPES[dtype])
    none = C if none is None else none
    cls = torch.where(torch.rand(shape[:-1], generator=gen) < objects, torch.randint(0, C, shape[:-1], generator=gen), none)
    return x, cls


def within(got, want, bound, dtype):
    fi = torch.finfo(dtype)
    bound = bound + (fi.eps / 2) * np.abs(want) + fi.smallest_normal * fi.eps + 2.0 ** -126
    off = np.abs(got.detach().double().cpu().numpy() - want)
    assert got.dtype == dtype
    assert (off <= bound).all(), (float((off / bound).max()), np.argwhere(off > bound)[:5].tolist())


def check_focal(x, cls, num_boxes=3.0, alpha=0.25, gamma=2.0, ignore_index=None, upstream=0.75, device_x=None):
    from detr_amd import losses

    dev = x.cuda().requires_grad_(True) if device_x is None else device_x
    loss = losses.focal_loss(dev, cls.cuda(), num_boxes, alpha, gamma, ignore_index=ignore_index, saved_bits=8)
    assert loss.dim() == 0 and loss.dtype == torch.float32
    (grad,) = torch.autograd.grad(loss, dev, torch.tensor(upstream).cuda())
    want, want_grad, decoded = oracle.focal(x.double().numpy(), cls.numpy(), num_boxes, alpha, gamma, ignore_index)
    z = np.abs(decoded)
    more = 0.0 if gamma == 2.0 else 4 * gamma
    far = float(x.double().abs().clamp(max=80).max()) if x.numel() else 0.0          # (beyond 80 a term is 0, or its size to a step)
    assert abs(loss.item() - want) <= (10 * far + 70 + more * (far + 10)) * U * abs(want) + 2.0 ** -126, (loss.item(), want)
    want_grad = want_grad * upstream
    within(grad, want_grad, (10 * z + 34 + more * (z + 10)) * U * np.abs(want_grad), x.dtype)
    return loss, grad


def check_ce(x, cls, weight=None, ignore_index=-100, upstream=0.75, device_x=None):
    from detr_amd import losses

    dev = x.cuda().requires_grad_(True) if device_x is None else device_x
    loss = losses.cross_entropy(dev, cls.cuda(), None if weight is None else weight.cuda(), ignore_index=ignore_index, saved_bits=8)
    assert loss.dim() == 0 and loss.dtype == torch.float32
    (grad,) = torch.autograd.grad(loss, dev, torch.tensor(upstream).cuda())
    want, want_grad, p = oracle.cross_entropy(x.double().numpy(), cls.numpy(), None if weight is None else weight.double().numpy(),
                                              ignore_index)
    finite = np.where(np.isfinite(x.double().numpy()), x.double().numpy(), 0.0).reshape(-1, x.shape[-1])
    largest = min(float(np.abs(finite).max()), 1e3)
    spread = min(float((finite.max(-1) - finite.min(-1)).max()), 104.0)
    t = 5 * spread + 40
    assert abs(loss.item() - want) <= (t + 4 * (2 * largest + 2 * largest + 8)) * U + 40 * U * abs(want), (loss.item(), want)
    # the weight of a row in the mean, from the gradient of its own logit's column: (p - 1) w or p w
    keep = ((cls != ignore_index) & (cls >= 0) & (cls < x.shape[-1])).numpy()
    w = keep * (1.0 if weight is None else weight.double().numpy()[np.where(keep, cls.numpy(), 0)])
    ws = (w / max(w.sum(), 1e-300))[..., None] * upstream
    within(grad, want_grad * upstream, ws * p * (5 * 33 + 40) * U + 46 * U * np.abs(want_grad * upstream), x.dtype)
    return loss, grad


# ---- the bytes ---------------------------------------------------------------------------------------------------------


def awkward(C, rows, dtype, seed):
    """Rows of every kind: ordinary, narrow, wide, far from zero, constant, with masked logits, on borders between codes."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=gen)
    scales = [2.0, 1e-3, 30.0, 1e-6, 0.0, 12.0, 1e5]
    for r in range(rows):
        x[r] = x[r] * scales[r % 7] + [0.0, 100.0, -7.0, 5.0, 3.25, -1000.0, 0.0][(r // 7) % 7]
    k = rows // 2
    x[k:k + 3] = torch.randint(-40, 41, (3, C), generator=gen) * 2.0 ** -5             # half-way between codes
    x[k + 3, ::2] = -float("inf")
    x[k + 4, ::3] = torch.finfo(DTYPES[dtype]).min
    x[k + 5] = torch.finfo(DTYPES[dtype]).min
    x[k + 6] = torch.linspace(-16, 15.9, C) if C > 1 else 1.0
    return x.to(DTYPES[dtype])


def raw_focal(x, cls, dtype):
    from detr_amd import _lib
    from detr_amd._lib import lib

    n, blocks = x.numel(), (x.numel() + 127) // 128
    codes = torch.full((128 * blocks + 16,), 77, dtype=torch.uint8, device="cuda")
    heads = torch.full((blocks + 1,), 77, dtype=torch.int32, device="cuda")
    out = torch.zeros(1, device="cuda")
    partials = torch.empty(_lib.CLS_LOSS_PARTIALS, dtype=torch.float64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = lib.dm_focal_loss_saved(x.data_ptr(), _lib.DTYPE_CODES[DTYPES[dtype]], cls.data_ptr(), cls.numel(), x.shape[-1], 0.25, 2.0,
                                 1.0, 0, 0, out.data_ptr(), codes.data_ptr(), heads.data_ptr(), partials.data_ptr(),
                                 status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert codes[128 * blocks:].eq(77).all() and int(heads[blocks]) == 77              # nothing behind the arrays
    return codes[:n].cpu().numpy(), heads[:blocks].cpu().numpy()


def raw_ce(x, cls, dtype):
    from detr_amd import _lib
    from detr_amd._lib import lib

    rows, C = x.shape
    codes = torch.full((rows * C + 16,), 77, dtype=torch.uint8, device="cuda")
    steps = torch.full((rows + 1,), 77, dtype=torch.int8, device="cuda")
    out = torch.zeros(2, device="cuda")
    partials = torch.empty(_lib.CLS_LOSS_PARTIALS, dtype=torch.float64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = lib.dm_cross_entropy_saved(x.data_ptr(), _lib.DTYPE_CODES[DTYPES[dtype]], cls.data_ptr(), None, rows, C, -100, out.data_ptr(),
                                    codes.data_ptr(), steps.data_ptr(), partials.data_ptr(), status.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert codes[rows * C:].eq(77).all() and int(steps[rows]) == 77
    return codes[:rows * C].view(rows, C).cpu().numpy(), steps[:rows].cpu().numpy()


CLASSES = [1, 2, 3, 4, 5, 7, 8, 12, 16, 17, 31, 33, 64, 65, 91, 92, 97, 128, 129, 255, 256, 257, 260, 300, 385, 512, 513, 700, 1023, 1024, 1025,
           1203, 1204, 1537, 2047, 2048, 2049, 3001, 5000]


@pytest.mark.parametrize("C", CLASSES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_bytes(C, dtype):
    rows = 60 if C <= 300 else 49
    x = awkward(C, rows, dtype, C)
    if dtype == "f16":
        x = torch.where(x.isfinite() | (x == -float("inf")), x, torch.full_like(x, 2.0))        # (1e5 is infinite there)
    cls = torch.zeros(rows, dtype=torch.int64).cuda()
    codes, heads, _ = oracle.focal_codes(x.double().numpy())
    got, got_heads = raw_focal(x.cuda(), cls, dtype)
    assert np.array_equal(got_heads, heads) and np.array_equal(got, codes)
    codes, steps, _ = oracle.ce_codes(x.double().numpy())
    got, got_steps = raw_ce(x.cuda(), cls, dtype)
    assert np.array_equal(got_steps, steps)
    known = steps != oracle.NOT_A_NUMBER
    assert np.array_equal(got[known], codes[known])


def test_the_bytes_of_rows_with_infinities_and_nan():
    x = torch.randn(6, 130)
    x[1, 5], x[2, 7], x[3, :], x[4, 129] = float("nan"), float("inf"), -float("inf"), float("nan")
    cls = torch.zeros(6, dtype=torch.int64).cuda()
    for C in (130, 2600):
        xc = x.repeat(1, C // 130)
        _, steps = raw_ce(xc.cuda(), cls, "f32")
        assert steps.tolist()[1:5] == [-128] * 4 and -128 not in (steps[0], steps[5])
        codes, heads, _ = oracle.focal_codes(xc.double().numpy())
        got, got_heads = raw_focal(xc.cuda(), cls, "f32")
        assert np.array_equal(got_heads, heads)
        fine = np.repeat(heads != (oracle.NOT_A_NUMBER & 255), 128)[:xc.numel()]
        assert np.array_equal(got[fine], codes[fine])


# ---- losses and gradients ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("C", CLASSES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_number_of_classes(C, dtype):
    rows = (3, 41) if C < 300 else (2, 11)
    x, cls = inputs((*rows, C), dtype, C, shift=-1.0)
    check_focal(x, cls)
    x, cls = inputs((*rows, C), dtype, C + 1, none=C - 1)
    w = torch.ones(C)
    w[-1] = 0.1
    check_ce(x, cls, w)
    check_ce(x, cls)


@pytest.mark.parametrize("C", CLASSES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_rows_than_one_workgroup_takes(C, dtype):
    rows = 1100 if C <= 16 else 600 if C <= 32 else 300 if C <= 128 else 70 if C <= 512 else 20
    x, cls = inputs((1, rows, C), dtype, 3 * C, shift=-1.0)
    cls[0, ::7] = -1
    check_focal(x, cls, ignore_index=-1)
    x, cls = inputs((1, rows, C), dtype, 3 * C + 1, none=C - 1)
    cls[0, ::5] = -1
    check_ce(x, cls, torch.rand(C, generator=torch.Generator().manual_seed(C)) + 0.1, ignore_index=-1)


@pytest.mark.parametrize("rows", [(1, 1), (1, 43), (7, 300), (64, 600)])
@pytest.mark.parametrize("C", [1, 2, 3, 9])
def test_few_classes_many_rows(rows, C):
    x, cls = inputs((*rows, C), "f32", rows[1] + C)
    check_focal(x, cls)
    x, cls = inputs((*rows, C), "f32", rows[1] + C, none=C - 1)
    check_ce(x, cls)


@pytest.mark.parametrize("gamma", [0.0, 0.5, 1.0, 1.5, 2.0, 3.0])
@pytest.mark.parametrize("alpha", [0.25, -1.0, 0.0])
def test_gamma_and_alpha(gamma, alpha):
    x, cls = inputs((3, 50, 7), "f32", 3, spread=5.0)
    x[0, 0, :4] = torch.tensor([18.0, -19.5, 0.0, 70.0])
    check_focal(x, cls, alpha=alpha, gamma=gamma)


@pytest.mark.parametrize("C", [1, 2, 3, 11, 91, 128, 300])
@pytest.mark.parametrize("filled", [float("nan"), float("inf"), -float("inf"), 3e4])
def test_what_rows_that_do_not_count_hold_changes_nothing(C, filled):
    """A block of the focal code spans several rows: the others keep their gradients, to the bit."""
    from detr_amd import losses

    x, cls = inputs((5, 37, C), "f32", 6 * C)
    ignored = torch.rand(5, 37, generator=torch.Generator().manual_seed(C)) < 0.4
    ignored[2] = True
    cls[ignored] = -1
    grads, sums = [], []
    for value in (0.0, filled):
        x[ignored] = value
        dev = x.cuda().requires_grad_(True)
        sums.append(losses.focal_loss(dev, cls.cuda(), 3.0, ignore_index=-1, saved_bits=8))
        grads.append(torch.autograd.grad(sums[-1], dev)[0])
    assert torch.equal(sums[0], sums[1]) and torch.equal(grads[0], grads[1])
    assert bool((grads[1][ignored.cuda()] == 0).all()) and bool(grads[1][~ignored.cuda()].ne(0).all())
    x[ignored] = 0.0
    check_focal(x, cls, ignore_index=-1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_ignored_rows(dtype):
    x, cls = inputs((4, 33, 11), dtype, 1)
    cls[torch.rand(4, 33, generator=torch.Generator().manual_seed(1)) < 0.4] = -1
    x[cls == -1] = float("nan")
    from detr_amd import losses

    want, _, _ = oracle.focal(torch.nan_to_num(x).double().numpy(), cls.numpy(), 3.0, ignore_index=-1)
    loss = losses.focal_loss(x.cuda(), cls.cuda(), 3.0, ignore_index=-1, saved_bits=8)
    assert abs(loss.item() - want) <= 200 * U * want
    x = torch.nan_to_num(x)
    check_focal(x, cls, ignore_index=-1)
    x, cls = inputs((4, 33, 11), dtype, 2, none=10)
    cls[1] = -1
    x[1] = float("nan")
    _, grad = check_ce(torch.where(torch.isnan(x), torch.zeros_like(x), x), cls, ignore_index=-1)
    dev = x.cuda().requires_grad_(True)
    loss = losses.cross_entropy(dev, cls.cuda(), ignore_index=-1, saved_bits=8)
    (again,) = torch.autograd.grad(loss, dev, torch.tensor(0.75).cuda())
    assert torch.equal(again, grad) and bool((again[1] == 0).all())


@pytest.mark.parametrize("C", [5, 300, 3001])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_masked_classes(C, dtype):
    """Logits at -inf and at the type's lowest value; a row that is left with one class; a row at the lowest value everywhere."""
    x, cls = inputs((2, 9, C), dtype, C, none=C - 1)
    gen = torch.Generator().manual_seed(C)
    out = torch.rand(x.shape, generator=gen) < 0.3
    out.scatter_(-1, cls[..., None], False)
    low = torch.finfo(x.dtype).min
    x = torch.where(out, torch.where(torch.rand(x.shape, generator=gen) < 0.5, -float("inf"), low).to(x.dtype), x)
    x[0, 3] = -float("inf")
    x[0, 3, cls[0, 3]] = 1.5
    check_ce(x, cls)
    # the lowest value everywhere: even probabilities
    x[1, 4] = low
    from detr_amd import losses

    dev = x.cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(losses.cross_entropy(dev, cls.cuda(), saved_bits=8), dev)
    want = torch.full((C,), 1.0 / C, dtype=torch.float64)
    want[cls[1, 4]] -= 1.0
    within(grad[1, 4], (want / 18).numpy(), 60 * U / 18, x.dtype)
    # the focal loss: the masked logit is saturated, not lost
    fx = x.clone()
    fx[1, 4] = 0.5
    check_focal(torch.where(fx == low, torch.full_like(fx, -60.0), fx), cls)


def test_nan_is_not_lost():
    from detr_amd import losses

    x, cls = inputs((2, 20, 30), "f32", 5)
    x[1, 3, 4] = float("nan")
    for fn in (lambda d: losses.focal_loss(d, cls.cuda(), 1.0, saved_bits=8),
               lambda d: losses.cross_entropy(d, torch.zeros_like(cls).cuda(), saved_bits=8)):
        dev = x.cuda().requires_grad_(True)
        loss = fn(dev)
        (grad,) = torch.autograd.grad(loss, dev)
        assert loss.isnan() and grad[1, 3].isnan().any() and not grad[0, 0].isnan().any()


def test_nothing_to_learn_from():
    from detr_amd import losses

    for shape in ((0, 5, 4), (3, 0, 4)):
        dev = torch.zeros(*shape, device="cuda", requires_grad=True)
        cls = torch.zeros(shape[:-1], dtype=torch.int64, device="cuda")
        loss = losses.focal_loss(dev, cls, 1.0, saved_bits=8)
        assert loss.item() == 0.0
        loss.backward()
        assert dev.grad.shape == dev.shape
        dev = torch.zeros(*shape, device="cuda", requires_grad=True)
        loss = losses.cross_entropy(dev, cls, saved_bits=8)
        assert loss.isnan()                        # the mean of nothing, as torch has it
        loss.backward()
        assert dev.grad.shape == dev.shape
    dev = torch.randn(2, 5, 4, device="cuda").requires_grad_(True)
    cls = torch.full((2, 5), -1, device="cuda")
    loss = losses.cross_entropy(dev, cls, ignore_index=-1, saved_bits=8)
    loss.backward()
    assert loss.isnan() and bool((dev.grad == 0).all())
    dev.grad = None
    loss = losses.focal_loss(dev, cls, 1.0, ignore_index=-1, saved_bits=8)
    loss.backward()
    assert loss.item() == 0.0 and bool((dev.grad == 0).all())


@pytest.mark.parametrize("name", golden_io.cls_case_names())
def test_the_loss_is_the_references(name):
    """The loss is of the logits as they came: the golden values of the reference's own modules, at the tolerance the
    32-bit calls are held to."""
    from detr_amd import losses

    case = golden_io.ClsLossCase(name)
    x, cls = torch.from_numpy(case.logits).cuda(), torch.from_numpy(case.target_cls).cuda()
    if case.kind == "focal":
        loss = losses.focal_loss(x, cls, case.num_boxes, case.alpha, case.gamma, ignore_index=case.ignore_index, saved_bits=8)
    else:
        loss = losses.cross_entropy(x, cls, torch.from_numpy(case.weight).cuda(), saved_bits=8)
    assert abs(loss.item() - case.loss) <= 1e-5 * abs(case.loss) + 1e-7


@pytest.mark.parametrize("kind", ["focal", "ce"])
def test_the_largest_sizes(kind):
    """Just below 2^31 logits, the rows of a short pattern (of whole blocks) over and over: the same gradients everywhere."""
    from detr_amd import losses

    C, times = 91, 184365
    x, cls = inputs((128, C), "bf16", 7, none=C - 1)
    big = x.cuda().expand(times, 128, C).reshape(-1, C).requires_grad_(True)
    assert (1 << 31) - 128 * C < big.numel() < 1 << 31
    maps = cls.cuda().expand(times, 128).reshape(-1)
    small = x.cuda().requires_grad_(True)

    def loss(x, cls, n):
        return losses.focal_loss(x, cls, n, saved_bits=8) if kind == "focal" else losses.cross_entropy(x, cls, saved_bits=8)

    # (a lane adds up to 2^31 / (1280 x 256) logits in float32, or the rows' terms: 6600 additions)
    got, want = loss(big, maps, float(times)), loss(small, cls.cuda(), 1.0)
    assert abs(got.item() - want.item()) <= (6600 + 200) * U * want.item()
    (grad,) = torch.autograd.grad(got, big, torch.tensor(float(times)).cuda())
    tiles = grad.view(times, 128, C)
    assert bool((tiles == tiles[:1]).all())
    (few,) = torch.autograd.grad(want, small)
    if kind == "focal":                      # (the same scale, exactly or but for the rounding of 1 / times, and of its product)
        off = (tiles[0].float() - few.float()).abs()
        assert bool((off <= (2 * 2.0 ** -8 + 4 * U) * few.float().abs()).all())
    with pytest.raises(NotImplementedError):
        loss(torch.empty(1, 1, dtype=torch.bfloat16, device="cuda").expand(1 << 31, 1), maps[:1].expand(1 << 31), 1.0)


def test_gradient_against_differences():
    """Central differences of the loss (the 32-bit call's) at logits that the bytes hold exactly (multiples of 1/16 over a
    range below 15.9).  h = 2^-5: off by h^2 / 6 times a third derivative (of a focal term or a row's loss: below 4, over the
    normaliser) and by the rounding of two losses over 2 h."""
    from detr_amd import losses

    gen = torch.Generator().manual_seed(6)
    h = 2.0 ** -5
    x = torch.randint(-60, 61, (1, 4, 6), generator=gen) / 16.0
    cls = torch.tensor([[0, 5, 2, 3]])
    for fn, share in ((lambda d, bits: losses.focal_loss(d, cls.cuda(), 2.0, saved_bits=bits), 0.5),
                      (lambda d, bits: losses.cross_entropy(d, cls.cuda(), saved_bits=bits), 0.25)):
        dev = x.cuda().requires_grad_(True)
        loss = fn(dev, 8)
        (grad,) = torch.autograd.grad(loss, dev)
        bound = h * h / 6 * 4 * share + 2 * 200 * U * loss.item() / (2 * h)
        for q in range(4):
            for c in range(6):
                up, down = x.clone(), x.clone()
                up[0, q, c] += h
                down[0, q, c] -= h
                d = (fn(up.cuda(), 32) - fn(down.cuda(), 32)).item() / (2 * h)
                assert abs(d - grad[0, q, c].item()) <= bound, (q, c, d, grad[0, q, c].item(), bound)


def test_what_is_kept_is_a_quarter():
    from detr_amd import losses

    def kept(fn, x):
        loss = fn(x)                               # (warm: status word, workspaces)
        del loss
        before = torch.cuda.memory_allocated()
        loss = fn(x)
        held = torch.cuda.memory_allocated() - before
        loss.backward()
        return held

    x = torch.randn(64, 900, 91, device="cuda", requires_grad=True)
    cls = torch.full((64, 900), 90, device="cuda")
    n = x.numel()
    for fn in (lambda t, b: losses.focal_loss(t, cls, 1.0, saved_bits=b), lambda t, b: losses.cross_entropy(t, cls, saved_bits=b)):
        assert kept(lambda t: fn(t, 32), x) >= 4 * n
        assert kept(lambda t: fn(t, 8), x) <= n + n // 16 + (1 << 20) + 8192          # (the allocator hands out up to 1 MB more)


def test_views_streams_and_repeats():
    from detr_amd import losses

    x, cls = inputs((3, 40, 9), "f32", 9)
    flat = torch.zeros(1 + x.numel(), device="cuda")
    odd = flat[1:].view(x.shape)
    odd.copy_(x)
    first = check_focal(x, cls, device_x=odd.detach().requires_grad_(True))
    turned = x.transpose(1, 2).contiguous().cuda().transpose(1, 2).detach().requires_grad_(True)
    second = check_focal(x, cls, device_x=turned)
    assert first[0].item() == second[0].item() and torch.equal(first[1], second[1])
    check_ce(x, cls.clamp(max=8), device_x=odd.detach().requires_grad_(True))
    half = torch.zeros(1 + x.numel(), dtype=torch.bfloat16, device="cuda")[1:].view(x.shape)
    half.copy_(x)
    check_ce(x.bfloat16(), cls.clamp(max=8), device_x=half.detach().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = check_focal(x, cls)
    side.synchronize()
    assert torch.equal(first[1], third[1])
    # a gradient of the gradient is refused
    dev = x.cuda().requires_grad_(True)
    (grad,) = torch.autograd.grad(losses.focal_loss(dev, cls.cuda(), 1.0, saved_bits=8), dev, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_the_graph_is_kept_or_not():
    from detr_amd import losses

    x, cls = inputs((3, 40, 9), "f32", 9)
    for fn in (lambda d: losses.focal_loss(d, cls.cuda(), 1.0, saved_bits=8),
               lambda d: losses.cross_entropy(d, cls.clamp(max=8).cuda(), saved_bits=8)):
        dev = x.cuda().requires_grad_(True)
        loss = fn(dev)
        (first,) = torch.autograd.grad(loss, dev, retain_graph=True)
        # (the bytes are kept, not the logits: they may change)
        with torch.no_grad():
            dev.zero_()
        (second,) = torch.autograd.grad(loss, dev)
        assert torch.equal(first, second)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(loss, dev)


def test_two_captured_steps_side_by_side():
    from detr_amd import losses

    w = torch.ones(21, device="cuda")
    w[-1] = 0.1

    def step(x, cls):
        a = losses.focal_loss(x, cls, 7.0, saved_bits=8)
        b = losses.cross_entropy(x, cls.clamp(max=20), w, saved_bits=8)
        return [a, b, *torch.autograd.grad([a, b], [x], [torch.ones_like(a), torch.ones_like(b)])]

    data = [(torch.zeros(16, 300, 21, device="cuda", requires_grad=True), torch.zeros(16, 300, dtype=torch.int64, device="cuda"))
            for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in data:
            step(*d)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(5):
        for i, (x, cls) in enumerate(data):
            new_x, new_cls = inputs((16, 300, 21), "f32", 100 * turn + i)
            with torch.no_grad():
                x.copy_(new_x)
                cls.copy_(new_cls)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream if turn % 2 else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        for d, result in zip(data, results):
            for got, want in zip(result, step(*d)):
                assert torch.equal(got, want)


def test_bad_classes_are_reported_and_arguments_refused():
    from detr_amd import losses

    losses.check_cls_status()
    x, cls = inputs((2, 9, 4), "f32", 0)
    bad = cls.clone()
    bad[1, 3] = 5
    for fn in (losses.focal_loss, lambda a, b, _, **k: losses.cross_entropy(a, b, **k)):
        dev = x.cuda().requires_grad_(True)
        loss = fn(dev, bad.clamp(max=5).cuda() if fn is losses.focal_loss else torch.where(bad == 5, 5, bad.clamp(max=3)).cuda(), 1.0,
                  saved_bits=8)
        (grad,) = torch.autograd.grad(loss, dev)
        assert bool((grad[1, 3] == 0).all()) and bool(grad[0].abs().sum() > 0)
        with pytest.raises(RuntimeError):
            losses.check_cls_status()
        losses.check_cls_status()
    xc, cc = x.cuda(), cls.cuda()
    for bits in (16, 0, "8", None):
        with pytest.raises(ValueError):
            losses.focal_loss(xc, cc, 1.0, saved_bits=bits)
        with pytest.raises(ValueError):
            losses.cross_entropy(xc, cc, saved_bits=bits)
    with pytest.raises(ValueError):
        losses.FocalLoss(0.25, 2.0, 4, saved_bits=4)
    with pytest.raises(ValueError):
        losses.CrossEntropy(saved_bits=4)
    for fn in (lambda a, b: losses.focal_loss(a, b, 1.0, saved_bits=8), lambda a, b: losses.cross_entropy(a, b, saved_bits=8)):
        with pytest.raises(TypeError):
            fn(xc.double(), cc)
        with pytest.raises(TypeError):
            fn(xc, cc.int())
        with pytest.raises(TypeError):
            fn(xc, cls)
        with pytest.raises(ValueError):
            fn(xc, cc[:, :5])
        with pytest.raises(ValueError):
            fn(xc[..., :0], cc)
        with pytest.raises(RuntimeError):
            fn(x, cls)
    with pytest.raises(ValueError):
        losses.cross_entropy(xc, cc, torch.ones(3, device="cuda"), saved_bits=8)
    # the class map must still be the one of the forward pass
    dev = x.cuda().requires_grad_(True)
    loss = losses.focal_loss(dev, cc, 1.0, saved_bits=8)
    cc[0, 0] = 1
    with pytest.raises(RuntimeError):
        loss.backward()


# ---- as a training step uses them -----------------------------------------------------------------------------------------


def test_modules():
    from detr_amd import losses

    x, cls = inputs((2, 30, 5), "bf16", 4)
    dev = x.cuda().requires_grad_(True)
    want = losses.focal_loss(dev, cls.cuda(), 3, 0.3, 1.5, saved_bits=8)
    for layout in (dev, dev.transpose(1, 2)):
        got = losses.FocalLoss(0.3, 1.5, 5, saved_bits=8)(layout, cls.cuda(), 3)
        assert got.item() == want.item()
    with pytest.raises(RuntimeError):
        losses.FocalLoss(0.3, 1.5, 5)(dev, cls.cuda(), 3)                  # 16-bit logits need the 8-bit form
    w = torch.rand(5) + 0.1
    y = cls.clamp(max=4).cuda()
    want = losses.cross_entropy(dev, y, w.cuda(), saved_bits=8)
    got = losses.CrossEntropy(w, saved_bits=8).cuda()(dev.transpose(1, 2), y)
    assert got.item() == want.item()


@pytest.mark.parametrize("kind", ["focal", "ce"])
def test_a_whole_step(kind):
    """set_loss_total with 8-bit classification losses and routers: matching, pair losses, class maps, classification losses
    and balance loss of a group of output sets, the same as its parts one by one; the sets' losses equal the 32-bit ones."""
    import detr_amd
    from detr_amd import losses, synth

    wl, sets, targets = synth.make_workload("cfg1" if kind == "ce" else "cfg2", device="cuda", batch=6)
    n_cls = wl.n_label_classes
    weight = None
    if kind == "ce":
        weight = torch.ones(n_cls + 1, device="cuda")
        weight[-1] = 0.1
    matcher = detr_amd.HungarianMatcher(**wl.matcher_kwargs)
    routers = [make_router(6, s["pred_logits"].shape[1], i) for i, s in enumerate(sets)]

    def leaves():
        return [{k: v.detach().clone().requires_grad_(True) for k, v in s.items()} for s in sets]

    common = dict(cls_loss=kind, class_weight=weight)
    whole, router_leaves = leaves(), [r.clone().requires_grad_(True) for r in routers]
    total = losses.set_loss_total(matcher, whole, targets, n_cls, l1_weight=5.0, giou_weight=2.0, cls_weight=2.0, saved_bits=8,
                                  router_logits=router_leaves, router_top_k=2, balance_weight=0.02, router_z_weight=0.001, **common)
    total.backward()
    parts, router_parts = leaves(), [r.clone().requires_grad_(True) for r in routers]
    sets8 = losses.set_losses(matcher, parts, targets, n_cls, saved_bits=8, **common)
    by_hand = sum(5.0 * a + 2.0 * b + 2.0 * c for a, b, c in sets8) / len(sets8) + \
        losses.balance_loss_total(router_parts, 2, 0.02, 0.001)
    by_hand.backward()
    matcher.check_status()
    losses.check_cls_status()
    torch.testing.assert_close(total, by_hand, rtol=64 * U, atol=0)
    for a, b in zip(whole, parts):
        for key in a:
            # (the two losses of a box may cancel: over the largest gradient)
            torch.testing.assert_close(a[key].grad, b[key].grad, rtol=8 * U, atol=16 * U * float(b[key].grad.abs().max()))
    for a, b in zip(router_leaves, router_parts):
        torch.testing.assert_close(a.grad, b.grad, rtol=8 * U, atol=2.0 ** -126)
    # the same losses as with 32 bits, and gradients of nearby logits: |z| < 12 here, so steps of 1/16 at most for two or three
    # classes (a range of 24: 1/8); a slope changes by at most its second derivative (below 1 per unit) times half a step
    sets32 = losses.set_losses(matcher, leaves(), targets, n_cls, **common)
    for x8, x32 in zip(sets8, sets32):
        for a, b in zip(x8, x32):
            torch.testing.assert_close(a, b, rtol=300 * U, atol=0)
    plain = leaves()
    losses.set_loss_total(matcher, plain, targets, n_cls, l1_weight=5.0, giou_weight=2.0, cls_weight=2.0, **common).backward()
    for a, b in zip(whole, plain):
        assert torch.equal(a["pred_boxes"].grad, b["pred_boxes"].grad)
        # (the normaliser is one of the same for every logit of a set: compare over the largest gradient)
        size = float(b["pred_logits"].grad.abs().max())
        assert float((a["pred_logits"].grad - b["pred_logits"].grad).abs().max()) <= 0.25 * size


def make_router(B, Q, seed):
    return torch.randn(B, Q, 8, generator=torch.Generator().manual_seed(seed)).cuda()


def test_attached_criterion():
    """`attach(criterion, fused_consumers=True, saved_bits=8)` puts the 8-bit form in front of the criterion's own module."""
    from detr_amd import criterion as crit
    from detr_amd import losses

    class FocalLoss(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.alpha, self.gamma, self.n_cls = 0.25, 2.0, 6

        def forward(self, inputs, targets, num_boxes):
            raise AssertionError("the module's own forward was called")

    class CrossEntropy(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.criterion = torch.nn.CrossEntropyLoss(weight=torch.rand(6) + 0.5)

        def forward(self, inputs, targets, num_boxes):
            raise AssertionError("the module's own forward was called")

    x, cls = inputs((2, 30, 6), "f32", 4)
    dev = x.cuda().requires_grad_(True)
    module = FocalLoss()
    assert crit.fuse_cls_criterion(module, saved_bits=8)
    loss = module(dev.transpose(1, 2), cls.cuda(), 3)
    want = losses.focal_loss(dev, cls.cuda(), 3, saved_bits=8)
    assert torch.equal(*(torch.autograd.grad(v, dev)[0] for v in (loss, want)))
    module = CrossEntropy().cuda()
    assert crit.fuse_cls_criterion(module, saved_bits=8)
    y = cls.clamp(max=5).cuda()
    loss = module(dev.transpose(1, 2), y, 3)
    want = losses.cross_entropy(dev, y, module.criterion.weight, saved_bits=8)
    assert torch.equal(*(torch.autograd.grad(v, dev)[0] for v in (loss, want)))
    with pytest.raises(ValueError):
        crit.fuse_cls_criterion(FocalLoss(), saved_bits=16)
