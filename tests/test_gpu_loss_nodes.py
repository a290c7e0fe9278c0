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
def test_hooks_see_all_that_is_saved(name):
    x, cls = data()
    mask = torch.rand(cls.shape, generator=torch.Generator().manual_seed(1)).cuda() < 0.8
    loss, least = calls(cls, mask)[name]
    x.requires_grad_(True)
    (want,) = torch.autograd.grad(loss(x), x)
    packed, unpacked = [], []

    def pack(t):
        packed.append(t.numel() * t.element_size())
        return t.cpu(), t.device

    def unpack(p):
        unpacked.append(p[0].numel() * p[0].element_size())
        return p[0].to(p[1])

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        value = loss(x)
    # (what is kept, the classes or logits, the mask; beside what torch's own nodes around it save)
    inputs = 8 * cls.numel() if name in ("focal", "ce") else 2 * 4 * x.numel() + 2 * mask.numel()
    assert sum(packed) >= least + inputs and not unpacked
    (got,) = torch.autograd.grad(value, x)
    assert torch.equal(got, want) and sum(unpacked) >= least + inputs


@pytest.mark.parametrize("name", ["focal", "ce"])
def test_saved_bytes_leave_the_gpu(name):
    gen = torch.Generator(device="cuda").manual_seed(3)
    cls = torch.zeros(64, 3000, dtype=torch.int64, device="cuda")
    x = torch.randn(64, 3000, 21, device="cuda", generator=gen, requires_grad=True)
    loss, n = calls(cls)[name]
    (want,) = torch.autograd.grad(loss(x), x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        value = loss(x)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < n // 8
    (got,) = torch.autograd.grad(value, x)
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoints(name, reentrant):
    """Without reentrance what is saved is dropped, and computed again when the backward pass asks for it."""
    from torch.utils.checkpoint import checkpoint

    x, cls = data()
    loss, _ = calls(cls)[name]
    results = []
    for how in (lambda f, *a: f(*a), lambda f, *a: checkpoint(f, *a, use_reentrant=reentrant)):
        a, b = x.clone().requires_grad_(True), torch.linspace(0.5, 1.5, 21, device="cuda").requires_grad_(True)
        value = how(lambda a, b: loss(a * b), a, b)
        value.backward()
        results.append((value.detach(), a.grad, b.grad))
    for plain, again in zip(*results):
        assert torch.equal(plain, again)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("wrong", ["device", "type", "shape"])
def test_a_hook_that_hands_back_another_tensor_is_refused(name, wrong):
    x, cls = data()
    loss, _ = calls(cls)[name]
    x.requires_grad_(True)
    other = {"device": lambda t: t.cpu(), "type": lambda t: t.double(), "shape": lambda t: t.flatten()[1:]}[wrong]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
        value = loss(x).view(1)          # (no node of torch's own below saves a tensor)
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(value.sum(), x)


def test_a_hook_may_hand_back_other_strides():
    x, cls = data()
    for name in NAMES:
        loss, _ = calls(cls)[name]
        leaf = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(loss(leaf), leaf)

        def apart(t):
            wide = torch.zeros(*t.shape, 3, dtype=t.dtype, device=t.device)
            wide[..., 1] = t
            return wide[..., 1]

        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart):
            value = loss(leaf)
        (got,) = torch.autograd.grad(value, leaf)
        assert torch.equal(got, want)


def test_the_loss_may_be_changed_in_place():
    """The loss shares its memory with what is kept for the backward pass, not its version."""
    x, cls = data()
    for name in NAMES:
        loss, _ = calls(cls)[name]
        leaf = x.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(loss(leaf), leaf)
        value = loss(leaf)
        value *= 2.0
        (got,) = torch.autograd.grad(value, leaf)
        torch.testing.assert_close(got, 2 * want, rtol=2.0 ** -22, atol=2.0 ** -126)


@pytest.mark.parametrize("name", NAMES)
def test_class_maps_and_masks_of_inference_mode(name):
    """What a data pipeline made in inference mode cannot be saved as it is: it is copied."""
    x, cls = data()
    mask = torch.rand(cls.shape, generator=torch.Generator().manual_seed(1)).cuda() < 0.8
    results = []
    for made in (lambda t: t, lambda t: t.clone()):
        with torch.inference_mode():
            c, m = made(cls), made(mask)
        leaf = x.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(calls(c, m)[name][0](leaf), leaf)
        results.append(grad)
    assert c.is_inference() and m.is_inference() and torch.equal(*results)
    if name in ("balance", "sigmoid"):        # logits of a frozen router
        with torch.inference_mode():
            frozen = x.clone()
        scores = "softmax" if name == "balance" else name
        leaf = x.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(losses.balance_losses([frozen, leaf], 3, scores=scores).balance[1], leaf)
        (want,) = torch.autograd.grad(losses.balance_losses([x, leaf], 3, scores=scores).balance[1], leaf)
        assert torch.equal(grad, want)


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


@pytest.mark.parametrize("name", ["focal32", "focal", "balance"])
def test_first_call_inside_a_capture(name):
    """The word that findings are reported in is neither part of the graph nor cleared by its replays."""
    x, cls = data()
    fn = {"focal32": lambda: losses.focal_loss(x, cls, 3.0), "focal": lambda: losses.focal_loss(x, cls, 3.0, saved_bits=8),
          "balance": lambda: losses.balance_losses(x, 2).balance}[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = fn().clone()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    index = torch.cuda.current_device()
    word = losses._cls_status.pop(index)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn()
        losses.check_cls_status()
        good = cls.clone()
        cls[0, 0] = 99
        losses.focal_loss(x, cls, 3.0)
        losses.focal_loss(x, cls, 3.0, saved_bits=8)
        cls.copy_(good)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        with pytest.raises(RuntimeError):
            losses.check_cls_status()
        graph.replay()
        losses.check_cls_status()
        if name != "balance":            # what the graph's own kernels find is reported as well
            cls[0, 0] = 99
            graph.replay()
            with pytest.raises(RuntimeError):
                losses.check_cls_status()
        assert losses._cls_status[index] is not word
    finally:
        losses._cls_status[index] = word


@pytest.mark.parametrize("kind", ["focal", "ce"])
def test_captured_graphs_share_no_workspace(kind, monkeypatch):
    """The 32-bit losses in two graphs that were captured on one stream: their partial sums lie apart, and apart from those of
    eager calls, so that replays on two streams do not meet."""
    x, cls = data(B=64, Q=900)
    name = "dm_focal_loss_f32" if kind == "focal" else "dm_cross_entropy_f32"
    real, used = getattr(losses.lib, name), []

    class Spy:
        def __getattr__(self, n):
            return getattr(lib, n)

    def spy(*args):
        used.append(args[-3])
        return real(*args)

    lib = losses.lib
    setattr(Spy, name, staticmethod(spy))
    monkeypatch.setattr(losses, "lib", Spy())
    xs = [x.clone(), x.clone() * 0.5]

    def fn(x):
        return losses.focal_loss(x, cls, 3.0) if kind == "focal" else losses.cross_entropy(x, cls)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [fn(x).clone() for x in xs]
    torch.cuda.synchronize()
    del used[:]
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(fn(x))
        graphs.append(graph)
    assert len(set(used)) == 2 and not set(used) & {p.data_ptr() for p in losses._cls_partials.values()}
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for got, value in zip(outs, want):
            assert torch.equal(got, value)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("per_image", [False, True])
def test_routers_that_need_no_gradient_are_left_out(scores, per_image):
    """The gradients of the others are the same, and nothing is allocated for a set that needs none."""
    sets, B, Q, E = 6, 8, 4096, 32
    gen = torch.Generator(device="cuda").manual_seed(4)
    xs = [torch.randn(B, Q + 8 * s, E, device="cuda", generator=gen, requires_grad=True) for s in range(sets)]
    groups = (sets, B) if per_image else (sets,)
    upstream = torch.rand(groups, device="cuda", generator=gen)

    def value():
        out = losses.balance_losses(xs, 2, scores=scores, per_image=per_image)
        return (out.balance * upstream).sum() if out.z is None else (out.balance * upstream).sum() + (out.z * upstream).sum()

    want = torch.autograd.grad(value(), xs)
    for wanted in ([0], [5], [2, 3], [0, 2, 5], [1, 2, 4]):
        loss = value()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        got = torch.autograd.grad(loss, [xs[i] for i in wanted])
        torch.cuda.synchronize()
        most = sum(xs[i].numel() * 4 for i in wanted) + (1 << 21)
        assert torch.cuda.max_memory_allocated() - before <= most
        for i, g in zip(wanted, got):
            assert torch.equal(g, want[i])
        del loss, got
    # one that is not a leaf's, one that is frozen
    mixed = [xs[0], xs[1].detach(), xs[2]]
    out = losses.balance_losses(mixed, 2, scores=scores, per_image=per_image)
    got = torch.autograd.grad((out.balance * upstream[:3]).sum(), [xs[0], xs[2]])
    out = losses.balance_losses(xs[:3], 2, scores=scores, per_image=per_image)
    both = torch.autograd.grad((out.balance * upstream[:3]).sum(), xs[:3])
    assert torch.equal(got[0], both[0]) and torch.equal(got[1], both[2])


def test_what_a_total_takes_of_the_routers():
    """set_loss_total hands the model's own choice, the counts of all ranks, the scores and the images on to the balance loss."""
    import detr_amd
    from detr_amd import synth

    wl, sets, targets = synth.make_workload("cfg2", device="cuda", batch=4)
    matcher = detr_amd.HungarianMatcher(**wl.matcher_kwargs)
    gen = torch.Generator().manual_seed(6)
    Q = sets[0]["pred_logits"].shape[1]
    routers = [torch.randn(4, Q, 8, generator=gen).cuda() for _ in sets]
    chosen = [torch.randint(-1, 8, (4, Q, 2), generator=gen).cuda() for _ in sets]
    plain = losses.set_loss_total(matcher, sets, targets, wl.n_label_classes)
    for extra in (dict(experts=chosen), dict(counts=torch.randint(1, 50, (len(sets), 8), generator=gen).cuda()),
                  dict(scores="sigmoid"), dict(per_image=True), dict(per_image=True, scores="sigmoid", experts=chosen)):
        total = losses.set_loss_total(matcher, sets, targets, wl.n_label_classes, router_logits=routers, router_top_k=2,
                                      balance_weight=0.5, **{"router_" + k: v for k, v in extra.items()})
        part = losses.balance_loss_total(routers, 2, 0.5, **extra)
        # (the sum of the two, rounded once)
        torch.testing.assert_close(total, plain + part, rtol=2.0 ** -23, atol=0)
        assert not torch.equal(part, losses.balance_loss_total(routers, 2, 0.5))
