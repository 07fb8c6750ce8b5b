"""Block operators as a program uses them: whole blocks against float64, streams, threads, graphs, large tensors, modules."""

import copy
import io
import threading

import pytest
import torch
import torch.nn.functional as F

import miniworld_b200 as mw
from miniworld_b200 import blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _block(d=64, seed=0, **kw):
    torch.manual_seed(seed)
    m = mw.SandwichTransition(d, scale=0.5, **kw).to(DEV)
    with torch.no_grad():
        m.feed_forward.squeeze.weight.normal_(std=0.3 * m.feed_forward.hidden**-0.5)
        for n in (m.ln_in, m.join.norm_out):
            if n is not None:
                n.weight.add_(0.1 * torch.randn_like(n.weight))
    return m


def _plain(m, p, x, gate, mask, kind="layer"):
    """The block in float64 from parameters ``p`` (linear weights rounded to bf16, as the products take them)."""
    def norm(v, name):
        if kind == "rms":
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * p[name + ".weight"]
        return F.layer_norm(v, v.shape[-1:], p[name + ".weight"], p[name + ".bias"], 1e-5)

    h = norm(x, "ln_in")
    a, b = F.linear(h, p["feed_forward.expand_a.weight"]), F.linear(h, p["feed_forward.expand_b.weight"])
    u = F.linear((F.silu(a) if m.feed_forward.activation == "silu" else F.gelu(a)) * b, p["feed_forward.squeeze.weight"])
    t = norm(u, "join.norm_out") * p["join.scale"] * torch.sigmoid(gate)
    return x + torch.where(mask[..., None], t, torch.zeros_like(t))


@pytest.mark.parametrize("shape,d,kw", [((2, 150), 64, {}), ((1, 203), 384, {}), ((2, 40, 40), 72, {"kind": "rms", "kind_out": "rms"}),
                                        ((2, 5000), 128, {"activation": "gelu"}), ((3,), 256, {}), ((2, 1100), 512, {"n": 2})])
def test_block_against_float64(shape, d, kw):
    """Norm, feed-forward, norm, gate, scale, mask and residual in one module with all gradients. bf16 between the operators: h, the
    hidden activations, u and their gradients are each rounded once, 2^-9 / sqrt(3) = 1.1e-3 of their norm; the norms pass relative
    errors on unchanged, a gradient goes through at most five of these roundings and sums of independent terms: sqrt(5) 1.1e-3 = 2.5e-3,
    and 8e-3 with a margin of three. The output is mostly the residual: 1.1e-3 and three times that."""
    m = _block(d, **kw)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(*shape, d, generator=g, device=DEV).bfloat16().requires_grad_(True)
    gate = torch.randn(shape[0], *[1] * (len(shape) - 1), d, generator=g, device=DEV).bfloat16().requires_grad_(True)
    mask = torch.rand(*shape, generator=g, device=DEV) > 0.2
    dy = torch.randn(*shape, d, generator=g, device=DEV).bfloat16()
    y = m(x, gate, mask)
    names = [n for n, _ in m.named_parameters()]
    got = torch.autograd.grad(y, [x, gate, *m.parameters()], dy)
    p = {n: (v.detach().bfloat16() if "feed_forward" in n else v.detach()).double().requires_grad_(True) for n, v in m.named_parameters()}
    xd, gd = x.detach().double().requires_grad_(True), gate.detach().double().requires_grad_(True)
    yd = _plain(m, p, xd, gd, mask, kw.get("kind", "layer"))
    want = torch.autograd.grad(yd, [xd, gd, *p.values()], dy.double())
    assert torch.equal(y[~mask], x[~mask])
    assert float((y.double() - yd).norm() / yd.norm()) <= 3.3e-3
    for n, a, b in zip(["x", "gate", *names], got, want):
        assert a.dtype == (torch.float32 if n not in ("x", "gate") else torch.bfloat16), n
        assert float((a.double() - b).norm() / b.norm()) <= 8e-3, n


def test_stack_with_joined_norms():
    """Blocks with the next block's norm in the join: three launches a block in the forward instead of four, the same function."""
    d, rows = 128, 600
    norms = [mw.BlockNorm(d).to(DEV) for _ in range(3)]
    joins = [mw.BlockJoin(d, "rms", scale=0.3).to(DEV) for _ in range(3)]
    torch.manual_seed(3)
    ffs = [mw.GatedFeedForward(d, n=2).to(DEV).bfloat16() for _ in range(3)]
    for f in ffs:
        torch.nn.init.normal_(f.squeeze.weight, std=0.1)
    x = torch.randn(rows, d, device=DEV).bfloat16().requires_grad_(True)

    def joined():
        a, h = x, norms[0](x)
        for i in range(3):
            u = ffs[i](h)
            a, h = joins[i](a, u, next_norm=norms[i + 1]) if i < 2 else (joins[i](a, u), None)
        return a

    def apart():
        a = x
        for i in range(3):
            a = joins[i](a, ffs[i](norms[i](a)))
        return a

    params = [p for ms in (norms, joins, ffs) for m in ms for p in m.parameters()]
    dy = torch.randn(rows, d, device=DEV).bfloat16()
    y, z = joined(), apart()
    gy, gz = torch.autograd.grad(y, [x, *params], dy), torch.autograd.grad(z, [x, *params], dy)
    # (the joined norm sees y before it is rounded: a relative 2^-9 of its input, through two more blocks)
    assert float((y.float() - z.float()).norm() / z.float().norm()) <= 4e-3
    for a, b in zip(gy, gz):
        assert float((a.float() - b.float()).norm() / b.float().norm().clamp_min(1e-6)) <= 1.5e-2


def _step(m, x, gate, dy):
    y = m(x, gate)
    return [y.detach(), *torch.autograd.grad(y, [x, gate, *m.parameters()], dy)]


@pytest.mark.parametrize("rows,d", [(3, 64), (300, 64), (9600, 64), (700, 384), (1200, 512)])
def test_training_step_replays_from_a_graph(rows, d):
    m = _block(d)
    x = torch.randn(rows, d, device=DEV).bfloat16().requires_grad_(True)
    gate = torch.randn(1, d, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(rows, d, device=DEV).bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _step(m, x, gate, dy)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs with scratch of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(m, x, gate, dy)
        graphs.append((graph, out))
    for round in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
            m.feed_forward.expand_a.weight.mul_(1.0 + 0.1 * round)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = _step(m, x, gate, dy)
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_calls_on_streams_and_threads():
    """Calls at the same time, on streams of their own and on a shared one, forward and backward, give what they give alone."""
    m = _block(64)
    inputs = [torch.randn(400 + 100 * i, 64, device=DEV).bfloat16().requires_grad_(True) for i in range(4)]
    gate = torch.randn(1, 64, device=DEV).bfloat16().requires_grad_(True)
    grads = [torch.randn_like(x) for x in inputs]
    want = [_step(m, x, gate, g) for x, g in zip(inputs, grads)]
    torch.cuda.synchronize()
    for own in (True, False):
        got, errors = [[] for _ in inputs], []

        def work(i):
            try:
                stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
                with torch.cuda.stream(stream):
                    for _ in range(25):
                        got[i].append(_step(m, inputs[i], gate, grads[i]))
                    stream.synchronize()
            except Exception as e:  # (an exception would be lost with its thread)
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(inputs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors, errors
        for steps, w in zip(got, want):
            assert len(steps) == 25
            for step in steps:
                for a, b in zip(step, w):
                    assert torch.equal(a, b)


def test_inputs_that_the_launch_before_has_written():
    """A chain of calls with nothing between them, each reading what the one before wrote over its own input's memory."""
    torch.manual_seed(0)
    n = blocks.Norm("rms", torch.rand(128, device=DEV) + 0.5)
    buffers = [torch.empty(3000, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    start = torch.randn(3000, 128, device=DEV).bfloat16()
    w = [(torch.randn(256, 128, device=DEV) * 0.1).bfloat16(), (torch.randn(256, 128, device=DEV) * 0.1).bfloat16(), (torch.randn(128, 256, device=DEV) * 0.1).bfloat16()]

    def chain(wait):
        a = start.clone()
        for i in range(20):
            h = blocks.block_norm(a, n.weight, kind="rms")
            if wait:
                torch.cuda.synchronize()
            u = blocks.gated_feed_forward(h, *w)
            if wait:
                torch.cuda.synchronize()
            b = blocks.block_join(a, u, post=n)
            if wait:
                torch.cuda.synchronize()
            buffers[i % 2].copy_(b)
            a = buffers[i % 2]
        return a.clone()

    want = chain(True)
    for _ in range(5):
        assert torch.equal(chain(False), want)


def test_soak_is_bit_identical():
    m = _block(96)
    x = torch.randn(5000, 96, device=DEV).bfloat16().requires_grad_(True)
    gate = torch.randn(5000, 96, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(5000, 96, device=DEV).bfloat16()
    want = _step(m, x, gate, dy)
    for _ in range(40):
        for a, b in zip(_step(m, x, gate, dy), want):
            assert torch.equal(a, b)


def test_join_of_more_elements_than_32_bits_count():
    rows, d = (1 << 24) + 37, 130
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    u = torch.empty_like(x)
    part = torch.randn(1 << 16, d, device=DEV).bfloat16()
    for r in range(0, rows, 1 << 16):
        n = min(1 << 16, rows - r)
        x[r : r + n] = part[:n]
        u[r : r + n] = part[:n].flip(0)
    w = 1 + 0.1 * torch.randn(d, device=DEV)
    N = blocks.Norm("layer", w)
    y, h = blocks.block_join(x, u, post=N, pre=N)
    for lo, hi in ((0, 500), (rows // 2, rows // 2 + 500), (rows - 500, rows)):
        ys, hs = blocks.block_join(x[lo:hi].clone(), u[lo:hi].clone(), post=N, pre=N)
        assert torch.equal(y[lo:hi], ys) and torch.equal(h[lo:hi], hs)
    del y, h
    xg, ug = x.requires_grad_(True), u.requires_grad_(True)
    out = blocks.block_join(xg, ug, post=N)
    gx, gu = torch.autograd.grad(out, [xg, ug], x.detach())
    assert torch.equal(gx, x)
    lo = rows - 500
    xs, us = x.detach()[lo:].clone().requires_grad_(True), u.detach()[lo:].clone().requires_grad_(True)
    gs = torch.autograd.grad(blocks.block_join(xs, us, post=N), [xs, us], xs.detach())
    assert torch.equal(gu[lo:], gs[1])


def test_feed_forward_of_more_elements_than_32_bits_count():
    rows, d, hidden = (1 << 23) + 300, 264, 8
    part = torch.randn(1 << 16, d, device=DEV).bfloat16()
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    for r in range(0, rows, 1 << 16):
        n = min(1 << 16, rows - r)
        x[r : r + n] = part[:n]
    w = [(torch.randn(hidden, d, device=DEV) * d**-0.5).bfloat16(), (torch.randn(hidden, d, device=DEV) * d**-0.5).bfloat16(), torch.randn(d, hidden, device=DEV).bfloat16()]
    y = blocks.gated_feed_forward(x, *w)
    lo = rows - 70000
    a = blocks.gated_feed_forward(x[lo:].clone(), *w)
    assert torch.equal(y[lo:], a) and torch.equal(y[:70000], blocks.gated_feed_forward(x[:70000].clone(), *w))
    x.requires_grad_(True)
    wg = [v.requires_grad_(True) for v in w]
    g = torch.autograd.grad(blocks.gated_feed_forward(x, *wg), [x, *wg], y)
    xs = x.detach()[lo:].clone().requires_grad_(True)
    (gs,) = torch.autograd.grad(blocks.gated_feed_forward(xs, *wg), xs, y[lo:].clone())
    assert torch.equal(g[0][lo:], gs) and all(bool(torch.isfinite(v).all()) for v in g)


def test_modules_copy_pickle_and_load():
    m = _block(64, n=2)
    x = torch.randn(10, 64, device=DEV).bfloat16()
    want = m(x)
    assert torch.equal(copy.deepcopy(m)(x), want)
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    assert torch.equal(torch.load(buf, weights_only=False)(x), want)
    other = mw.SandwichTransition(64, n=2, scale=0.1).to(DEV)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), want)
    half = copy.deepcopy(m).to(torch.bfloat16)
    assert half.join.scale.dtype == torch.float32 and half.ln_in.weight.dtype == torch.float32
    assert torch.equal(half.ln_in.weight, m.ln_in.weight) and torch.equal(half(x), want)  # (the weights are rounded to bf16 either way)


def test_same_operator_as_the_pair_transition():
    """Without a norm after the block, a scale and a gate it is the Transition: width 128 against its kernel, which holds its weights,
    normalised input and hidden activations in fp16 instead of bf16: 2^-9 / sqrt(3) for each of three roundings of the update."""
    t = mw.Transition(128).to(DEV).bfloat16()
    torch.nn.init.normal_(t.squeeze.weight, std=0.05)
    m = mw.SandwichTransition(128, kind_out=None).to(DEV).bfloat16()
    m.load_state_dict({**{"ln_in." + k: v for k, v in t.ln_in.state_dict().items()},
                       **{"feed_forward." + k: v for k, v in t.state_dict().items() if not k.startswith("ln_in")}})
    x = torch.randn(1, 60, 60, 128, device=DEV).bfloat16()
    with torch.no_grad():
        a, b = m(x).float(), t(x).float()
    assert float((a - b).norm() / (b - x.float()).norm()) <= 3 * (3**0.5) * 2.0**-9


def test_refused_under_transforms():
    x = torch.randn(4, 64, device=DEV)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: blocks.block_norm(v).sum())(x)
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        with pytest.raises(RuntimeError):
            blocks.block_norm(mode.from_tensor(x))


def test_second_derivatives_are_refused():
    """A gradient under ``create_graph`` is right and raises an error where it would be differentiated again."""
    x = torch.randn(5, 64, device=DEV).bfloat16().requires_grad_(True)
    w = [torch.randn(*s, device=DEV).mul_(0.1).requires_grad_(True) for s in ((72, 64), (72, 64), (64, 72))]
    for f, leaves in ((lambda: blocks.block_join(x, x * 2, post=blocks.Norm(), pre=blocks.Norm())[1], [x]),
                      (lambda: blocks.gated_feed_forward(x, *w), [x, *w])):
        y = f()
        dy = torch.randn_like(y)
        want = torch.autograd.grad(f(), leaves, dy)
        got = torch.autograd.grad(y, leaves, dy, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(RuntimeError, match="no second derivative"):
            sum(g.float().square().sum() for g in got).backward()


def test_forward_mode_and_lazy_negation_are_refused():
    import torch.autograd.forward_ad as fwad

    x = torch.randn(5, 64, device=DEV).bfloat16()
    with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        blocks.block_norm(fwad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="plain dense"):
        blocks.block_norm(torch._neg_view(x))
    # a gradient that arrives so is taken for what it stands for
    x.requires_grad_(True)
    dy = torch.randn(5, 64, device=DEV).bfloat16()
    (want,) = torch.autograd.grad(blocks.block_norm(x), x, -dy)
    (got,) = torch.autograd.grad(blocks.block_norm(x), x, torch._neg_view(dy))
    assert torch.equal(got, want)


def _allocated():
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated()


def _wide():
    """A feed-forward that keeps 6 bytes a hidden value for its backward, and what it keeps."""
    m = mw.GatedFeedForward(512, n=4).to(DEV).bfloat16()
    torch.nn.init.normal_(m.squeeze.weight, std=0.02)
    return m, torch.randn(4096, 512, device=DEV).bfloat16().requires_grad_(True), 6 * 4096 * 2048


def test_what_is_kept_goes_with_the_backward():
    """... although the output (a logged loss) still holds the node."""
    m, x, kept = _wide()
    before = _allocated()
    y = m(x)
    assert _allocated() - before >= kept
    torch.autograd.grad(y, [x, *m.parameters()], torch.ones_like(y))
    assert _allocated() - before <= y.numel() * 2 + 4096
    x = torch.randn(1 << 18, 16, device=DEV).bfloat16().requires_grad_(True)
    before = _allocated()
    y, h = blocks.block_join(x, x, post=blocks.Norm(), pre=blocks.Norm())
    torch.autograd.grad([y, h], [x], [y.detach(), h.detach()])
    assert _allocated() - before <= 4 * y.numel() + 8192  # (not the statistics, 8 bytes a row of each norm)


def test_checkpoints_hold_nothing_of_a_block():
    from torch.utils.checkpoint import checkpoint

    m, x, kept = _wide()
    norm = blocks.Norm("rms")

    def f(x):
        y, h = blocks.block_join(x, m(x), post=norm, pre=norm)
        return y + h

    dy = torch.randn(4096, 512, device=DEV).bfloat16()
    leaves = [x, *m.parameters()]
    want = torch.autograd.grad(f(x), leaves, dy)
    before = _allocated()
    y = checkpoint(f, x, use_reentrant=False)
    assert _allocated() - before <= y.numel() * 2 + 4096
    for a, b in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(a, b)


def test_what_is_kept_may_be_moved():
    """Saved-tensor hooks that copy to the host and back, to memory that begins at any 16-byte boundary."""
    m, x, kept = _wide()
    norm = blocks.Norm("layer")

    def f():
        return blocks.block_join(x, m(x), post=norm, pre=norm)

    dy, dh = torch.randn(4096, 512, device=DEV).bfloat16(), torch.randn(4096, 512, device=DEV).bfloat16()
    leaves = [x, *m.parameters()]
    want = torch.autograd.grad(f(), leaves, [dy, dh])

    def moved(t):
        room = torch.empty(t.numel() * t.element_size() + 16, dtype=torch.uint8, device=DEV)
        return room[16:].view(t.dtype).view(t.shape).copy_(t)

    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, moved)):
        with hooks:
            out = f()
        for a, b in zip(torch.autograd.grad(out, leaves, [dy, dh]), want):
            assert torch.equal(a, b)


def test_what_is_kept_comes_back_as_something_else():
    m, x, _ = _wide()
    f = torch.randn(6, 64, device=DEV).requires_grad_(True)
    for make, leaf, unpack in (
            (lambda: m(x), x, lambda t: t[:1024] if t.dtype == torch.uint8 else t),
            (lambda: m(x), x, lambda t: t.cpu() if t.dtype == torch.uint8 else t),
            (lambda: blocks.block_norm(f), f, lambda t: t[:5] if t.shape == (6, 2) else t),
            (lambda: blocks.block_join(f, f, post=blocks.Norm()), f, lambda t: t.double() if t.shape == (6, 2) else t)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = make()
        with pytest.raises(RuntimeError, match="came back with another"):
            torch.autograd.grad(y, leaf, torch.ones_like(y))
