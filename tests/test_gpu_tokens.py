"""Token operators as a program uses them: together, on streams and threads, in graphs, on large tensors, and what they refuse."""

import copy
import threading

import pytest
import torch
import torch.nn.functional as F

import miniworld_b200 as mw
from miniworld_b200 import blocks
from tests.token_reference import attention, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


class Stack(torch.nn.Module):
    """A token block: norm, attention with a bias of the relative position, dropout and residual, feed-forward."""

    def __init__(self, d, heads, **kw):
        super().__init__()
        self.norm = mw.BlockNorm(d)
        self.qkv = torch.nn.Parameter(torch.randn(3 * d, d) * d**-0.5)
        self.out = torch.nn.Parameter(torch.randn(d, d) * d**-0.5)
        self.attention = mw.TokenAttention(heads, **kw)
        self.dropout = mw.BlockDropout(0.2)
        self.transition = mw.SandwichTransition(d, n=2, scale=0.5)
        torch.nn.init.normal_(self.transition.feed_forward.squeeze.weight, std=0.3 * (2 * d) ** -0.5)
        torch.nn.init.normal_(self.attention.table, std=0.5)
        self.heads = heads

    def forward(self, x, key, mask=None, offsets=None):
        q, k, v = F.linear(self.norm(x), self.qkv.to(x.dtype)).unflatten(-1, (3, self.heads, -1)).unbind(-3)
        u = F.linear(self.attention(q, k, v, mask, offsets).flatten(-2), self.out.to(x.dtype))
        return self.transition(self.dropout(x, u, key))


def _plain(m, p, x, keep, mask, causal):
    d, n = x.shape[-1], x.shape[-2]
    h = F.layer_norm(x, (d,), p["norm.weight"], p["norm.bias"], 1e-5)
    q, k, v = F.linear(h, p["qkv"]).unflatten(-1, (3, m.heads, -1)).unbind(-3)
    place = torch.arange(n, device=DEV)
    reach = m.attention.bucket_of.numel() // 2
    bias = p["attention.table"][m.attention.bucket_of.long()[(place[None, :] - place[:, None]).clamp(-reach, reach) + reach]].permute(2, 0, 1)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * q.shape[-1] ** -0.5 + bias
    counts = mask[:, None, None, :].expand_as(s)
    if causal:
        counts = counts & (place[:, None] >= place[None, :])
    o = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~counts, -1e30), -1), v) * mask[..., None, None]
    x = x + keep * F.linear(o.flatten(-2), p["out"]) * (65536 / (65536 - round(0.2 * 65536)))
    h = F.layer_norm(x, (d,), p["transition.ln_in.weight"], p["transition.ln_in.bias"], 1e-5)
    u = F.linear(F.silu(F.linear(h, p["transition.feed_forward.expand_a.weight"])) * F.linear(h, p["transition.feed_forward.expand_b.weight"]),
                 p["transition.feed_forward.squeeze.weight"])
    u = F.layer_norm(u, (d,), p["transition.join.norm_out.weight"], p["transition.join.norm_out.bias"], 1e-5)
    return x + u * p["transition.join.scale"]


@pytest.mark.parametrize("b,n,d,heads,kw", [(2, 150, 64, 4, {}), (1, 300, 384, 16, {"reach": 128, "exact": 8}), (3, 70, 128, 2, {"causal": True})])
def test_a_block_of_all_operators_against_float64(b, n, d, heads, kw):
    """bf16 between the operators: about twelve roundings lie on the way of a gradient, 2^-9 / sqrt(3) = 1.1e-3 of their norm each and
    independent: sqrt(12) 1.1e-3 = 4e-3, and 1.2e-2 with a margin of three. The output is mostly the residual: a third of that."""
    torch.manual_seed(n)
    m = Stack(d, heads, **kw).to(DEV)
    x = torch.randn(b, n, d, device=DEV).bfloat16().requires_grad_(True)
    mask = torch.rand(b, n, device=DEV) > 0.15
    mask[:, 0] = True
    dy = torch.randn(b, n, d, device=DEV).bfloat16()
    key = blocks.dropout_key(DEV)
    y = m(x, key, mask)
    names = [k for k, _ in m.named_parameters()]
    got = torch.autograd.grad(y, [x, *m.parameters()], dy)
    keep = (blocks.block_dropout(None, torch.ones(b, n, d, device=DEV), key, p=0.2) != 0).double()
    cast = lambda k, v: (v.detach().bfloat16() if k in ("qkv", "out") or "feed_forward" in k else v.detach()).double().requires_grad_(True)  # noqa: E731
    p = {k: cast(k, v) for k, v in m.named_parameters()}
    xd = x.detach().double().requires_grad_(True)
    yd = _plain(m, p, xd, keep, mask, kw.get("causal", False))
    want = torch.autograd.grad(yd, [xd, *p.values()], dy.double())
    assert float((y.detach().double() - yd.detach()).norm() / yd.detach().norm()) <= 4e-3
    for k, a, w in zip(["x", *names], got, want):
        assert float((a.double() - w).norm() / w.norm()) <= 1.2e-2, k


def test_packed_and_padded_batches_agree():
    """The same sequences packed and padded: outputs and gradients of the tokens are those of the other form, bit for bit."""
    lengths, n, h, d = [130, 1, 77, 256], 256, 4, 32
    t = [torch.randn(4, n, h, d, device=DEV).bfloat16() for _ in range(4)]
    mask = torch.arange(n, device=DEV)[None] < torch.tensor(lengths, device=DEV)[:, None]
    padded = [v.clone().requires_grad_(True) for v in t[:3]]
    packed = [v[mask].clone().requires_grad_(True) for v in t[:3]]
    a = blocks.token_attention(*padded, mask=mask)
    b = blocks.token_attention(*packed, offsets=torch.tensor([0, *lengths]).cumsum(0).to(DEV))
    assert torch.equal(a[mask], b) and not a[~mask].any()
    for x, y in zip(torch.autograd.grad(a, padded, t[3]), torch.autograd.grad(b, packed, t[3][mask])):
        assert torch.equal(x[mask], y) and not x[~mask].any()


def test_sequences_do_not_see_one_another():
    """What one sequence of a pack holds changes no bit of another's results (bf16; in fp16 the gradients' common power of two may)."""
    lengths, h, d = [100, 300, 64, 129], 2, 64
    ends = torch.tensor([0, *lengths]).cumsum(0)
    t = [torch.randn(sum(lengths), h, d, device=DEV).bfloat16() for _ in range(4)]

    def step(v):
        leaves = [x.clone().requires_grad_(True) for x in v[:3]]
        o = blocks.token_attention(*leaves, offsets=ends.to(DEV), causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, v[3])]

    want = step(t)
    lo, hi = int(ends[1]), int(ends[2])
    for fill in (float("nan"), float("inf"), 1e30):
        other = [x.clone() for x in t]
        for x in other:
            x[lo:hi] = fill
        for a, b in zip(step(other), want):
            assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:])


def _step(m, x, key, dy, offsets=None, mask=None):
    y = m(x, key, mask, offsets)
    return [y.detach(), *torch.autograd.grad(y, [x, *m.parameters()], dy)]


@pytest.mark.parametrize("packed", [False, True])
def test_training_steps_replay_from_graphs(packed):
    m = Stack(64, 2).to(DEV)
    rows = 333
    x = torch.randn(rows if packed else 3, 64, device=DEV).bfloat16() if packed else torch.randn(3, 111, 64, device=DEV).bfloat16()
    x.requires_grad_(True)
    offsets = torch.tensor([0, 100, 101, 300], dtype=torch.int32, device=DEV) if packed else None
    mask = None if packed else torch.rand(3, 111, device=DEV) > 0.2
    dy, key = torch.randn_like(x), blocks.dropout_key(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _step(m, x, key, dy, offsets, mask)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs with scratch of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(m, x, key, dy, offsets, mask)
        graphs.append((graph, out))
    for turn in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
            key.add_(turn + 1)
            m.attention.table.normal_()
            if packed:  # other lengths in the same tensor
                offsets.copy_(torch.tensor([[0, 5, 200, 333], [0, 0, 0, 290], [0, 128, 256, 257]][turn], dtype=torch.int32))
            else:
                mask.copy_(torch.rand(3, 111, device=DEV) > 0.1 * turn)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = _step(m, x, key, dy, offsets, mask)
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_new_masks_in_every_replay():
    x, u = torch.zeros(1000, device=DEV), torch.ones(1000, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = blocks.block_dropout(x, u, blocks.dropout_key(DEV), p=0.5)
    seen = []
    for _ in range(3):
        graph.replay()
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_calls_on_streams_and_threads():
    m = Stack(64, 4, reach=16).to(DEV)
    key = blocks.dropout_key(DEV)
    inputs = [torch.randn(2, 130 + 100 * i, 64, device=DEV).bfloat16().requires_grad_(True) for i in range(4)]
    grads = [torch.randn_like(x) for x in inputs]
    want = [_step(m, x, key, g) for x, g in zip(inputs, grads)]
    torch.cuda.synchronize()
    for own in (True, False):
        got, errors = [[] for _ in inputs], []

        def work(i):
            try:
                stream = torch.cuda.Stream() if own else torch.cuda.current_stream()
                with torch.cuda.stream(stream):
                    for _ in range(15):
                        got[i].append(_step(m, inputs[i], key, grads[i]))
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
            assert len(steps) == 15
            for step in steps:
                for a, b in zip(step, w):
                    assert torch.equal(a, b)


def test_inputs_that_the_launch_before_has_written():
    """A chain of calls with nothing between them, each on what the one before wrote, in memory that both have read."""
    where, table, pair = blocks.relative_buckets(8, device=DEV), torch.randn(17, 2, device=DEV), torch.randn(17, 64, device=DEV)
    index, key = torch.arange(50, device=DEV), blocks.dropout_key(DEV)
    start = torch.randn(50, 50, 2, 32, device=DEV).bfloat16()

    def chain(wait):
        a = start.clone()
        pause = torch.cuda.synchronize if wait else lambda: None
        for i in range(12):
            o = blocks.token_attention(a, a, a, table=table, bucket_of=where, causal=i % 2 == 1)
            pause()
            z = blocks.relative_position(o.view(50, 50, 64), pair, index, bucket_of=where)
            pause()
            a.copy_(blocks.block_dropout(a.view(50, 50, 64), z, key, p=0.3, call=i, shared=0).view_as(a) * 0.5)
            pause()
        return a

    want = chain(True)
    for _ in range(4):
        assert torch.equal(chain(False), want)


def test_soak_is_bit_identical():
    m = Stack(96, 4).to(DEV)
    x, key = torch.randn(7, 513, 96, device=DEV).bfloat16().requires_grad_(True), blocks.dropout_key(DEV)
    mask = torch.rand(7, 513, device=DEV) > 0.1
    dy = torch.randn_like(x)
    want = _step(m, x, key, dy, mask=mask)
    for _ in range(30):
        for a, b in zip(_step(m, x, key, dy, mask=mask), want):
            assert torch.equal(a, b)


def test_more_than_32_bits_of_elements():
    """Rows beyond 2^31 elements of a tensor: the last sequences against a call of their own."""
    length, h, d = 200, 16, 128
    s = (1 << 31) // (length * h * d) + 3
    part = [torch.randn(8, length, h, d, device=DEV).bfloat16() for _ in range(4)]
    q, k, v, do = (p.repeat((s + 7) // 8, 1, 1, 1)[:s] for p in part)
    assert q.numel() > 1 << 31
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = blocks.token_attention(*leaves, causal=True)
    grads = torch.autograd.grad(o, leaves, do)
    for at in (slice(0, 3), slice(s - 3, s)):
        few = [t.detach()[at].clone().requires_grad_(True) for t in (q, k, v)]
        of = blocks.token_attention(*few, causal=True)
        assert torch.equal(o[at], of)
        for a, b in zip(grads, torch.autograd.grad(of, few, do[at])):
            assert torch.equal(a[at], b)


def test_more_blocks_than_a_grid_dimension_counts():
    """70000 sequences of two tokens, packed and not."""
    n = 70000
    q = torch.randn(n, 2, 1, 8, device=DEV).bfloat16()
    a = blocks.token_attention(q, q, q)
    b = blocks.token_attention(*[q.view(-1, 1, 8)] * 3, offsets=torch.arange(0, 2 * n + 1, 2, device=DEV))
    assert torch.equal(a.view(-1, 1, 8), b)
    want, off = attention(*[q[-50:].view(-1, 1, 8)] * 3, [2] * 50)
    check(b[-100:], want["o"], off["o"], "o")


def test_second_derivatives_transforms_and_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwad

    q = torch.randn(1, 9, 2, 16, device=DEV).bfloat16().requires_grad_(True)
    z, table = torch.randn(1, 5, 5, 8, device=DEV).requires_grad_(True), torch.randn(9, 8, device=DEV).requires_grad_(True)
    where, index, key = blocks.relative_buckets(4, device=DEV), torch.arange(5, device=DEV), blocks.dropout_key(DEV)
    calls = [(lambda x: blocks.token_attention(x, x * 1, x * 2), q), (lambda x: blocks.relative_position(x, table, index, bucket_of=where), z),
             (lambda x: blocks.block_dropout(x, x * 3, key, p=0.5), z)]
    for f, x in calls:
        y = f(x)
        dy = torch.randn_like(y)
        (want,) = torch.autograd.grad(f(x), x, dy)
        (got,) = torch.autograd.grad(y, x, dy, create_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="no second derivative"):
            got.float().square().sum().backward()
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: f(v).float().sum())(x.detach())
        with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwad.make_dual(x.detach(), torch.ones_like(x)))
    from torch._subclasses.fake_tensor import FakeTensorMode

    plain = q.detach()
    with FakeTensorMode() as mode, pytest.raises(RuntimeError):
        blocks.token_attention(*[mode.from_tensor(plain)] * 3)


def test_saved_tensors():
    """Hooks see what the backward needs: moved tensors give the same gradients, others are refused, and a checkpoint runs again."""
    q, k, v = (torch.randn(2, 140, 2, 40, device=DEV).bfloat16().requires_grad_(True) for _ in range(3))
    table, where = torch.randn(65, 2, device=DEV).requires_grad_(True), blocks.relative_buckets(32, device=DEV)
    mask = torch.rand(2, 140, device=DEV) > 0.3
    leaves = [q, k, v, table]
    f = lambda: blocks.token_attention(q, k, v, mask=mask, table=table, bucket_of=where)  # noqa: E731
    do = torch.randn_like(f())
    want = torch.autograd.grad(f(), leaves, do)
    with torch.autograd.graph.save_on_cpu():
        y = f()
    for a, b in zip(torch.autograd.grad(y, leaves, do), want):
        assert torch.equal(a, b)
    y = torch.utils.checkpoint.checkpoint(lambda: f(), use_reentrant=False)
    for a, b in zip(torch.autograd.grad(y, leaves, do), want):
        assert torch.equal(a, b)
    for change in (lambda t: t[:1], lambda t: t.float() if t.dtype == torch.bfloat16 else t.half() if t.dtype == torch.float32 else t.long(), lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            y = f()
            with pytest.raises(RuntimeError, match="saved for the backward"):
                torch.autograd.grad(y, leaves, do)
    y = f()
    with torch.no_grad():
        k.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves, do)


def test_only_the_gradients_that_are_asked_for():
    q, k, v = (torch.randn(1, 70, 2, 16, device=DEV).bfloat16() for _ in range(3))
    table, where = torch.randn(9, 2, device=DEV), blocks.relative_buckets(4, device=DEV)
    do = torch.randn_like(q)
    every = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
    want = torch.autograd.grad(blocks.token_attention(*every[:3], table=every[3], bucket_of=where), every, do)
    for i in range(4):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v, table))]
        (got,) = torch.autograd.grad(blocks.token_attention(*some[:3], table=some[3], bucket_of=where), some[i], do)
        assert torch.equal(got, want[i])


def test_refusals():
    bf = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    q, where, table = bf(2, 6, 4, 16), blocks.relative_buckets(4, device=DEV), torch.zeros(9, 4, device=DEV)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    z, pair, index, key = bf(1, 5, 5, 8), torch.zeros(9, 8, device=DEV), torch.arange(5, device=DEV), blocks.dropout_key(DEV)
    A, R, D = blocks.token_attention, blocks.relative_position, blocks.block_dropout
    bad = [
        lambda: A(q[0, 0], q[0, 0], q[0, 0]), lambda: A(q, q[:, :5], q[:, :5]), lambda: A(q, q, q[:, :, :2]), lambda: A(q, q[:, :, :3], q[:, :, :3]),
        lambda: A(q, q[..., :8], q[..., :8]), lambda: A(*[bf(2, 6, 4, 12)] * 3), lambda: A(*[bf(2, 6, 4, 136)] * 3), lambda: A(q.long(), q, q),
        lambda: A(q, q, q, scale=float("inf")), lambda: A(q, q, q, scale=1e300), lambda: A(q, q, q, offsets=ints(0, 6)), lambda: A(*[q[0]] * 3, offsets=ints(0)),
        lambda: A(*[q[0]] * 3, offsets=ints(0, 6).float()), lambda: A(*[q[0]] * 3, offsets=ints(0, 6).cpu()), lambda: A(q, q, q, mask=torch.ones(3, 6, device=DEV)),
        lambda: A(q, q, q, mask=torch.ones(2, 6)), lambda: A(q, q, q, table=table), lambda: A(q, q, q, bucket_of=where), lambda: A(q, q, q, table=table[:, :3], bucket_of=where),
        lambda: A(q, q, q, table=table.half(), bucket_of=where), lambda: A(q, q, q, table=table, bucket_of=where[:4]), lambda: A(q, q, q, table=table, bucket_of=where.long()),
        lambda: A(q, q, q, table=torch.zeros(600, 4, device=DEV), bucket_of=where), lambda: A(q, q, q, table=table.t().contiguous().t(), bucket_of=where),
        lambda: A(q, q, q, table=table, bucket_of=torch.zeros(515, dtype=torch.int32, device=DEV)), lambda: A(*[bf(2, 6, 0, 16)] * 3),
        lambda: R(z[0, 0], pair, index, bucket_of=where), lambda: R(bf(1, 5, 6, 8), pair, index, bucket_of=where), lambda: R(z.double(), pair, index, bucket_of=where),
        lambda: R(z, pair.half(), index, bucket_of=where), lambda: R(z, pair[:, :4], index, bucket_of=where), lambda: R(z, pair, index[:4], bucket_of=where),
        lambda: R(z, pair, index.float(), bucket_of=where), lambda: R(z, pair, index.cpu(), bucket_of=where), lambda: R(z, pair, index, bucket_of=where, chain=index.bool()),
        lambda: R(z, torch.zeros(513, 8, device=DEV), index, bucket_of=where), lambda: R(z, pair, index, bucket_of=where.cpu()),
        lambda: D(z, z[:, :4], key, p=0.5), lambda: D(z, z, key, p=1.5), lambda: D(z, z, key, p=-0.1), lambda: D(z, z, key, p=float("nan")), lambda: D(z, z, key.int(), p=0.5),
        lambda: D(z, z, key[:1], p=0.5), lambda: D(z, z, key.cpu(), p=0.5), lambda: D(z, z, key, p=0.5, shared=4), lambda: D(z, z, key, p=0.5, shared=-5), lambda: D(z.double(), z, key, p=0.5),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_modules_copy_and_load():
    m = Stack(64, 2).to(DEV)
    x, key = torch.randn(2, 40, 64, device=DEV).bfloat16(), blocks.dropout_key(DEV)
    want = m(x, key)
    assert torch.equal(copy.deepcopy(m)(x, key), want)
    other = Stack(64, 2).to(DEV)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x, key), want)
    m.eval()
    assert torch.equal(m(x, key), m(x, None))
    p = mw.RelativePosition(16, reach=4).to(DEV)
    index = torch.arange(9, device=DEV)
    y = p(torch.zeros(1, 9, 9, 16, device=DEV), index, index // 5)
    assert torch.equal(y[0, 0, 8], y[0, 8, 0]) and not torch.equal(y[0, 0, 1], y[0, 1, 0])


def test_relative_position_in_front_of_a_pair_stack():
    """The pair tensor with its relative position through a triangle update: the table gets its gradient through both."""
    torch.manual_seed(1)
    n = 40
    position, update = mw.RelativePosition(128).to(DEV), mw.TriangleMultiplication(128).to(DEV).bfloat16()
    torch.nn.init.normal_(update.to_out.weight, std=0.1)
    z, index = torch.randn(1, n, n, 128, device=DEV).bfloat16(), torch.arange(n, device=DEV)
    dy = torch.randn_like(z)
    y = position(z, index)
    (got,) = torch.autograd.grad(update(y), position.table, dy)
    leaf = y.detach().requires_grad_(True)
    (dz,) = torch.autograd.grad(update(leaf), leaf, dy)
    d = (index[None, :] - index[:, None]).clamp(-32, 32) + 32
    want = torch.zeros(66, 128, dtype=torch.float64, device=DEV).index_add_(0, d.view(-1), dz.view(-1, 128).double())
    assert float((got.double() - want).abs().max()) <= 2.0**-24 * n * n * float(dz.abs().max())
