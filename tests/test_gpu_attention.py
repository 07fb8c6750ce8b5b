"""Attention over tokens against float64: lengths, heads, widths, masks, biases, packed sequences, layouts."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_reference import attention, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _inputs(rows, h, hk, d, type, seed=0, table=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    t = {"q": rand(rows, h, d), "k": rand(rows, hk, d), "v": rand(rows, hk, d) + 0.5, "do": 0.1 * rand(rows, h, d)}
    t = {k: v.to(type) for k, v in t.items()}
    t["table"] = None if table is None else (0.5 * rand(table, h)).to(type)
    return t


def _bucket_of(bias):
    return {"none": None, "near": blocks.relative_buckets(32, device=DEV), "log": blocks.relative_buckets(128, 8, device=DEV),
            "far": blocks.relative_buckets(255, device=DEV), "one": blocks.relative_buckets(0, device=DEV)}[bias]


def _run(t, lengths, packed, mask, causal, bucket_of, scale=None, train=True):
    names = [n for n in ("q", "k", "v", "table") if t[n] is not None]
    leaves = {n: t[n].detach().clone().requires_grad_(train) for n in names}
    kw = dict(causal=causal, scale=scale, table=leaves.get("table"), bucket_of=bucket_of)
    if packed:
        ends = torch.tensor([0, *lengths]).cumsum(0).to(DEV, torch.int32)
        o = blocks.token_attention(leaves["q"], leaves["k"], leaves["v"], offsets=ends, mask=mask, **kw)
    else:
        cut = lambda x: x.view(len(lengths), lengths[0], *x.shape[1:])  # noqa: E731
        o = blocks.token_attention(cut(leaves["q"]), cut(leaves["k"]), cut(leaves["v"]), mask=None if mask is None else cut(mask), **kw)
        o = o.view(t["q"].shape)
    got = {"o": o.detach()}
    if train:
        got.update(zip(names, torch.autograd.grad(o, [leaves[n] for n in names], t["do"])))
    return got


def _compare(t, lengths, packed=False, mask=None, causal=False, bias="none", scale=None):
    bucket_of = _bucket_of(bias)
    got = _run(t, lengths, packed, mask, causal, bucket_of, scale)
    want, off = attention(t["q"], t["k"], t["v"], lengths, mask, causal, scale, t["table"], bucket_of, t["do"])
    for n, v in got.items():
        check(v, want[n], off[n], n)
    alone = _run(t, lengths, packed, mask, causal, bucket_of, scale, train=False)["o"]
    assert torch.equal(alone, got["o"])  # the forward without a graph is the same
    return got


BUCKETS = {"none": None, "near": 65, "log": 32, "far": 511, "one": 1}


@pytest.mark.parametrize("m", [1, 2, 7, 8, 31, 32, 33, 64, 127, 128, 129, 200, 255, 256, 257, 384, 511, 640])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(m, causal):
    _compare(_inputs(2 * m, 2, 2, 32, torch.bfloat16, m, 65), [m] * 2, causal=causal, bias="near")


@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 127, 128, 129, 192, 200, 255, 256, 257, 384, 385, 512, 640])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_lengths_of_wide_heads(m, causal, type):
    """Widths beyond 64: two query tiles to a block, of which the second may be short or not there."""
    _compare(_inputs(2 * m, 4, 2, 96, type, m, 65), [m] * 2, causal=causal, bias="near")


@pytest.mark.parametrize("kind", ["tail", "holes", "first", "none"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,type", [(128, torch.bfloat16), (72, torch.float16)])
def test_masks_of_wide_heads_in_packed_sequences(kind, causal, d, type):
    lengths = [300, 5, 0, 129, 256]
    rows = sum(lengths) + 50
    place = torch.arange(rows, device=DEV)
    mask = {"tail": place % 300 < 220, "holes": torch.rand(rows, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) > 0.3,
            "first": place % 300 > 140, "none": place < 0}[kind]
    t = _inputs(rows, 8, 2, d, type, 7, 32)
    for n in ("q", "k", "v", "do"):
        t[n][~mask] = float("nan")
    got = _compare(t, lengths, packed=True, mask=mask, causal=causal, bias="log")
    for n in ("o", "q", "k", "v"):
        assert not got[n][~mask].any() and not got[n][sum(lengths):].any()


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_widths(d, type):
    _compare(_inputs(150 + 33, 3, 3, d, type, d), [150, 33], packed=True)
    _compare(_inputs(300, 2, 1, d, type, d + 1, 32), [300], causal=True, bias="log")


@pytest.mark.parametrize("h,hk", [(1, 1), (4, 4), (4, 1), (6, 3), (16, 4), (5, 5), (12, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_heads(h, hk, causal):
    _compare(_inputs(3 * 140, h, hk, 64, torch.bfloat16, h, 32), [140] * 3, causal=causal, bias="log")


@pytest.mark.parametrize("bias", ["near", "log", "far", "one"])
@pytest.mark.parametrize("m", [5, 130, 700])
@pytest.mark.parametrize("causal", [False, True])
def test_biases(bias, m, causal):
    _compare(_inputs(m, 3, 3, 32, torch.bfloat16, m, BUCKETS[bias]), [m], causal=causal, bias=bias)


@pytest.mark.parametrize("lengths", [[1], [0], [0, 5, 0], [1, 1, 1, 1], [128, 128], [1, 300, 2, 129, 64, 0, 257], [513, 3], [40] * 20, [0, 0, 260, 0]])
@pytest.mark.parametrize("spare", [0, 1, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_packed_sequences(lengths, spare, causal):
    rows = sum(lengths) + spare
    t = _inputs(rows, 4, 2, 40, torch.bfloat16, rows, 65)
    for n in ("q", "k", "v", "do"):  # what lies behind the last sequence is never used
        t[n][sum(lengths):] = float("nan")
    got = _compare(t, lengths, packed=True, causal=causal, bias="near")
    for n in ("o", "q", "k", "v"):
        assert not got[n][sum(lengths):].any()


@pytest.mark.parametrize("kind", ["tail", "holes", "first", "one", "none", "third"])
@pytest.mark.parametrize("m", [20, 128, 300])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fill", [None, float("nan"), float("inf"), -3.0e38])
def test_masks(kind, m, causal, fill):
    """Tokens that the mask leaves out, with whatever they hold: rows without a key are zero, and so are their gradients."""
    place = torch.arange(m, device=DEV)
    mask = {"tail": place < (2 * m) // 3, "holes": torch.rand(m, generator=torch.Generator(device=DEV).manual_seed(m), device=DEV) > 0.3,
            "first": place >= m // 2, "one": place == m // 3, "none": place < 0, "third": place % 3 != 0}[kind]
    mask = torch.cat([mask, mask.flip(0)])
    t = _inputs(2 * m, 4, 2, 64, torch.bfloat16, m, 32)
    if fill is not None:
        for n in ("q", "k", "v", "do"):
            t[n][~mask] = fill
    got = _compare(t, [m] * 2, mask=mask, causal=causal, bias="log")
    for n in ("o", "q", "k", "v"):
        assert not got[n][~mask].any()


@pytest.mark.parametrize("type,d", [(torch.float16, 64), (torch.bfloat16, 24), (torch.bfloat16, 96)])
@pytest.mark.parametrize("left", [1, 44, 64, 65, 100])
def test_many_blocks_with_short_last_tiles(type, d, left):
    """Last tiles with keys for one half of the columns only, in more blocks than the GPU holds at once: warps that have nothing to do
    for a tile keep step with those that have."""
    lengths = [256 + left] * 40 + [left] * 40 + [384 + left] * 20
    t = _inputs(sum(lengths), 8, 4, d, type, left, 32)
    bucket_of = _bucket_of("log")
    first = _run(t, lengths, True, None, False, bucket_of)
    want, off = attention(t["q"], t["k"], t["v"], lengths, None, False, None, t["table"], bucket_of, t["do"])
    for n, v in first.items():
        check(v, want[n], off[n], n)
    for _ in range(5):
        for n, v in _run(t, lengths, True, None, False, bucket_of).items():
            assert torch.equal(v, first[n]), n
        assert blocks.read_status(DEV) == 0


def test_a_masked_packed_batch():
    lengths = [200, 0, 77, 130]
    t = _inputs(sum(lengths) + 9, 4, 4, 48, torch.float16, 5, 65)
    mask = torch.rand(sum(lengths) + 9, device=DEV) > 0.4
    mask[200:277] = False  # one sequence without a token
    _compare(t, lengths, packed=True, mask=mask, bias="near")


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-3, 4.0, 12.0])
def test_magnitudes(type, size):
    """Flat softmaxes and ones with a single key: scores up to about +-400."""
    t = _inputs(2 * 330, 2, 2, 64, type, 9)
    t["q"], t["k"] = t["q"] * size, t["k"] * size
    _compare(t, [330] * 2)
    t["do"] *= 1e-3
    _compare(t, [330] * 2, causal=True)


def test_a_growing_maximum():
    """Every later key scores higher than those before it, so the running maximum moves with every one of them, and by much."""
    m, d = 700, 64
    t = _inputs(m, 2, 2, d, torch.bfloat16, 3)
    ramp = torch.linspace(0, 60, m, device=DEV)[:, None, None]
    t["q"] = torch.full_like(t["q"], 1.0)
    t["k"] = (t["k"] * 0.05 + ramp / 8).to(torch.bfloat16)
    _compare(t, [m])
    t["k"] = t["k"].flip(0).contiguous()
    _compare(t, [m])


def test_scale_and_sign():
    t = _inputs(260, 2, 2, 32, torch.bfloat16, 4, 65)
    for scale in (1.0, -0.3, 0.0, 1e-4):
        _compare(t, [260], scale=scale, bias="near")


def test_gradients_of_fp16_keep_small_values():
    """Gradients of a long flat softmax lie far below 1: a probability of 1/2000 of a gradient of 1e-3."""
    t = _inputs(2000, 1, 1, 64, torch.float16, 6)
    t["q"] *= 0.1
    t["do"] *= 0.01
    got = _run(t, [2000], False, None, False, None)
    want, _ = attention(t["q"], t["k"], t["v"], [2000], do=t["do"])
    for n in ("q", "k", "v"):
        # against the result before it is rounded to fp16, of which most is subnormal there
        error = (got[n].double() - want[n]).abs()
        assert float((error - 2.0**-11 * want[n].abs() - 2.0**-25).max()) <= 0.02 * float(want[n].abs().mean()), n


def test_slices_of_one_projection_and_other_strides():
    m, h, d = 200, 4, 48
    qkv = torch.randn(2, m, 3, h, d, device=DEV).bfloat16()
    q, k, v = qkv.unbind(2)
    want = blocks.token_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(blocks.token_attention(q, k, v), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]  # [2, h, m, d] in memory
    assert torch.equal(blocks.token_attention(*heads_first), want)
    wide = [torch.nn.functional.pad(t, (0, 4))[..., :d] for t in (q, k, v)]  # rows 52 elements apart: copied
    assert torch.equal(blocks.token_attention(*wide), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)  # starts on 2 bytes
    assert torch.equal(blocks.token_attention(odd, k, v), want)
    same = k[:, :, :1].expand(-1, -1, h, -1)  # one head for all by a stride of zero
    assert torch.equal(blocks.token_attention(q, same, same), blocks.token_attention(q, k[:, :, :1], k[:, :, :1]))
    qkv.requires_grad_(True)
    q, k, v = qkv.unbind(2)
    do = torch.randn(2, m, h, d, device=DEV).bfloat16()
    (got,) = torch.autograd.grad(blocks.token_attention(q, k, v), qkv, do)
    apart = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    for i, g in enumerate(torch.autograd.grad(blocks.token_attention(*apart), apart, do.transpose(1, 2).contiguous().transpose(1, 2))):
        assert torch.equal(got[:, :, i], g)


def test_converted_types():
    x = [torch.randn(2, 50, 4, 32, device=DEV) for _ in range(3)]
    got = blocks.token_attention(*x)
    assert got.dtype == torch.float32 and torch.equal(got, blocks.token_attention(*(t.bfloat16() for t in x)).float())
    mixed = blocks.token_attention(x[0].half(), x[1], x[2].bfloat16())
    assert torch.equal(mixed, blocks.token_attention(x[0].half(), x[1].half(), x[2].bfloat16().half()))
    table, where = torch.randn(65, 4, device=DEV), blocks.relative_buckets(32, device=DEV)
    a = blocks.token_attention(*(t.half() for t in x), table=table, bucket_of=where)
    b = blocks.token_attention(*(t.half() for t in x), table=table.half(), bucket_of=where)
    assert float((a - b).abs().max()) < 2e-2 and not torch.equal(a, b)


def test_the_fp32_tables_gradient():
    lengths = [300, 65]
    t = _inputs(365, 4, 2, 32, torch.bfloat16, 8, 65)
    t["table"] = t["table"].float() * 1.01
    _compare(t, lengths, packed=True, bias="near")


def test_empty_calls():
    where, table = blocks.relative_buckets(4, device=DEV), torch.randn(9, 2, device=DEV, requires_grad=True)
    for shape in ((0, 5, 2, 16), (3, 0, 2, 16)):
        q = torch.zeros(shape, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        o = blocks.token_attention(q, q, q, table=table, bucket_of=where)
        g = torch.autograd.grad(o, [q, table], torch.zeros_like(o))
        assert o.shape == g[0].shape == shape and not g[1].any()


def test_gradients_against_differences():
    """d/dt of a weighted sum of the outputs along a direction, from gradients and from central differences of the float64 function whose
    values the kernels' outputs are within their bounds of (so the gradients are those of the function that is computed)."""
    lengths = [60, 35]
    t = _inputs(95, 4, 2, 32, torch.bfloat16, 11, 32)
    where = _bucket_of("log")
    got = _run(t, lengths, True, None, True, where)
    f = lambda v: float((attention(v["q"], v["k"], v["v"], lengths, None, True, None, v["table"], where)[0]["o"] * t["do"].double()).sum())  # noqa: E731
    for n in ("q", "k", "v", "table"):
        step = torch.randn(t[n].shape, device=DEV, dtype=torch.float64)
        near = [f({**{m: x.double() if x is not None else None for m, x in t.items()}, n: t[n].double() + s * step}) for s in (1e-5, -1e-5)]
        slope = (near[0] - near[1]) / 2e-5
        # every element of the gradient within 4 half steps of its size: their random sum within as many of the norms' product
        size = float(got[n].double().norm() * step.norm())
        assert abs(float((got[n].double() * step).sum()) - slope) <= 4 * 2.0**-8 * size / step.numel() ** 0.5 * 5, n


def test_offsets_beyond_the_rows_stay_inside():
    """Offsets that the host cannot check: out of order or beyond the tensor. The result means nothing, but every access stays in bounds
    and rows of other tensors keep their values."""
    around = torch.zeros(3, 100, 2, 32, dtype=torch.bfloat16, device=DEV)
    q = around[1]
    for ends in ([0, 50, 1000], [0, -7, 100], [0, 80, 20, 100], [5, 50, 100], [0, 2**31 - 1], [0, -(2**31), 30]):
        blocks.token_attention(q, q, q, offsets=torch.tensor(ends, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert not around.any()


def test_bucket_numbers_beyond_the_table_stay_inside():
    q = torch.randn(1, 40, 2, 32, device=DEV).bfloat16()
    where = torch.tensor([-5, 0, 7, 1 << 30, -(1 << 31)], dtype=torch.int32, device=DEV)
    table = torch.randn(3, 2, device=DEV, requires_grad=True)
    o = blocks.token_attention(q, q, q, table=table, bucket_of=where)
    (g,) = torch.autograd.grad(o.float().sum(), table)
    assert torch.isfinite(o).all() and torch.isfinite(g).all()


@pytest.mark.parametrize("shape", [(5, 0, 2, 16), (0, 2, 16), (2, 0, 3, 4, 128), (3, 2, 0, 1, 8)])
def test_calls_without_tokens_in_any_dimension(shape):
    q = torch.zeros(shape, device=DEV, dtype=torch.float16, requires_grad=True)
    for mask in (None, torch.ones(shape[:-2], device=DEV)):
        o = blocks.token_attention(q, q, q, mask=mask)
        (g,) = torch.autograd.grad(o, q, torch.zeros_like(o))
        assert o.shape == g.shape == shape


@pytest.mark.parametrize("d", [32, 96])
def test_backward_of_offsets_that_mean_nothing_stays_inside(d):
    """As the forward's: in bounds whatever the offsets are, and tensors beside the inputs and the table keep their values."""
    around = torch.zeros(3, 300, 2, d, dtype=torch.bfloat16, device=DEV)
    q, table = around[1].requires_grad_(True), torch.zeros(9, 2, device=DEV, requires_grad=True)
    where = blocks.relative_buckets(4, device=DEV)
    many = torch.randint(-400, 700, (1200,), generator=torch.Generator().manual_seed(3)).tolist()
    for ends in ([0, 150, 1000], [0, -7, 300], [0, 280, 20, 300], [5, 250, 300], [0, 2**31 - 1], [0, -(2**31), 30], many, many[:33], many[:32]):
        o = blocks.token_attention(q, q, q, offsets=torch.tensor(ends, dtype=torch.int32, device=DEV), table=table, bucket_of=where)
        g = torch.autograd.grad(o, [q, table], torch.ones_like(o))
        assert g[0].shape == q.shape
    torch.cuda.synchronize()
    assert not around.detach().any() and not table.detach().any()


def test_many_sequences_of_every_count():
    """The search for a block's sequence in up to 32 candidates, and in rounds above: 31 to 34 and 1023 to 1026 sequences."""
    for count in (31, 32, 33, 34, 63, 64, 1023, 1024, 1025, 1026):
        lengths = [(7 * i) % 5 + (140 if i in (0, 30, 31, 32, count - 1) else 0) for i in range(count)]
        _compare(_inputs(sum(lengths) + 3, 1, 1, 16, torch.bfloat16, count), lengths, packed=True)
