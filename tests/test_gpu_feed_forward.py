"""The gated feed-forward of any width, forward and backward, against float64.

Tolerances. h, da and db are rounded to the type T of the input once, then summed: each relative rounding error lies within
eps_T / 2 and has a standard deviation of at most eps_T / sqrt(12), so a sum of n products with the other operand is off by a
standard deviation of eps_T / sqrt(12) * sqrt(sum of the squared products); six of these bound it (for n <= 12 they are above the
worst case, eps_T / 2 times the sum of the magnitudes). On top come the rounding of the result, eps / 2 of it, and fp32 arithmetic:
the products' sums and the activation (a few units of 2^-24 each, and 2^-21 for the fast exponential and division), 2^-16 of the
sum of the magnitudes."""

import math

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _status():
    yield
    assert blocks.read_status(DEV) == 0


def _make(rows, d, hidden, type, weights=None, seed=0):
    g = torch.Generator().manual_seed(seed + math.prod(rows if isinstance(rows, tuple) else (rows,)) * 31 + d * 7 + hidden)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    weights = type if weights is None else weights
    rows = rows if isinstance(rows, tuple) else (rows,)
    return {"x": r(*rows, d).to(type).to(DEV), "w_a": (r(hidden, d) * d**-0.5).to(weights).to(DEV),
            "w_b": (r(hidden, d) * d**-0.5).to(weights).to(DEV), "w_s": (r(d, hidden) * hidden**-0.5).to(weights).to(DEV),
            "dy": (r(*rows, d) * 0.1).to(type).to(DEV)}


def _want(t, act, type):
    """name -> (value, bound without the result's rounding)."""
    d = t["x"].shape[-1]
    x, dy = t["x"].to(type).double().reshape(-1, d), t["dy"].double().reshape(-1, d)
    wa, wb, ws = (t[k].to(type).double() for k in ("w_a", "w_b", "w_s"))  # (fp32 weights are rounded first)
    a, b = x @ wa.t(), x @ wb.t()
    if act == "silu":
        s = torch.sigmoid(a)
        f, slope = a * s, s * (1 + a * (1 - s))
    else:
        c = 0.5 * torch.erfc(-a * 0.5**0.5)
        f, slope = a * c, c + a * torch.exp(-a * a / 2) * (2 * torch.pi) ** -0.5
    h = f * b
    dh = dy @ ws
    da, db = dh * b * slope, dh * f
    eps, small = torch.finfo(type).eps, 2.0**-16
    # what a, b, dh themselves are off by in fp32, through the following products
    fa, fb, fd = small * (x.abs() @ wa.abs().t()), small * (x.abs() @ wb.abs().t()), small * (dy.abs() @ ws.abs())
    eh = f.abs() * fb + 1.2 * fa * b.abs() + small * h.abs()
    eda = fd * (b * slope).abs() + dh.abs() * (fb + b.abs() * fa) + small * da.abs()
    edb = fd * f.abs() + 1.2 * dh.abs() * fa + small * db.abs()

    def product(p, ep, q):  # p [m, k] rounded to the type and off by ep, q [k, n] as it is
        return p @ q, 6 * eps / 12**0.5 * (p.square() @ q.square()).sqrt() + small * (p.abs() @ q.abs()) + ep @ q.abs()

    dx1, dx2 = product(da, eda, wa), product(db, edb, wb)
    shape = t["x"].shape
    out = {"y": product(h, eh, ws.t()), "x": (dx1[0] + dx2[0], dx1[1] + dx2[1]), "w_a": product(da.t(), eda.t(), x),
           "w_b": product(db.t(), edb.t(), x)}
    s = product(h.t(), eh.t(), dy)
    out["w_s"] = (s[0].t(), s[1].t())
    for k in ("y", "x"):
        out[k] = tuple(v.reshape(shape) for v in out[k])
    return out


def _run(t, act):
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if k != "dy"}
    y = blocks.gated_feed_forward(*leaves.values(), activation=act)
    with torch.no_grad():
        assert torch.equal(y, blocks.gated_feed_forward(*leaves.values(), activation=act))
    g = torch.autograd.grad(y, list(leaves.values()), t["dy"], retain_graph=True)
    for a, b in zip(g, torch.autograd.grad(y, list(leaves.values()), t["dy"])):
        assert torch.equal(a, b)  # the same bits again
    return {"y": y.detach(), **dict(zip(leaves, g))}


def _compare(got, want, what):
    for k, (ref, bound) in want.items():
        g = got[k]
        assert g.shape == ref.shape, (what, k)
        assert torch.isfinite(g).all(), (what, k)
        # (a subnormal result of a 16-bit type is rounded to a multiple of the smallest one)
        bound = bound + torch.finfo(g.dtype).eps / 2 * ref.abs() + torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps
        bad = (g.double() - ref).abs() / bound
        assert float(bad.max()) <= 1.0, (what, k, float(bad.max()), int(bad.argmax()))


@pytest.mark.parametrize("rows,d,hidden", [
    (1, 8, 8), (1, 64, 256), (1, 768, 2048), (2, 72, 136), (3, 384, 1536), (7, 128, 512), (8, 200, 536), (9, 256, 1024), (31, 64, 64),
    (64, 136, 72), (127, 64, 256), (128, 128, 128), (129, 384, 1536), (255, 192, 320), (257, 320, 264), (384, 384, 1536), (609, 384, 1536),
    (1000, 64, 256), (1100, 1000, 2000), (2048, 512, 2048), (5000, 96, 384), (9001, 64, 256), (40000, 24, 40), (20011, 256, 1024),
])
def test_against_float64(rows, d, hidden):
    t = _make(rows, d, hidden, torch.bfloat16)
    _compare(_run(t, "silu"), _want(t, "silu", torch.bfloat16), (rows, d, hidden))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows,d,hidden", [(7200, 64, 64), (9473, 8, 8), (9473, 128, 64), (100001, 16, 64), (120000, 8, 136), (60003, 64, 256), (19000, 72, 72),
                                           (40001, 120, 320), (30000, 128, 512), (7169, 56, 1000), (70007, 24, 192)])
def test_narrow_tensors_of_many_rows(rows, d, hidden, act):
    """Several tiles a CTA pair, one to sixteen blocks of hidden units, odd numbers of them among these."""
    type = torch.float16 if hidden % 3 == 0 else torch.bfloat16
    t = _make(rows, d, hidden, type)
    _compare(_run(t, act), _want(t, act, type), (rows, d, hidden, act))


def test_narrow_rows_do_not_touch_one_another():
    t = _make(20000, 64, 128, torch.bfloat16)
    w = [t[k] for k in ("w_a", "w_b", "w_s")]
    want = blocks.gated_feed_forward(t["x"], *w)
    x = t["x"].clone()
    x[777::1000] = float("nan")
    got = blocks.gated_feed_forward(x, *w)
    keep = torch.ones(20000, dtype=torch.bool, device=DEV)
    keep[777::1000] = False
    assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[~keep]).any()


@pytest.mark.parametrize("rows,d,hidden", [(1, 64, 128), (5, 384, 1536), (300, 200, 536), (2100, 256, 768), (12000, 128, 512)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("weights", ["same", "fp32"])
def test_types_and_activations(rows, d, hidden, type, act, weights):
    t = _make(rows, d, hidden, type, torch.float32 if weights == "fp32" else None)
    got = _run(t, act)
    assert got["w_a"].dtype == t["w_a"].dtype and got["y"].dtype == type
    _compare(got, _want(t, act, type), (rows, d, hidden, type, act, weights))


def test_other_float_types_run_through_bf16():
    t = _make(50, 64, 128, torch.bfloat16)
    want = blocks.gated_feed_forward(t["x"], t["w_a"], t["w_b"], t["w_s"])
    for type in (torch.float32, torch.float64):
        y = blocks.gated_feed_forward(t["x"].to(type), t["w_a"], t["w_b"], t["w_s"])
        assert y.dtype == type and torch.equal(y, want.to(type))
    x = t["x"].float().requires_grad_(True)
    (g,) = torch.autograd.grad(blocks.gated_feed_forward(x, t["w_a"], t["w_b"], t["w_s"]).sum(), x)
    assert g.dtype == torch.float32


@pytest.mark.parametrize("rows", [1, 4, 200, 3000])
def test_large_activations(rows):
    """Arguments of the activation far on both sides: no overflow on the way, exact zeros and identities."""
    t = _make(rows, 64, 128, torch.bfloat16)
    t["w_a"] *= 64
    for act in ("silu", "gelu"):
        _compare(_run(t, act), _want(t, act, torch.bfloat16), (rows, act))


@pytest.mark.parametrize("rows", [2, 200])
def test_fp16_saturates(rows):
    x = torch.full((rows, 64), 60.0, dtype=torch.float16, device=DEV)
    w = torch.full((64, 64), 1.0, dtype=torch.float16, device=DEV)
    y = blocks.gated_feed_forward(x, w, w, torch.eye(64, dtype=torch.float16, device=DEV))
    assert (y == 65504).all()  # a = b = 3840, h = 65504 instead of infinity


@pytest.mark.parametrize("rows", [3, 150])
def test_rows_do_not_touch_one_another(rows):
    t = _make(rows, 128, 256, torch.bfloat16)
    w = [t[k] for k in ("w_a", "w_b", "w_s")]
    want = blocks.gated_feed_forward(t["x"], *w)
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[1] = bad
        got = blocks.gated_feed_forward(x, *w)
        assert not torch.isfinite(got[1]).any()
        keep = torch.arange(rows, device=DEV) != 1
        assert torch.equal(got[keep], want[keep])


def test_only_what_is_asked_for():
    t = _make(70, 64, 128, torch.bfloat16)
    full = _run(t, "silu")
    names = ["x", "w_a", "w_b", "w_s"]
    for wanted in (["x"], ["w_a"], ["w_s"], ["x", "w_b"], ["w_a", "w_b", "w_s"]):
        leaves = {k: t[k].clone().requires_grad_(k in wanted) for k in names}
        y = blocks.gated_feed_forward(*leaves.values())
        for k, g in zip(wanted, torch.autograd.grad(y, [leaves[k] for k in wanted], t["dy"])):
            assert torch.equal(g, full[k]), (wanted, k)


def test_no_rows():
    t = _make((2, 0), 64, 128, torch.bfloat16)
    got = _run(t, "silu")
    assert got["y"].shape == (2, 0, 64) and got["x"].shape == (2, 0, 64)
    assert not got["w_a"].any() and not got["w_b"].any() and not got["w_s"].any()


def test_layouts_are_converted():
    t = _make((6, 50), 64, 128, torch.bfloat16)
    w = [t[k] for k in ("w_a", "w_b", "w_s")]
    want = blocks.gated_feed_forward(t["x"], *w)
    swapped = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(blocks.gated_feed_forward(swapped, *w), want)
    flat = torch.zeros(6 * 50 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    flat[1:] = t["x"].flatten()
    assert torch.equal(blocks.gated_feed_forward(flat[1:].view(6, 50, 64), *w), want)
    # gradients that arrive expanded or off a boundary
    x = t["x"].clone().requires_grad_(True)
    y = blocks.gated_feed_forward(x, *w)
    (a,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    (b,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    assert torch.equal(a, b)
    odd = torch.zeros(y.numel() + 1, dtype=torch.bfloat16, device=DEV)
    odd[1:] = 1
    assert torch.equal(torch.autograd.grad(y, x, odd[1:].view_as(y))[0], a)


def test_refusals():
    t = _make(4, 64, 128, torch.bfloat16)
    x, wa, wb, ws = (t[k] for k in ("x", "w_a", "w_b", "w_s"))
    f = blocks.gated_feed_forward
    off = torch.zeros(128 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(128, 64)
    for call, word in [
        (lambda: f(x.cpu(), wa, wb, ws), "CUDA"), (lambda: f(x, wa.cpu(), wb, ws), "CUDA"), (lambda: f(x.long(), wa, wb, ws), "float"),
        (lambda: f(x, wa.half(), wb.half(), ws.half()), "weights"), (lambda: f(x, wa, wb.float(), ws), "one type"),
        (lambda: f(x[:, :32], wa, wb, ws), "w_a must be"), (lambda: f(x, wa, wb[:64], ws), "w_b must be"), (lambda: f(x, wa, wb, ws.t()), "w_s must be"),
        (lambda: f(x, wa, wb, ws.t().contiguous().t()), "contiguous"), (lambda: f(x, off, wb, ws), "16-byte"),
        (lambda: f(x[:, :60], wa[:, :60].contiguous(), wb[:, :60].contiguous(), ws[:60].contiguous()), "multiples of 8"),
        (lambda: f(x, wa[:100], wb[:100], ws[:, :100].contiguous()), "multiples of 8"), (lambda: f(x, wa[:0], wb[:0], ws[:, :0]), "multiples of 8"),
    ]:
        with pytest.raises(RuntimeError, match=word):
            call()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda r: f(r, wa, wb, ws))(x)


def test_module_matches_the_function():
    m = mw.GatedFeedForward(64, n=2, activation="gelu", check_status=True).to(DEV)
    torch.nn.init.normal_(m.squeeze.weight, std=0.1)
    x = torch.randn(3, 5, 64, device=DEV).bfloat16()
    want = blocks.gated_feed_forward(x, m.expand_a.weight, m.expand_b.weight, m.squeeze.weight, activation="gelu")
    y = m(x)
    assert torch.equal(y, want)
    y.float().square().sum().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and bool(p.grad.any()) for p in m.parameters())


@pytest.mark.parametrize("rows,d,hidden", [(2048, 512, 2048), (1025, 520, 72)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("scale_a,scale_b", [(1e-3, 1e-3), (1e-6, 1e-6), (1e-8, 1e-8), (1.0, 1e-12), (2.0**18, 1.0), (1.0, 2.0**40), (1e-25, 1e25)])
def test_expanded_inputs_of_any_magnitude(rows, d, hidden, act, scale_a, scale_b):
    """Widths and rows for which the forward leaves its expanded inputs for the backward: they keep their precision over bf16's range."""
    t = _make(rows, d, hidden, torch.bfloat16)
    t["w_a"] *= scale_a
    t["w_b"] *= scale_b
    _compare(_run(t, act), _want(t, act, torch.bfloat16), (rows, d, hidden, act, scale_a, scale_b))


def _with_kept(want, t, type):
    """Bounds of a backward that takes a and b from the forward, which keeps them to a relative e of 2^-11 at most (uniform within it, of
    either sign): db = dh f(a) is off by dh a f'(a) e, da = dh b f'(a) by dh b f'(a) e and dh b a f''(a) e. |f'| <= 1.13 and |a f''| <= 0.32
    for SiLU and GELU (sqrt(1.13^2 + 0.32^2) < 1.2): standard deviations of 1.2 * 2^-11 / sqrt(3) of |dh a| and |dh b|, six of them as above."""
    d = t["x"].shape[-1]
    x, dy = t["x"].double().reshape(-1, d), t["dy"].double().reshape(-1, d)
    wa, wb, ws = (t[k].to(type).double() for k in ("w_a", "w_b", "w_s"))
    dh, six = dy @ ws, 6 * 1.2 * 2.0**-11 / 3**0.5
    da, db = (dh * (x @ wb.t())).square(), (dh * (x @ wa.t())).square()
    more = {"x": ((da @ wa.square()).sqrt() + (db @ wb.square()).sqrt()).reshape(t["x"].shape), "w_a": (da.t() @ x.square()).sqrt(),
            "w_b": (db.t() @ x.square()).sqrt()}
    return {k: (v, bound + six * more[k] if k in more else bound) for k, (v, bound) in want.items()}


@pytest.mark.parametrize("rows,d,hidden", [(2048, 512, 2048), (1025, 520, 72)])
def test_expanded_inputs_beyond_fp16(rows, d, hidden):
    """fp16, |a| up to 2^19 with h, da and db within the type. The subnormal ones among these are rounded to multiples of 2^-24: the
    products get 2^-25 of the other operand's magnitudes more."""
    t = _make(rows, d, hidden, torch.float16, torch.float32)
    t["w_a"] *= 2.0**17
    t["w_b"] *= 2.0**-6
    t["dy"] *= 2.0**-4
    want = _with_kept(_want(t, "silu", torch.float16), t, torch.float16)
    half = 2.0**-25
    wa, wb, ws = (t[k].half().double().abs() for k in ("w_a", "w_b", "w_s"))
    x, dy = t["x"].double().abs(), t["dy"].double().abs()
    more = {"y": half * ws.sum(1).expand(rows, d), "x": half * (wa.sum(0) + wb.sum(0)).expand(rows, d), "w_a": half * x.sum(0).expand(hidden, d),
            "w_b": half * x.sum(0).expand(hidden, d), "w_s": half * dy.sum(0)[:, None].expand(d, hidden)}
    _compare(_run(t, "silu"), {k: (v, b + more[k]) for k, (v, b) in want.items()}, (rows, d, hidden))


@pytest.mark.parametrize("rows,hidden", [(2048, 2048), (1025, 72)])
def test_expanded_inputs_of_neighbours_that_differ(rows, hidden):
    """Neighbouring units of which one is 2^20 times the other: each unit's own gradients keep their precision."""
    t = _make(rows, 512, hidden, torch.bfloat16)
    t["w_b"][::2] *= 2.0**-20
    t["w_a"][1::3] *= 2.0**-20
    _compare(_run(t, "silu"), _want(t, "silu", torch.bfloat16), (rows, hidden))


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_expanded_inputs_that_are_not_finite(bad):
    """An infinite or undefined weight of one unit: its gradients are not finite, its neighbours' are what they are without it."""
    t = _make(1100, 512, 128, torch.bfloat16)
    want = _run(t, "silu")
    dirty = {k: v.clone() for k, v in t.items()}
    dirty["w_b"][37, 5] = bad
    leaves = {k: v.requires_grad_(True) for k, v in dirty.items() if k != "dy"}
    got = dict(zip(leaves, torch.autograd.grad(blocks.gated_feed_forward(*leaves.values()), list(leaves.values()), dirty["dy"])))
    keep = torch.arange(128, device=DEV) != 37
    for k in ("w_a", "w_b"):
        assert torch.equal(got[k][keep], want[k][keep]), k
    assert not torch.isfinite(got["w_a"][37]).any()


@pytest.mark.parametrize("rows,d,hidden", [(1025, 512, 72), (4100, 520, 1544)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("weights", ["same", "fp32"])
def test_expanded_inputs_that_the_forward_keeps(rows, d, hidden, type, act, weights):
    """Single CTAs and pairs of the backward that takes a and b from the forward."""
    t = _make(rows, d, hidden, type, torch.float32 if weights == "fp32" else None)
    _compare(_run(t, act), _with_kept(_want(t, act, type), t, type), (rows, d, hidden, type, act, weights))


@pytest.mark.parametrize("rows,d", [(3, 64), (200, 64), (9500, 64), (1100, 512)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_closed_units(rows, d, type):
    """a = -4096: act(a) and its slope are zero in any precision, and so are the output and every gradient."""
    make = lambda *s, v: torch.full(s, v, dtype=type, device=DEV, requires_grad=True)  # noqa: E731
    t = [make(rows, d, v=1.0), make(128, d, v=-4096.0 / d), make(128, d, v=64.0 / d), make(d, 128, v=1.0)]
    for act in ("silu", "gelu"):
        y = blocks.gated_feed_forward(*t, activation=act)
        assert not y.any(), act
        for g in torch.autograd.grad(y, t, torch.ones_like(y)):
            assert not g.any(), act


@pytest.mark.parametrize("rows,d", [(3, 64), (150, 64), (20000, 64), (1100, 512)])
def test_fp16_rows_that_are_not_finite(rows, d):
    """An infinite element of a row: nothing finite comes out of that row, the others are what they are without it."""
    t = _make(rows, d, 256, torch.float16)
    w = [t[k] for k in ("w_a", "w_b", "w_s")]
    keep = torch.arange(rows, device=DEV) != 1
    want = blocks.gated_feed_forward(t["x"], *w)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = t["x"].clone()
        x[1, 3] = bad
        for act in ("silu", "gelu"):
            got = blocks.gated_feed_forward(x, *w, activation=act)
            assert not torch.isfinite(got[1]).any(), (bad, act)
            assert act == "gelu" or torch.equal(got[keep], want[keep]), bad


@pytest.mark.parametrize("rows,d", [(8, 64), (150, 64), (20000, 64), (1100, 512), (5000, 1024)])
def test_fp16_results_overflow_to_infinity(rows, d):
    """Results beyond the type are infinite, as a loss scaler expects, with operands (h, da, db) inside it."""
    full = lambda *s, v: torch.full(s, v, dtype=torch.float16, device=DEV, requires_grad=True)  # noqa: E731
    # a = b = 32, h = 1024, y = 128 * 1024 = 2^17;  dh = d, da = db = 32 d, dx = 128 * 2 * 32 d * 32 / d = 2^18
    x, w_a, w_b, w_s = full(rows, d, v=1.0), full(128, d, v=32.0 / d), full(128, d, v=32.0 / d), full(d, 128, v=1.0)
    y = blocks.gated_feed_forward(x, w_a, w_b, w_s)
    assert (y == float("inf")).all()
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (dx == float("inf")).all()


@pytest.mark.parametrize("rows,d", [(3, 64), (150, 64), (20000, 64), (1100, 512), (5000, 1024)])
def test_fp16_gradients_of_units_overflow(rows, d):
    """da and db beyond the type: every gradient formed from them says so."""
    full = lambda *s, v: torch.full(s, v, dtype=torch.float16, device=DEV, requires_grad=True)  # noqa: E731
    # a = b = 64, dh = 2048: da = db = 2^17
    t = [full(rows, d, v=1.0), full(64, d, v=64.0 / d), full(64, d, v=64.0 / d), full(d, 64, v=2048.0 / d)]
    y = blocks.gated_feed_forward(*t)
    g = torch.autograd.grad(y, t[:3], torch.ones_like(y))
    assert not any(torch.isfinite(v).any() for v in g)


@pytest.mark.parametrize("rows", [2, 100])
def test_fp32_weights_beyond_fp16(rows):
    """A master weight that the type of the products cannot hold is infinite there, as a conversion makes it."""
    t = _make(rows, 64, 64, torch.float16, torch.float32)
    t["w_a"][3, 2] = 1e6
    got = blocks.gated_feed_forward(t["x"], t["w_a"], t["w_b"], t["w_s"])
    assert not torch.isfinite(got).any()


@pytest.mark.parametrize("rows,d,hidden", [(1100, 512, 128), (50, 64, 128)])
def test_saved_tensors_that_come_back_as_others(rows, d, hidden):
    """Saved-tensor hooks that give back tensors which fit one another, but not the forward: refused before anything is launched."""
    t = _make(rows, d, hidden, torch.bfloat16)
    shapes = {(hidden, d): (2 * hidden, d), (d, hidden): (d, 2 * hidden)}
    leaves = [t[k].clone().requires_grad_(True) for k in ("x", "w_a", "w_b", "w_s")]

    def wider(v):
        return torch.zeros(shapes.get(tuple(v.shape), tuple(v.shape)), dtype=v.dtype, device=DEV)

    def narrower(v):
        return v[:hidden // 2].contiguous() if tuple(v.shape) == (hidden, d) else v[:, :hidden // 2].contiguous() if tuple(v.shape) == (d, hidden) else v

    for unpack in (wider, narrower, lambda v: v.half(), lambda v: v.float(), lambda v: v[: v.shape[0] // 2], lambda v: v.cpu(),
                   lambda v: v.t().contiguous().t(), lambda v: v.flatten()):
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
            y = blocks.gated_feed_forward(*leaves)
        with pytest.raises(RuntimeError, match="came back with another|must be"):
            torch.autograd.grad(y, leaves, t["dy"])


@pytest.mark.parametrize("rows,d", [(200, 64), (9500, 64), (1100, 512), (5000, 1024)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_units_that_are_not_finite_do_not_touch_their_neighbours(rows, d, type, act):
    """Units share powers of two and reciprocals (of a product, whose rounding and so whose last bits depend on all four factors): one
    whose a is infinite or a NaN leaves the others' gradients within the bounds that they have without it, since a sigmoid's relative
    error is the same few units of 2^-24 for any factors of the product."""
    t = _make(rows, d, 128, type)
    want = _want(t, act, type)
    if d >= 512:
        want = _with_kept(want, t, type)
    keep = torch.arange(128, device=DEV) != 37
    want = {"w_a": tuple(v[keep] for v in want["w_a"]), "w_b": tuple(v[keep] for v in want["w_b"]), "w_s": tuple(v[:, keep] for v in want["w_s"])}
    for bad in (float("inf"), float("-inf"), float("nan")):
        leaves = {k: v.clone() for k, v in t.items() if k != "dy"}
        leaves["w_a"][37, 5] = bad
        for v in leaves.values():
            v.requires_grad_(True)
        y = blocks.gated_feed_forward(*leaves.values(), activation=act)
        got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"])))
        assert not torch.isfinite(y).any() and not torch.isfinite(got["w_a"][37]).any(), bad
        _compare({"w_a": got["w_a"][keep], "w_b": got["w_b"][keep], "w_s": got["w_s"][:, keep]}, want, (rows, d, type, act, bad))
