"""The join of two blocks (norms, gate, scale, mask, residual) and the norm alone against float64.

Tolerances. An output of type T is rounded once: eps_T / 2 of its value. Before that stand a few dozen fp32 operations, each 2^-24 of
the terms that are added: 2^-18 (64 of them) times the sum of the terms' magnitudes ``amp``, which the reference forms beside each
result; a mean or variance adds up d <= 4096 values in at most 8 NV + log2(threads) + 4 steps (< 64). A sum over rows adds at most
rows / teams + teams + blocks / 8 + 8 (< 256) rounded terms in a chain: 2^-16 times the sum of the terms' magnitudes."""

import math

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def _norm64(v, w, b, kind, eps):
    """Result, its terms' magnitudes, normalised values, 1 / sigma."""
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = c * r
    w = torch.ones_like(v[0]) if w is None else w
    res = n * w + (0 if b is None else b)
    # values are rounded relative to the largest of their row and its mean
    big = (v.abs().amax(-1, keepdim=True) * r) * w.abs() + (0 if b is None else b.abs())
    return res, big, n, r


def _back64(n, r, w, g, kind):
    q = g if w is None else g * w
    res = q - n * (q * n).mean(-1, keepdim=True)
    if kind == "layer":
        res = res - q.mean(-1, keepdim=True)
    amp = q.abs() + n.abs() * (q * n).abs().mean(-1, keepdim=True) + q.abs().mean(-1, keepdim=True)
    return r * res, r * amp


def _make(rows, d, type, gate, scale, mask, post, pre, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + math.prod(rows_shape(rows)) * 7919 + d)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": (r(*rows_shape(rows), d) * 1.5 + 0.3).to(type).to(DEV), "u": (r(*rows_shape(rows), d) * 0.8).to(type).to(DEV)}
    if gate is not None:
        t["gate"] = r(*gate, d).to(type).to(DEV)
    if scale:
        t["scale"] = (0.5 + 0.2 * r(d)).to(DEV)
    if mask:
        t["mask"] = (torch.rand(rows_shape(rows), generator=g) > 0.3).to(DEV)
    for name, kind in (("post", post), ("pre", pre)):
        if kind is not None:
            t[name + "_w"] = (1 + 0.2 * r(d)).to(DEV)
            if bias:
                t[name + "_b"] = (0.1 * r(d)).to(DEV)
    t["dy"] = r(*rows_shape(rows), d).to(type).to(DEV)
    t["dh"] = r(*rows_shape(rows), d).to(type).to(DEV)
    return t


def rows_shape(rows):
    return rows if isinstance(rows, tuple) else (rows,)


def _run(t, post, pre, eps=1e-5):
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items() if k not in ("mask", "dy", "dh")}
    get = leaves.get
    kw = dict(gate=get("gate"), scale=get("scale"), mask=t.get("mask"),
              post=None if post is None else blocks.Norm(post, get("post_w"), get("post_b"), eps),
              pre=None if pre is None else blocks.Norm(pre, get("pre_w"), get("pre_b"), eps))
    out = blocks.block_join(leaves["x"], leaves["u"], **kw)
    y, h = out if pre is not None else (out, None)
    with torch.no_grad():
        again = blocks.block_join(leaves["x"], leaves["u"], **kw)
    again = again if pre is not None else (again,)
    assert torch.equal(y, again[0]) and (h is None or torch.equal(h, again[1]))
    outs, grads = ([y], [t["dy"]]) if pre is None else ([y, h], [t["dy"], t["dh"]])
    g = torch.autograd.grad(outs, list(leaves.values()), grads, retain_graph=True)
    for a, b in zip(g, torch.autograd.grad(outs, list(leaves.values()), grads)):
        assert torch.equal(a, b)  # the same bits again
    return {"y": y.detach(), **({} if h is None else {"h": h.detach()}), **dict(zip(leaves, g))}


def _want(t, post, pre, eps=1e-5):
    """name -> (value, bound without the output's rounding)."""
    v = {k: x.double() for k, x in t.items() if k != "mask"}
    small, sums = 2.0**-18, 2.0**-16
    d, shape = v["x"].shape[-1], v["x"].shape
    valid = t["mask"][..., None].double() if "mask" in t else torch.ones(*shape[:-1], 1, dtype=torch.float64, device=DEV)
    u = v["u"] * valid if "mask" in t else v["u"]
    sig = torch.sigmoid(v["gate"]).expand(shape) if "gate" in v else torch.ones_like(u)
    s = v.get("scale", torch.ones(d, dtype=torch.float64, device=DEV))
    if post is None:
        tt, ta, n, r, w = u, u.abs(), u, None, None
    else:
        w = v["post_w"]
        tt, ta, n, r = _norm64(u, w, v.get("post_b"), post, eps)
    f = valid * s * sig
    y, ya = v["x"] + f * tt, v["x"].abs() + f.abs() * ta
    out = {"y": (y, small * ya)}
    e, ea = v["dy"], torch.zeros_like(y)
    rows = tuple(range(len(shape) - 1))
    if pre is not None:
        h, ha, ny, ry = _norm64(y, v["pre_w"], v.get("pre_b"), pre, eps)
        yerr = ya.amax(-1, keepdim=True) * ry  # of the normalised values: what y itself is off by
        out["h"] = (h, small * (ha + yerr * v["pre_w"].abs()))
        back, ba = _back64(ny, ry, v["pre_w"], v["dh"], pre)
        e, ea = e + back, ba * (1 + yerr)
        out["pre_w"] = ((v["dh"] * ny).sum(rows), (sums * (v["dh"] * ny).abs() + small * v["dh"].abs() * (1 + yerr)).sum(rows))
        if "pre_b" in v:
            out["pre_b"] = (v["dh"].sum(rows), sums * v["dh"].abs().sum(rows))
    ea = e.abs() + ea
    out["x"] = (e, small * ea)
    dt, da = e * f, ea * f.abs()
    if post is None:
        out["u"] = (dt, small * da)
    else:
        back, ba = _back64(n, r, w, dt, post)
        extra = _back64(n.abs(), r, w.abs(), da, post)[1] * (1 + (u.abs().amax(-1, keepdim=True) * r))
        out["u"] = (back, small * (ba + extra))
        out["post_w"] = ((dt * n).sum(rows), (sums * (dt * n).abs() + small * da * (n.abs() + u.abs().amax(-1, keepdim=True) * r)).sum(rows))
        if "post_b" in v:
            out["post_b"] = (dt.sum(rows), (sums * dt.abs() + small * da).sum(rows))
    if "scale" in v:
        out["scale"] = ((e * valid * sig * tt).sum(rows), (sums * (e * sig * tt).abs() + small * ea * ta).sum(rows))
    if "gate" in v:
        dg, ga = dt * tt * (1 - sig), da * ta
        own = [i for i in range(len(shape) - 1) if v["gate"].dim() < len(shape) - i or v["gate"].shape[i - len(shape)] != shape[i]]
        if own:
            dg, ga = dg.sum(own, keepdim=True), ga.sum(own, keepdim=True) + 4 * (dg.abs()).sum(own, keepdim=True)
        out["gate"] = (dg.reshape(v["gate"].shape), small * ga.reshape(v["gate"].shape))
    return out


def _compare(got, want, what):
    assert set(got) == set(want), (set(got) ^ set(want), what)
    for k, (ref, bound) in want.items():
        g = got[k]
        assert g.shape == ref.shape, (what, k)
        bound = bound + torch.finfo(g.dtype).eps / 2 * ref.abs() + torch.finfo(g.dtype).tiny
        bad = (g.double() - ref).abs() / bound
        assert torch.isfinite(g).all(), (what, k)
        assert float(bad.max() if bad.numel() else 0) <= 1.0, (what, k, float(bad.max()), int(bad.argmax()))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 5), (1, 8), (5, 24), (257, 64), (100, 72), (33, 128), (19, 203), (700, 256), (40, 384), (9, 520),
                                    (21, 768), (333, 1024), (6, 1500), (5, 2048), (3, 4095), (2, 4096)])
def test_join_against_float64(type, rows, d):
    t = _make(rows, d, type, (rows,), True, True, "layer", "layer")
    _compare(_run(t, "layer", "layer"), _want(t, "layer", "layer"), (type, rows, d))


PARTS = [
    # gate, scale, mask, post, pre, bias
    (None, False, False, None, None, True), (None, False, False, None, "layer", True), (None, True, False, "rms", None, False),
    ("row", False, False, None, "rms", False), ("row", False, True, "layer", None, True), ("row", True, True, "rms", "rms", True),
    ("one", True, False, "layer", "rms", True), (None, False, True, "rms", "layer", False), ("one", False, True, None, None, True),
]


@pytest.mark.parametrize("d", [96, 130])
@pytest.mark.parametrize("gate,scale,mask,post,pre,bias", PARTS)
def test_join_of_any_parts(gate, scale, mask, post, pre, bias, d):
    rows = 150
    t = _make(rows, d, torch.bfloat16, {None: None, "row": (rows,), "one": (1,)}[gate], scale, mask, post, pre, bias)
    _compare(_run(t, post, pre), _want(t, post, pre), (gate, scale, mask, post, pre, bias, d))


@pytest.mark.parametrize("d", [64, 100, 384, 1024])
@pytest.mark.parametrize("shape,gate", [((4, 50), (4, 1)), ((4, 50), (1,)), ((4, 50), ()), ((3, 7, 11), (3, 7, 1)), ((3, 7, 11), (3, 1, 1)),
                                        ((1200, 3), (1200, 1)), ((2, 5000), (2, 1)), ((1, 9), (1, 1))])
def test_gate_rows_that_several_rows_share(shape, gate, d):
    """A gate row per sample, per row of a pair tensor, one for all."""
    t = _make(shape, d, torch.float16, gate, True, True, "rms", "layer")
    _compare(_run(t, "rms", "layer"), _want(t, "rms", "layer"), (shape, gate, d))


def test_gate_rows_inside_one_team():
    """So many rows that a team walks several whole gate rows, and parts of them."""
    t = _make((9000, 3), 16, torch.bfloat16, (9000, 1), False, True, "layer", None)
    _compare(_run(t, "layer", None), _want(t, "layer", None), "inside")
    t = _make((700, 129), 8, torch.float32, (700, 1), False, False, None, "rms")
    _compare(_run(t, None, "rms"), _want(t, None, "rms"), "parts")


def test_many_gate_rows():
    """More gate rows than one dimension of a grid may have blocks (65535), each of many rows."""
    g = torch.Generator(device=DEV).manual_seed(5)
    n, m, d = 66000, 257, 8
    x, u, dy = (torch.randn(n, m, d, generator=g, device=DEV, dtype=torch.float32).bfloat16() for _ in range(3))
    gate = torch.randn(n, 1, d, generator=g, device=DEV).bfloat16().requires_grad_(True)
    (got,) = torch.autograd.grad(blocks.block_join(x, u, gate=gate), gate, dy)
    s = torch.sigmoid(gate.detach().double())
    terms = dy.double() * u.double()
    slope = s * (1 - s)
    ref, amp = terms.sum(1, keepdim=True) * slope, terms.abs().sum(1, keepdim=True) * slope
    assert float(((got.double() - ref).abs() / (2.0**-16 * amp + 2.0**-8 * ref.abs() + 1e-30)).max()) <= 1.0


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 64), (1000, 64), (24, 384), (7, 33), (200, 1536)])
def test_norm_alone(rows, d, type, kind):
    t = _make(rows, d, type, None, False, False, None, kind)
    x, w, b = (t[k].clone().requires_grad_(True) for k in ("x", "pre_w", "pre_b"))
    h = blocks.block_norm(x, w, b, kind=kind)
    g = torch.autograd.grad(h, [x, w, b], t["dh"])
    res, amp, n, r = _norm64(t["x"].double(), w.detach().double(), b.detach().double(), kind, 1e-5)
    back, ba = _back64(n, r, w.detach().double(), t["dh"].double(), kind)
    big = 1 + t["x"].double().abs().amax(-1, keepdim=True) * r
    dh = t["dh"].double()
    want = {"h": (res, 2.0**-18 * amp), "x": (back, 2.0**-18 * ba * big),
            "w": ((dh * n).sum(0), (2.0**-16 * (dh * n).abs() + 2.0**-18 * dh.abs() * big).sum(0)), "b": (dh.sum(0), 2.0**-16 * dh.abs().sum(0))}
    _compare({"h": h.detach(), "x": g[0], "w": g[1], "b": g[2]}, want, (rows, d, type, kind))


def test_masked_rows_may_hold_anything():
    t = _make(64, 128, torch.bfloat16, (64,), True, True, "layer", "rms")
    clean = _run(t, "layer", "rms")
    for bad in (float("nan"), float("inf"), torch.finfo(torch.bfloat16).min):
        dirty = {k: v.clone() for k, v in t.items()}
        for k in ("u", "gate"):
            dirty[k][~t["mask"]] = bad
        got = _run(dirty, "layer", "rms")
        for k in clean:
            assert torch.equal(got[k], clean[k]), (bad, k)
    assert torch.equal(clean["y"][~t["mask"]], t["x"][~t["mask"]])
    assert not clean["u"][~t["mask"]].any() and not clean["gate"][~t["mask"]].any()


def test_no_row_is_valid():
    t = _make(40, 64, torch.float16, (1,), True, True, "layer", "layer")
    t["mask"].zero_()
    got = _run(t, "layer", "layer")
    assert torch.equal(got["y"], t["x"])
    for k in ("u", "gate", "scale", "post_w", "post_b"):
        assert not got[k].any(), k


def test_closed_and_open_gates():
    """Logits at the ends of the range: the gate is 0 or 1 and its gradient 0, never a NaN."""
    t = _make(8, 64, torch.float32, (8,), False, False, None, None)
    t["gate"] = torch.tensor([-1e30, -200.0, -88.5, -40.0, 40.0, 88.5, 200.0, 1e30], device=DEV)[:, None].expand(8, 64).contiguous()
    got = _run(t, None, None)
    assert torch.equal(got["y"][:3], t["x"][:3]) and torch.equal(got["y"][4:], t["x"][4:] + t["u"][4:])
    assert torch.isfinite(got["gate"]).all() and not got["gate"][[0, 1, 5, 6, 7]].any()


def test_rows_of_one_value():
    """Variance zero: the layer norm gives its bias."""
    x = torch.full((5, 96), 3.25, device=DEV, dtype=torch.bfloat16)
    b = torch.randn(96, device=DEV)
    assert torch.equal(blocks.block_norm(x, None, b), b.to(torch.bfloat16).expand(5, 96))


def test_a_common_offset_does_not_cancel():
    x = (torch.randn(50, 384, device=DEV) + 4000.0)  # fp32: the offset is exact to 2^-12, the variance is not lost
    want = torch.nn.functional.layer_norm(x.double(), (384,))
    assert float((blocks.block_norm(x).double() - want).abs().max()) < 4000 * 2.0**-18


@pytest.mark.parametrize("rows", [0])
def test_no_rows(rows):
    t = _make(rows, 64, torch.bfloat16, (rows,), True, False, "layer", "layer")
    got = _run(t, "layer", "layer")
    assert got["y"].shape == (0, 64) and got["h"].shape == (0, 64)
    for k in ("scale", "post_w", "post_b", "pre_w", "pre_b"):
        assert not got[k].any(), k


@pytest.mark.parametrize("shape,gate", [((4, 0), (4, 1)), ((0, 5), (1, 1)), ((0,), ())])
def test_gate_rows_of_no_rows(shape, gate):
    """The gradient of a gate row that no row shares is zero, whatever the memory held."""
    x = torch.zeros(*shape, 64, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(*gate, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    torch.full((4 * 64,), float("nan"), dtype=torch.bfloat16, device=DEV)  # (freed: what the next allocation finds)
    (got,) = torch.autograd.grad(blocks.block_join(x, x, gate=g), g, x)
    assert got.shape == g.shape and not got.any()


def test_layouts_and_types_are_converted():
    t = _make(60, 64, torch.bfloat16, (60,), True, False, "layer", "layer")
    want = _run(t, "layer", "layer")
    # rows of a wider tensor, a transposed tensor, an odd start
    wide = torch.zeros(60, 80, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:67] = t["x"]
    flat = torch.zeros(60 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    flat[1:] = t["u"].flatten()
    tr = t["gate"].t().contiguous().t()
    kw = dict(scale=t["scale"], post=blocks.Norm("layer", t["post_w"], t["post_b"]), pre=blocks.Norm("layer", t["pre_w"], t["pre_b"]))
    y, h = blocks.block_join(wide[:, 3:67], flat[1:].view(60, 64), gate=tr, **kw)
    # (an odd start takes single elements: the sums are formed in another order)
    assert float((y.float() - want["y"].float()).abs().max()) <= 2.0**-7 * float(want["y"].abs().max())
    y, h = blocks.block_join(wide[:, 3:67], t["u"], gate=tr, **kw)
    assert torch.equal(y, want["y"]) and torch.equal(h, want["h"])
    y, h = blocks.block_join(t["x"], t["u"].float(), gate=t["gate"].double(), **kw)
    assert torch.equal(y, want["y"]) and torch.equal(h, want["h"])
    u = t["u"].float().requires_grad_(True)
    (g,) = torch.autograd.grad(blocks.block_join(t["x"], u, gate=t["gate"], **kw)[0], u, t["dy"])
    assert g.dtype == torch.float32


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(64, device=DEV)
    N = blocks.Norm
    for call, word in [
        (lambda: blocks.block_join(x, x[:2]), "shape"), (lambda: blocks.block_join(x, x.long()), "float"),
        (lambda: blocks.block_join(x.double(), x), "bf16, fp16 or fp32"), (lambda: blocks.block_join(x, x.cpu()), "CUDA"),
        (lambda: blocks.block_join(x, x, gate=x[:3]), "leading dimensions"), (lambda: blocks.block_join(x, x, gate=x[:, :1]), "gate"),
        (lambda: blocks.block_join(x.view(2, 2, 64), x.view(2, 2, 64), gate=x[:2]), "leading dimensions"),
        (lambda: blocks.block_join(x, x, gate=x.view(1, 4, 64)), "at most"),
        (lambda: blocks.block_join(x, x, mask=torch.ones(3, device=DEV)), "mask"),
        (lambda: blocks.block_join(x, x, mask=torch.ones(4, 64, device=DEV)), "mask"),
        (lambda: blocks.block_join(x, x, scale=w.bfloat16()), "scale"), (lambda: blocks.block_join(x, x, scale=w[:8]), "scale"),
        (lambda: blocks.block_join(x, x, post=N("layer", w.half())), "fp32"), (lambda: blocks.block_norm(x, w.cpu()), "CUDA"),
        (lambda: blocks.block_norm(torch.zeros(2, 4097, device=DEV)), "4096"), (lambda: blocks.block_norm(x, eps=-1.0), "eps"),
        (lambda: blocks.block_norm(torch.zeros((), device=DEV)), "x must be"), (lambda: blocks.block_norm(torch.zeros(2, 0, device=DEV)), "x must be"),
        (lambda: blocks.block_norm(x.to_sparse()), "dense"),
    ]:
        with pytest.raises(RuntimeError, match=word):
            call()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda r: blocks.block_norm(r))(x)


def test_what_changes_before_the_backward_is_noticed():
    x = torch.randn(6, 64, device=DEV).bfloat16().requires_grad_(True)
    mask = torch.ones(6, dtype=torch.bool, device=DEV)
    y = blocks.block_join(x, x, mask=mask)
    mask[2] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(torch.ones_like(y))
    # hooks that give back other tensors than were saved
    f = torch.randn(6, 64, device=DEV).requires_grad_(True)
    for unpack in (lambda t: t.bfloat16(), lambda t: t[:3], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = blocks.block_join(f, f * 2, scale=torch.ones(64, device=DEV), mask=torch.ones(6, dtype=torch.bool, device=DEV))
        with pytest.raises(RuntimeError, match="came back with another"):
            y.backward(torch.ones_like(y))


def test_no_gradient_arrives():
    class Cut(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a):
            return a * 1

        @staticmethod
        def backward(ctx, g):
            return None

    x = torch.randn(6, 64, device=DEV).bfloat16().requires_grad_(True)
    u = torch.randn(6, 64, device=DEV).bfloat16().requires_grad_(True)
    y, h = blocks.block_join(x, u, post=blocks.Norm(), pre=blocks.Norm())
    g = torch.autograd.grad(Cut.apply(y).sum() + Cut.apply(h).sum(), [x, u], allow_unused=True)
    assert all(i is None or not i.any() for i in g)


def test_gradients_against_differences():
    """fp32, directional: (f(x + e v) - f(x - e v)) / 2e in double steps of the fp32 forward is off by 2^-24 |f| / e + e^2."""
    t = _make(16, 48, torch.float32, (16,), True, True, "layer", "rms")
    got = _run(t, "layer", "rms")
    e = 2.0**-7
    g = torch.Generator(device=DEV).manual_seed(5)

    def f(s):
        out = blocks.block_join(s["x"], s["u"], gate=s["gate"], scale=s["scale"], mask=s["mask"], post=blocks.Norm("layer", s["post_w"], s["post_b"]),
                                pre=blocks.Norm("rms", s["pre_w"], s["pre_b"]))
        return float((out[0].double() * t["dy"].double()).sum() + (out[1].double() * t["dh"].double()).sum())

    for k in ("x", "u", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b"):
        v = torch.randn(t[k].shape, generator=g, device=DEV)
        num = (f({**t, k: t[k] + e * v}) - f({**t, k: t[k] - e * v})) / (2 * e)
        want = float((got[k].double() * v.double()).sum())
        scale = float((got[k].double().square() * v.double().square()).sum().sqrt())
        assert abs(num - want) <= 40 * e * e * scale + 1e-2 * e * scale + 2e-3, (k, num, want)


def test_stack_of_modules():
    """norm, then blocks joined with the next norm: the same as norms and joins apart, to the rounding of y that the joined form does
    not see."""
    torch.manual_seed(0)
    x = torch.randn(2, 30, 64, device=DEV, dtype=torch.float32)
    norms = [mw.BlockNorm(64, "rms").to(DEV) for _ in range(3)]
    joins = [mw.BlockJoin(64, "rms", scale=0.5).to(DEV) for _ in range(3)]
    h, a = norms[0](x), x
    for i in range(3):
        u = torch.tanh(h)
        if i < 2:
            a, h = joins[i](a, u, next_norm=norms[i + 1])
        else:
            a = joins[i](a, u)
    b = x
    for i in range(3):
        b = joins[i](b, torch.tanh(norms[i](b)))
    assert float((a - b).abs().max()) <= 64 * 2.0**-24 * float(a.abs().max())


@pytest.mark.parametrize("d", [100, 130, 200, 203, 250, 1000])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("gate,bias", [(None, False), ("row", False), ("one", True), (None, True)])
def test_norms_without_weights(gate, bias, type, d):
    """No weight after the block and no scale: nothing but the width keeps the registers past it out of the next norm's mean."""
    rows = 70
    t = _make(rows, d, type, {None: None, "row": (rows,), "one": (1,)}[gate], False, True, "layer", "layer", bias)
    t["u"] += 1  # (a mean, which those registers take with its sign turned)
    ones = torch.ones(d, device=DEV)
    want = _want({**t, "post_w": ones, "pre_w": ones}, "layer", "layer")
    del t["post_w"], t["pre_w"], want["post_w"], want["pre_w"]
    _compare(_run(t, "layer", "layer"), want, (gate, bias, type, d))


def test_c_calls_without_a_norm_do_not_read_its_parameters():
    """post_kind 0: t = u, whatever post_w and post_b point to, on tiles and (one element off a boundary) on the first kernels."""
    import ctypes

    from miniworld_b200 import _lib

    lib = _lib.load()
    t = _make(50, 100, torch.bfloat16, None, True, False, None, "layer")
    w, b = torch.full((100,), 3.0, device=DEV), torch.full((100,), 5.0, device=DEV)
    need = ctypes.c_size_t(0)
    assert lib.b200_block_join_workspace_bytes(50, 100, 1, ctypes.byref(need)) == 0
    ws = torch.empty(need.value + 1024, dtype=torch.uint8, device=DEV)
    at = (ws.data_ptr() + 1023) // 1024 * 1024
    p = lambda v: None if v is None else v.data_ptr()  # noqa: E731

    def run(post_w, post_b, off):
        def place(v):
            room = torch.zeros(v.numel() + 8, dtype=v.dtype, device=DEV)[off:off + v.numel()].view(v.shape)
            return room.copy_(v)

        x, u, dy, dh = (place(t[k]) for k in ("x", "u", "dy", "dh"))
        y, h, dx, du = (place(torch.zeros_like(x)) for _ in range(4))
        stats, dscale = torch.zeros(50, 2, device=DEV), torch.zeros(100, device=DEV)
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.b200_block_join_forward(p(x), p(u), None, None, p(t["scale"]), p(post_w), p(post_b), p(t["pre_w"]), p(t["pre_b"]), p(y), p(h), None,
                                           p(stats), 50, 100, 1, 0, 0, 1, 1e-5, 1e-5, stream) == 0
        assert lib.b200_block_join_backward(p(dy), p(dh), p(x), p(u), None, None, p(t["scale"]), p(post_w), p(post_b), p(t["pre_w"]), p(t["pre_b"]), None,
                                            p(stats), p(dx), p(du), None, p(dscale), None, None, None, None, at, need.value, 50, 100, 1, 0, 0, 1,
                                            stream) == 0
        torch.cuda.synchronize()
        return [v.clone() for v in (y, h, stats, dx, du, dscale)]

    for off in (0, 1):
        for a, b_ in zip(run(w, b, off), run(None, None, off)):
            assert torch.equal(a, b_), off
