"""Workloads of the block operators: the norms around a block joined with its gate, residual scale and residual, and the gated
feed-forward of any width.

A case is one call that a model makes on its token, pair or alignment tensors, seen as ``[samples, rows, width]``. The keys:

  op      "norm": the norm in front of a block; "join": residual add of a block's output through a norm, a sigmoid gate, a scale
          per channel and a row mask, with the norm in front of the next block; "ff": the gated feed-forward
  mode    "infer", or "train" (forward and backward: outputs and every gradient come back)
  type    "bf16", "fp16" or "fp32" of the activations (and of the feed-forward's weights); norm parameters are fp32
  b, m    samples and rows per sample;  d: width
  kind    "layer" or "rms" (norm and join);  gate: "none", "row" (logits per element) or "sample" (one vector per sample)
  mask    rows at the end of each sample are padding (join);  next: the join also gives the next block's normalised input
  h, act  hidden width and activation, "silu" or "gelu" (ff)
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def _norm(name, mode, type, b, m, d, kind):
    return {"name": name, "op": "norm", "mode": mode, "type": type, "b": b, "m": m, "d": d, "kind": kind}


def _join(name, mode, type, b, m, d, kind, gate, mask, next):
    return {"name": name, "op": "join", "mode": mode, "type": type, "b": b, "m": m, "d": d, "kind": kind, "gate": gate, "mask": mask,
            "next": next}


def _ff(name, mode, type, b, m, d, h, act):
    return {"name": name, "op": "ff", "mode": mode, "type": type, "b": b, "m": m, "d": d, "h": h, "act": act}


def listed():
    return [
        # the single representation of a short peptide: the call is a launch
        _norm("norm_infer_m24_d384", "infer", "bf16", 1, 24, 384, "layer"),
        # training on a crop's alignment: 512 sequences of 384 tokens, 64 channels
        _norm("norm_train_msa_d64", "train", "bf16", 512, 384, 64, "layer"),
        # a whole sequence in full precision, at a width of no round size
        _join("join_infer_m203_d203_fp32", "infer", "fp32", 1, 203, 203, "layer", "row", False, True),
        # the pair tensor of a 384-token crop between two blocks
        _join("join_infer_pair384_d128", "infer", "bf16", 1, 384 * 384, 128, "layer", "row", False, True),
        # a batch of token tensors conditioned by one gate vector a sample, padded at the end
        _join("join_train_b4_m768_d768", "train", "fp16", 4, 768, 768, "rms", "sample", True, True),
        # training on two pair tensors of 256 tokens, padded rows masked
        _join("join_train_pair256_d128", "train", "bf16", 2, 256 * 256, 128, "layer", "row", True, True),
        # a wide trunk, the last join of a stack (no norm follows)
        _join("join_train_m8192_d1024", "train", "bf16", 1, 8192, 1024, "rms", "row", False, False),
        # one token
        _ff("ff_infer_m1_d768", "infer", "bf16", 1, 1, 768, 2048, "silu"),
        # the single representation of a 384-token crop
        _ff("ff_infer_m384_d384", "infer", "bf16", 1, 384, 384, 1536, "silu"),
        # a crop's alignment, 512 sequences of 384 tokens, 64 channels
        _ff("ff_infer_msa_d64", "infer", "bf16", 512, 384, 64, 256, "silu"),
        # training on three short sequences
        _ff("ff_train_b3_m203_d384", "train", "fp16", 3, 203, 384, 1536, "gelu"),
        # training on the tokens of a wide trunk
        _ff("ff_train_m16384_d1024", "train", "bf16", 1, 16384, 1024, 4096, "silu"),
    ]


_MOST_ELEMENTS = 384 * 384 * 128  # of a norm's or a join's tensors: the largest listed one
_MOST_FLOPS = 18.0 * 16384 * 1024 * 4096  # of a feed-forward: likewise
_MOST_HIDDEN = 16384 * 4096


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "join", "join", "ff", "ff"))
    mode = rng.choice(("infer", "train"))
    b = rng.choice((1, 1, 2, 3, 4, 8))
    while True:
        if op == "ff":
            d = _spread(rng, 8, 128) * 8  # tensor rows of whole 16-byte pieces
            h = max(8, int(d * rng.choice((2.0, 2.667, 4.0))) // 8 * 8)
            case = _ff(None, mode, rng.choice(("bf16", "bf16", "fp16")), b, _spread(rng, 1, 100000), d, h, rng.choice(("silu", "silu", "gelu")))
            if work(case)["flops"] <= _MOST_FLOPS and b * case["m"] * h <= _MOST_HIDDEN:
                break
        else:
            d = _spread(rng, 32, 1024)
            if rng.random() < 0.6:  # widths are round more often than not
                d = (d + 31) // 32 * 32
            m, type, kind = _spread(rng, 1, 100000), rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice(("layer", "rms"))
            if op == "norm":
                case = _norm(None, mode, type, b, m, d, kind)
            else:
                case = _join(None, mode, type, b, m, d, kind, rng.choice(("none", "row", "sample")), rng.random() < 0.4, rng.random() < 0.7)
            if b * m * d <= _MOST_ELEMENTS:
                break
    del case["name"]
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    b, m, d, type, train = case["b"], case["m"], case["d"], TYPES[case["type"]], case["mode"] == "train"

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    # the residual stream: channels of different magnitude, a common offset
    x = (normal(b, m, d) * (0.5 + 1.5 * torch.rand(d, generator=gen, device="cuda")) + 0.1 * normal(d)).to(type)
    s = {"case": case, "x": x}
    leaves = ["x"]
    if case["op"] == "ff":
        h = case["h"]
        s["w_a"], s["w_b"], s["w_s"] = ((normal(h, d) * d**-0.5).to(type), (normal(h, d) * d**-0.5).to(type), (normal(d, h) * h**-0.5).to(type))
        leaves += ["w_a", "w_b", "w_s"]
        grads = ["dy"]
    else:
        def norm(name):
            s[name + "_w"] = 1.0 + 0.1 * normal(d)
            leaves.append(name + "_w")
            s[name + "_b"] = 0.02 * normal(d) if case["kind"] == "layer" else None
            if s[name + "_b"] is not None:
                leaves.append(name + "_b")

        if case["op"] == "norm":
            norm("pre")
            grads = ["dh"]
        else:
            s["u"] = (0.7 * normal(b, m, d)).to(type)
            s["scale"] = 0.1 + 0.05 * normal(d)
            leaves += ["u", "scale"]
            norm("post")
            if case["gate"] != "none":
                s["gate"] = normal(b, m if case["gate"] == "row" else 1, d).to(type)
                leaves.append("gate")
            if case["mask"]:
                length = torch.randint((3 * m + 3) // 4, m + 1, (b, 1), generator=gen, device="cuda")
                s["mask"] = torch.arange(m, device="cuda")[None, :] < length
            grads = ["dy"]
            if case["next"]:
                norm("pre")
                grads.append("dh")
    if train:
        for name in grads:
            s[name] = (0.01 * normal(b, m, d)).to(type)
        for name in leaves:
            s[name].requires_grad_(True)
        s["leaves"] = leaves
    return s


def _plain_norm(v, w, b, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * w
    return n if b is None else n + b


def _plain(s):
    """The operators in fp32, rounded once at the end: their outputs before that rounding."""
    case, x = s["case"], s["x"].float()
    if case["op"] == "norm":
        return {"h": _plain_norm(x, s["pre_w"], s["pre_b"], case["kind"])}
    if case["op"] == "ff":
        a, b = x @ s["w_a"].float().t(), x @ s["w_b"].float().t()
        if case["act"] == "silu":
            g = a * torch.sigmoid(a)
        else:
            g = 0.5 * a * (1.0 + torch.erf(a * 0.5**0.5))
        return {"y": (g * b) @ s["w_s"].float().t()}
    t = _plain_norm(s["u"].float(), s["post_w"], s["post_b"], case["kind"]) * s["scale"]
    if "gate" in s:
        t = t * torch.sigmoid(s["gate"].float())
    if "mask" in s:
        t = torch.where(s["mask"][..., None], t, torch.zeros((), device=t.device))
    y = x + t
    out = {"y": y}
    if case["next"]:
        out["h"] = _plain_norm(y, s["pre_w"], s["pre_b"], case["kind"])
    return out


def _own(s):
    from miniworld_b200 import blocks

    case = s["case"]
    if case["op"] == "norm":
        return {"h": blocks.block_norm(s["x"], s["pre_w"], s["pre_b"], kind=case["kind"], eps=EPS)}
    if case["op"] == "ff":
        return {"y": blocks.gated_feed_forward(s["x"], s["w_a"], s["w_b"], s["w_s"], activation=case["act"])}
    post = blocks.Norm(case["kind"], s["post_w"], s["post_b"], EPS)
    pre = blocks.Norm(case["kind"], s["pre_w"], s["pre_b"], EPS) if case["next"] else None
    out = blocks.block_join(s["x"], s["u"], gate=s.get("gate"), scale=s["scale"], mask=s.get("mask"), post=post, pre=pre)
    return dict(zip(("y", "h"), out)) if case["next"] else {"y": out}


def run(state):
    s = state
    type = s["x"].dtype
    if "leaves" not in s:
        with torch.no_grad():
            out = _own(s) if own else _plain(s)
            return {k: v.to(type) for k, v in out.items()}
    out = {k: v.to(type) for k, v in (_own(s) if own else _plain(s)).items()}
    names = s["leaves"]
    grads = torch.autograd.grad(list(out.values()), [s[n] for n in names], [s["d" + k] for k in out])
    return {**{k: v.detach() for k, v in out.items()}, **dict(zip(names, grads))}


def _exact_norm(v, w, b, kind):
    """(normalised values without the affine part, rstd, result) of the last dimension."""
    d = v.shape[-1]
    c = v - v.sum(-1, keepdim=True) / d if kind == "layer" else v
    r = ((c**2).sum(-1, keepdim=True) / d + EPS) ** -0.5
    return c * r, r, c * r * w + (0 if b is None else b)


def _exact_norm_back(n, r, w, g, kind):
    """Gradient of the norm's input from that of its result ``g``."""
    d = n.shape[-1]
    q = g * w
    back = q - n * ((q * n).sum(-1, keepdim=True) / d)
    if kind == "layer":
        back = back - q.sum(-1, keepdim=True) / d
    return r * back


def exact(case, seed):
    """What ``run`` returns, in float64 by the formulas of the operators and of their gradients."""
    s = prepare(case, seed)
    v = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.dtype != torch.bool}
    train, kind = case["mode"] == "train", case.get("kind")
    v.setdefault("pre_b", None)
    v.setdefault("post_b", None)
    rows = (0, 1)
    if case["op"] == "norm":
        n, r, h = _exact_norm(v["x"], v["pre_w"], v["pre_b"], kind)
        out = {"h": h}
        if train:
            out["x"] = _exact_norm_back(n, r, v["pre_w"], v["dh"], kind)
            out["pre_w"] = (v["dh"] * n).sum(rows)
            if v["pre_b"] is not None:
                out["pre_b"] = v["dh"].sum(rows)
    elif case["op"] == "ff":
        x = v["x"].reshape(-1, case["d"])
        a, b = torch.einsum("md,hd->mh", x, v["w_a"]), torch.einsum("md,hd->mh", x, v["w_b"])
        if case["act"] == "silu":
            sg = 1.0 / (1.0 + torch.exp(-a))
            act, slope = a * sg, sg * (1.0 + a * (1.0 - sg))
        else:
            cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
            act, slope = a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
        out = {"y": torch.einsum("mh,dh->md", act * b, v["w_s"]).reshape(s["x"].shape)}
        if train:
            dy = v["dy"].reshape(-1, case["d"])
            dh = torch.einsum("md,dh->mh", dy, v["w_s"])
            da, db = dh * b * slope, dh * act
            out["x"] = (torch.einsum("mh,hd->md", da, v["w_a"]) + torch.einsum("mh,hd->md", db, v["w_b"])).reshape(s["x"].shape)
            out["w_a"], out["w_b"] = torch.einsum("mh,md->hd", da, x), torch.einsum("mh,md->hd", db, x)
            out["w_s"] = torch.einsum("md,mh->dh", dy, act * b)
    else:
        n, r, t = _exact_norm(v["u"], v["post_w"], v["post_b"], kind)
        g = 1.0 / (1.0 + torch.exp(-v["gate"])) if "gate" in v else torch.ones(1, 1, 1, dtype=torch.float64, device="cuda")
        valid = s["mask"][..., None].double() if "mask" in s else 1.0
        y = v["x"] + t * g * v["scale"] * valid
        out = {"y": y}
        if case["next"]:
            ny, ry, out["h"] = _exact_norm(y, v["pre_w"], v["pre_b"], kind)
        if train:
            e = v["dy"]
            if case["next"]:
                e = e + _exact_norm_back(ny, ry, v["pre_w"], v["dh"], kind)
            dt = e * g * v["scale"] * valid
            out["x"] = e
            out["u"] = _exact_norm_back(n, r, v["post_w"], dt, kind)
            out["scale"] = (e * g * t * valid).sum(rows)
            out["post_w"] = (dt * n).sum(rows)
            if v["post_b"] is not None:
                out["post_b"] = dt.sum(rows)
            if "gate" in v:
                dg = e * t * v["scale"] * valid * g * (1.0 - g)
                out["gate"] = dg if case["gate"] == "row" else dg.sum(1, keepdim=True)
            if case["next"]:
                out["pre_w"] = (v["dh"] * ny).sum(rows)
                if v["pre_b"] is not None:
                    out["pre_b"] = v["dh"].sum(rows)
    return out


def work(case):
    """One read of every input and one write of every output; the products of the feed-forward and of its gradients (twice the
    forward's: nothing that is computed again counts), and the few operations per element of a norm."""
    b, m, d, size = case["b"], case["m"], case["d"], {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    train, rows = case["mode"] == "train", b * m
    if case["op"] == "ff":
        weights, flops = 3 * case["h"] * d, 6.0 * rows * d * case["h"]
        if train:
            return {"bytes": size * (4 * rows * d + 2 * weights), "flops": 3.0 * flops}
        return {"bytes": size * (2 * rows * d + weights), "flops": flops}
    params = 4 * d * (2 if case["kind"] == "layer" else 1)
    if case["op"] == "norm":
        tensors, flops = (4 if train else 2) * rows * d, (18.0 if train else 8.0) * rows * d
    else:
        gates = {"none": 0, "row": rows * d, "sample": b * d}[case["gate"]]
        outs = 2 if case["next"] else 1
        tensors = (2 + outs) * rows * d + gates
        if train:
            tensors += (outs + 2) * rows * d + gates
        flops = (50.0 if train else 20.0) * rows * d
        params = params * outs + 4 * d
    return {"bytes": size * tensors + params * (2 if train else 1) + (rows if case.get("mask") else 0), "flops": flops}
