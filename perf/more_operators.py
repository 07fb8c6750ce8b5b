"""Workloads of the token operators: attention over the tokens of a batch or of packed sequences with a learned bias of their relative
position, the relative position added to the pair tensor, and dropout whose mask is drawn again wherever it is needed.

A case is one call that a model makes. The keys:

  op       "attention"; "position": the pair tensor with the bucket of every pair's distance added to it; "dropout": a residual add of
           a block's output with some of its elements dropped
  mode     "infer", or "train" (forward and backward: outputs and every gradient come back)
  type     "bf16", "fp16" or "fp32" of the activations (attention: 16 bits; its table of biases has the same type)
  form     attention: "batch", ``b`` samples of ``m`` tokens, or "packed", ``b`` sequences of many lengths up to ``m`` in one tensor
  b, m     samples and tokens of a sample (of the longest sequence)
  spare    packed: rows behind the last sequence
  h, hk, d  heads of the queries, heads of keys and values, their width
  causal   a token attends to itself and those before it
  bias     "none"; "near": one bucket for each distance up to 32, those beyond in the outer two; "log": 32 buckets, exact for short
           distances, then wider and wider up to 128
  mask     attention: "none"; "tail": samples are padded at the end (one of several to nothing); "holes": single tokens are missing
  n, c     position: tokens and channels of the pair tensor;  chains: chains of the sample, whose pairs share one bucket
  shape, width, shared  dropout: rows, channels, and how many rows in a sequence share one mask (1: none do)
  p        share of the elements that are dropped
"""

import math
import random

import numpy
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
REACH = 32  # distances of one bucket each


def _attention(name, mode, type, form, b, m, h, hk, d, causal, bias, mask, spare=0):
    return {"name": name, "op": "attention", "mode": mode, "type": type, "form": form, "b": b, "m": m, "h": h, "hk": hk, "d": d,
            "causal": causal, "bias": bias, "mask": mask, "spare": spare}


def _position(name, mode, type, b, n, c, chains):
    return {"name": name, "op": "position", "mode": mode, "type": type, "b": b, "n": n, "c": c, "chains": chains}


def _dropout(name, mode, type, rows, width, shared, p):
    return {"name": name, "op": "dropout", "mode": mode, "type": type, "rows": rows, "width": width, "shared": shared, "p": p}


def listed():
    return [
        # the single representation of a short peptide: the call is a launch
        _attention("attention_infer_m24_h16_d24", "infer", "bf16", "batch", 1, 24, 16, 16, 24, False, "near", "none"),
        # four crops, padded at the end, through a wide token trunk
        _attention("attention_infer_b4_m384_h16_d48", "infer", "bf16", "batch", 4, 384, 16, 16, 48, False, "near", "tail"),
        # the rows of a crop's alignment
        _attention("attention_infer_msa512_m384_h8_d32", "infer", "bf16", "batch", 512, 384, 8, 8, 32, False, "none", "none"),
        # sequences of a database read by a causal model, four query heads to one of the keys
        _attention("attention_infer_packed48_causal_h16_d128", "infer", "bf16", "packed", 48, 8192, 16, 4, 128, True, "none", "none"),
        # training on whole proteins, packed without padding
        _attention("attention_train_packed64_h8_d64", "train", "fp16", "packed", 64, 1400, 8, 8, 64, False, "log", "none", 37),
        # training on two long complexes
        _attention("attention_train_b2_m4096_h16_d64", "train", "bf16", "batch", 2, 4096, 16, 16, 64, False, "near", "none"),
        # a small crop before the first block
        _position("position_infer_n128_c128", "infer", "bf16", 1, 128, 128, 1),
        # training crops of a protein of no round length in full precision, on a template stack's width
        _position("position_train_b4_n203_c64_fp32", "train", "fp32", 4, 203, 64, 2),
        # training on a crop of a complex
        _position("position_train_n768_c128", "train", "bf16", 1, 768, 128, 3),
        # a step on the single representation of a short peptide
        _dropout("dropout_train_m24_d384", "train", "bf16", 24, 384, 1, 0.15),
        # the update of a pair tensor, one mask for all rows as the triangle updates drop theirs
        _dropout("dropout_train_pair384_row", "train", "bf16", 384 * 384, 128, 384, 0.25),
        # the tokens of a wide trunk
        _dropout("dropout_train_m16384_d1024", "train", "fp16", 16384, 1024, 1, 0.1),
    ]


_MOST_FLOPS = 12.0 * 2 * 4096 * 4096 * 16 * 64  # of an attention: the largest listed one
_MOST_TOKENS = 512 * 384 * 8 * 32  # elements of its queries
_MOST_PAIRS = 768 * 768 * 128  # of a pair tensor
_MOST_ELEMENTS = 384 * 384 * 128


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "position", "dropout"))
    mode = rng.choice(("infer", "train"))
    while True:
        if op == "attention":
            hk, group = _spread(rng, 1, 16), rng.choice((1, 1, 1, 2, 4))
            form = rng.choice(("batch", "packed"))
            b, m = (_spread(rng, 1, 512) if rng.random() < 0.5 else rng.choice((1, 2, 3))), _spread(rng, 1, 8192)
            case = _attention(None, mode, rng.choice(("bf16", "bf16", "fp16")), form, b, m, hk * group, hk, _spread(rng, 1, 16) * 8,
                              rng.random() < 0.4, rng.choice(("none", "near", "log")),
                              rng.choice(("none", "tail", "holes")) if form == "batch" else "none",
                              rng.choice((0, 5, 200)) if form == "packed" else 0)
            if work(case)["flops"] <= _MOST_FLOPS and sum(lengths(case)) * case["h"] * case["d"] <= _MOST_TOKENS:
                break
        elif op == "position":
            case = _position(None, mode, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice((1, 1, 2, 4)), _spread(rng, 1, 1024),
                             rng.choice((64, 128, 128, _spread(rng, 16, 256))), rng.choice((1, 2, 5)))
            if case["b"] * case["n"] ** 2 * case["c"] <= _MOST_PAIRS:
                break
        else:
            shared, width = rng.choice((1, 1, _spread(rng, 2, 512))), _spread(rng, 32, 1024)
            if rng.random() < 0.7:  # widths are round more often than not
                width = (width + 31) // 32 * 32
            case = _dropout(None, mode, rng.choice(("bf16", "bf16", "fp16", "fp32")), shared * _spread(rng, 1, 50000), width, shared,
                            rng.choice((0.05, 0.1, 0.15, 0.25, 0.5)))
            if case["rows"] * width <= _MOST_ELEMENTS:
                break
    del case["name"]
    return case


def lengths(case):
    """Tokens of each sequence, the same for every seed: a packed batch is a few long sequences and many short ones."""
    if case["form"] == "batch":
        return [case["m"]] * case["b"]
    rng = random.Random(case["b"] * 10007 + case["m"])
    return [case["m"]] + [_spread(rng, 1, case["m"]) for _ in range(case["b"] - 1)]


def _bucket_map(kind):
    """Bucket of the distances -reach .. reach of the key from the query (those beyond count as the outer two)."""
    if kind == "near":
        return list(range(2 * REACH + 1))
    exact, half, reach = 8, 16, 128

    def bucket(d):
        far = abs(d)
        if far >= exact:
            far = min(half - 1, exact + int(math.log(far / exact) / math.log(reach / exact) * (half - exact)))
        return far + (half if d > 0 else 0)

    return [bucket(d) for d in range(-reach, reach + 1)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    type, train = TYPES[case["type"]], case["mode"] == "train"

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "attention":
        h, hk, d = case["h"], case["hk"], case["d"]
        own_lengths = lengths(case)
        lead = (case["b"], case["m"])
        if case["form"] == "packed":
            lead = (sum(own_lengths) + case["spare"],)
            ends = torch.tensor([0] + own_lengths, dtype=torch.int64).cumsum(0)
            s["offsets"] = ends.to(device="cuda", dtype=torch.int32)
        # (normalised projections: logits of about one, a common part of the values)
        s["q"], s["k"] = normal(*lead, h, d).to(type), normal(*lead, hk, d).to(type)
        s["v"] = (normal(*lead, hk, d) + 0.3 * normal(hk, d)).to(type)
        leaves = ["q", "k", "v"]
        if case["bias"] != "none":
            buckets = _bucket_map(case["bias"])
            s["bucket_of"] = torch.tensor(buckets, dtype=torch.int32, device="cuda")
            s["table"] = (0.5 * normal(max(buckets) + 1, h)).to(type)
            leaves.append("table")
        if case["mask"] == "tail":
            length = torch.randint((case["m"] + 1) // 2, case["m"] + 1, (case["b"], 1), generator=gen, device="cuda")
            if case["b"] > 3:
                length[-1] = 0
            s["mask"] = torch.arange(case["m"], device="cuda")[None, :] < length
        elif case["mask"] == "holes":
            s["mask"] = torch.rand(case["b"], case["m"], generator=gen, device="cuda") >= 0.1
        grads = {"o": normal(*lead, h, d)}
    elif case["op"] == "position":
        b, n, c, chains = case["b"], case["n"], case["c"], case["chains"]
        s["z"] = (normal(b, n, n, c) * (0.5 + 1.5 * torch.rand(c, generator=gen, device="cuda"))).to(type)
        s["table"] = 0.3 * normal(2 * REACH + 2, c)
        # residues of a chain follow one another, with a gap here and there where a crop left some out
        step = torch.where(torch.rand(b, n, generator=gen, device="cuda") < 0.02, 40, 1)
        s["chain"] = (torch.arange(n, device="cuda") * chains // n).expand(b, n).contiguous()
        s["index"] = step.cumsum(1) - 700 * s["chain"]
        s["bucket_of"] = torch.tensor(_bucket_map("near"), dtype=torch.int32, device="cuda")
        leaves, grads = ["z", "table"], {"y": normal(b, n, n, c)}
    else:
        shape = (case["rows"] // case["shared"], case["shared"], case["width"])
        s["x"], s["u"] = normal(*shape).to(type), (0.7 * normal(*shape)).to(type)
        s["key"] = torch.randint(-(2**62), 2**62, (2,), generator=gen, device="cuda")
        leaves, grads = ["x", "u"], {"y": normal(*shape)}
    if train:
        for k, g in grads.items():
            s["d" + k] = (0.01 * g).to(type)
        for name in leaves:
            s[name].requires_grad_(True)
        s["leaves"] = leaves
    return s


# ---------------------------------------------------------------------------------------------- plain forms
_SCORES = 1 << 28  # scores at a time


def _plain_scores(s, q, k, valid, at):
    """Scores in fp32 of sequences [n, heads, tokens, d] of one length, and which of them count; ``at``: their heads."""
    case, m = s["case"], q.shape[2]
    scores = (q * case["d"] ** -0.5) @ k.transpose(-1, -2)
    if "table" in s:
        reach = s["bucket_of"].numel() // 2
        place = torch.arange(m, device="cuda")
        distance = (place[None, :] - place[:, None]).clamp(-reach, reach) + reach
        scores = scores + s["table"].detach().float()[s["bucket_of"].long()[distance]][..., at].permute(2, 0, 1)
    counts = torch.ones(m, m, dtype=torch.bool, device="cuda")
    if case["causal"]:
        counts = counts.tril()
    counts = counts[None, None]
    if valid is not None:
        counts = counts & valid[:, None, None, :] & valid[:, None, :, None]
    return scores, counts


def _plain_softmax(scores, counts):
    scores = torch.where(counts, scores, torch.full((), -math.inf, device="cuda"))
    most = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(most), most, torch.zeros_like(most)))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _groups(case):
    """(first sequence, its first row, sequences, tokens of each) of the sequences that are worked on together."""
    all_lengths = lengths(case)
    if case["form"] == "packed":
        row = 0
        for i, m in enumerate(all_lengths):
            yield i, row, 1, m
            row += m
        return
    m = case["m"]
    most = max(1, _SCORES // (m * m))
    for i in range(0, case["b"], most):
        yield i, i * m, min(most, case["b"] - i), m


def _plain_attention(s):
    case = s["case"]
    h, hk, d = case["h"], case["hk"], case["d"]
    group, train = h // hk, "leaves" in s
    q, k, v = (s[t].detach().reshape(-1, s[t].shape[-2], d) for t in "qkv")
    do = s["do"].reshape(-1, h, d) if train else None
    out = {"o": torch.zeros(q.shape, device="cuda")}
    if train:
        out.update(q=torch.zeros(q.shape, device="cuda"), k=torch.zeros(k.shape, device="cuda"), v=torch.zeros(v.shape, device="cuda"))
        if "table" in s:
            out["table"] = torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda")
    mask = s["mask"].reshape(-1) if "mask" in s else None
    for first, row, n, m in _groups(case):
        rows = slice(row, row + n * m)
        valid = mask[rows].view(n, m) if mask is not None else None
        heads = max(1, min(hk, _SCORES // (n * m * m * group)))

        def part(t, at):  # [n, heads, m, d] in fp32
            return t[rows, at].float().view(n, m, -1, d).transpose(1, 2)

        def put(t, at, value):
            t[rows, at] = value.transpose(1, 2).reshape(n * m, -1, d)

        for at in range(0, hk, heads):
            atk = slice(at, min(at + heads, hk))
            atq = slice(atk.start * group, atk.stop * group)
            qp, kp, vp = part(q, atq), part(k, atk).repeat_interleave(group, 1), part(v, atk).repeat_interleave(group, 1)
            if valid is not None:
                vp = torch.where(valid[:, None, :, None], vp, torch.zeros((), device="cuda"))
            prob = _plain_softmax(*_plain_scores(s, qp, kp, valid, atq))
            o = prob @ vp
            put(out["o"], atq, o)
            if not train:
                continue
            dop = part(do, atq)
            if valid is not None:
                dop = torch.where(valid[:, None, :, None], dop, torch.zeros((), device="cuda"))
            dv = prob.transpose(-1, -2) @ dop
            ds = prob * (dop @ vp.transpose(-1, -2) - (dop * o).sum(-1, keepdim=True))
            del prob
            put(out["q"], atq, ds @ kp * d**-0.5)
            dk = ds.transpose(-1, -2) @ qp * d**-0.5
            put(out["k"], atk, dk.unflatten(1, (-1, group)).sum(2))
            put(out["v"], atk, dv.unflatten(1, (-1, group)).sum(2))
            if "table" in s:
                # diagonals of [m, m] are columns of [m, 2 m - 1] once every row is moved one place less than the row before it
                reach, total = s["bucket_of"].numel() // 2, ds.sum(0, dtype=torch.float64).flip(1)
                skewed = torch.nn.functional.pad(total, (0, m)).flatten(1)[:, : m * (2 * m - 1)].view(-1, m, 2 * m - 1)
                distance = torch.arange(1 - m, m, device="cuda").clamp(-reach, reach) + reach
                number = torch.arange(s["table"].shape[0], device="cuda")
                one = (s["bucket_of"][distance][:, None] == number).double()
                out["table"][:, atq] += (skewed.sum(1) @ one).t()
    return {name: t.view(s[name if name != "o" else "q"].shape) for name, t in out.items()}


def _plain_buckets(s):
    reach = s["bucket_of"].numel() // 2
    distance = (s["index"][:, None, :] - s["index"][:, :, None]).clamp(-reach, reach) + reach
    bucket = s["bucket_of"].long()[distance]
    same = s["chain"][:, None, :] == s["chain"][:, :, None]
    return torch.where(same, bucket, s["table"].shape[0] - 1)


def _plain_position(s):
    bucket = _plain_buckets(s)
    out = {"y": s["z"].detach().float() + s["table"].detach()[bucket]}
    if "leaves" in s:
        out["z"] = s["dy"].float()
        buckets, c = s["table"].shape
        total = torch.zeros(buckets, c, dtype=torch.float64, device="cuda")
        rows = s["dy"].reshape(-1, c)
        number = torch.arange(buckets, device="cuda")
        for at in range(0, rows.shape[0], 1 << 18):
            one = (bucket.view(-1)[at : at + (1 << 18), None] == number).double()
            total += one.t() @ rows[at : at + (1 << 18)].double()
        out["table"] = total
    return out


_MASK32 = 0xFFFFFFFF


def _plain_numbers(key, count):
    """``count`` 16-bit numbers of the counter-based generator Philox-4x32-10 (Salmon et al. 2011): block i of eight from the counter
    (i, second word of the key) and the first word as its key, the low half of every word first."""
    i = torch.arange((count + 7) // 8, device="cuda")
    word = [i & _MASK32, i >> 32, (key[1] & _MASK32).expand_as(i), (key[1] >> 32 & _MASK32).expand_as(i)]
    k0, k1 = key[0] & _MASK32, key[0] >> 32 & _MASK32
    for _ in range(10):
        a, b = word[0] * 0xD2511F53, word[2] * 0xCD9E8D57
        word = [(b >> 32 & _MASK32) ^ word[1] ^ k0, b & _MASK32, (a >> 32 & _MASK32) ^ word[3] ^ k1, a & _MASK32]
        k0, k1 = k0 + 0x9E3779B9 & _MASK32, k1 + 0xBB67AE85 & _MASK32
    halves = [w >> shift & 0xFFFF for w in word for shift in (0, 16)]
    return torch.stack(halves, 1).view(-1)[:count]


def _threshold(p):
    return int(round(p * 65536))


def _plain_dropout(s):
    outer, _, width = s["x"].shape
    shared = s["case"]["shared"]
    limit = _threshold(s["case"]["p"])
    shape = (outer, 1, width) if shared > 1 else s["x"].shape
    keep = _plain_numbers(s["key"], math.prod(shape)).view(shape) >= limit
    scale = 65536.0 / (65536 - limit)
    zero = torch.zeros((), device="cuda")
    out = {"y": s["x"].detach().float() + torch.where(keep, s["u"].detach().float() * scale, zero)}
    if "leaves" in s:
        out["x"] = s["dy"].float()
        out["u"] = torch.where(keep, s["dy"].float() * scale, zero)
    return out


def _own(s):
    from miniworld_b200 import blocks

    case = s["case"]
    if case["op"] == "attention":
        return {"o": blocks.token_attention(s["q"], s["k"], s["v"], offsets=s.get("offsets"), mask=s.get("mask"), causal=case["causal"],
                                            table=s.get("table"), bucket_of=s.get("bucket_of"))}
    if case["op"] == "position":
        return {"y": blocks.relative_position(s["z"], s["table"], s["index"], bucket_of=s["bucket_of"], chain=s["chain"])}
    return {"y": blocks.block_dropout(s["x"], s["u"], s["key"], p=case["p"], shared=1 if case["shared"] > 1 else None)}


def run(state):
    s = state
    if not own:
        plain = {"attention": _plain_attention, "position": _plain_position, "dropout": _plain_dropout}[s["case"]["op"]]
        type = TYPES[s["case"]["type"]]
        with torch.no_grad():
            return {k: v.to(s[k].dtype if k in s else type) for k, v in plain(s).items()}
    if "leaves" not in s:
        with torch.no_grad():
            return _own(s)
    out = _own(s)
    grads = torch.autograd.grad(list(out.values()), [s[n] for n in s["leaves"]], [s["d" + k] for k in out])
    return {**{k: v.detach() for k, v in out.items()}, **dict(zip(s["leaves"], grads))}


# ---------------------------------------------------------------------------------------------- exact values
def _exact_attention(s):
    """Query head by query head, sequence by sequence, from softmax(x)_j = exp(x_j - log sum exp x) and its derivative."""
    case = s["case"]
    d, group = case["d"], case["h"] // case["hk"]
    q, k, v = (s[t].detach().reshape(-1, s[t].shape[-2], d) for t in "qkv")
    train = "leaves" in s
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v))
    table = s["table"].detach().double() if "table" in s else None
    dtable = torch.zeros_like(table) if table is not None else None
    mask = s["mask"].reshape(-1) if "mask" in s else None
    m_most = max(lengths(case))
    buckets = None
    if table is not None:
        reach = (s["bucket_of"].numel() - 1) // 2
        far = torch.arange(-(m_most - 1), m_most, device="cuda")
        buckets = s["bucket_of"].long()[torch.minimum(torch.maximum(far, torch.tensor(-reach, device="cuda")), torch.tensor(reach, device="cuda")) + reach]
    # (sequences of one length together, a bounded number of scores at a time)
    starts = [0]
    for m in lengths(case):
        starts.append(starts[-1] + m)
    by_length = {}
    for i, m in enumerate(lengths(case)):
        by_length.setdefault(m, []).append(starts[i])
    for m, firsts in by_length.items():
        i = torch.arange(m, device="cuda")
        allowed = torch.ones(m, m, dtype=torch.bool, device="cuda") if not case["causal"] else i[:, None] >= i[None, :]
        most = max(1, (1 << 26) // (m * m))
        for at in range(0, len(firsts), most):
            rows = torch.tensor(firsts[at : at + most], device="cuda")[:, None] + i  # [n, m]
            ok = allowed[None]
            if mask is not None:
                there = mask[rows]
                ok = ok & there[:, :, None] & there[:, None, :]
            empty = ~ok.any(-1)
            if buckets is not None:
                bucket = buckets[(i[None, :] - i[:, None]) + m_most - 1]
            for head in range(case["h"]):
                qh, kh, vh = q[rows, head].double(), k[rows, head // group].double(), v[rows, head // group].double()
                x = torch.einsum("nid,njd->nij", qh, kh) / math.sqrt(d)
                if buckets is not None:
                    x += table[bucket, head]
                x.masked_fill_(~ok, -math.inf)
                norm = torch.logsumexp(x, -1, keepdim=True).masked_fill(empty[..., None], 0.0)
                prob = torch.exp_(x.sub_(norm))
                vz = vh if mask is None else vh.masked_fill(~there[..., None], 0.0)
                oh = torch.einsum("nij,njd->nid", prob, vz)
                o[rows, head] = oh
                if not train:
                    continue
                g = s["do"].reshape(-1, case["h"], d)[rows, head].double()
                if mask is not None:
                    g = g.masked_fill(~there[..., None], 0.0)
                dv[rows, head // group] += torch.einsum("nij,nid->njd", prob, g)
                dx = torch.einsum("nid,njd->nij", g, vz)
                dx -= (g * oh).sum(-1, keepdim=True)
                dx *= prob
                dq[rows, head] = torch.einsum("nij,njd->nid", dx, kh) / math.sqrt(d)
                dk[rows, head // group] += torch.einsum("nij,nid->njd", dx, qh) / math.sqrt(d)
                if buckets is not None:
                    dtable[:, head] += torch.bincount(bucket.reshape(-1), dx.sum(0).reshape(-1), minlength=table.shape[0])
    out = {"o": o}
    if train:
        out.update(q=dq, k=dk, v=dv)
        if table is not None:
            out["table"] = dtable
    return {name: t.view(s["q" if name == "o" else name].shape) for name, t in out.items()}


def _exact_position(s):
    b, n, _, c = s["z"].shape
    rows = s["table"].shape[0]
    reach = (s["bucket_of"].numel() - 1) // 2
    y = torch.empty(s["z"].shape, dtype=torch.float64, device="cuda")
    dtable = torch.zeros(rows, c, dtype=torch.float64, device="cuda")
    table = s["table"].detach().double()
    for sample in range(b):
        index, chain = s["index"][sample].cpu().numpy(), s["chain"][sample].cpu().numpy()
        far = numpy.clip(index[None, :] - index[:, None], -reach, reach)
        bucket = s["bucket_of"].cpu().numpy()[far + reach]
        bucket = torch.from_numpy(numpy.where(chain[None, :] == chain[:, None], bucket, rows - 1).astype(numpy.int64)).cuda()
        y[sample] = s["z"].detach()[sample].double() + torch.nn.functional.embedding(bucket, table)
        if "leaves" in s:
            dy, flat = s["dy"][sample].reshape(-1, c).double(), bucket.reshape(-1)
            for number in range(rows):
                dtable[number] += dy[flat == number].sum(0)
    if "leaves" not in s:
        return {"y": y}
    return {"y": y, "z": s["dy"].double(), "table": dtable}


def _exact_numbers(key, count):
    """The same numbers by unsigned 64-bit products on the host."""
    low = numpy.uint64(_MASK32)
    seed, second = (int(w) & (2**64 - 1) for w in key.tolist())
    with numpy.errstate(over="ignore"):
        block = numpy.arange(-(-count // 8), dtype=numpy.uint64)
        c = [block & low, block >> numpy.uint64(32), numpy.full_like(block, second & _MASK32), numpy.full_like(block, second >> 32)]
        for turn in range(10):
            k0 = numpy.uint64(((seed & _MASK32) + turn * 0x9E3779B9) & _MASK32)
            k1 = numpy.uint64(((seed >> 32) + turn * 0xBB67AE85) & _MASK32)
            first, other = c[0] * numpy.uint64(0xD2511F53), c[2] * numpy.uint64(0xCD9E8D57)
            c = [(other >> numpy.uint64(32)) ^ c[1] ^ k0, other & low, (first >> numpy.uint64(32)) ^ c[3] ^ k1, first & low]
    words = numpy.stack(c, 1).astype("<u4")
    return words.view("<u2").reshape(-1)[:count]


def _exact_dropout(s):
    case, x = s["case"], s["x"]
    shape = (x.shape[0], 1 if case["shared"] > 1 else x.shape[1], x.shape[2])
    dropped = round(case["p"] * 65536)
    keep = _exact_numbers(s["key"], shape[0] * shape[1] * shape[2]) >= dropped
    factor = torch.from_numpy(keep.reshape(shape)).cuda().double() * (1.0 / (1.0 - dropped / 65536))
    out = {"y": x.detach().double() + s["u"].detach().double() * factor}
    if "leaves" in s:
        out["x"] = s["dy"].double()
        out["u"] = s["dy"].double() * factor
    return out


def exact(case, seed):
    """What ``run`` returns, in float64 by the formulas of the operators and of their gradients."""
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "position": _exact_position, "dropout": _exact_dropout}[case["op"]](s)


def work(case):
    """One read of every input and one write of every output (a gradient that is another tensor as it came counts once); the
    products of the attention over the pairs of tokens that its lengths and its order leave (a mask does not change them), and of its
    gradients twice as many, none counted that is computed again."""
    train = case["mode"] == "train"
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["type"]]
    if case["op"] == "attention":
        pairs = sum(m * (m + 1) / 2 if case["causal"] else m * m for m in lengths(case))
        tokens = sum(lengths(case)) + case["spare"]
        q, kv = tokens * case["h"] * case["d"], 2 * tokens * case["hk"] * case["d"]
        table = {"none": 0, "near": 2 * REACH + 1, "log": 32}[case["bias"]] * case["h"]
        more = tokens if case["mask"] != "none" else 0
        return {"bytes": size * ((2 * q + kv + table) + (2 * q + kv + table if train else 0)) + more,
                "flops": (12.0 if train else 4.0) * pairs * case["h"] * case["d"]}
    if case["op"] == "position":
        pair = case["b"] * case["n"] ** 2 * case["c"]
        table = 4 * (2 * REACH + 2) * case["c"]
        return {"bytes": size * pair * (3 if train else 2) + table * (2 if train else 1) + 16 * case["b"] * case["n"],
                "flops": (2.0 if train else 1.0) * pair}
    elements = case["rows"] * case["width"]
    return {"bytes": size * elements * (5 if train else 3), "flops": (4.0 if train else 2.0) * elements}
