"""Attention over tokens in float64, head by head, with bounds that follow what the kernels keep: the gradient of the scores from an output
before it was rounded, and sums of the outer buckets without what the probabilities' rounding leaves in it. Tables may hold -inf."""

import torch

from tests.token_reference import half_step, smallest

F32 = 2.0**-24
LOST = 2.0**-126  # below that exp2 gives 0


def attention(q, k, v, do, lengths, mask=None, causal=False, scale=None, table=None, bucket_of=None, exact=False):
    """(results, bounds) for ``o`` and the gradients ``q``, ``k``, ``v``, ``table``, from [rows, heads, d] tensors.

    With u the half step of the type and f = 2^-24:

    - an exponential is off by the fp32 errors of its score, (d + 8) f of the sum of its terms' magnitudes and of 8 (exp2 and the
      difference with the row's maximum), relatively; the denominator by the mean of those over the row and (m / 8 + 16) f for its own
      sum (a thread adds a quarter of half a row). Together ``eps``.
    - o before it is rounded: sum p (u + eps) |v| for the rounded probabilities, m f sum p |v| for the products' sums.
    - delta = dO . o with o's rounding error kept to u of itself: D = sum p (u + eps) |dO . v| + |dO| (m f sum p |v| + (u^2 + 4 f) |o|)
      + d f |dO| |o|.
    - ds before it is rounded: |ds| (eps + 4 f) + p (t + D), t = (d + 8) f |dO| |v| for the product dO . v; after it u |ds| more.
    - a distance within the reach adds its ds up, in sums of at most 64 + m / 64 terms one after the other.
    - of the outer buckets a row's sum of all its ds, times their probabilities, is taken off. It is -D but for the ds' other errors, so of
      the row's error is left: those of the bucket, as many of the whole row as the bucket has probability, and D times what the row's
      probabilities are off from one together.
    - fp16: p is held times 2^15 (2^7 in the forward) and ds times a power of two that brings 2 max |dO| max |v| to 2^14 .. 2^15: what is
      subnormal then is off by 2^-25 of that unit.

    ``exact``: every probability is, relative to its row's greatest, a number of the type, which rounding it does not change. (That is the
    forward's operand, on which o and delta rest; the backward's, for dv, is the probability itself.)
    """
    type, rows, heads, d = q.dtype, q.shape[0], q.shape[1], q.shape[2]
    f16 = type == torch.float16
    group = heads // k.shape[1]
    scale = d**-0.5 if scale is None else scale
    u, tiny = half_step(type), smallest(type)
    u_p = 0.0 if exact else u
    dev = q.device
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)  # noqa: E731
    r = {n: zeros(t) for n, t in (("o", q), ("q", q), ("k", k), ("v", v))}
    e = {n: zeros(t) for n, t in r.items()}
    if table is not None:
        r["table"], e["table"] = zeros(table), zeros(table)
        reach = bucket_of.numel() // 2
    zero = torch.zeros((), dtype=torch.float64, device=dev)
    ends = [0]
    for m in lengths:
        ends.append(ends[-1] + m)
    there = torch.ones(rows, dtype=torch.bool, device=dev) if mask is None else mask
    there = there & (torch.arange(rows, device=dev) < ends[-1])
    clean = lambda t: torch.where(there[:, None, None], t.double(), zero)  # noqa: E731
    qd, kd, vd, gd = clean(q), clean(k), clean(v), clean(do)
    unit_p, unit_f = (2.0**-40, 2.0**-32) if f16 else (0.0, 0.0)
    for h in range(heads):
        kh = h // group
        own = slice(kh * group, (kh + 1) * group)
        unit_ds = 0.0
        if f16 and rows > 0:
            unit_ds = 2.0**-39 * 2 * float(gd[:, own].norm(dim=-1).max()) * float(vd[:, kh].norm(dim=-1).max())
        for at, m in zip(ends, lengths):
            if m == 0:
                continue
            at = slice(at, at + m)
            place = torch.arange(m, device=dev)
            here = there[at]
            counts = here[None, :] & here[:, None]
            if causal:
                counts = counts & (place[:, None] >= place[None, :])
            qs, ks, vs, g = qd[at, h], kd[at, kh], vd[at, kh], gd[at, h]
            s, size = scale * qs @ ks.t(), abs(scale) * qs.abs() @ ks.abs().t()
            if table is not None:
                distance = (place[None, :] - place[:, None]).clamp(-reach, reach)
                bucket = bucket_of.long()[distance + reach]
                bias = table.double()[bucket, h]
                counts = counts & ~torch.isneginf(bias)
                bias = torch.where(counts, bias, zero)
                s, size = s + bias, size + bias.abs()
            some = counts.any(1, keepdim=True)
            p = torch.softmax(torch.where(some, s.masked_fill(~counts, float("-inf")), zero), -1)
            p = torch.where(some, p, zero)
            loss = (d + 8) * F32 * (size + 8)
            eps = loss + (loss * p).sum(-1, keepdim=True) + (m / 8 + 16) * F32
            eps = torch.where(counts, eps, zero)
            held = lambda unit, step: torch.where(counts, p * (step + eps) + unit + LOST, zero)  # noqa: E731
            o, weight = p @ vs, p @ vs.abs()
            r["o"][at, h] = o
            e["o"][at, h] = (u * o.abs() + (held(unit_f, u_p) @ vs.abs() + m * F32 * weight) * (1 + u) + tiny)
            dp, size_dp = g @ vs.t(), g.abs() @ vs.abs().t()
            delta = (g * o).sum(-1, keepdim=True)
            off_delta = (held(unit_f, u_p) * dp.abs()).sum(-1, keepdim=True) + (g.abs() * (m * F32 * weight + (u * u + (d + 4) * F32) * o.abs() + tiny * u)).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            lone = ds.abs() * (eps + 4 * F32) + p * (d + 8) * F32 * size_dp + torch.where(counts, LOST * (size_dp + delta.abs() + 1), zero)  # all but D's
            exact_off = lone + p * off_delta * (1 + 2.0**-10)
            ds_off = exact_off * (1 + u) + u * ds.abs() + torch.where(counts, unit_ds + zero, zero)
            sums = (m + 16) * F32
            r["q"][at, h] = scale * ds @ ks
            e["q"][at, h] = abs(scale) * (ds_off + sums * ds.abs()) @ ks.abs()
            r["k"][at, kh] += scale * ds.t() @ qs
            e["k"][at, kh] += abs(scale) * (ds_off + group * sums * ds.abs()).t() @ qs.abs()
            r["v"][at, kh] += p.t() @ g
            e["v"][at, kh] += (held(unit_p, u) + group * sums * p).t() @ g.abs()
            if table is not None:
                deep = (64 + m / 64) * F32
                size_ds = ds.abs() + p * off_delta
                row = lone.sum(-1, keepdim=True) + deep * size_ds.sum(-1, keepdim=True) + off_delta * (p * eps).sum(-1, keepdim=True)
                outer = distance.abs() == reach
                off = torch.where(outer, lone + p * row * (1 + 2.0**-10), exact_off) + deep * size_ds
                r["table"][:, h].index_add_(0, bucket.reshape(-1), ds.reshape(-1))
                e["table"][:, h].index_add_(0, bucket.reshape(-1), off.reshape(-1))
    for n in ("q", "k", "v"):
        e[n] = u * r[n].abs() + e[n] * (1 + u) + tiny
    if table is not None:
        t = half_step(table.dtype)
        e["table"] += t * (r["table"].abs() + e["table"]) + smallest(table.dtype)
    return r, e


def imitated(q, k, v, do, m, table, bucket_of, causal=False, rest=True, outer=True):
    """The kernels' arithmetic for one sequence of ``m`` tokens, with its roundings: float64 otherwise. Returns the table's gradient.
    ``rest`` false: delta from the rounded output; ``outer`` false: nothing is taken off the outer buckets."""
    type, heads, d = q.dtype, q.shape[1], q.shape[2]
    group, reach = heads // k.shape[1], bucket_of.numel() // 2
    place = torch.arange(m)
    distance = (place[None, :] - place[:, None]).clamp(-reach, reach)
    bucket = bucket_of.long()[distance + reach]
    total = torch.zeros(table.shape, dtype=torch.float64)
    for h in range(heads):
        qs, ks, vs, g = q[:, h].double(), k[:, h // group].double(), v[:, h // group].double(), do[:, h].double()
        s = qs @ ks.t() * d**-0.5 + table.double()[bucket, h]
        if causal:
            s = s.masked_fill(place[:, None] < place[None, :], float("-inf"))
        ex = torch.exp(s - s.amax(1, keepdim=True))
        den = ex.sum(1, keepdim=True)
        o = (ex.to(type).double() @ vs) / den
        rounded = o.to(type).double()
        kept = rounded + (o - rounded).to(type).double() if rest else rounded
        p = ex / den
        ds = p * (g @ vs.t() - (g * kept).sum(-1, keepdim=True))
        if outer:
            ds = torch.where(distance.abs() == reach, ds - p * ds.sum(-1, keepdim=True), ds)
        total[:, h].index_add_(0, bucket.reshape(-1), ds.reshape(-1))
    return total


def flat(m, d, type, seed=0, device="cpu", heads=2):
    """Scores of zero, so that every probability is 1 / m, and values of which every output lies a quarter of a step above a number of the
    type: the rounding of the outputs shifts every row's delta the same way."""
    g = torch.Generator().manual_seed(seed)
    step = torch.finfo(type).eps
    q, k = torch.zeros(m, heads, d), torch.zeros(m, 1, d)
    v = 1 + step * (torch.rand(m, 1, d, generator=g) < 0.25)
    v[:, :, 0] = torch.randint(-3, 4, (m, 1), generator=g).float()  # what the true gradients come from
    do = torch.full((m, heads, d), 0.25)
    do[:, :, 0] = step * torch.randint(-2, 3, (m, heads), generator=g).float()
    from miniworld_b200 import blocks

    return [t.to(type).to(device) for t in (q, k, v, do)] + [torch.zeros(17, heads, device=device), blocks.relative_buckets(8, device=device)]


def coherent(m, d, type, seed=0, device="cpu", heads=2):
    """All but the nearest key score the same, with a probability that loses nearly a half step of the type to its rounding, and every
    dO . v is positive: what the rounding leaves in delta has one sign in all rows."""
    g = torch.Generator().manual_seed(seed)
    u = half_step(type)
    q, k = torch.zeros(m, heads, d), torch.zeros(m, 1, d)
    v, do = 1 + 0.5 * torch.rand(m, 1, d, generator=g), 0.1 + 0.05 * torch.rand(m, heads, d, generator=g)
    table = torch.full((17, heads), float(torch.log(torch.tensor(0.75 + 0.45 * u, dtype=torch.float64))))
    table[8] = 0.0
    from miniworld_b200 import blocks

    return [t.to(type).to(device) for t in (q, k, v, do)] + [table.to(device), blocks.relative_buckets(8, device=device)]
