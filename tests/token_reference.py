"""The token operators in float64, with bounds for what the kernels may be off by."""

import numpy
import torch


def half_step(type) -> float:
    """The most that one rounding to ``type`` is off, relative to the value."""
    return torch.finfo(type).eps / 2


def smallest(type) -> float:
    """The most that one rounding to ``type`` is off where the value is subnormal."""
    return torch.finfo(type).tiny * torch.finfo(type).eps / 2


def attention(q, k, v, lengths, mask=None, causal=False, scale=None, table=None, bucket_of=None, do=None):
    """(results, bounds): ``o`` and, with ``do``, ``q``, ``k``, ``v``, ``table`` gradients, in float64, from [rows, heads, d] tensors.

    Bounds, with u the half step of the type. The kernels round each probability once (relative u) before the product with v, and the
    result once: |do| <= u |o| + u P|v|. delta = dO . o sees the rounded o: e = |dO| . (that bound). ds is rounded once and carries p e, so
    dq is off by u |dq| + scale sum (u |ds| + p e) |k|, likewise dk; dv by u |dv| + u sum p |dO|; dtable by the sum of p e (and u |dtable|
    in 16 bits). What fp32 adds: scores are sums of d products and exponents of up to a few hundred, each to 2^-24 of their magnitude, so
    a probability to a relative (d + 8) 2^-24 (scale |q| . |k| + |bias| + 8); sums to (rows + d) 2^-24 of the sum of their magnitudes.
    Below 2^-126 fp32 has no normal numbers and exp2 gives 0: a probability may be off by that much, and so may a product of it.
    """
    type, rows, heads, d = q.dtype, q.shape[0], q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    scale = d**-0.5 if scale is None else scale
    u, tiny, f32, lost = half_step(type), smallest(type), 2.0**-24, 2.0**-126
    r = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("o", q), ("q", q), ("k", k), ("v", v))}
    e = {n: torch.zeros_like(t) for n, t in r.items()}
    if table is not None:
        r["table"], e["table"] = (torch.zeros(table.shape, dtype=torch.float64, device=q.device) for _ in range(2))
        reach = bucket_of.numel() // 2
    start = 0
    for m in lengths:
        at = slice(start, start + m)
        start += m
        if m == 0:
            continue
        place = torch.arange(m, device=q.device)
        counts = torch.ones(m, m, dtype=torch.bool, device=q.device)
        if causal:
            counts = counts.tril()
        here = torch.ones(m, dtype=torch.bool, device=q.device) if mask is None else mask[at]
        counts = counts & here[None, :] & here[:, None]
        clean = lambda t: torch.where(here[:, None, None], t[at].double(), torch.zeros((), dtype=torch.float64, device=q.device)).transpose(0, 1)  # noqa: E731
        qs, ks, vs = clean(q), clean(k).repeat_interleave(group, 0), clean(v).repeat_interleave(group, 0)
        s = scale * qs @ ks.transpose(1, 2)
        size = abs(scale) * qs.abs() @ ks.abs().transpose(1, 2)
        if table is not None:
            bucket = bucket_of.long()[(place[None, :] - place[:, None]).clamp(-reach, reach) + reach]
            bias = table.double()[bucket].permute(2, 0, 1)
            s, size = s + bias, size + bias.abs()
        s = s.masked_fill(~counts, float("-inf"))
        some = counts.any(1)
        p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], s, torch.zeros_like(s)), -1), torch.zeros_like(s))
        # what fp32 leaves of a probability: its own exponent's error and the greatest of its row (through the denominator)
        loss = (d + 8) * f32 * (size.masked_fill(~counts, 0.0) + 8)
        loss = loss + (loss * p).sum(-1, keepdim=True)
        o = p @ vs
        p_off = p * (u + loss + m * f32) + lost
        r["o"][at] = o.transpose(0, 1)
        o_off = u * o.abs() + p_off @ vs.abs() * (1 + u) + m * f32 * (p @ vs.abs()) + tiny
        e["o"][at] = o_off.transpose(0, 1)
        if do is None:
            continue
        g = clean(do)
        dp, delta = g @ vs.transpose(1, 2), (g * o).sum(-1, keepdim=True)
        dp_size = g.abs() @ vs.abs().transpose(1, 2)
        ds = p * (dp - delta)
        delta_off = (g.abs() * o_off).sum(-1, keepdim=True) + d * f32 * (g.abs() * o.abs()).sum(-1, keepdim=True)
        exact_off = p * (delta_off + d * f32 * dp_size) + ds.abs() * (loss + m * f32) + lost * (dp_size + delta.abs() + 1)  # before ds is rounded
        ds_off = exact_off * (1 + u) + u * ds.abs()
        sums = (m + 16) * f32

        def put(name, value, off):
            if name in ("k", "v"):
                value, off = value.unflatten(0, (-1, group)).sum(1), off.unflatten(0, (-1, group)).sum(1)
            r[name][at] = value.transpose(0, 1)
            e[name][at] = (u * value.abs() + off * (1 + u) + tiny).transpose(0, 1)

        put("q", scale * ds @ ks, abs(scale) * (ds_off + sums * ds.abs()) @ ks.abs())
        put("k", scale * ds.transpose(1, 2) @ qs, abs(scale) * (ds_off + sums * ds.abs()).transpose(1, 2) @ qs.abs())
        put("v", p.transpose(1, 2) @ g, (p_off + sums * p).transpose(1, 2) @ g.abs())
        if table is not None:
            one = torch.nn.functional.one_hot(bucket, table.shape[0]).double()
            r["table"] += torch.einsum("hij,ijb->bh", ds, one)
            e["table"] += torch.einsum("hij,ijb->bh", exact_off + (sums + 2.0**-20) * p * (dp_size + delta.abs()), one)
    if table is not None:
        t = half_step(table.dtype)
        e["table"] += t * (r["table"].abs() + e["table"]) + smallest(table.dtype)
    return r, e


def check(got, want, off, what=""):
    """``got`` within ``off`` of ``want`` everywhere."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    excess = (got.double() - want).abs() - off
    bad = ~(excess <= 0)  # (NaN counts)
    if bool(bad.any()):
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements, first {i}: {float(got[i])} for {float(want[i])}, bound {float(off[i])}; "
                             f"relative L2 error {float((got.double() - want).norm() / want.norm().clamp_min(1e-300)):.2e}")


def philox_halves(seed: int, second: int, count: int) -> numpy.ndarray:
    """16-bit numbers of Philox-4x32-10, in Python integers of any size (key ``seed``, counter (block, ``second``))."""
    out = []
    low = 0xFFFFFFFF
    for block in range((count + 7) // 8):
        c = [block & low, block >> 32, second & low, second >> 32 & low]
        k = [seed & low, seed >> 32 & low]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        for w in c:
            out += [w & 0xFFFF, w >> 16]
    return numpy.array(out[:count], dtype=numpy.int64)
