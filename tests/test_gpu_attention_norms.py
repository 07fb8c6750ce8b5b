"""The attention's errors as a whole: the norm of what o, dq, dk and dv are off by, against what independent roundings give.

One rounding to a type with the half step u is off by at most u of the value and by u / sqrt(3) in the mean square, and by as much of the
least number's half step below the normal range. With independent roundings of the probabilities p, of ds and of the results

    |off o|^2  = u^2/3 (|o|^2 + sum p^2 v^2)                    D_i^2 = u^2/3 sum_j p_ij^2 (dO_i . v_j)^2 (what dO . o is off by)
    |off dv|^2 = u^2/3 (|dv|^2 + sum p^2 dO^2)
    |off dq|^2 = u^2/3 (|dq|^2 + scale^2 sum ds^2 k^2) + scale^2 sum_i D_i^2 (sum_j p_ij k_j)^2
    |off dk|^2 = u^2/3 (|dk|^2 + scale^2 sum ds^2 q^2) + scale^2 sum_ij D_i^2 p_ij^2 q_i^2

The mean over a value's place between two powers of two is less by a quarter, so a tenth more than these leaves room for chance (there are
thousands of elements) and for fp32's own errors, 2^-24 of similar sums."""

import pytest
import torch

from miniworld_b200 import blocks
from tests.token_reference import half_step, smallest

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("m,h,hk,d", [(100, 4, 4, 64), (640, 4, 2, 32), (700, 2, 1, 128), (2048, 2, 2, 64)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_errors_are_those_of_independent_roundings(m, h, hk, d, type, causal):
    g = torch.Generator(device=DEV).manual_seed(m + d)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    q, k, v, do = (t.to(type) for t in (rand(m, h, d), rand(m, hk, d), rand(m, hk, d) + 0.5, rand(m, h, d)))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = blocks.token_attention(*(t.unsqueeze(0) for t in leaves), causal=causal)[0]
    got = dict(zip(("o", "q", "k", "v"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    c, least, scale2 = half_step(type) ** 2 / 3, smallest(type) ** 2 / 3, 1.0 / d
    group = h // hk
    qd, gd = q.double().transpose(0, 1), do.double().transpose(0, 1)
    kd, vd = (t.double().transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
    s = qd @ kd.transpose(1, 2) * d**-0.5
    if causal:
        s = s.masked_fill(torch.ones(m, m, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
    p = torch.softmax(s, -1)
    out, dp = p @ vd, gd @ vd.transpose(1, 2)
    ds = p * (dp - (gd * out).sum(-1, keepdim=True))
    d2 = c * (p * dp).square().sum(-1, keepdim=True)
    shared = lambda t: t.unflatten(0, (hk, group)).sum(1)  # noqa: E731
    want = {"o": out, "q": ds @ kd * d**-0.5, "k": shared(ds.transpose(1, 2) @ qd) * d**-0.5, "v": shared(p.transpose(1, 2) @ gd)}
    off = {"o": c * (p.square() @ vd.square()).sum(), "v": c * (p.square().transpose(1, 2) @ gd.square()).sum(),
           "q": scale2 * (c * (ds.square() @ kd.square()).sum() + (d2 * (p @ kd).square()).sum()),
           "k": scale2 * (c * (ds.square().transpose(1, 2) @ qd.square()).sum() + ((d2 * p.square()).transpose(1, 2) @ qd.square()).sum())}
    for n, w in want.items():
        w = w.transpose(0, 1)
        limit = 1.1 * float(off[n] + c * w.square().sum() + least * w.numel()) ** 0.5
        error = float((got[n].double() - w).norm())
        assert error <= limit, (n, error / float(w.norm()), limit / float(w.norm()))
        assert limit < 0.004 * float(w.norm()), n
    assert blocks.read_status(DEV) == 0
