"""Dropout with a residual add: the mask bit for bit, one rounding, the same mask in the backward."""

import math

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import blocks
from tests.token_reference import check, half_step, philox_halves, smallest

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _key(seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-(2**63), 2**63 - 1, (2,), generator=g).to(DEV)


def _mask(key, p, shape, shared, call=0):
    shape = list(shape)
    if shared is not None:
        shape[shared] = 1
    seed, second = (int(v) % 2**64 for v in key.tolist())
    halves = philox_halves(seed, (second + call) % 2**64, math.prod(shape))
    return torch.from_numpy(halves >= round(p * 65536)).to(DEV).view(shape)


@pytest.mark.parametrize("shape,shared", [((1,), None), ((7,), None), ((8,), None), ((3, 5), None), ((40, 384), None), ((2, 33, 65), None), ((24, 20, 64), 1),
                                          ((2, 9, 31, 16), 1), ((2, 9, 31, 16), -2), ((5, 7, 3), 1), ((3, 70, 11), 1), ((6, 8), 0), ((6, 8), 1), ((300, 13), 0),
                                          ((3, 1, 24), 1), ((2, 100, 40, 2), 1)])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [True, False])
def test_values_mask_and_gradients(shape, shared, type, residual):
    g = torch.Generator(device=DEV).manual_seed(3)
    x, u, dy = (torch.randn(shape, generator=g, device=DEV).to(type) for _ in range(3))
    leaves = [u.requires_grad_(True)] + ([x.requires_grad_(True)] if residual else [])
    key, p = _key(len(shape)), 0.3
    y = blocks.block_dropout(x if residual else None, u, key, p=p, shared=shared, call=5)
    grads = torch.autograd.grad(y, leaves, dy)
    keep, scale = _mask(key, p, shape, shared, 5).expand(shape), 65536.0 / (65536 - round(p * 65536))
    want = torch.where(keep, u.detach().double() * scale, torch.zeros((), dtype=torch.float64, device=DEV)) + (x.detach().double() if residual else 0)
    size = u.detach().abs().double() * scale + x.detach().abs().double()
    check(y, want, half_step(type) * want.abs() + smallest(type) + 2.0**-23 * size, "y")
    base = x.detach() if residual else torch.zeros_like(u)
    assert torch.equal(y.detach()[~keep], base[~keep])
    du = torch.where(keep, dy.double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
    check(grads[0], du, half_step(type) * du.abs() + smallest(type) + 2.0**-23 * du.abs(), "u")
    if residual:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("p", [0.0, 1e-7, 1.0 / 65536, 0.5, 65535 / 65536, 1.0])
def test_shares(p):
    u = torch.randn(1000, 64, device=DEV)
    x = torch.randn(1000, 64, device=DEV)
    keep = _mask(_key(), p, u.shape, None)
    y = blocks.block_dropout(x, u, _key(), p=p)
    t = round(p * 65536)
    want = x.double() + torch.where(keep, u.double() * (65536 / (65536 - t) if t < 65536 else 0.0), torch.zeros((), dtype=torch.float64, device=DEV))
    check(y, want, 2.0**-23 * (x.abs() + u.abs() * (65536 / max(1, 65536 - t))).double(), "y")
    if p in (0.0, 1e-7):
        assert torch.equal(y, x + u)
    if p == 1.0:
        assert torch.equal(y, x)


def test_dropped_elements_hold_anything():
    x, u = torch.randn(64, 128, device=DEV).bfloat16(), torch.randn(64, 128, device=DEV).bfloat16()
    keep = _mask(_key(), 0.5, u.shape, None)
    u[~keep] = float("nan")
    y = blocks.block_dropout(x, u.requires_grad_(True), _key(), p=0.5)
    assert torch.isfinite(y).all() and torch.equal(y.detach()[~keep], x[~keep])
    dy = torch.ones_like(y)
    dy[~keep] = float("inf")
    (g,) = torch.autograd.grad(y, u, dy)
    assert torch.isfinite(g).all() and not g[~keep].any()


def test_keys_and_calls_are_different_masks():
    u = torch.ones(1 << 20, device=DEV)
    kept = [blocks.block_dropout(None, u, key, p=0.5, call=call) != 0 for key, call in ((_key(1), 0), (_key(2), 0), (_key(1), 1))]
    for i, a in enumerate(kept):
        # 2^20 fair draws: six standard deviations of their mean are 0.003; of two masks' agreement too
        assert abs(float(a.float().mean()) - 0.5) < 0.003
        for b in kept[i + 1 :]:
            assert abs(float((a == b).float().mean()) - 0.5) < 0.003
    assert torch.equal(kept[0], blocks.block_dropout(None, u, _key(1), p=0.5) != 0)


def test_layouts_types_and_alignment():
    x, u = torch.randn(40, 64, device=DEV).bfloat16(), torch.randn(64, 40, device=DEV)
    want = blocks.block_dropout(x, u.t().bfloat16().contiguous(), _key(), p=0.25)
    assert torch.equal(blocks.block_dropout(x, u.t(), _key(), p=0.25), want)  # converted
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    assert torch.equal(blocks.block_dropout(odd, u.t(), _key(), p=0.25), want)
    shared = blocks.block_dropout(x.view(5, 8, 64), u.t().reshape(5, 8, 64), _key(), p=0.25, shared=1)
    assert torch.equal(blocks.block_dropout(odd.view(5, 8, 64), u.t().reshape(5, 8, 64), _key(), p=0.25, shared=1), shared)
    for shape in ((0, 8), (4, 0), (3, 0, 8)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        y = blocks.block_dropout(e, e, _key(), p=0.5, shared=0)
        assert y.shape == torch.autograd.grad(y, e, torch.zeros_like(y))[0].shape == shape


def test_a_key_changed_before_the_backward_is_refused():
    u, key = torch.randn(64, device=DEV, requires_grad=True), _key()
    y = blocks.block_dropout(None, u, key, p=0.5)
    key += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_module():
    torch.manual_seed(0)
    m = mw.BlockDropout(0.25, shared=1)
    x, u = torch.randn(2, 30, 30, 32, device=DEV).bfloat16(), torch.randn(2, 30, 30, 32, device=DEV).bfloat16()
    assert torch.equal(m.eval()(x, u), x + u) and torch.equal(mw.BlockDropout(0.0)(x, u), x + u)
    m.train()
    a, b = m(x, u), m(x, u)
    dropped = (a == x).all(1, keepdim=True)
    assert not torch.equal(a, b) and abs(float(dropped.float().mean()) - 0.25) < 0.06  # 1920 draws: six standard deviations
    assert torch.equal((a == x) | dropped, dropped.expand_as(a) | (a == x)) and torch.equal(m(x, u, _key()), m(x, u, _key()))
    torch.manual_seed(7)
    first = m(x, u)
    torch.manual_seed(7)
    assert torch.equal(first, m(x, u))


def test_more_than_32_bits_of_elements():
    n = (1 << 31) + 40
    u = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = blocks.block_dropout(None, u, _key(), p=0.5)
    seed, second = (int(v) % 2**64 for v in _key().tolist())
    low = 0xFFFFFFFF
    for block in (0, (1 << 28) - 1, 1 << 28, n // 8 - 1):
        c, k = [block & low, block >> 32, second & low, second >> 32], [seed & low, seed >> 32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
            k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
        want = [2.0 if h >= 32768 else 0.0 for w in c for h in (w & 0xFFFF, w >> 16)]
        assert y[block * 8 : block * 8 + 8].tolist() == want, block
