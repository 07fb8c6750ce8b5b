"""Block operators without a GPU: the C ABI's symbols and refusals, the modules' constructors."""

import ctypes
import os
import re

import pytest
import torch

import miniworld_b200 as mw
from miniworld_b200 import _lib, blocks, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.fixture
def p():
    """An aligned address that no refused call reads."""
    buf = ctypes.create_string_buffer(4096)
    yield (ctypes.addressof(buf) + 1023) // 1024 * 1024


def test_header_symbols_are_exported_and_bound(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "b200_blocks.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(b200_\w+)\s*\(", text))
    assert names == set(_lib.BLOCKS_SIGNATURES)
    assert all(hasattr(lib, n) for n in names)


def _join_forward(lib, p, x=0, u=0, y=0, h=0, rows=4, d=64, gate_rows=1, dtype=0, post=1, pre=1, gate=None, stats=None):
    at = lambda v: p if v == 0 else v  # noqa: E731
    return lib.b200_block_join_forward(at(x), at(u), gate, None, None, None, None, None, None, at(y), at(h), stats, None, rows, d, gate_rows,
                                       dtype, post, pre, 1e-5, 1e-5, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), -2), (dict(d=0), -2), (dict(gate_rows=0), -2), (dict(rows=5, gate_rows=2), -2), (dict(rows=1 << 41), -2),
    (dict(d=4097), -3), (dict(dtype=3), -3), (dict(post=3), -3), (dict(pre=-1), -3),
    (dict(x=None), -1), (dict(y=None), -1), (dict(h=None), -1), (dict(u=None), -1), (dict(pre=0), -1),
    (dict(u=None, y=None, post=0, pre=0, h=None), -1),
])
def test_join_forward_refuses(lib, p, kw, code):
    assert _join_forward(lib, p, **kw) == code


def test_join_without_rows_is_done_at_once(lib):
    assert lib.b200_block_join_forward(*[None] * 13, 0, 64, 1, 0, 1, 1, 1e-5, 1e-5, None) == 0


def test_join_backward_refuses(lib, p):
    need = ctypes.c_size_t(0)
    assert lib.b200_block_join_workspace_bytes(10, 64, 1, None) == -1
    assert lib.b200_block_join_workspace_bytes(10, 5000, 1, ctypes.byref(need)) == -3
    assert lib.b200_block_join_workspace_bytes(10, 64, 3, ctypes.byref(need)) == -2
    assert lib.b200_block_join_workspace_bytes(10, 64, 1, ctypes.byref(need)) == 0
    plain = need.value
    assert lib.b200_block_join_workspace_bytes(10, 64, 10, ctypes.byref(need)) == 0 and need.value > plain >= 160 * 5 * 64 * 4

    def call(dy=p, dh=p, u=p, gate=None, post_stats=p, pre_stats=p, dgate=None, ws=p, n=1 << 40, rows=4, post=1, pre=1, du=p):
        return lib.b200_block_join_backward(dy, dh, p, u, gate, None, None, None, None, None, None, post_stats, pre_stats, p, du, dgate,
                                            *[None] * 5, ws, n, rows, 64, 1, 0, post, pre, None)

    assert call(ws=None) == -1 and call(post_stats=None) == -1 and call(pre_stats=None) == -1
    assert call(dgate=p) == -1  # a gradient of a gate that is not there
    assert call(pre=0, pre_stats=None) == -1  # ... of a norm that is not there
    assert call(u=None, post=0, post_stats=None) == -1  # dy or du without u
    assert call(ws=p + 16) == -4 and call(n=8) == -5


def test_feed_forward_refuses(lib, p):
    need = ctypes.c_size_t(0)
    sizes = lib.b200_ff_workspace_bytes
    assert sizes(100, 64, 256, 0, 0, None) == -1
    assert sizes(-1, 64, 256, 0, 0, ctypes.byref(need)) == -2 and sizes(1 << 31, 64, 256, 0, 0, ctypes.byref(need)) == -2
    assert sizes(10, 0, 256, 0, 0, ctypes.byref(need)) == -2 and sizes(10, 60, 256, 0, 0, ctypes.byref(need)) == -3
    assert sizes(10, 64, 100, 0, 0, ctypes.byref(need)) == -3 and sizes(10, 64, 256, 3, 0, ctypes.byref(need)) == -3
    assert sizes(100, 64, 256, 0, 0, ctypes.byref(need)) == 0 and need.value >= 100 * 256 * 2
    forward = need.value
    assert sizes(0, 64, 256, 0, 0, ctypes.byref(need)) == 0 and sizes(0, 64, 256, 0, 1, ctypes.byref(need)) == 0  # no rows
    assert sizes(100, 64, 256, 1, 0, ctypes.byref(need)) == 0 and need.value >= forward + 3 * 64 * 256 * 2
    assert sizes(100, 64, 256, 0, 1, ctypes.byref(need)) == 0 and need.value >= 3 * 100 * 256 * 2

    def call(x=p, w=p, y=p, kept=None, ws=p, n=1 << 40, rows=10, d=64, hidden=256, dtype=0, weights=0, act=0):
        return lib.b200_ff_forward(x, w, p, p, y, kept, ws, n, rows, d, hidden, dtype, weights, act, None)

    assert call(dtype=1) == -3 and call(dtype=2, weights=0) == -3 and call(act=2) == -3 and call(d=12) == -3 and call(rows=-1) == -2
    assert call(x=None) == -1 and call(w=None) == -1 and call(y=None) == -1 and call(ws=None) == -1
    assert call(x=p + 8) == -4 and call(w=p + 2) == -4 and call(ws=p + 16) == -4 and call(kept=p + 16) == -4
    assert call(rows=0, x=None) == 0
    assert lib.b200_ff_kept_bytes(4096, 1024, 4096, ctypes.byref(need)) == 0 and need.value == 3 * 4096 * 4096 * 2
    assert lib.b200_ff_kept_bytes(4096, 384, 1536, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.b200_ff_kept_bytes(64, 1024, 4096, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.b200_ff_kept_bytes(64, 1020, 4096, ctypes.byref(need)) == -3 and lib.b200_ff_kept_bytes(64, 1024, 4096, None) == -1

    def back(dy=p, dx=p, dw=p, ws=p, d=64, dtype=0, act=0):
        return lib.b200_ff_backward(dy, p, p, p, p, None, dx, dw, p, p, ws, 1 << 40, 10, d, 256, dtype, 0, act, None)

    assert back(dy=None) == -1 and back(ws=None) == -1 and back(dx=p + 8) == -4 and back(dw=p + 4) == -4 and back(d=4) == -3
    assert back(dtype=1) == -3 and back(act=-1) == -3


def test_no_cpu_implementation():
    x = torch.zeros(2, 64, dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: blocks.block_norm(x), lambda: blocks.block_join(x, x), lambda: mw.GatedFeedForward(64)(x),
                 lambda: mw.SandwichTransition(64)(x), lambda: mw.BlockNorm(64)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_constructors_refuse():
    for make in (lambda: mw.GatedFeedForward(60), lambda: mw.GatedFeedForward(64, hidden=100), lambda: mw.GatedFeedForward(0)):
        with pytest.raises(NotImplementedError):
            make()
    for make in (lambda: mw.GatedFeedForward(64, activation="relu"), lambda: mw.GatedFeedForward(64, implementation="triton"),
                 lambda: mw.BlockNorm(64, kind="batch"), lambda: mw.BlockJoin(64, kind="batch")):
        with pytest.raises(ValueError):
            make()
    with pytest.raises(ValueError):
        blocks.block_norm(torch.zeros(1, 8), kind="none")
    with pytest.raises(ValueError):
        blocks.gated_feed_forward(*[torch.zeros(8, 8)] * 4, activation="tanh")


def test_parameters_of_the_modules():
    m = mw.SandwichTransition(64, n=2, scale=0.1).to(torch.bfloat16)
    kinds = {k: (tuple(v.shape), v.dtype) for k, v in m.state_dict().items()}
    assert kinds == {
        "ln_in.weight": ((64,), torch.float32), "ln_in.bias": ((64,), torch.float32),
        "feed_forward.expand_a.weight": ((128, 64), torch.bfloat16), "feed_forward.expand_b.weight": ((128, 64), torch.bfloat16),
        "feed_forward.squeeze.weight": ((64, 128), torch.bfloat16), "join.norm_out.weight": ((64,), torch.float32),
        "join.norm_out.bias": ((64,), torch.float32), "join.scale": ((64,), torch.float32),
    }
    assert mw.BlockNorm(64, "rms").bias is None and mw.BlockNorm(64, "rms", bias=True).bias is not None
    assert mw.BlockJoin(64, None).norm_out is None and mw.BlockJoin(64).scale is None


@pytest.mark.parametrize("names,post", [(("d_scale",), 0), (("d_post_w",), 0), (("d_post_b",), 0), (("d_post_w",), None), (("d_post_b",), None)])
def test_join_backward_refuses_sums_of_what_is_not_there(lib, p, names, post):
    """Gradients of the scale and of the norm after the block without the block's output (``post`` 0: a plain norm), or without that norm."""
    u = None if post == 0 else p
    d = [p if n in names else None for n in ("d_scale", "d_post_w", "d_post_b", "d_pre_w", "d_pre_b")]
    code = lib.b200_block_join_backward(None if u is None else p, p, p, u, None, None, None, None, None, None, None, None, p, p, u, None, *d, p, 1 << 40,
                                        4, 64, 1, 0, 0, 1, None)
    assert code == -1


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16, torch.float64])
def test_conversions_leave_the_fp32_parameters_and_their_gradients(type):
    """``.to(type)`` between steps: values and accumulated gradients of norms and scale stay as they are, bit for bit."""
    m = mw.SandwichTransition(64, n=2, scale=0.1)
    for p in m.parameters():
        torch.nn.init.normal_(p)
        p.grad = torch.randn_like(p)
    want = {k: (p.detach().clone(), p.grad.clone()) for k, p in m.named_parameters()}
    m.to(type)
    for k, p in m.named_parameters():
        kept = not k.startswith("feed_forward")
        assert p.dtype == p.grad.dtype == (torch.float32 if kept else type), k
        assert not kept or (torch.equal(p, want[k][0]) and torch.equal(p.grad, want[k][1])), k
    moved = m.to("meta")
    assert moved.join.scale.is_meta and moved.join.scale.dtype == torch.float32
    assert moved.to_empty(device="cpu").join.scale.device.type == "cpu"
