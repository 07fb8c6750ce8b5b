"""Token operators without a GPU: the C ABI's symbols and refusals, the modules' constructors, buckets."""

import ctypes
import math
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
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "b200_tokens.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(b200_\w+)\s*\(", text))
    assert names == set(_lib.TOKENS_SIGNATURES)
    assert all(hasattr(lib, n) for n in names)


def _call(p, **kw):
    c = dict(rows=20, sequences=2, length=10, heads=4, kv_heads=2, d=32, dtype=0, causal=0, scale=0.1, offsets=None, mask=None, table=None,
             table_dtype=0, bucket_of=None, buckets=0, reach=0)
    c.update({k: p if v == "p" else v for k, v in kw.items()})
    return _lib.AttentionCall(**c)


REFUSED_CALLS = [
    (dict(rows=-1), -2), (dict(rows=1 << 31), -2), (dict(heads=3), -2), (dict(heads=0), -2), (dict(kv_heads=0), -2), (dict(rows=21), -2),
    (dict(sequences=-2, length=-10), -2), (dict(offsets="p", sequences=0), -2), (dict(d=4), -3), (dict(d=36), -3), (dict(d=136), -3), (dict(dtype=1), -3),
    (dict(dtype=3), -3), (dict(scale=math.inf), -3), (dict(scale=math.nan), -3), (dict(heads=40000, kv_heads=40000), -3),
    (dict(table="p", buckets=5, reach=2), -1), (dict(table="p", bucket_of="p", buckets=0), -2), (dict(table="p", bucket_of="p", buckets=5, reach=-1), -2),
    (dict(table="p", bucket_of="p", buckets=513, reach=2), -3), (dict(table="p", bucket_of="p", buckets=5, reach=257), -3),
    (dict(table="p", bucket_of="p", buckets=5, reach=2, table_dtype=2), -3),
]


@pytest.mark.parametrize("kw,code", REFUSED_CALLS)
def test_attention_refuses_calls(lib, p, kw, code):
    c, t = _call(p, **kw), _lib.AttentionTensor(p, 128, 32)
    need = ctypes.c_size_t(0)
    assert lib.b200_token_attention_forward(c, t, t, t, p, None, None, None) == code
    assert lib.b200_token_attention_workspace_bytes(c, ctypes.byref(need)) == code
    assert lib.b200_token_attention_backward(c, t, t, t, p, p, p, t, p, p, p, None, p, 1 << 40, None) == code


def test_attention_refuses_tensors(lib, p):
    c, good = _call(p), _lib.AttentionTensor(p, 128, 32)
    bad = [(_lib.AttentionTensor(None, 128, 32), -1), (_lib.AttentionTensor(p + 8, 128, 32), -4), (_lib.AttentionTensor(p, 132, 32), -4),
           (_lib.AttentionTensor(p, 128, 12), -4), (_lib.AttentionTensor(p, -128, 32), -2), (_lib.AttentionTensor(p, 128, -32), -2), (None, -1)]
    for t, code in bad:
        for at in range(4):
            four = [t if i == at else good for i in range(4)]
            if at < 3:
                assert lib.b200_token_attention_forward(c, *four[:3], p, None, None, None) == code
            assert lib.b200_token_attention_backward(c, *four[:3], p, p, p, four[3], p, p, p, None, p, 1 << 40, None) == code
    assert lib.b200_token_attention_forward(None, good, good, good, p, None, None, None) == -1
    assert lib.b200_token_attention_forward(c, good, good, good, None, None, None, None) == -1
    assert lib.b200_token_attention_forward(c, good, good, good, p, p, None, None) == -1  # both are kept, or none
    assert lib.b200_token_attention_forward(c, good, good, good, p, p + 8, p, None) == -4
    assert lib.b200_token_attention_forward(c, good, good, good, p + 2, None, None, None) == -4
    assert lib.b200_token_attention_forward(_call(p, rows=0, sequences=0), None, None, None, None, None, None, None) == 0

    def back(o=p, rest=p, lse=p, dq=p, dk=p, dv=p, dtable=None, ws=p, n=1 << 40, call=c):
        return lib.b200_token_attention_backward(call, good, good, good, o, rest, lse, good, dq, dk, dv, dtable, ws, n, None)

    assert back(o=None) == back(rest=None) == back(lse=None) == back(dq=None) == back(dk=None) == back(dv=None) == back(ws=None) == -1
    assert back(dtable=p) == -1  # the gradient of a table that is not there
    assert back(o=p + 8) == back(rest=p + 2) == back(dq=p + 8) == back(dk=p + 4) == back(dv=p + 2) == back(ws=p + 16) == -4
    assert back(n=8) == -5
    need = ctypes.c_size_t(0)
    assert lib.b200_token_attention_workspace_bytes(c, None) == -1
    assert lib.b200_token_attention_workspace_bytes(c, ctypes.byref(need)) == 0 and need.value >= 20 * 4 * 4
    plain = need.value
    assert lib.b200_token_attention_workspace_bytes(_call(p, table="p", bucket_of="p", buckets=65, reach=32), ctypes.byref(need)) == 0 and need.value > plain


def test_position_refuses(lib, p):
    def forward(z=p, table=p, index=p, where=p, y=p, b=2, n=10, c=64, buckets=65, reach=32, dtype=0):
        return lib.b200_relative_position_forward(z, table, index, None, where, y, b, n, c, buckets, reach, 0, dtype, None)

    def back(dy=p, index=p, where=p, dt=p, ws=p, n_ws=1 << 40, b=2, n=10, c=64, buckets=65, reach=32, dtype=0):
        return lib.b200_relative_position_backward(dy, index, None, where, dt, ws, n_ws, b, n, c, buckets, reach, 0, dtype, None)

    for f in (forward, back):
        assert f(b=-1) == f(n=-1) == f(c=0) == f(buckets=0) == f(reach=-1) == -2
        assert f(b=1 << 30, n=1 << 30) == f(n=1 << 20, c=4000) == -2
        assert f(buckets=513) == f(reach=257) == f(c=4097) == f(dtype=3) == f(dtype=-1) == -3
        assert f(index=None) == f(where=None) == -1
    assert forward(z=None) == forward(table=None) == forward(y=None) == -1
    assert back(dy=None) == back(dt=None) == back(ws=None) == -1 and back(ws=p + 16) == -4
    assert forward(b=0, z=None) == 0
    need = ctypes.c_size_t(0)
    assert lib.b200_relative_position_workspace_bytes(2, 10, 64, 65, None) == -1
    assert lib.b200_relative_position_workspace_bytes(2, 10, 64, 600, ctypes.byref(need)) == -3
    assert lib.b200_relative_position_workspace_bytes(2, 100, 64, 65, ctypes.byref(need)) == 0 and need.value >= 65 * 64 * 4


def test_dropout_refuses(lib, p):
    def f(x=p, u=p, key=p, y=p, outer=2, shared=3, inner=8, threshold=100, dtype=0):
        return lib.b200_block_dropout(x, u, key, 0, y, outer, shared, inner, threshold, dtype, None)

    assert f(outer=-1) == f(shared=-1) == f(inner=-1) == f(inner=1 << 41) == f(outer=1 << 30, inner=1 << 30) == -2
    assert f(outer=1 << 62, inner=0) == f(shared=1 << 62, inner=0) == -2
    assert f(threshold=-1) == f(threshold=65537) == f(dtype=3) == -3
    assert f(u=None) == f(key=None) == f(y=None) == -1
    assert f(outer=0, u=None) == f(inner=0, u=None) == f(shared=0, u=None) == 0
    code = ctypes.c_int(0)
    assert lib.b200_tokens_read_status(None, None) == -1 and code.value == 0


def test_no_cpu_implementation():
    q, key = torch.zeros(2, 5, 4, 16, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    z, table, where = torch.zeros(1, 4, 4, 8), torch.zeros(9, 8), blocks.relative_buckets(4)
    for call in (lambda: blocks.token_attention(q, q, q), lambda: blocks.relative_position(z, table, torch.arange(4), bucket_of=where),
                 lambda: blocks.block_dropout(None, q, key, p=0.5), lambda: blocks.block_dropout(q, q, key, p=0.5), lambda: mw.TokenAttention(4)(q, q, q),
                 lambda: mw.RelativePosition(8)(z, torch.arange(4)), lambda: mw.BlockDropout(0.5)(q, q, key)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_constructors_refuse():
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            mw.BlockDropout(p)
    for args in ((-1,), (257,), (16, 0), (16, 16), (256, 129)):
        with pytest.raises(ValueError):
            blocks.relative_buckets(*args)


def test_buckets():
    assert blocks.relative_buckets(3).tolist() == [0, 1, 2, 3, 4, 5, 6] and blocks.relative_buckets(0).tolist() == [0]
    where = blocks.relative_buckets(128, 8).tolist()
    middle = 128
    assert where[middle - 7 : middle + 8] == [7, 6, 5, 4, 3, 2, 1, 0, 17, 18, 19, 20, 21, 22, 23]
    assert set(where) == set(range(32)) - {16} and where[0] == 15 and where[-1] == 31
    for d in range(1, 129):
        assert where[middle + d] == where[middle - d] + 16
        assert where[middle - d] >= where[middle - d + 1]


def test_parameters_of_the_modules():
    m = torch.nn.ModuleDict({"a": mw.TokenAttention(8), "b": mw.TokenAttention(8, reach=None), "c": mw.RelativePosition(64, reach=16), "d": mw.BlockDropout(0.1)})
    m = m.to(torch.bfloat16)
    assert {k: (tuple(v.shape), v.dtype) for k, v in m.state_dict().items()} == {"a.table": ((65, 8), torch.float32), "c.table": ((34, 64), torch.float32)}
    assert m["a"].bucket_of.dtype == m["c"].bucket_of.dtype == torch.int32 and m["b"].bucket_of is None
    assert m.to("meta")["a"].bucket_of.is_meta


@pytest.mark.parametrize("u", [torch.float32, torch.float16, torch.bfloat16])
def test_dropout_that_drops_nothing_keeps_the_type_of_training(u):
    x, u = torch.randn(3, 4).bfloat16(), torch.randn(3, 4).to(u)
    for m in (mw.BlockDropout(0.3).eval(), mw.BlockDropout(0.0)):
        y = m(x, u)
        assert y.dtype == x.dtype and torch.equal(y, x + u.bfloat16()) and torch.equal(m(None, u), u)


def test_tables_that_no_kernel_takes_are_refused_at_once():
    assert mw.TokenAttention(2, reach=255).table.shape == (511, 2) and mw.RelativePosition(8, reach=255).table.shape == (512, 8)
    assert mw.TokenAttention(2, reach=256, exact=128).table.shape == (512, 2)
    for build in (lambda: mw.TokenAttention(2, reach=256), lambda: mw.RelativePosition(8, reach=256), lambda: mw.RelativePosition(8, reach=256, exact=128)):
        with pytest.raises(ValueError, match="512 buckets"):
            build()
