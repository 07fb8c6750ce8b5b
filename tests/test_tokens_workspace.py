"""The attention's backward takes no room for a table's gradient that is not asked for."""

import ctypes

import pytest
import torch

from miniworld_b200 import _lib, blocks, build


def _call(p, table, rows=4000, sequences=2000, heads=4, kv_heads=2, d=32, reach=32):
    return _lib.AttentionCall(rows=rows, sequences=sequences, length=0, heads=heads, kv_heads=kv_heads, d=d, dtype=0, causal=0, scale=0.1, offsets=p, mask=None,
                              table=p if table else None, table_dtype=1, bucket_of=p if table else None, buckets=2 * reach + 1 if table else 0,
                              reach=reach if table else 0)


def test_sizes():
    build.build()
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 1023) // 1024 * 1024
    need = {}
    for table in (False, True):
        n = ctypes.c_size_t(0)
        assert lib.b200_token_attention_workspace_bytes(_call(p, table), ctypes.byref(n)) == 0
        need[table] = n.value
    assert need[True] - need[False] >= 4 * 65 * 4 * 2001
    t = _lib.AttentionTensor(p, 128, 32)

    def back(dtable, bytes, rows=4000):
        return lib.b200_token_attention_backward(_call(p, True, rows), t, t, t, p, p, p, t, p, p, p, dtable, p, bytes, None)

    assert back(p, need[True] - 1024) == back(p, need[False]) == back(None, need[False] - 1024) == -5
    if not torch.cuda.is_available():  # (no device: what is refused for its workspace is refused before)
        assert back(None, need[False]) not in (0, -5) and back(p, need[True]) not in (0, -5)


@pytest.mark.gpu
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
def test_the_other_gradients_are_the_same(type):
    dev = "cuda:0"
    q, k, v, do = (torch.randn(400, n, 64, device=dev).to(type) for n in (4, 2, 2, 4))
    offsets = torch.arange(0, 401, 4, device=dev)
    where, table = blocks.relative_buckets(32, device=dev), torch.randn(65, 4, device=dev)
    results = []
    for wanted in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        bias = table.clone().requires_grad_(wanted)
        o = blocks.token_attention(*leaves, offsets=offsets, table=bias, bucket_of=where)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        g = torch.autograd.grad(o, leaves + [bias] * wanted, do)
        results.append((g, torch.cuda.max_memory_allocated() - before))
    for a, b in zip(results[0][0], results[1][0]):
        assert torch.equal(a, b)
    assert results[0][1] - results[1][1] > 4 * 65 * 4 * 100
    assert blocks.read_status(dev) == 0
