"""Attention through the C ABI with every output and the workspace in the middle of a larger allocation: nothing around them is written,
whatever the offsets on the device are."""

import ctypes

import pytest
import torch

from miniworld_b200 import _lib, blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
AROUND, FILL = 1 << 16, 0xA5

MANY = torch.randint(-400, 700, (1200,), generator=torch.Generator().manual_seed(3)).tolist()
OFFSETS = [[0, 300], [0, 100, 100, 290], [0, 128, 256, 300], [0, 150, 1000], [0, -7, 300], [0, 280, 20, 300], [5, 250, 300], [300, 0], [0, 2**31 - 1],
           [0, -(2**31), 30], [2**31 - 1, -(2**31)], [0] * 70, [300] * 70, MANY, MANY[:33], MANY[:32], None]


class Guarded:
    """``count`` elements with filled bytes before and behind."""

    def __init__(self, count, type):
        self.bytes = count * torch.empty(0, dtype=type).element_size()
        raw = torch.full((self.bytes + 2 * AROUND + 1024,), FILL, dtype=torch.uint8, device=DEV)
        start = AROUND + -(raw.data_ptr() + AROUND) % 1024
        self.raw, self.start = raw, start
        self.ptr = raw.data_ptr() + start
        self.view = raw[start : start + self.bytes].view(type)

    def untouched(self):
        return bool((self.raw[: self.start] == FILL).all()) and bool((self.raw[self.start + self.bytes :] == FILL).all())


@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [0, 1])
def test_nothing_around_the_outputs_is_written(d, type, causal):
    lib, rows, h, hk, reach = _lib.load(), 300, 4, 2, 9
    stream = torch.cuda.current_stream().cuda_stream
    mask = (torch.arange(rows, device=DEV) % 5 != 2).to(torch.uint8)
    where, table = blocks.relative_buckets(reach, device=DEV), torch.zeros(2 * reach + 1, h, device=DEV)
    q, k, v, do = (torch.randn(rows, n, d, device=DEV).to(type) for n in (h, hk, hk, h))
    tensor = lambda t: _lib.AttentionTensor(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    tq, tk, tv, td = (tensor(t) for t in (q, k, v, do))
    for ends in OFFSETS:
        offsets = None if ends is None else torch.tensor(ends, dtype=torch.int32, device=DEV)
        c = _lib.AttentionCall(rows=rows, sequences=3 if ends is None else len(ends) - 1, length=100 if ends is None else 0, heads=h, kv_heads=hk, d=d,
                               dtype=0 if type == torch.bfloat16 else 2, causal=causal, scale=0.1, offsets=None if ends is None else offsets.data_ptr(),
                               mask=mask.data_ptr(), table=table.data_ptr(), table_dtype=1, bucket_of=where.data_ptr(), buckets=2 * reach + 1, reach=reach)
        need = ctypes.c_size_t(0)
        assert lib.b200_token_attention_workspace_bytes(c, ctypes.byref(need)) == 0
        out = {n: Guarded(rows * heads * d, type) for n, heads in (("o", h), ("rest", h), ("dq", h), ("dk", hk), ("dv", hk))}
        out.update(lse=Guarded(h * rows, torch.float32), dtable=Guarded((2 * reach + 1) * h, torch.float32), ws=Guarded(need.value, torch.uint8))
        p = {n: g.ptr for n, g in out.items()}
        assert lib.b200_token_attention_forward(c, tq, tk, tv, p["o"], p["rest"], p["lse"], stream) == 0
        assert lib.b200_token_attention_backward(c, tq, tk, tv, p["o"], p["rest"], p["lse"], td, p["dq"], p["dk"], p["dv"], p["dtable"], p["ws"], need.value, stream) == 0
        torch.cuda.synchronize()
        for n, g in out.items():
            assert g.untouched(), (n, ends)
        if ends is None or ends[:2] in ([0, 300], [0, 100], [0, 128]):  # offsets in order: every row is written
            for n in ("o", "dq", "dk", "dv"):
                assert bool(torch.isfinite(out[n].view.float()).all()) and not out[n].view.view(rows, -1)[2].any(), n
        assert blocks.read_status(DEV) == 0
