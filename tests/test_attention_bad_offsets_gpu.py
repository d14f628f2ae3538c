"""Offsets that decrease, or run out of the arrays, leave results unspecified; nothing outside the arrays is read or
written. Inputs lie between rows of NaN, outputs between rows that have to stay."""
import ctypes

import pytest
import torch

import torchlib_xpu_b200
from torchlib_xpu_b200 import cabi

pytestmark = pytest.mark.gpu

torchlib_xpu_b200.load_torch_ops()
append = torch.ops.fbgemm.b200tbe_paged_cache_append
answer = torch.ops.fbgemm.b200tbe_paged_attention
pop = torch.ops.fbgemm.b200tbe_pop_device_status
PAD = 150   # more rows than a tile
CODES = {torch.float32: cabi.FP32, torch.float16: cabi.FP16, torch.bfloat16: cabi.BF16}

OFFSETS = [
    # rows, offsets
    (100, [0, 60, 20, 100]),
    (128, [128, 0, 128, 0, 128]),
    (300, [0, 300, 0, 300, 0, 300, 300]),
    (700, [-5, 690, 3, 5000, 129, 1, 700, -(1 << 31)]),
    (700, [650] + [(i * 389) % 701 for i in range(200)] + [10]),
    (5000, [(i * 2111) % 5001 for i in range(30)]),
]


def _between(rows, heads, D, dtype, outside, seed):
    """[rows, heads, D] inside a larger buffer whose other rows hold `outside`: (buffer, slice)."""
    wide = torch.full((rows + 2 * PAD, heads, D), outside, dtype=dtype, device="cuda")
    inner = wide[PAD:PAD + rows]
    if seed is not None:
        inner.copy_(torch.randn(inner.shape, generator=torch.Generator().manual_seed(seed)))
    return wide, inner


@pytest.mark.parametrize("rows,offsets", OFFSETS)
@pytest.mark.parametrize("dtype,heads,kv,D", [(torch.bfloat16, 2, 1, 64), (torch.float16, 3, 3, 128), (torch.bfloat16, 2, 2, 36),
                                              (torch.float32, 2, 1, 32)])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("wide_offsets", [True, False])
def test_jagged_attention(dtype, heads, kv, D, causal, rows, offsets, wide_offsets):
    nan, stays = float("nan"), 7.0
    (_, q), (_, g) = (_between(rows, heads, D, dtype, nan, s) for s in (1, 2))
    (_, k), (_, v) = (_between(rows, kv, D, dtype, nan, s) for s in (3, 4))
    outs = [_between(rows, h, D, dtype, stays, None) for h in (heads, heads, kv, kv)]
    lse = torch.full((heads * rows + 2 * PAD,), stays, device="cuda")
    lse[PAD:PAD + heads * rows] = 0
    dev = torch.tensor(offsets, dtype=torch.int64 if wide_offsets else torch.int32, device="cuda")
    k_dev = dev.flip(0).contiguous() if wide_offsets else dev
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = cabi.AttentionParams()
    p.q, p.k, p.v, p.out, p.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[0][1].data_ptr(), lse[PAD:].data_ptr()
    p.q_offsets, p.k_offsets, p.status = dev.data_ptr(), k_dev.data_ptr(), status.data_ptr()
    p.q_stride = p.out_stride = heads * D
    p.k_stride = p.v_stride = kv * D
    p.q_head_stride = p.k_head_stride = p.v_head_stride = p.out_head_stride = D
    p.total_q = p.total_k = rows
    p.batch, p.heads, p.kv_heads, p.head_dim, p.dtype = len(offsets) - 1, heads, kv, D, CODES[dtype]
    p.offset_bytes, p.causal, p.scale = dev.element_size(), causal, D ** -0.5
    stream = torch.cuda.current_stream().cuda_stream
    lib = cabi.lib()
    forward_bytes = lib.b200tbe_jagged_attention_scratch_bytes(rows, p.batch)
    backward_bytes = lib.b200tbe_jagged_attention_backward_scratch_bytes(rows, rows, p.batch, heads)
    guard = 1 << 12
    for with_scratch in (False, True):
        scratch = torch.full((max(forward_bytes, backward_bytes) + 2 * guard,), 7, dtype=torch.uint8, device="cuda")
        p.scratch, p.scratch_bytes = (scratch[guard:].data_ptr(), forward_bytes) if with_scratch else (None, 0)
        cabi.check(lib.b200tbe_jagged_attention(ctypes.byref(p), stream), "forward")
        assert (scratch[:guard] == 7).all() and (scratch[guard + forward_bytes:] == 7).all()
    assert not torch.isnan(outs[0][1]).any()
    # a row of two sequences has one log-sum, which may be -infinity where the other sequence's scores are finite: exp(s - lse)
    # is infinite then, and dS NaN, without a look outside. With log-sums that are finite NaN can only come from there.
    lse[PAD:PAD + heads * rows] = 5
    b = cabi.AttentionBackwardParams()
    b.forward = p
    b.grad_out, b.grad_q, b.grad_k, b.grad_v = g.data_ptr(), outs[1][1].data_ptr(), outs[2][1].data_ptr(), outs[3][1].data_ptr()
    b.grad_out_stride = b.grad_q_stride = heads * D
    b.grad_k_stride = b.grad_v_stride = kv * D
    b.grad_out_head_stride = b.grad_q_head_stride = b.grad_k_head_stride = b.grad_v_head_stride = D
    b.scratch, b.scratch_bytes = scratch[guard:].data_ptr(), backward_bytes
    cabi.check(lib.b200tbe_jagged_attention_backward(ctypes.byref(b), stream), "backward")
    assert (scratch[:guard] == 7).all() and (scratch[guard + backward_bytes:] == 7).all()
    assert int(status) == 0
    for wide, inner in outs:
        assert (wide[:PAD] == stays).all() and (wide[PAD + rows:] == stays).all()
        assert not torch.isnan(inner).any()
    assert (lse[:PAD] == stays).all() and (lse[PAD + heads * rows:] == stays).all()


@pytest.mark.parametrize("rows,offsets", OFFSETS)
def test_append(rows, offsets):
    """Rows whose place a decreasing pair of offsets leaves open go somewhere in their sequence's pages, or nowhere."""
    batch, page = len(offsets) - 1, 16
    pages = 4
    table = torch.arange(batch * pages, dtype=torch.int32).view(batch, pages) + 3
    total = batch * pages + 6
    caches = [torch.full((total, page, 2, 32), 7.0, device="cuda") for _ in range(2)]
    (_, k), (_, v) = (_between(rows, 2, 32, torch.float32, float("nan"), s) for s in (5, 6))
    lengths = torch.tensor([(i * 13) % 60 for i in range(batch)], device="cuda")
    pop(k)
    append(k, v, torch.tensor(offsets, device="cuda"), *caches, table.cuda(), lengths)
    assert pop(k) in (0, 1)   # rows before position 0 are reported
    for c in caches:
        assert not torch.isnan(c).any() and (c[:3] == 7).all() and (c[-3:] == 7).all()
    out = answer(k[:1].expand(batch, 2, 32), *caches, table.cuda(), lengths)
    assert torch.isfinite(out).all() and pop(k) == 0
