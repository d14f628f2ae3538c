"""The attention and cache entry points refuse what they cannot take before anything is launched: no GPU needed
(the pointers are never followed on the host)."""
import ctypes

import pytest
import torch

import torchlib_xpu_b200
from torchlib_xpu_b200 import cabi

torchlib_xpu_b200.load_torch_ops()
BAD_ARG, SCRATCH, UNSUPPORTED, TOO_LARGE = -1, -2, -4, -5
AT = 1 << 20


def _attention(**changes):
    p = cabi.AttentionParams()
    p.q = p.k = p.v = p.out = p.q_offsets = p.k_offsets = AT
    p.total_q = p.total_k = 10
    p.batch, p.heads, p.kv_heads, p.head_dim, p.dtype, p.offset_bytes, p.scale = 1, 4, 2, 64, cabi.BF16, 8, 1.0
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), BAD_ARG), (dict(k=None), BAD_ARG), (dict(v=None), BAD_ARG), (dict(out=None), BAD_ARG),
    (dict(q_offsets=None), BAD_ARG), (dict(k_offsets=None), BAD_ARG), (dict(heads=3), BAD_ARG), (dict(heads=0), BAD_ARG),
    (dict(kv_heads=0), BAD_ARG), (dict(batch=-1), BAD_ARG), (dict(total_q=-1), BAD_ARG), (dict(total_k=-1), BAD_ARG),
    (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=257), UNSUPPORTED), (dict(dtype=cabi.INT8), UNSUPPORTED),
    (dict(offset_bytes=2), UNSUPPORTED), (dict(total_q=1 << 31), TOO_LARGE), (dict(total_k=1 << 31), TOO_LARGE),
])
def test_attention_refuses(changes, status):
    lib = cabi.lib()
    p = _attention(**changes)
    assert lib.b200tbe_jagged_attention(ctypes.byref(p), None) == status
    b = cabi.AttentionBackwardParams()
    b.forward = p
    b.grad_out = b.grad_q = b.grad_k = b.grad_v = b.scratch = AT
    b.forward.lse, b.scratch_bytes = AT, 1 << 40
    assert lib.b200tbe_jagged_attention_backward(ctypes.byref(b), None) == status


def test_attention_backward_refuses():
    lib = cabi.lib()

    def status(lse=AT, scratch=AT, scratch_bytes=1 << 20, **changes):
        b = cabi.AttentionBackwardParams()
        b.forward = _attention(lse=lse)
        b.grad_out = b.grad_q = b.grad_k = b.grad_v = AT
        b.scratch, b.scratch_bytes = scratch, scratch_bytes
        for name, value in changes.items():
            setattr(b, name, value)
        return lib.b200tbe_jagged_attention_backward(ctypes.byref(b), None)

    assert lib.b200tbe_jagged_attention(None, None) == BAD_ARG
    assert lib.b200tbe_jagged_attention_backward(None, None) == BAD_ARG
    for name in ("grad_out", "grad_q", "grad_k", "grad_v"):
        assert status(**{name: None}) == BAD_ARG
    assert status(lse=None) == BAD_ARG
    assert status(scratch=None) == SCRATCH
    assert status(scratch=AT + 8) == SCRATCH
    need = lib.b200tbe_jagged_attention_backward_scratch_bytes(10, 10, 1, 4)
    assert need >= 10 * 4 * 4
    assert status(scratch_bytes=need - 1) == SCRATCH
    assert lib.b200tbe_jagged_attention_backward_scratch_bytes(10, 10, 1, 0) == 0


def test_forward_scratch():
    lib = cabi.lib()
    need = lib.b200tbe_jagged_attention_scratch_bytes(10, 1)
    assert need > 0 and lib.b200tbe_jagged_attention_scratch_bytes(-1, 1) == 0
    for at, n in ((AT + 8, need), (AT, need - 1)):
        p = _attention(scratch=at, scratch_bytes=n)
        assert lib.b200tbe_jagged_attention(ctypes.byref(p), None) == SCRATCH


def test_nothing_to_do():
    lib = cabi.lib()
    p = _attention(total_q=0, q=None, out=None)
    assert lib.b200tbe_jagged_attention(ctypes.byref(p), None) == 0


def _cache(**changes):
    c = cabi.PagedCache()
    c.k_cache = c.v_cache = c.page_table = c.lengths = AT
    c.num_pages, c.max_pages, c.page_size, c.batch, c.kv_heads, c.head_dim, c.dtype, c.length_bytes = 4, 2, 16, 2, 2, 64, cabi.FP16, 4
    for name, value in changes.items():
        setattr(c, name, value)
    return c


CACHE_REFUSALS = [
    (dict(k_cache=None), BAD_ARG), (dict(v_cache=None), BAD_ARG), (dict(page_table=None), BAD_ARG), (dict(lengths=None), BAD_ARG),
    (dict(page_size=0), BAD_ARG), (dict(batch=-1), BAD_ARG), (dict(kv_heads=0), BAD_ARG), (dict(max_pages=-1), BAD_ARG),
    (dict(num_pages=-1), BAD_ARG), (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=257), UNSUPPORTED),
    (dict(dtype=cabi.INT4), UNSUPPORTED), (dict(length_bytes=1), UNSUPPORTED),
]


@pytest.mark.parametrize("changes,status", CACHE_REFUSALS)
def test_cache_refuses(changes, status):
    lib = cabi.lib()
    c = _cache(**changes)
    assert lib.b200tbe_paged_cache_append(ctypes.byref(c), AT, AT, 128, 64, 128, 64, AT, 8, 5, None) == status
    assert lib.b200tbe_paged_attention(ctypes.byref(c), AT, AT, 256, 64, 256, 64, 4, 1.0, AT, 1 << 40, None) == status


def test_append_and_attention_refuse():
    lib = cabi.lib()
    c = _cache()
    append = lambda k=AT, v=AT, o=AT, ob=8, n=5: lib.b200tbe_paged_cache_append(  # noqa: E731
        ctypes.byref(c), k, v, 128, 64, 128, 64, o, ob, n, None)
    assert append(k=None) == BAD_ARG and append(v=None) == BAD_ARG and append(o=None) == BAD_ARG and append(n=-1) == BAD_ARG
    assert append(ob=2) == UNSUPPORTED
    assert append(k=None, n=0) == 0
    need = lib.b200tbe_paged_attention_scratch_bytes(64)
    answer = lambda q=AT, out=AT, heads=4, scratch=AT, n=need: lib.b200tbe_paged_attention(  # noqa: E731
        ctypes.byref(c), q, out, 256, 64, 256, 64, heads, 1.0, scratch, n, None)
    assert answer(q=None) == BAD_ARG and answer(out=None) == BAD_ARG and answer(heads=3) == BAD_ARG and answer(heads=0) == BAD_ARG
    assert answer(scratch=None) == SCRATCH and answer(n=need - 1) == SCRATCH and answer(scratch=AT + 4) == SCRATCH
    assert lib.b200tbe_paged_cache_append(None, AT, AT, 0, 0, 0, 0, AT, 8, 1, None) == BAD_ARG
    assert lib.b200tbe_paged_attention(None, AT, AT, 0, 0, 0, 0, 4, 1.0, AT, need, None) == BAD_ARG
    c = _cache(batch=0)
    assert answer(q=None) == 0
    assert lib.b200tbe_paged_attention_scratch_bytes(0) == 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 1, 8)
    o = torch.tensor([0, 4])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.fbgemm.b200tbe_jagged_attention(q, q, q, o)
    cache = torch.zeros(1, 4, 1, 8)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([4])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.fbgemm.b200tbe_paged_cache_append(q, q, o, cache, cache, table, lengths)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.fbgemm.b200tbe_paged_attention(q[:1], cache, cache, table, lengths)
