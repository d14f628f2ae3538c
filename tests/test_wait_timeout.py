"""What becomes of a wait inside a kernel that nothing ends: it gives up, is reported, and the GPU goes on."""
import ctypes
import os
import subprocess

import pytest
import torch

import torchlib_xpu_b200
from tests.test_attention_gpu import CASES, CROSS
from torchlib_xpu_b200 import _build

WAIT_TIMEOUT = 8


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("waits") / "wait_timeout.so")
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "wait_timeout.cu")
    subprocess.run([_build._nvcc(), *_build.NVCC_FLAGS, "-shared", source, "-o", path, "-cudart", "static"], check=True)
    return ctypes.CDLL(path)


def test_it_builds(waits):
    assert waits.wait_out


@pytest.mark.gpu
def test_a_wait_that_nothing_ends(waits):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def run(blocks, complete):
        waited = torch.full((blocks, 128), -1, dtype=torch.int32, device="cuda")
        events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        events[0].record()
        assert waits.wait_out(blocks, complete, ctypes.c_void_p(status.data_ptr()), ctypes.c_void_p(waited.data_ptr()), stream) == 0
        events[1].record()
        torch.cuda.synchronize()
        bits = int(status.item())
        status.zero_()
        return waited.cpu(), bits, events[0].elapsed_time(events[1])

    run(1, 1)
    waited, bits, ms = run(4, 1)
    assert (waited == 1).all() and bits == 0
    waited, bits, ms = run(3, 0)
    assert (waited == 0).all() and bits == WAIT_TIMEOUT
    assert 500 < ms < 10000   # 2^32 cycles at 1 to 2 GHz, and the millisecond in which copies would land
    # every SM's tensor memory can be had again, by this kernel and by the attention's
    waited, bits, ms = run(4 * 148, 1)
    assert (waited == 1).all() and bits == 0
    torchlib_xpu_b200.load_torch_ops()
    q = torch.randn(300, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    out = torch.ops.fbgemm.b200tbe_jagged_attention(q, q, q, torch.tensor([0, 300], device="cuda"))
    want = torch.softmax(torch.einsum("ihd,jhd->hij", q.double(), q.double()) / 8, -1)
    want = torch.einsum("hij,jhd->ihd", want, q.double())
    # the weights and the result are rounded to bf16 (by 2^-8 each of at most max|v| < 8), all else is far smaller
    assert (out.double() - want).abs().max() < 2 * 2.0 ** -8 * 8
    assert torch.ops.fbgemm.b200tbe_pop_device_status(q) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,q_lengths,k_lengths,heads,kv,D,causal",
                         [(c[0], c[1], c[1], *c[2:]) for c in CASES] + [c[:7] for c in CROSS])
def test_no_wait_of_the_attention_gives_up(dtype, q_lengths, k_lengths, heads, kv, D, causal):
    torchlib_xpu_b200.load_torch_ops()
    offsets = [torch.tensor([0] + n, device="cuda").cumsum(0) for n in (q_lengths, k_lengths)]
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(n, h, D, generator=gen, device="cuda").to(dtype).requires_grad_()
               for n, h in ((sum(q_lengths), heads), (sum(k_lengths), kv), (sum(k_lengths), kv)))
    torch.ops.fbgemm.b200tbe_pop_device_status(q)
    out = torch.ops.fbgemm.b200tbe_jagged_attention(q, k, v, *offsets, causal)
    torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert torch.ops.fbgemm.b200tbe_pop_device_status(q) == 0
