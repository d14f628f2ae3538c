"""The status word inside graph captures."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

# in a process of its own: the word is made once a process
PROGRAM = """
import torch, torchlib_xpu_b200
torchlib_xpu_b200.load_torch_ops()
ops = torch.ops.fbgemm
k = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
q = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
table, lengths = torch.tensor([[1, 9]], dtype=torch.int32, device="cuda"), torch.tensor([20], device="cuda")
made = %r
if made:
    assert ops.b200tbe_pop_device_status(q) == 0   # makes the word; no attention or cache call has run
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.b200tbe_paged_attention(q, k, k, table, lengths)
graph.replay()
torch.cuda.synchronize()
assert (out == 0).all()
assert ops.b200tbe_pop_device_status(q) == (1 if made else 0)
graph.replay()
assert ops.b200tbe_pop_device_status(q) == (1 if made else 0)
print("done")
"""


@pytest.mark.parametrize("made", [True, False], ids=["made by another operator", "not made"])
def test_a_first_call_under_capture(made):
    run = subprocess.run([sys.executable, "-c", PROGRAM % made], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stderr[-2000:]


INFERENCE = """
import torch, torchlib_xpu_b200
torchlib_xpu_b200.load_torch_ops()
ops = torch.ops.fbgemm
with torch.inference_mode():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    table, lengths = torch.tensor([[1, 9]], dtype=torch.int32, device="cuda"), torch.tensor([20], device="cuda")
    ops.b200tbe_paged_attention(q, k, k, table, lengths)   # makes the word
assert ops.b200tbe_pop_device_status(q) == 1
assert ops.b200tbe_pop_device_status(q) == 0
print("done")
"""


def test_a_word_made_in_inference_mode_is_cleared_outside():
    run = subprocess.run([sys.executable, "-c", INFERENCE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "done" in run.stdout, run.stderr[-2000:]
