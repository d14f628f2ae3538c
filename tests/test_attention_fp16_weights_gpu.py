"""fp16 weights far below a row's largest: many of them together may be what the result is made of, and fp16 itself holds
what is under 2^-14 with ever fewer bits. The kernels therefore lift the weights by a power of two before they round them: by
2^6 over whole sequences (whose maximum in use may lag by 2^8) and over a cache, by 2^14 where the maximum is the row's own and
in the backward pass. The reference allows 2^-25 for each weight; here it is 2^-25 over the lift."""
import pytest
import torch

import torchlib_xpu_b200
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

FP16 = torch.float16
torchlib_xpu_b200.load_torch_ops()
attention = torch.ops.fbgemm.b200tbe_jagged_attention
answer = torch.ops.fbgemm.b200tbe_paged_attention
T = ref.tiny(FP16)


def _keys(n, every):
    """Keys whose score with a query [4, 0, ..] is -13.46875, but for each `every`-th one's, which is 0: a weight of exp(-13.46875),
    23.73 steps of 2^-24, would be rounded to 24 of them, off by 1.1 %. Values 64, and 0 where the score is 0."""
    k, v = torch.zeros(n, 1, 64, dtype=FP16), torch.full((n, 1, 64), 64.0, dtype=FP16)
    k[..., 0] = -13.46875 / 4
    k[::every] = 0
    v[::every] = 0
    return k, v


def _queries(n, heads=1):
    q = torch.zeros(n, heads, 64, dtype=FP16)
    q[..., 0] = 4
    return q


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("rows,keys,lift", [(100, 120, 14), (100, 2000, 6), (300, 128, 6), (700, 2000, 6)])
def test_sequences(rows, keys, lift, heads):
    q, (k, v) = _queries(rows, heads), _keys(keys, 5000)
    parts = [t.cuda().requires_grad_() for t in (q, k, v)]
    offsets = [torch.tensor([0, n], device="cuda") for n in (rows, keys)]
    g = torch.full((rows, heads, 64), 64.0, dtype=FP16, device="cuda")
    out = attention(*parts, *offsets, False, 1.0)
    dv, = torch.autograd.grad(out, parts[2], g)
    want = ref.one_sequence(q, k, v, False, 1.0, g)
    per_weight = T * float(v.double().sum(0).max())
    ref.assert_within(out, want["o"], want["o_off"] - per_weight * (1 - 2.0 ** -lift), "out")
    per_weight = T * float(g.double().sum((0, 1)).max())
    # the key with the score 0 has nearly all of every query's weight: 64 for each, 89 600 for 1400, which fp16 cannot hold
    fits = want["dv"][:, 0, 0] < 65504
    assert fits[1:].all() and (dv[0] == float("inf")).all().item() == (not fits[0])
    ref.assert_within(dv[fits.cuda()], want["dv"][fits], (want["dv_off"] - per_weight * (1 - 2.0 ** -14))[fits], "dv")


def test_gradient_of_values_over_many_keys():
    """Scores of 0 over 307 700 keys: every weight is 1 / 307700 = 54.52 steps of 2^-24. All sums on the way to it are
    exact, its logarithm and exponential are off by a few units of fp32 (64 allowed)."""
    keys, rows = 307700, 8
    q = torch.zeros(rows, 1, 64, dtype=FP16, device="cuda")
    k, v = (torch.zeros(keys, 1, 64, dtype=FP16, device="cuda").requires_grad_() for _ in range(2))
    g = torch.full((rows, 1, 64), 64.0, dtype=FP16, device="cuda")
    out = attention(q, k, v, torch.tensor([0, rows], device="cuda"), torch.tensor([0, keys], device="cuda"))
    dv, = torch.autograd.grad(out, v, g)
    want = rows * 64.0 / keys
    u = ref.U[FP16]
    off = want * (2 * u + (64 + rows) * ref.W) + 2.0 ** -14 * T * rows * 64 + T
    assert (dv.double() - want).abs().max() <= off


def test_answers():
    n, page = 3001, 16
    k, v = _keys(n, 8)
    pages = (n + page - 1) // page
    caches = [torch.nn.functional.pad(t, (0, 0, 0, 0, 0, pages * page - n)).view(pages, page, 1, 64).cuda() for t in (k, v)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    q = _queries(1, 4)
    out = answer(q.cuda(), *caches, table, torch.tensor([n], device="cuda"), 1.0)
    want = ref.one_sequence(q, k, v, False, 1.0)
    # a weight is rounded as a part of the largest one: over the sum of all, which are more than n / 8 of those
    per_weight = T * float(v.double().sum(0).max())
    off = want["o_off"] - per_weight + per_weight * 2.0 ** -6 / (n / 8)
    ref.assert_within(out, want["o"], off, "out")
