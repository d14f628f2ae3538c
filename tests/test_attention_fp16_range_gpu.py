"""fp16 gradients of the jagged attention whose 64-bit values fp16 can hold, from output gradients near both ends of
fp16's range: dS = P (dP - delta) may lie far outside of it."""
import math

import pytest
import torch

import torchlib_xpu_b200
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

FP16 = torch.float16
torchlib_xpu_b200.load_torch_ops()
attention = torch.ops.fbgemm.b200tbe_jagged_attention
pop = torch.ops.fbgemm.b200tbe_pop_device_status


def _normal(shape, seed, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * size).to(FP16).cuda()


def _want(q, k, v, causal, scale, grad):
    """The reference's results and bounds with what dS loses below fp16's normal range put in its place.

    The kernels hold dS times a power of two that keeps 2 max|dO| max|v| of a sequence (lengths of the rows) at or under
    2^15 and, since it is the largest such power or its half, over 2^13: a dS below fp16's normal range is then off by at most
    2^-25 of that unit, or max|dO| max|v| 2^-38. The reference allows 2^-25 of dS itself. The gradients are
    linear in dO, so it is asked for dO times the power of two 2^m that makes the two the same, and its results
    and bounds are divided again; what an output below the normal range is rounded by (2^-25) comes back on top."""
    size = float(grad.double().norm(dim=-1).max() * v.double().norm(dim=-1).max())
    m = 13 - math.ceil(math.log2(size)) if size > 0 else 0
    want = ref.one_sequence(q, k, v, causal, scale, grad.double() * 2.0 ** m)
    for n in ("dq", "dk", "dv"):
        want[n] = want[n] * 2.0 ** -m
        want[n + "_off"] = want[n + "_off"] * 2.0 ** -m + 2.0 ** -25
    return want


LENGTHS = [
    ([2, 100, 1, 37, 128, 0, 64], "one tile each"),
    ([200, 130, 256, 3], "two tiles at most"),
    ([700, 129, 300], "several tiles"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,D", [(2, 2, 64), (4, 1, 64), (2, 1, 128), (2, 1, 36)])
@pytest.mark.parametrize("lengths,what", LENGTHS, ids=[w for _, w in LENGTHS])
@pytest.mark.parametrize("grad_size,q_size,v_size", [(1e4, 0.25, 4.0), (3e3, 0.05, 40.0), (1e-4, 1.0, 1.0), (1e-4, 1.0, 0.01)])
def test_output_gradients_near_the_ends_of_the_range(grad_size, q_size, v_size, lengths, what, heads, kv, D, causal):
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    q, k = _normal((o[-1], heads, D), 1, q_size), _normal((o[-1], kv, D), 2, q_size)
    v, g = _normal((o[-1], kv, D), 3, v_size), _normal((o[-1], heads, D), 4, grad_size)
    # the query heads of a key head differ in size, the later ones larger: their sums share a unit
    g = (g * 2.0 ** (torch.arange(heads, device="cuda") - heads + 1)[:, None]).to(FP16)
    parts = [t.detach().requires_grad_() for t in (q, k, v)]
    pop(q)
    out = attention(*parts, torch.tensor(o, device="cuda"), None, causal)
    got = torch.autograd.grad(out, parts, g)
    assert pop(q) == 0
    for b in range(len(lengths)):
        s = slice(o[b], o[b + 1])
        if lengths[b] == 0:
            continue
        want = _want(q[s], k[s], v[s], causal, D ** -0.5, g[s])
        for name, x in zip(("dq", "dk", "dv"), got):
            assert want[name].abs().max() < 65504 * (1 - 2.0 ** -8), "the case is to have finite gradients"
            ref.assert_within(x[s], want[name], want[name + "_off"], "%s of sequence %d" % (name, b))


@pytest.mark.parametrize("lengths", [[60, 61, 100], [300, 200, 400]])
def test_a_neighbour_of_another_size_changes_nothing(lengths):
    """The unit in which a sequence's dS is held is its own: neighbours whose gradients are larger by 2^20 leave
    every bit as it was."""
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    q, k, v = (_normal((o[-1], 2, 64), s) for s in (11, 12, 13))
    g = _normal((o[-1], 2, 64), 14, 1e-4)
    dev = torch.tensor(o, device="cuda")

    def run(grad):
        parts = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(attention(*parts, dev, None, True), parts, grad)

    alone = run(g)
    large = g.clone()
    for a, b in ((0, 1), (2, 3)):
        large[o[a]:o[b]] *= 2.0 ** 20
    for x, y in zip(alone, run(large)):
        assert torch.equal(x[o[1]:o[2]], y[o[1]:o[2]])
        assert torch.isfinite(y).all()


def test_no_gradient_at_all():
    """An output gradient of zeros, and values of zeros: nothing to divide by."""
    for lengths in ([50, 100], [300, 200]):
        o = torch.tensor([0, lengths[0], sum(lengths)], device="cuda")
        parts = [_normal((sum(lengths), 2, 64), s).requires_grad_() for s in (21, 22, 23)]
        out = attention(*parts, o, None, True)
        for x in torch.autograd.grad(out, parts, torch.zeros_like(out)):
            assert (x == 0).all()
        zero = torch.zeros_like(parts[2]).requires_grad_()
        out = attention(parts[0], parts[1], zero, o, None, True)
        dq, dk = torch.autograd.grad(out, parts[:2], torch.ones_like(out))
        assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("lengths", [[150, 64], [300, 200, 1000]])
def test_a_replayed_graph_finds_its_units_again(lengths):
    """One captured backward pass, replayed with output gradients of 10^4, of 10^-4 and of 10^4 again: nothing is left of
    the pass before, and each is what an eager call gives."""
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    dev = torch.tensor(o, device="cuda")
    q, k, v = (_normal((o[-1], h, 64), s, 0.25) for h, s in ((4, 31), (2, 32), (2, 33)))
    sizes = [_normal((o[-1], 4, 64), 34, x) for x in (1e4, 1e-4, 1e4)]

    def run(g):
        parts = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(attention(*parts, dev, None, True), parts, g)

    want = [run(g) for g in sizes]
    held = sizes[1].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for g, w in zip(sizes, want):
        held.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(w, got))
    assert all(torch.isfinite(t).all() for w in want for t in w)
