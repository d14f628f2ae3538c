"""Jagged attention and its gradients on a B200 against 64-bit attention, through torch.ops.fbgemm and the C ABI."""
import ctypes

import pytest
import torch

import torchlib_xpu_b200
from tests import attention_reference as ref
from torchlib_xpu_b200 import cabi

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
torchlib_xpu_b200.load_torch_ops()
attention = torch.ops.fbgemm.b200tbe_jagged_attention


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _normal(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(dtype).cuda()


def _check(q, k, v, qo, ko, causal, scale=None, grad=None, odtype=torch.int64):
    """One forward (and backward) pass against the reference; returns what the operator gave."""
    dq_off = torch.tensor(qo, dtype=odtype, device="cuda")
    dk_off = torch.tensor(ko, dtype=odtype, device="cuda")
    if grad is not None:
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = attention(q, k, v, dq_off, dk_off, causal, scale)
    want = ref.jagged(q, k, v, qo, ko, causal, q.shape[2] ** -0.5 if scale is None else scale, grad)
    assert out.dtype == q.dtype
    ref.assert_within(out, want["o"], want["o_off"], "out")
    if grad is None:
        return out
    got = torch.autograd.grad(out, (q, k, v), grad)
    for name, x in zip(("dq", "dk", "dv"), got):
        ref.assert_within(x, want[name], want[name + "_off"], name)
    return (out, *got)


EDGES = [1, 0, 2, 127, 128, 129, 0, 255, 256, 257, 63, 64, 65, 1, 0]

CASES = [
    # dtype, lengths, heads, kv heads, D, causal
    (BF16, [1], 1, 1, 64, True),
    (BF16, EDGES, 2, 1, 64, True),
    (FP16, EDGES, 2, 2, 128, False),
    (BF16, EDGES, 4, 1, 128, True),
    (FP32, EDGES, 2, 1, 32, True),
    (FP32, [200, 3], 3, 3, 48, False),
    (FP16, [300, 5, 64], 6, 2, 80, True),
    (BF16, [140, 31], 2, 2, 17, True),      # rows of odd size
    (FP16, [70, 150], 1, 1, 256, False),
    (FP32, [70, 33], 2, 1, 200, True),
    (BF16, [513, 1000], 3, 1, 96, False),
    (FP16, [1025, 0, 40], 2, 1, 32, True),
    (BF16, [129, 250], 7, 7, 8, True),
    (FP32, [1, 1, 1], 1, 1, 1, True),
    (BF16, [2100], 2, 1, 128, True),        # many tiles of keys, and of queries
    (FP16, [1700, 90], 2, 2, 64, False),
]


@pytest.mark.parametrize("dtype,lengths,heads,kv,D,causal", CASES)
def test_self_attention_and_gradients(dtype, lengths, heads, kv, D, causal):
    o = _offsets(lengths)
    q, g = (_normal((o[-1], heads, D), dtype, s) for s in (1, 2))
    k, v = (_normal((o[-1], kv, D), dtype, s) for s in (3, 4))
    _check(q, k, v, o, o, causal, grad=g)


CROSS = [
    # dtype, query lengths, key lengths, heads, kv heads, D, causal, offsets
    (BF16, [5, 0, 130, 1, 257, 3], [300, 40, 0, 1, 128, 129], 4, 2, 64, False, torch.int32),
    (FP16, [5, 0, 130, 1, 257, 300], [300, 40, 0, 1, 128, 20], 2, 1, 128, True, torch.int64),   # rows that see nothing
    (FP32, [65, 200, 7], [64, 3, 90], 2, 2, 32, True, torch.int32),
    (FP32, [65, 200, 7], [64, 0, 90], 2, 1, 40, False, torch.int64),
    (BF16, [1, 1, 1, 1], [700, 1, 128, 129], 8, 2, 128, True, torch.int64),
    (BF16, [0, 0], [10, 200], 1, 1, 64, False, torch.int64),                                   # no query at all
    (FP16, [10, 200], [0, 0], 1, 1, 64, True, torch.int64),                                    # no key at all
]


@pytest.mark.parametrize("dtype,ql,kl,heads,kv,D,causal,odtype", CROSS)
def test_queries_and_keys_of_different_lengths(dtype, ql, kl, heads, kv, D, causal, odtype):
    qo, ko = _offsets(ql), _offsets(kl)
    q, g = (_normal((qo[-1], heads, D), dtype, s) for s in (11, 12))
    k, v = (_normal((ko[-1], kv, D), dtype, s) for s in (13, 14))
    _check(q, k, v, qo, ko, causal, grad=g, odtype=odtype)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128), (FP32, 32), (BF16, 36)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_no_sequence_are_zero_and_never_read(dtype, D, causal):
    """Rows before the first sequence and behind the last hold NaN and infinity: the sequences' results do not
    change, and the rows' own results and gradients are 0."""
    lengths, before, behind = [100, 1, 260], 3, 70
    o = [before + x for x in _offsets(lengths)]
    total = o[-1] + behind
    q, g = (_normal((total, 2, D), dtype, s) for s in (21, 22))
    k, v = (_normal((total, 1, D), dtype, s) for s in (23, 24))
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (g, float("nan"))):
        t[:before] = bad
        t[o[-1]:] = bad
    out, dq, dk, dv = _check(q, k, v, o, o, causal, grad=g)
    inner = slice(before, o[-1])
    rows = torch.ones(total, dtype=torch.bool)
    rows[inner] = False
    for t in (out, dq, dk, dv):
        assert (t[rows.cuda()] == 0).all()


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128), (FP32, 32), (BF16, 128)])
def test_neighbours_that_are_not_finite(dtype, D):
    """A sequence full of NaN between two others changes nothing in theirs."""
    o = _offsets([100, 61, 200])
    q, g = (_normal((o[-1], 2, D), dtype, s) for s in (31, 32))
    k, v = (_normal((o[-1], 2, D), dtype, s) for s in (33, 34))
    dev = torch.tensor(o, device="cuda")

    def both():
        parts = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = attention(*parts, dev, dev, True)
        return (out.detach(), *torch.autograd.grad(out, parts, g))

    clean = both()
    for t in (q, k, v, g):
        t[o[1]:o[2]] = float("nan")
    for a, b in zip(clean, both()):
        assert torch.equal(a[:o[1]], b[:o[1]]) and torch.equal(a[o[2]:], b[o[2]:])


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128), (FP32, 48), (BF16, 20)])
def test_slices_of_one_projection(dtype, D):
    o = _offsets([130, 0, 77])
    rows = _normal((o[-1], 4 + 2 + 2, D), dtype, 41)
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    g = _normal((4, o[-1], D), dtype, 42).transpose(0, 1)   # heads outermost
    a = _check(q, k, v, o, o, True, grad=g)
    b = _check(q.contiguous(), k.contiguous(), v.contiguous(), o, o, True, grad=g.contiguous())
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 64), (FP32, 64)])
def test_odd_addresses_and_broadcast_heads(dtype, D):
    """Rows that begin off every 16-byte boundary, a last dimension that is not dense, and one key head
    expanded to all of them."""
    o = _offsets([90, 150])
    q = _normal((o[-1], 2, D + 3), dtype, 51)[..., 1:1 + D]
    k = _normal((o[-1], D, 2), dtype, 52).transpose(1, 2)
    v = _normal((o[-1], 1, D), dtype, 53).expand(-1, 2, -1)
    g = _normal((1, 1, 1), dtype, 54).expand(o[-1], 2, D)
    _check(q, k, v, o, o, True, grad=g)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_scale_and_large_scores(dtype):
    """Scores from -300 to 300: the maximum runs far ahead of a tile's, and whole tiles weigh nothing."""
    o = _offsets([700])
    q, k, v, g = (_normal((o[-1], 1, 64), dtype, s) for s in (61, 62, 63, 64))
    ramp = torch.linspace(0.05, 2.0, o[-1], device="cuda")[:, None, None]
    k = (k.float() * ramp).to(dtype)
    _check(q, k, v, o, o, True, scale=2.0, grad=g)
    _check(q, k.flip(0), v, o, o, False, scale=-1.5, grad=g)
    _check(q, k, v, o, o, False, scale=0.0, grad=g)


def test_gradients_against_differences():
    """d loss along random directions, in fp32, against central differences of the operator itself: the loss
    is about 10, rounded to 2^-24 of its terms, and a step of 2^-6 leaves a third-derivative term of about
    step^2 / 6 of the slope's own size."""
    o = _offsets([40, 0, 23, 70])
    q, k, v, g = (_normal((o[-1], 2, 32), FP32, s) for s in (71, 72, 73, 74))
    dev = torch.tensor(o, device="cuda")
    for causal in (True, False):
        parts = [t.clone().requires_grad_() for t in (q, k, v)]
        grads = torch.autograd.grad(attention(*parts, dev, dev, causal), parts, g)
        for i, t in enumerate((q, k, v)):
            d = _normal(t.shape, FP32, 80 + i)
            d = d / d.norm()
            step = 2.0 ** -6

            def loss(x):
                a = [q, k, v]
                a[i] = x
                return (attention(*a, dev, dev, causal).double() * g.double()).sum()

            slope = float((loss(t + step * d) - loss(t - step * d)) / (2 * step))
            want = float((grads[i].double() * d.double()).sum())
            # each output element is off by at most 2^-20 of its size (a few units of fp32): the two losses' roundings
            # add like noise of 2^-20 * |g . out| / step; the curvature adds step^2 of the gradient's norm
            noise = 2.0 ** -20 * float((attention(q, k, v, dev, dev, causal).abs() * g.abs()).sum()) ** 0.5 * 4 / step
            assert abs(slope - want) <= noise + step ** 2 * float(grads[i].double().norm()), (i, causal, slope, want)


def test_only_what_needs_a_gradient():
    o = _offsets([33, 100])
    q, k, v, g = (_normal((o[-1], 2, 64), BF16, s) for s in (91, 92, 93, 94))
    dev = torch.tensor(o, device="cuda")
    full = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(attention(*full, dev, None, True), full, g)
    for i in range(3):
        parts = [q, k, v]
        parts[i] = parts[i].clone().requires_grad_()
        got, = torch.autograd.grad(attention(*parts, dev, None, True), parts[i], g)
        assert torch.equal(got, want[i])
    with torch.no_grad():
        assert not attention(*full, dev, None, True).requires_grad


def test_a_second_derivative_is_refused():
    o = torch.tensor([0, 8], device="cuda")
    q = _normal((8, 1, 16), FP32, 95).requires_grad_()
    out = attention(q, q, q, o)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64), (FP32, 32)])
def test_repeats_bit_for_bit(dtype, D):
    o = _offsets([400, 10, 333])
    dev = torch.tensor(o, device="cuda")
    q, g = (_normal((o[-1], 4, D), dtype, s) for s in (101, 102))
    k, v = (_normal((o[-1], 2, D), dtype, s) for s in (103, 104))
    first = None
    for _ in range(4):
        parts = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention(*parts, dev, None, True)
        got = (out.detach(), *torch.autograd.grad(out, parts, g))
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, got))
        first = got


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_streams_and_graphs(dtype):
    """A side stream, then a captured forward and backward pass replayed on new inputs while an eager graph of
    other leaves lives; two captured graphs side by side."""
    o = _offsets([150, 64])
    dev = torch.tensor(o, device="cuda")
    make = lambda s: [_normal((o[-1], 2, 64), dtype, s + i) for i in range(4)]  # noqa: E731

    def step(q, k, v, g):
        parts = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention(*parts, dev, None, True)
        return (out.detach(), *torch.autograd.grad(out, parts, g))

    first, second = make(111), make(121)
    want = [step(*first), step(*second)]
    alive = attention(*[t.clone().requires_grad_() for t in first[:3]], dev, None, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*first)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want[0], got))
    held = [[t.clone() for t in first] for _ in range(2)]
    graphs, outs = [], []
    for inputs in held:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*inputs))
        graphs.append(graph)
    for t, new in zip(held[1], second):
        t.copy_(new)
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want[i], outs[i]))
    alive.sum().backward()


def test_empty_batches():
    for rows, offsets in ((0, [0]), (0, [0, 0, 0]), (5, [0])):
        q = _normal((rows, 2, 64), BF16, 131).requires_grad_()
        out = attention(q, q, q, torch.tensor(offsets, device="cuda"))
        assert out.shape == q.shape and (out == 0).all()
        g, = torch.autograd.grad(out.sum(), q)
        assert (g == 0).all()


def test_offsets_beyond_the_rows_read_and_write_nothing_outside():
    """Offsets that run past the arrays are cut to them."""
    q = _normal((100, 1, 64), BF16, 141)
    want = attention(q, q, q, torch.tensor([0, 40, 100], device="cuda"))
    got = attention(q, q, q, torch.tensor([-7, 40, 1 << 40], device="cuda"))
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv,D,causal", [(4, 2, 128, True), (3, 1, 64, False), (2, 2, 40, True)])
def test_many_tiles_for_every_cta(heads, kv, D, causal):
    """More tiles than the GPU has CTAs, of long and short sequences mixed, so that CTAs take several after one another:
    some sequences against the reference, and the whole a second time, bit for bit."""
    gen = torch.Generator().manual_seed(6)
    lengths = torch.randint(100, 700, (90,), generator=gen).tolist() + [0, 1, 1500]
    o = _offsets(lengths)
    q, g = (_normal((o[-1], heads, D), BF16, s) for s in (181, 182))
    k, v = (_normal((o[-1], kv, D), BF16, s) for s in (183, 184))
    dev = torch.tensor(o, device="cuda")
    parts = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*parts, dev, None, causal)
    grads = torch.autograd.grad(out, parts, g)
    for b in (0, 17, 55, 89, 91, 92):
        s = slice(o[b], o[b + 1])
        one = ref.one_sequence(q[s], k[s], v[s], causal, D ** -0.5, g[s])
        for name, x in zip(("o", "dq", "dk", "dv"), (out, *grads)):
            ref.assert_within(x[s], one[name], one[name + "_off"], "%s of sequence %d" % (name, b))
    again = attention(*parts, dev, None, causal)
    assert torch.equal(out, again)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(again, parts, g)))


def test_many_short_sequences():
    """More sequences than one search step covers, single rows among them."""
    gen = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 9, (2500,), generator=gen).tolist()
    o = _offsets(lengths)
    q, g = (_normal((o[-1], 2, 64), BF16, s) for s in (151, 152))
    k, v = (_normal((o[-1], 1, 64), BF16, s) for s in (153, 154))
    _check(q, k, v, o, o, True, grad=g)


def test_refusals():
    q = _normal((6, 4, 16), FP32, 161)
    k = _normal((6, 2, 16), FP32, 162)
    o = torch.tensor([0, 6], device="cuda")
    bad = [
        ((q, k, k[:, :1], o), "same shape"),
        ((q, k[:5], k[:5], o), "same number of rows"),
        ((q, k[..., :8], k[..., :8], o, o), "head_dim"),
        ((q[:, :3], k, k, o, o), "multiple"),
        ((q.half(), k, k, o, o), "dtype"),
        ((q.double(), k.double(), k.double(), o, o), "float32"),
        ((q[0], k, k, o, o), "head_dim"),
        ((q, k, k, o.float(), o.float()), "int64 or int32"),
        ((q, k, k, o, o.int()), "same length and dtype"),
        ((q, k, k, o, torch.tensor([0, 3, 6], device="cuda")), "same length"),
        ((q, k, k, o.cpu(), o), "CUDA"),
        ((q, k.cpu(), k.cpu(), o, o), "CUDA"),
        ((q, k, k, o[:0], o[:0]), "at least one"),
        ((q, k, k, torch.tensor([0, 1, 6, 7], device="cuda")[::2], o), "contiguous"),
    ]
    for args, words in bad:
        with pytest.raises(RuntimeError, match=words):
            attention(*args)
    with pytest.raises(RuntimeError, match="head_dim"):
        wide = _normal((6, 1, 257), FP32, 163)
        attention(wide, wide, wide, o)


def test_c_abi_with_strided_output():
    """out and the gradients written into slices of wider buffers, whose other columns stay as they were."""
    o = _offsets([150, 3])
    n, H, D = o[-1], 2, 64
    q, k, v, g = (_normal((n, H, D), BF16, s) for s in (171, 172, 173, 174))
    dev = torch.tensor(o, device="cuda")
    wide = torch.full((n, 4 * H, D), 7.0, dtype=BF16, device="cuda")
    out, dq, dk, dv = (wide[:, i * H:(i + 1) * H] for i in range(4))
    lse = torch.empty(H, n, device="cuda")
    p = cabi.AttentionParams()
    p.q, p.k, p.v, p.out, p.lse = (t.data_ptr() for t in (q, k, v, out, lse))
    p.q_offsets = p.k_offsets = dev.data_ptr()
    p.q_stride = p.k_stride = p.v_stride = H * D
    p.q_head_stride = p.k_head_stride = p.v_head_stride = p.out_head_stride = D
    p.out_stride = 4 * H * D
    p.total_q = p.total_k = n
    p.batch, p.heads, p.kv_heads, p.head_dim, p.dtype, p.offset_bytes, p.causal, p.scale = 2, H, H, D, cabi.BF16, 8, 1, D ** -0.5
    stream = torch.cuda.current_stream().cuda_stream
    cabi.check(cabi.lib().b200tbe_jagged_attention(ctypes.byref(p), stream), "forward")
    want = ref.jagged(q, k, v, o, o, True, D ** -0.5, g)
    ref.assert_within(out, want["o"], want["o_off"], "out")
    for b in range(2):
        one = ref.one_sequence(q[o[b]:o[b + 1]], k[o[b]:o[b + 1]], v[o[b]:o[b + 1]], True, D ** -0.5)
        # the log-sum: its scores are off by (D + 8) 2^-24 of their terms' sizes (at most |q||k| / 8 < 25 here)
        assert (lse[:, o[b]:o[b + 1]].cpu().double() - one["lse"]).abs().max() < (D + 24) * 2.0 ** -24 * 25
    assert (wide[:, H:] == 7).all()
    b = cabi.AttentionBackwardParams()
    b.forward = p
    b.grad_out, b.grad_q, b.grad_k, b.grad_v = (t.data_ptr() for t in (g, dq, dk, dv))
    b.grad_out_stride, b.grad_out_head_stride = H * D, D
    b.grad_q_stride = b.grad_k_stride = b.grad_v_stride = 4 * H * D
    b.grad_q_head_stride = b.grad_k_head_stride = b.grad_v_head_stride = D
    need = cabi.lib().b200tbe_jagged_attention_backward_scratch_bytes(n, n, 2, H)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    b.scratch, b.scratch_bytes = scratch.data_ptr(), need - 1
    assert cabi.lib().b200tbe_jagged_attention_backward(ctypes.byref(b), stream) == -2
    b.scratch_bytes = need
    cabi.check(cabi.lib().b200tbe_jagged_attention_backward(ctypes.byref(b), stream), "backward")
    for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        ref.assert_within(t, want[name], want[name + "_off"], name)
    ref.assert_within(out, want["o"], want["o_off"], "out after backward")
