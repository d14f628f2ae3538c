"""The paged cache on a B200: rows appended to it, and the attention of one new token, against 64-bit attention."""
import pytest
import torch

import torchlib_xpu_b200
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
torchlib_xpu_b200.load_torch_ops()
append = torch.ops.fbgemm.b200tbe_paged_cache_append
answer = torch.ops.fbgemm.b200tbe_paged_attention
attention = torch.ops.fbgemm.b200tbe_jagged_attention
pop = torch.ops.fbgemm.b200tbe_pop_device_status


def _normal(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(dtype)


def _pages(lengths, page, seed, spare=2, width=None):
    """Shuffled pages for the lengths: (page table, number of pages). Unused entries hold ids of no page."""
    gen = torch.Generator().manual_seed(seed)
    counts = [(n + page - 1) // page for n in lengths]
    ids = torch.randperm(sum(counts) + spare, generator=gen, dtype=torch.int32)
    table = torch.full((len(lengths), max(1, width or max(counts, default=1))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, sum(counts) + spare


def _rows(cache, table, b, n, page):
    t = torch.arange(n)
    return cache[table[b, t // page].long(), t % page]


def _fill(cache, lengths, table, page):
    """Everything of the cache that no sequence owns becomes NaN."""
    owned = torch.zeros(cache.shape[:2], dtype=torch.bool)
    for b, n in enumerate(lengths):
        t = torch.arange(n)
        owned[table[b, t // page].long(), t % page] = True
    cache[~owned] = float("nan")


ANSWERS = [
    # dtype, lengths, heads, kv heads, D, page
    (BF16, [1], 1, 1, 64, 16),
    (BF16, [1, 0, 15, 16, 17, 63, 64, 65, 700], 8, 2, 128, 16),
    (FP16, [33, 127, 128, 129, 0, 1000], 4, 4, 64, 32),
    (FP32, [5, 0, 300, 64], 4, 2, 48, 16),
    (BF16, [5000, 3], 7, 1, 128, 100),       # pages that end inside a tile
    (FP16, [200, 77], 16, 1, 64, 1),         # one position a page; more query heads than one step takes
    (BF16, [300, 5], 12, 1, 80, 64),
    (BF16, [130, 257], 2, 2, 17, 7),         # rows of odd size
    (FP32, [100, 257], 3, 1, 256, 256),
    (FP16, [300], 9, 3, 256, 16),
    (BF16, [90, 300, 2], 64, 2, 32, 16),
    (FP16, [20000], 2, 1, 64, 64),           # one sequence over the whole GPU
    (BF16, [40000, 1, 12345], 8, 1, 128, 64),
    (FP16, [65, 66], 3, 3, 8, 16),
    (BF16, [64] * 40, 5, 1, 96, 16),
    (FP32, [9000, 10], 8, 8, 64, 32),
    (FP32, [300, 0, 65, 4000], 6, 1, 128, 16),
    (FP32, [129, 64], 18, 2, 100, 10),
    (FP16, [64, 128, 192, 1, 63, 65], 3, 1, 64, 64),
    (BF16, [1025, 700], 8, 8, 72, 48),
]


@pytest.mark.parametrize("ldtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,lengths,heads,kv,D,page", ANSWERS)
def test_one_new_token(dtype, lengths, heads, kv, D, page, ldtype):
    table, pages = _pages(lengths, page, 1)
    k, v = _normal((pages, page, kv, D), dtype, 2), _normal((pages, page, kv, D), dtype, 3)
    _fill(k, lengths, table, page)
    _fill(v, lengths, table, page)
    q = _normal((len(lengths), heads, D), dtype, 4)
    pop(torch.empty(0, device="cuda"))
    out = answer(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lengths, dtype=ldtype, device="cuda"))
    assert pop(out) == 0
    for b, n in enumerate(lengths):
        one = ref.one_sequence(q[b:b + 1], _rows(k, table, b, n, page), _rows(v, table, b, n, page), False, D ** -0.5)
        ref.assert_within(out[b:b + 1], one["o"], one["o_off"], "sequence %d" % b)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (FP16, 64), (FP32, 48)])
def test_strides_scale_and_streams(dtype, D):
    """Keys and values of one buffer, heads before positions, q a slice, on a side stream."""
    lengths, page, kv, heads = [70, 333, 1], 16, 2, 6
    table, pages = _pages(lengths, page, 5, width=40)
    both = _normal((pages, 2, kv, page, D), dtype, 6).cuda()
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    q = _normal((3, heads + 2, D), dtype, 7).cuda()[:, 1:1 + heads]
    wide = torch.full((3, 50), -1, dtype=torch.int32)
    wide[:, :40] = table
    side = torch.cuda.Stream()
    dev_table, dev_lengths = wide.cuda()[:, :40], torch.tensor(lengths, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = answer(q, k, v, dev_table, dev_lengths, 0.7)
    torch.cuda.current_stream().wait_stream(side)
    kc, vc, qc = k.cpu(), v.cpu(), q.cpu()
    for b, n in enumerate(lengths):
        one = ref.one_sequence(qc[b:b + 1], _rows(kc, table, b, n, page), _rows(vc, table, b, n, page), False, 0.7)
        ref.assert_within(out[b:b + 1], one["o"], one["o_off"], "sequence %d" % b)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_positions_far_into_a_large_cache(dtype):
    """Pages whose elements lie past 2^31 of the cache."""
    D, kv, page = 128, 8, 64
    pages = (1 << 31) // (D * kv * page) + 40
    k = torch.zeros((pages, page, kv, D), dtype=dtype, device="cuda")
    v = torch.zeros_like(k)
    lengths = [page * 3 + 5, 70]
    table = torch.tensor([[pages - 1, 0, pages - 7, pages - 3], [pages - 2, 1, -1, -1]], dtype=torch.int32)
    n = sum(lengths)
    rows_k, rows_v = _normal((n, kv, D), dtype, 8), _normal((n, kv, D), dtype, 9)
    offsets = torch.tensor([0, lengths[0], n])
    append(rows_k.cuda(), rows_v.cuda(), offsets.cuda(), k, v, table.cuda(), torch.tensor(lengths, device="cuda"))
    q = _normal((2, kv, D), dtype, 10)
    out = answer(q.cuda(), k, v, table.cuda(), torch.tensor(lengths, device="cuda"))
    for b in range(2):
        rows = slice(int(offsets[b]), int(offsets[b + 1]))
        one = ref.one_sequence(q[b:b + 1], rows_k[rows], rows_v[rows], False, D ** -0.5)
        ref.assert_within(out[b:b + 1], one["o"], one["o_off"], "sequence %d" % b)


def test_bad_pages_take_no_part_and_are_reported():
    """A page id outside the cache, and a length past the page table, as documented: those positions are left
    out, the others answer, the status word says so."""
    dtype, page, D = BF16, 16, 64
    lengths = [50, 40, 30]
    table, pages = _pages([64, 48, 32], page, 11, width=4)
    k, v = _normal((pages, page, 2, D), dtype, 12), _normal((pages, page, 2, D), dtype, 13)
    q = _normal((3, 4, D), dtype, 14)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = pages, -5
    long = torch.tensor([50, 40, 4 * page + 9], device="cuda")   # the third: more than its row of the table holds
    pop(torch.empty(0, device="cuda"))
    out = answer(q.cuda(), k.cuda(), v.cuda(), bad.cuda(), torch.tensor(lengths, device="cuda"))
    assert pop(out) == 1 and pop(out) == 0
    for b, n in enumerate(lengths):
        t = torch.arange(n)
        ids = bad[b, t // page].long()
        keep = (ids >= 0) & (ids < pages)
        kr, vr = k[ids[keep], t[keep] % page], v[ids[keep], t[keep] % page]
        one = ref.one_sequence(q[b:b + 1], kr, vr, False, D ** -0.5)
        ref.assert_within(out[b:b + 1], one["o"], one["o_off"], "sequence %d" % b)
    answer(q.cuda(), k.cuda(), v.cuda(), table.cuda(), long)
    assert pop(out) == 1
    for value in (-1, pages, -(1 << 31), (1 << 31) - 1):
        one_bad = table.clone()
        one_bad[2, 1] = value
        answer(q.cuda(), k.cuda(), v.cuda(), one_bad.cuda(), torch.tensor(lengths, device="cuda"))
        assert pop(out) == 1
    all_bad = torch.full_like(table, pages + 3)
    got = answer(q.cuda(), k.cuda(), v.cuda(), all_bad.cuda(), torch.tensor(lengths, device="cuda"))
    assert (got == 0).all() and pop(out) == 1
    # appended rows whose page is bad, or that would lie before position 0, are left out
    kc, vc = torch.zeros((pages, page, 2, D), dtype=dtype, device="cuda"), torch.zeros((pages, page, 2, D), dtype=dtype, device="cuda")
    rows = _normal((sum(lengths), 2, D), dtype, 15)
    offsets = torch.tensor([0, 50, 90, 120], device="cuda")
    append(rows.cuda(), rows.cuda(), offsets, kc, vc, bad.cuda(), torch.tensor([50, 40, 20], device="cuda"))
    assert pop(out) == 1
    want = torch.zeros((pages, page, 2, D), dtype=dtype)
    for b, n in enumerate([50, 40, 20]):
        for t in range(n):
            if 0 <= int(bad[b, t // page]) < pages:
                want[int(bad[b, t // page]), t % page] = rows[[0, 50, 100][b] + t]
    assert torch.equal(kc.cpu(), want) and torch.equal(vc.cpu(), want)


APPENDS = [
    # dtype, rows, before, kv heads, D, page
    (BF16, [1], [0], 1, 64, 16),
    (FP16, [1] * 40, [7 * i for i in range(40)], 4, 64, 16),
    (BF16, [0, 130, 3, 0, 1000], [5, 0, 15, 9, 77], 8, 128, 64),
    (FP32, [20, 33], [3, 0], 2, 48, 100),
    (BF16, [20, 33], [3, 0], 3, 17, 1),
    (FP16, [9, 300], [1, 2], 1, 2, 5),
]


@pytest.mark.parametrize("odtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,counts,before,kv,D,page", APPENDS)
def test_append(dtype, counts, before, kv, D, page, odtype):
    """Bit for bit; places no row goes to, and rows behind the last sequence, stay as they were."""
    lengths = [a + b for a, b in zip(counts, before)]
    table, pages = _pages(lengths, page, 21)
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    n = offsets[-1] + 3   # three rows of no sequence
    k, v = _normal((n, kv, D), dtype, 22), _normal((n, kv, D), dtype, 23)
    kc, vc = _normal((pages, page, kv, D), dtype, 24), _normal((pages, page, kv, D), dtype, 25)
    want_k, want_v = kc.clone(), vc.clone()
    for b, m in enumerate(counts):
        for i in range(m):
            at = before[b] + i
            want_k[int(table[b, at // page]), at % page] = k[offsets[b] + i]
            want_v[int(table[b, at // page]), at % page] = v[offsets[b] + i]
    dk, dv = kc.cuda(), vc.cuda()
    append(k.cuda(), v.cuda(), torch.tensor(offsets, dtype=odtype, device="cuda"), dk, dv, table.cuda(),
           torch.tensor(lengths, dtype=odtype, device="cuda"))
    assert torch.equal(dk.cpu(), want_k) and torch.equal(dv.cpu(), want_v)
    # strided rows into strided caches
    wide = torch.stack([k, v], 1).cuda()
    cache = torch.stack([kc, vc], 1).transpose(2, 3).contiguous().cuda()   # [pages, 2, kv, page, D]
    ck, cv = cache[:, 0].transpose(1, 2), cache[:, 1].transpose(1, 2)
    append(wide[:, 0], wide[:, 1], torch.tensor(offsets, dtype=odtype, device="cuda"), ck, cv, table.cuda(),
           torch.tensor(lengths, dtype=odtype, device="cuda"))
    assert torch.equal(ck.cpu(), want_k) and torch.equal(cv.cpu(), want_v)


@pytest.mark.parametrize("dtype,D,heads,kv", [(BF16, 128, 8, 2), (FP16, 64, 4, 4), (FP32, 48, 4, 2)])
def test_prompts_then_tokens(dtype, D, heads, kv):
    """A run as a server makes it: prompts attend and fill the cache, then each new token is appended and
    answered; every answer is what attention over the whole sequence gives at its last row."""
    page, prompts, steps = 16, [37, 1, 200], 5
    most = [n + steps for n in prompts]
    table, pages = _pages(most, page, 31)
    table = table.cuda()
    kc, vc = (torch.full((pages, page, kv, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    total = sum(most)
    q, k, v = _normal((total, heads, D), dtype, 32), _normal((total, kv, D), dtype, 33), _normal((total, kv, D), dtype, 34)
    starts = [0, most[0], most[0] + most[1]]
    rows = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, prompts)])
    offsets = torch.tensor([0, 37, 38, 238], device="cuda")
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    out = attention(q[rows].cuda(), k[rows].cuda(), v[rows].cuda(), offsets, None, True)
    append(k[rows].cuda(), v[rows].cuda(), offsets, kc, vc, table, lengths)
    at = 0
    for b, n in enumerate(prompts):
        s = slice(starts[b], starts[b] + n)
        one = ref.one_sequence(q[s], k[s], v[s], True, D ** -0.5)
        ref.assert_within(out[at:at + n], one["o"], one["o_off"], "prompt %d" % b)
        at += n
    step_offsets = torch.arange(4, device="cuda")
    hold = [torch.zeros(3, h, D, dtype=dtype, device="cuda") for h in (heads, kv, kv)]

    def step():
        lengths.add_(1)
        append(hold[1], hold[2], step_offsets, kc, vc, table, lengths)
        return answer(hold[0], kc, vc, table, lengths)

    graph = None
    for i in range(steps):
        new = torch.tensor([s + n + i for s, n in zip(starts, prompts)])
        for t, x in zip(hold, (q, k, v)):
            t.copy_(x[new])
        if i < 2:
            got = step()
        else:
            if graph is None:   # the other steps are replays of one graph
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    got = step()
            graph.replay()
        for b, n in enumerate(prompts):
            s = slice(starts[b], starts[b] + n + i + 1)
            last = starts[b] + n + i
            one = ref.one_sequence(q[last:last + 1], k[s], v[s], False, D ** -0.5)
            ref.assert_within(got[b:b + 1], one["o"], one["o_off"], "step %d, sequence %d" % (i, b))
    assert lengths.tolist() == most


def test_repeats_bit_for_bit():
    lengths = [3000, 1, 700, 64]
    table, pages = _pages(lengths, 16, 41)
    k, v = _normal((pages, 16, 2, 128), BF16, 42).cuda(), _normal((pages, 16, 2, 128), BF16, 43).cuda()
    q, n = _normal((4, 16, 128), BF16, 44).cuda(), torch.tensor(lengths, device="cuda")
    first = answer(q, k, v, table.cuda(), n)
    for _ in range(5):
        assert torch.equal(first, answer(q, k, v, table.cuda(), n))


def test_two_streams_at_once():
    """The operators on two streams at the same time, several calls deep, give what they give alone."""
    gen = torch.Generator().manual_seed(51)
    work = []
    for i, (dtype, D) in enumerate(((BF16, 128), (FP16, 64))):
        lengths = torch.randint(1, 700, (40,), generator=gen).tolist()
        table, pages = _pages(lengths, 32, 52 + i)
        cache = [_normal((pages, 32, 2, D), dtype, 53 + i).cuda(), _normal((pages, 32, 2, D), dtype, 55 + i).cuda()]
        n = sum(lengths)
        offsets = torch.tensor([0] + lengths, device="cuda").cumsum(0)
        rows = [_normal((n, h, D), dtype, 57 + i + j).cuda() for j, h in enumerate((4, 2, 2))]
        work.append((rows, offsets, cache, table.cuda(), torch.tensor(lengths, device="cuda"), _normal((40, 4, D), dtype, 61 + i).cuda()))

    def run(rows, offsets, cache, table, lengths, q):
        parts = [t.detach().requires_grad_() for t in rows]
        out = attention(*parts, offsets, None, True)
        grads = torch.autograd.grad(out, parts, torch.ones_like(out))
        got = answer(q, *cache, table, lengths)
        append(rows[1], rows[2], offsets, *cache, table, lengths)
        return (out.detach(), *grads, got, answer(q, *cache, table, lengths))

    want = [run(*w[:2], [c.clone() for c in w[2]], *w[3:]) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(3):
        got = []
        copies = [[c.clone() for c in w[2]] for w in work]
        torch.cuda.synchronize()
        for stream, w, cache in zip(streams, work, copies):
            with torch.cuda.stream(stream):
                got.append(run(*w[:2], cache, *w[3:]))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_many_sequences():
    gen = torch.Generator().manual_seed(45)
    lengths = torch.randint(0, 40, (1500,), generator=gen).tolist()
    table, pages = _pages(lengths, 8, 46)
    k, v = _normal((pages, 8, 1, 32), FP16, 47), _normal((pages, 8, 1, 32), FP16, 48)
    q = _normal((1500, 2, 32), FP16, 49)
    out = answer(q.cuda(), k.cuda(), v.cuda(), table.cuda(), torch.tensor(lengths, device="cuda"))
    for b, n in enumerate(lengths):
        one = ref.one_sequence(q[b:b + 1], _rows(k, table, b, n, 8), _rows(v, table, b, n, 8), False, 32 ** -0.5)
        ref.assert_within(out[b:b + 1], one["o"], one["o_off"], "sequence %d" % b)


def test_empty_and_refused():
    k = torch.zeros(4, 16, 2, 32, dtype=FP16, device="cuda")
    table, lengths = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.tensor([5, 0], device="cuda")
    q = torch.zeros(2, 4, 32, dtype=FP16, device="cuda")
    rows, offsets = torch.zeros(5, 2, 32, dtype=FP16, device="cuda"), torch.tensor([0, 5, 5], device="cuda")
    assert answer(q[:0], k, k, table[:0], lengths[:0]).shape == (0, 4, 32)
    append(rows[:0], rows[:0], offsets * 0, k, k.clone(), table, lengths)
    assert (answer(q, k, k, table[:, :0], lengths * 0) == 0).all()    # no pages at all
    assert (answer(q, k[:0], k[:0], table, lengths * 0) == 0).all()   # a cache without pages
    bad = [
        (lambda: answer(q, k, k[:2], table, lengths), "same shape"),
        (lambda: answer(q.float(), k, k, table, lengths), "dtype"),
        (lambda: answer(q[:, :3], k, k, table, lengths), "multiple"),
        (lambda: answer(q[:1], k, k, table, lengths), "batch"),
        (lambda: answer(q[..., :16], k, k, table, lengths), "head_dim"),
        (lambda: answer(q, k[0], k[0], table, lengths), "num_pages"),
        (lambda: answer(q, k, k, table.long(), lengths), "int32"),
        (lambda: answer(q, k, k, table[0], lengths), "int32"),
        (lambda: answer(q, k, k, table, lengths.float()), "int64 or int32"),
        (lambda: answer(q, k, k, table, lengths[:1]), "same batch"),
        (lambda: answer(q, k, k, table.cpu(), lengths), "page_table"),
        (lambda: answer(q, k.transpose(2, 3), k.transpose(2, 3), table, lengths), "side by side"),
        (lambda: append(rows[:, :1], rows[:, :1], offsets, k, k, table, lengths), "heads"),
        (lambda: append(rows, rows[:4], offsets, k, k, table, lengths), "same shape"),
        (lambda: append(rows, rows, offsets[:2], k, k, table, lengths), "one entry more"),
        (lambda: append(rows.float(), rows.float(), offsets, k, k, table, lengths), "dtype"),
    ]
    for call, words in bad:
        with pytest.raises(RuntimeError, match=words):
            call()
