"""Cases of the sequence operators: attention over jagged sequences with its gradients, rows into a paged
key-value cache, and the attention of one new token over that cache.

A user of the embedding path has a batch of histories as jagged rows; these operators are what comes next:
training a model over them, filling a cache with their keys and values, and answering one token at a time.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SCORES_AT_ONCE = 1 << 27     # scores the plain form holds at a time


def listed():
    return [
        # one short request's history, forward only: the call's latency is what counts
        {"name": "attend_request", "op": "attend", "train": False, "dtype": "bf16", "batch": 1, "low": 37, "high": 37,
         "skew": 1.0, "heads": 4, "kv_heads": 4, "dim": 64, "causal": True, "cross": 0, "packed": True},
        # scoring candidates against histories: queries and keys of different lengths, no mask between them
        {"name": "attend_candidates", "op": "attend", "train": False, "dtype": "fp16", "batch": 96, "low": 0, "high": 1500,
         "skew": 2.0, "heads": 6, "kv_heads": 2, "dim": 80, "causal": False, "cross": 200, "packed": False},
        # prompts of very different lengths, packed, with shared key and value heads: work in proportion to length squared
        {"name": "attend_prompts", "op": "attend", "train": False, "dtype": "bf16", "batch": 5, "low": 611, "high": 8192,
         "skew": 1.0, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "cross": 0, "packed": True},
        # a training batch of short histories: the jagged configuration's 4096 rows of 0 to 128 positions, 256 wide
        {"name": "train_histories", "op": "attend", "train": True, "dtype": "bf16", "batch": 4096, "low": 0, "high": 128,
         "skew": 1.0, "heads": 4, "kv_heads": 4, "dim": 64, "causal": True, "cross": 0, "packed": False},
        # a training batch of long histories with shared heads
        {"name": "train_long", "op": "attend", "train": True, "dtype": "fp16", "batch": 7, "low": 301, "high": 4099,
         "skew": 1.0, "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "cross": 0, "packed": False},
        # a small model trained in single precision
        {"name": "train_fp32", "op": "attend", "train": True, "dtype": "fp32", "batch": 48, "low": 1, "high": 257,
         "skew": 1.0, "heads": 4, "kv_heads": 4, "dim": 32, "causal": False, "cross": 0, "packed": False},
        # the prompts' keys and values go into the cache
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "batch": 9, "low": 100, "high": 6000, "skew": 1.0,
         "before": 77, "kv_heads": 8, "dim": 128, "page": 64},
        # one new row for each sequence of a serving batch
        {"name": "append_step", "op": "append", "dtype": "fp16", "batch": 64, "low": 1, "high": 1, "skew": 1.0,
         "before": 1000, "kv_heads": 4, "dim": 64, "page": 16},
        # one sequence is answered: latency
        {"name": "answer_one", "op": "answer", "dtype": "bf16", "batch": 1, "low": 701, "high": 701, "skew": 1.0,
         "heads": 16, "kv_heads": 4, "dim": 128, "page": 16},
        # a serving batch of very different lengths
        {"name": "answer_batch", "op": "answer", "dtype": "bf16", "batch": 64, "low": 1, "high": 8191, "skew": 1.0,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # few very long sequences: one of them alone has to fill the GPU
        {"name": "answer_long", "op": "answer", "dtype": "fp16", "batch": 2, "low": 50001, "high": 131072, "skew": 1.0,
         "heads": 8, "kv_heads": 8, "dim": 64, "page": 32},
        # many short sequences, in single precision
        {"name": "answer_fp32", "op": "answer", "dtype": "fp32", "batch": 300, "low": 0, "high": 400, "skew": 1.0,
         "heads": 8, "kv_heads": 4, "dim": 48, "page": 16},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "train", "train", "append", "answer", "answer"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    case = {"dtype": rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"]), "kv_heads": kv_heads, "skew": rng.choice([0.5, 1.0, 2.0])}
    if op in ("attend", "train"):
        case.update(op="attend", train=op == "train", heads=kv_heads * rng.choice([1, 1, 2, 4]),
                    dim=rng.choice([32, 48, 64, 64, 80, 96, 128, 128]), causal=rng.random() < 0.7, cross=0, packed=False)
        case["high"] = _log_int(rng, 1, 512 if case["dtype"] == "fp32" else 6000)
        case["low"] = rng.randint(0, case["high"])
        if not case["causal"] and rng.random() < 0.5:
            case["cross"] = _log_int(rng, 1, 700)
        elif not case["train"]:
            case["packed"] = rng.random() < 0.5
        # no more scores than the largest listed case of its direction, and no more rows
        scores = (1 << 25 if case["dtype"] == "fp32" else 1 << 30 if case["train"] else 1 << 31) // case["heads"]
        longest = max(case["high"], case["cross"])
        case["batch"] = _log_int(rng, 1, max(1, min(4096, (1 << 17) // longest, scores // longest ** 2)))
    elif op == "append":
        case.update(op="append", dim=rng.choice([32, 48, 64, 80, 128]), page=rng.choice([1, 16, 32, 64, 100, 256]),
                    before=rng.randint(0, 300), high=_log_int(rng, 1, 6000))
        case["low"] = rng.randint(0, case["high"])
        case["batch"] = _log_int(rng, 1, max(1, min(512, 27000 // (case["high"] + case["before"]))))
    else:
        case.update(op="answer", heads=kv_heads * rng.choice([1, 2, 4, 4, 7, 8]), dim=rng.choice([32, 48, 64, 64, 80, 128, 128]),
                    page=rng.choice([1, 16, 16, 32, 64, 100, 256]), high=_log_int(rng, 1, 60000))
        case["low"] = rng.randint(0, case["high"])
        width = kv_heads * case["dim"] * (2 if case["dtype"] == "fp32" else 1)
        case["batch"] = _log_int(rng, 1, max(1, min(512, (1 << 28) // (width * case["high"]))))
    return case


def _spread(low, high, batch, skew):
    """Lengths from low to high, both among them."""
    if batch == 1:
        return [high]
    return [low + int(round((high - low) * (i / (batch - 1)) ** skew)) for i in range(batch)]


def _lengths(case):
    """(of the queries, of the keys), before the seed has put them in an order"""
    keys = _spread(case["low"], case["high"], case["batch"], case["skew"])
    if case["op"] == "attend" and case["cross"]:
        return _spread(1, case["cross"], case["batch"], 1.0), keys
    return keys, keys


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    cpu = torch.Generator()
    cpu.manual_seed(seed * 7919 + 5)
    dtype = _DTYPES[case["dtype"]]
    order = torch.randperm(case["batch"], generator=cpu).tolist()
    q_len, k_len = ([lens[i] for i in order] for lens in _lengths(case))
    kv, dim = case["kv_heads"], case["dim"]
    s = {"case": case, "q_len": q_len, "k_len": k_len}
    if case["op"] == "attend":
        heads = case["heads"]
        qo, ko = _offsets(q_len), _offsets(k_len)
        if case["packed"]:   # the rows of one projection: heads' queries, then keys, then values
            rows = _normal(gen, (qo[-1], heads + 2 * kv, dim), dtype)
            s["q"], s["k"], s["v"] = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
        else:
            s["q"] = _normal(gen, (qo[-1], heads, dim), dtype)
            s["k"], s["v"] = _normal(gen, (ko[-1], kv, dim), dtype), _normal(gen, (ko[-1], kv, dim), dtype)
        s["q_offsets"] = torch.tensor(qo, device="cuda")
        s["k_offsets"] = torch.tensor(ko, device="cuda") if case["cross"] else s["q_offsets"]
        if case["train"]:
            for name in ("q", "k", "v"):
                s[name].requires_grad_()
            s["grad"] = _normal(gen, (qo[-1], heads, dim), dtype)
        return s
    # a cache whose pages belong to the sequences in no order, with some pages to spare
    page = case["page"]
    lengths = [n + case["before"] for n in k_len] if case["op"] == "append" else k_len
    pages = [(n + page - 1) // page for n in lengths]
    total = sum(pages) + 3
    ids = torch.randperm(total, generator=cpu, dtype=torch.int32)
    table = torch.zeros(case["batch"], max(1, max(pages)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = ids[at:at + n]
        at += n
    s["page_table"] = table.cuda()
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["k_cache"], s["v_cache"] = (_normal(gen, (total, page, kv, dim), dtype) for _ in range(2))
    if case["op"] == "append":
        offsets = _offsets(k_len)
        s["k"], s["v"] = (_normal(gen, (offsets[-1], kv, dim), dtype) for _ in range(2))
        s["offsets"] = torch.tensor(offsets, device="cuda")
    else:
        s["q"] = _normal(gen, (case["batch"], case["heads"], dim), dtype)
    return s


def run(s):
    case = s["case"]
    if own:
        import torchlib_xpu_b200  # noqa: F401

        ops = torch.ops.fbgemm
        if case["op"] == "append":
            ops.b200tbe_paged_cache_append(s["k"], s["v"], s["offsets"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])
            return s["k_cache"], s["v_cache"]
        if case["op"] == "answer":
            return ops.b200tbe_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])
        out = ops.b200tbe_jagged_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], case["causal"])
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["grad"]))
    with torch.no_grad():
        if case["op"] == "append":
            return _plain_append(s)
        if case["op"] == "answer":
            return _plain_answer(s)
        return _plain_attend(s)


def _rows_of(starts, lengths, width):
    """Row numbers [n, width] of n sequences, and which of them are theirs."""
    step = torch.arange(width, device=starts.device)
    inside = step[None, :] < lengths[:, None]
    return torch.where(inside, starts[:, None] + step[None, :], 0), inside


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    group, scale = heads // kv, case["dim"] ** -0.5
    q, k, v = s["q"], s["k"], s["v"]
    q_starts, k_starts = s["q_offsets"][:-1], s["k_offsets"][:-1]
    q_lens, k_lens = s["q_offsets"].diff(), s["k_offsets"].diff()
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    grads = [torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)] if case["train"] else None
    b = 0
    while b < case["batch"]:
        # as many sequences at once as their padded scores allow
        e, mq, mk = b, 0, 0
        while e < case["batch"]:
            nq, nk = max(mq, s["q_len"][e]), max(mk, s["k_len"][e])
            if e > b and (e + 1 - b) * heads * nq * nk > _SCORES_AT_ONCE:
                break
            e, mq, mk = e + 1, nq, nk
        n = e - b
        if mq and mk:
            per = max(1, min(kv, _SCORES_AT_ONCE // max(1, n * group * mq * mk)))   # kv heads at once
            qi, q_in = _rows_of(q_starts[b:e], q_lens[b:e], mq)
            ki, k_in = _rows_of(k_starts[b:e], k_lens[b:e], mk)
            allowed = (q_in[:, :, None] & k_in[:, None, :])[:, None, None]
            if case["causal"]:
                last = torch.arange(mq, device=q.device)[None, :] + (k_lens - q_lens)[b:e, None]
                allowed = allowed & (torch.arange(mk, device=q.device)[None, None, :] <= last[:, :, None])[:, None, None]
            for h in range(0, kv, per):
                hs, qs = slice(h, min(kv, h + per)), slice(h * group, min(kv, h + per) * group)

                def queries(t):
                    return t[:, qs][qi].float().view(n, mq, -1, group, dim).permute(0, 2, 3, 1, 4)

                def keys(t):
                    return t[:, hs][ki].float().permute(0, 2, 1, 3)[:, :, None]

                qf, kf, vf = queries(q), keys(k), keys(v)
                scores = (qf @ kf.transpose(-1, -2)) * scale
                scores = scores.masked_fill(~allowed, float("-inf"))
                top = scores.amax(-1, keepdim=True)
                p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
                del scores
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                o = p @ vf
                rows = qi[q_in]

                def back(t, to, where, index):   # [n, kv, group, m, dim] to the jagged rows
                    to[:, qs][index] = t.permute(0, 3, 1, 2, 4).reshape(n, t.shape[3], -1, dim)[where].to(to.dtype)

                back(o, out, q_in, rows)
                if case["train"]:
                    g = queries(s["grad"])
                    dp = g @ vf.transpose(-1, -2)
                    ds = p * (dp - (g * o).sum(-1, keepdim=True))
                    del dp
                    back((ds @ kf) * scale, grads[0], q_in, rows)
                    for t, to in ((((ds.transpose(-1, -2) @ qf) * scale).sum(2), grads[1]),
                                  ((p.transpose(-1, -2) @ g).sum(2), grads[2])):
                        to[:, hs][ki[k_in]] = t.permute(0, 2, 1, 3)[k_in].to(to.dtype)
        b = e
    return (out, *grads) if case["train"] else out


def _plain_append(s):
    starts, counts = s["offsets"][:-1], s["offsets"].diff()
    rows, inside = _rows_of(starts, counts, max(1, max(s["k_len"])))
    step = torch.arange(rows.shape[1], device=rows.device)
    at = (s["lengths"][:, None] - counts[:, None] + step[None, :])[inside]
    page = s["case"]["page"]
    seq = torch.arange(rows.shape[0], device=rows.device)[:, None].expand_as(rows)[inside]
    pages = s["page_table"][seq, at // page].long()
    s["k_cache"][pages, at % page] = s["k"][rows[inside]]
    s["v_cache"][pages, at % page] = s["v"][rows[inside]]
    return s["k_cache"], s["v_cache"]


def _plain_answer(s):
    case = s["case"]
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    b = 0
    while b < case["batch"]:
        e, most = b, 0
        while e < case["batch"]:
            most_e = max(most, s["k_len"][e])
            if e > b and (e + 1 - b) * most_e * kv * dim > 4 * _SCORES_AT_ONCE:
                break
            e, most = e + 1, most_e
        n, used = e - b, max(1, (most + page - 1) // page)
        pages = s["page_table"][b:e, :used].long()
        kf, vf = (s[c][pages].view(n, used * page, kv, dim).permute(0, 2, 1, 3).float() for c in ("k_cache", "v_cache"))
        qf = s["q"][b:e].float().view(n, kv, heads // kv, dim)
        scores = (qf @ kf.transpose(-1, -2)) * dim ** -0.5
        past = torch.arange(used * page, device=scores.device)[None, :] >= s["lengths"][b:e, None]
        scores = scores.masked_fill(past[:, None, None], float("-inf"))
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
        total = p.sum(-1, keepdim=True)
        # a sequence's values only: what lies behind its length in the last page takes no part
        o = (p / torch.where(total == 0, 1.0, total)) @ vf.masked_fill(past[:, None, :, None], 0.0)
        out[b:e] = o.reshape(n, heads, dim).to(out.dtype)
        b = e
    return out


def exact(case, seed):
    if case["op"] == "append":
        return None   # rows are moved, nothing is computed
    s = prepare(case, seed)
    group = case["heads"] // case["kv_heads"]
    if case["op"] == "answer":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["k_len"]):
            if n == 0:
                continue
            table = s["page_table"][b]
            where = torch.arange(n, device="cuda")
            pages, slots = table[where // case["page"]].long(), where % case["page"]
            k, v = (s[c][pages, slots].double().repeat_interleave(group, 1) for c in ("k_cache", "v_cache"))
            logits = torch.einsum("hd,thd->ht", s["q"][b].double(), k) / math.sqrt(case["dim"])
            out[b] = torch.einsum("ht,thd->hd", torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True)), v)
        return out
    q, k, v = (s[name].detach().double() for name in ("q", "k", "v"))
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    qo, ko = _offsets(s["q_len"]), _offsets(s["k_len"])
    for b in range(case["batch"]):
        nq, nk = s["q_len"][b], s["k_len"][b]
        if nq == 0 or nk == 0:
            continue
        qs, ks = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
        hidden = None
        if case["causal"]:   # a query sees the keys up to its own place, counted from the ends
            hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
        per = case["kv_heads"] if nq * nk <= 1 << 18 else 1
        for h in range(0, case["kv_heads"], per):
            hk, hq = slice(h, h + per), slice(h * group, (h + per) * group)
            parts = [t.clone().requires_grad_(case["train"]) for t in (q[qs, hq], k[ks, hk], v[ks, hk])]
            a, c, d = parts[0], parts[1].repeat_interleave(group, 1), parts[2].repeat_interleave(group, 1)
            logits = torch.einsum("ihd,jhd->hij", a, c) / math.sqrt(case["dim"])
            if hidden is not None:
                logits = logits.masked_fill(hidden, float("-inf"))
            o = torch.einsum("hij,jhd->ihd", torch.softmax(logits, -1), d)
            out[qs, hq] = o.detach()
            if case["train"]:
                got = torch.autograd.grad(o, parts, s["grad"][qs, hq].double())
                grads[0][qs, hq], grads[1][ks, hk], grads[2][ks, hk] = got
            del logits, o
    return (out, *grads) if case["train"] else out


def _pairs(case):
    """Pairs of a query and a key that it sees, over the batch."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        total += sum(max(0, min(nk, i + 1 + nk - nq)) for i in range(nq)) if case["causal"] else nq * nk
    return total


def work(case):
    q_len, k_len = _lengths(case)
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    row = case["kv_heads"] * case["dim"] * size      # of the keys, and of the values
    if case["op"] == "append":
        tokens = sum(k_len)
        pages = sum((n + case["before"]) // case["page"] - case["before"] // case["page"] + 1 for n in k_len if n)
        return {"bytes": 4 * tokens * row + 4 * pages + 12 * case["batch"], "flops": 0}
    q_row = case["heads"] * case["dim"] * size
    if case["op"] == "answer":
        pages = sum((n + case["page"] - 1) // case["page"] for n in k_len)
        return {"bytes": 2 * sum(k_len) * row + 2 * case["batch"] * q_row + 4 * pages + 4 * case["batch"],
                "flops": 4 * sum(k_len) * case["heads"] * case["dim"]}
    nq, nk = sum(q_len), sum(k_len)
    product = 2 * _pairs(case) * case["heads"] * case["dim"]
    moved = 2 * nq * q_row + 2 * nk * row
    if not case["train"]:
        return {"bytes": moved, "flops": 2 * product}
    # out and the three gradients are written; queries, keys, values and the output's gradient are read
    return {"bytes": 4 * nq * q_row + 4 * nk * row, "flops": 7 * product}
