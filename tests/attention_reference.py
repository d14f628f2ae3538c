"""Attention in 64 bits for the tests, with how far a kernel's rounded steps may take it off.

u is half a step of the operands' type, w half a step of fp32 (2^-24). The kernels hold scores, maxima and
sums in fp32 and may round two things to the operands' type before a product: the weights P and dS.

* a score is a sum of D fp32 products of exact operands: off by at most s = (D + 8) w scale sum |q||k| (the 8:
  scaling, the subtraction of the maximum, and the exponent's rounding, each of a number no larger). A weight
  is then off by the factor 1 +- r, r = 2 s_max + 2 w |log-sum| + 16 w (its own score and the log-sum's; the
  exponential's and the final quotient's roundings).
* O: P may be rounded (u), n terms are summed (n w), the result is rounded (u):
      |O - o| <= (u + r + n w) sum p|v| + u |o|
* dV likewise with the gradient's rows in place of v, over the queries of all heads that share the key.
* dP is a sum of D products: off by D w sum |g||v|. rowsum(g o) takes the rounded output: off by
  sum |g| |O - o| + D w sum |g||o|. Their difference e makes dS off by p e + r |dS|, and rounding adds u |dS|.
      |dQ - dq| <= scale sum (p e + (r + u + n w) |dS|) |k| + u |dq|,  dK likewise.
Where fp16 holds a weight below its normal range (2^-14), it is off by up to 2^-25 instead of u: that much is
added for every key. A result that small is stored that coarsely too.
"""
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
W = 2.0 ** -24


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133


def one_sequence(q, k, v, causal, scale, grad=None):
    """q [nq, H, D], k, v [nk, Hkv, D], any type -> dict of 64-bit results and bounds (o; dq, dk, dv)."""
    dtype, nq, H, D = q.dtype, q.shape[0], q.shape[1], q.shape[2]
    nk, kv = k.shape[0], k.shape[1]
    group, u, t = H // kv, U[dtype], tiny(dtype)
    q, k, v = (x.detach().cpu().double().transpose(0, 1) for x in (q, k, v))   # [H, n, D]
    kx, vx = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    sees = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        sees = torch.arange(nk)[None, :] <= torch.arange(nq)[:, None] + nk - nq
    s = torch.where(sees, q @ kx.transpose(1, 2) * scale, torch.tensor(-float("inf"), dtype=torch.float64))
    if nk == 0:
        p = s.clone()
        lse = torch.full((H, nq, 1), -float("inf"), dtype=torch.float64)
    else:
        lse = torch.logsumexp(s, -1, keepdim=True)
        p = torch.where(sees, torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)), torch.zeros_like(s))
    o = p @ vx
    far = (D + 8) * W * abs(scale) * (q.abs() @ kx.abs().transpose(1, 2))
    far = far.amax(-1, keepdim=True) if nk else torch.zeros(H, nq, 1, dtype=torch.float64)
    r = 2 * far + 2 * W * torch.where(torch.isinf(lse), torch.zeros_like(lse), lse.abs()) + 16 * W
    small = t * (vx.abs().sum(1, keepdim=True))
    o_off = (u + r + nk * W) * (p @ vx.abs()) + u * o.abs() + small + t
    back = lambda x: x.transpose(0, 1)  # noqa: E731
    out = {"o": back(o), "o_off": back(o_off), "lse": lse[..., 0]}
    if grad is None:
        return out
    g = grad.detach().cpu().double().transpose(0, 1)
    dp = g @ vx.transpose(1, 2)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e = D * W * (g.abs() @ vx.abs().transpose(1, 2)) + (g.abs() * o_off).sum(-1, keepdim=True) + \
        D * W * (g.abs() * o.abs()).sum(-1, keepdim=True) + 2 * W * (dp.abs() + delta.abs())
    n = max(nk, nq * group)
    ds_off = p * e + (r + u + n * W) * ds.abs() + t
    dq = scale * ds @ kx
    dq_off = abs(scale) * (ds_off @ kx.abs()) + u * dq.abs() + t
    shared = lambda x: x.view(kv, group, nk, D).sum(1)  # noqa: E731
    dk = shared(scale * ds.transpose(1, 2) @ q)
    dk_off = shared(abs(scale) * (ds_off.transpose(1, 2) @ q.abs())) + u * dk.abs() + t
    dv = shared(p.transpose(1, 2) @ g)
    dv_off = shared((p * (u + r + n * W) + t).transpose(1, 2) @ g.abs()) + u * dv.abs() + t
    out.update(dq=back(dq), dq_off=back(dq_off), dk=back(dk), dk_off=back(dk_off), dv=back(dv), dv_off=back(dv_off))
    return out


def jagged(q, k, v, q_offsets, k_offsets, causal, scale, grad=None):
    """The whole batch: dict of tensors like one_sequence's, rows of no sequence 0 (bound 0)."""
    names = {"o": q, "dq": q, "dk": k, "dv": v} if grad is not None else {"o": q}
    out = {}
    for n, like in names.items():
        out[n] = torch.zeros(like.shape, dtype=torch.float64)
        out[n + "_off"] = torch.zeros(like.shape, dtype=torch.float64)
    for b in range(len(q_offsets) - 1):
        qs, ks = slice(q_offsets[b], q_offsets[b + 1]), slice(k_offsets[b], k_offsets[b + 1])
        one = one_sequence(q[qs], k[ks], v[ks], causal, scale, None if grad is None else grad[qs])
        for n in names:
            rows = ks if n in ("dk", "dv") else qs
            out[n][rows], out[n + "_off"][rows] = one[n], one[n + "_off"]
    return out


def assert_within(got, want, off, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), "%s: not finite" % what
    worst = ((got - want).abs() - off)
    assert (worst <= 0).all(), "%s: %d of %d beyond the bound, worst by a factor of %.3g" % (
        what, int((worst > 0).sum()), worst.numel(), float(((got - want).abs() / off.clamp_min(1e-300)).max()))
