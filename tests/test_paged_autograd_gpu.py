"""Writes to a paged cache count as writes, and derivatives through it are refused."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import torchlib_xpu_b200

pytestmark = pytest.mark.gpu

torchlib_xpu_b200.load_torch_ops()
append = torch.ops.fbgemm.b200tbe_paged_cache_append
answer = torch.ops.fbgemm.b200tbe_paged_attention


def _arguments():
    """Two sequences of 3 and 5 positions in pages of 4: rows, their offsets, caches, page table, lengths, one query each."""
    gen = torch.Generator().manual_seed(2)
    rows = [torch.randn(8, 2, 16, generator=gen).cuda() for _ in range(2)]
    caches = [torch.zeros(3, 4, 2, 16, device="cuda") for _ in range(2)]
    table = torch.tensor([[2, 0], [0, 1]], dtype=torch.int32, device="cuda")
    return rows, torch.tensor([0, 3, 8], device="cuda"), caches, table, torch.tensor([3, 5], device="cuda"), torch.randn(2, 4, 16, generator=gen).cuda()


def test_an_append_is_seen_by_graphs_that_saved_the_cache():
    rows, offsets, caches, table, lengths, _ = _arguments()
    append(*rows, offsets, *caches, table, lengths)
    assert caches[0]._version == 1 and caches[1]._version == 1
    w = torch.ones(3, 4, 2, 16, device="cuda", requires_grad=True)
    for saved in (caches[0], caches[1][:2]):   # whole, and a view of it
        loss = (w[:saved.shape[0]] * saved).sum()
        append(*rows, offsets, *caches, table, lengths)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.no_grad():
        append(*rows, offsets, *caches, table, lengths)
    assert caches[0]._version == 4
    with torch.inference_mode():
        append(*rows, offsets, *caches, table, lengths)
    assert caches[0]._version == 5


def test_caches_of_inference_mode():
    """They have no version; they are written as before, inside the mode and outside."""
    rows, offsets, caches, table, lengths, q = _arguments()
    append(*rows, offsets, *caches, table, lengths)
    with torch.inference_mode():
        inner = [torch.zeros_like(c) for c in caches]
        append(*rows, offsets, *inner, table, lengths)
        a = answer(q, *inner, table, lengths)
    assert all(torch.equal(x, y) for x, y in zip(caches, inner))
    with torch.no_grad():
        append(*rows, offsets, *inner, table, lengths)
    assert torch.equal(a, answer(q, *caches, table, lengths))


def test_rows_and_caches_that_require_gradients():
    rows, offsets, caches, table, lengths, q = _arguments()
    # rows are stored as values: the cache takes no part in their graph
    append(rows[0].clone().requires_grad_() * 2, rows[1], offsets, *caches, table, lengths)
    assert not caches[0].requires_grad and torch.equal(caches[0][2, :3], rows[0][:3] * 2)
    for i in range(2):
        trained = list(caches)
        trained[i] = caches[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="requires grad"):
            append(*rows, offsets, *trained, table, lengths)
        trained[i] = trained[i] * 1.0   # a result of a graph
        with pytest.raises(RuntimeError, match="requires grad"):
            append(*rows, offsets, *trained, table, lengths)
        with torch.no_grad():
            append(*rows, offsets, *trained, table, lengths)
        assert trained[i]._version == 1


def test_answers_have_no_gradient():
    rows, offsets, caches, table, lengths, q = _arguments()
    append(*rows, offsets, *caches, table, lengths)
    plain = answer(q, *caches, table, lengths)
    assert not plain.requires_grad
    leaf = q.clone().requires_grad_()
    got = answer(leaf, *caches, table, lengths)
    assert torch.equal(got, plain)
    with pytest.raises(RuntimeError, match="b200tbe_paged_attention has no gradient"):
        got.sum().backward()
    trained = caches[1].clone().requires_grad_()
    got = answer(q, caches[0], trained, table, lengths)
    with pytest.raises(RuntimeError, match="b200tbe_paged_attention has no gradient"):
        got.sum().backward()
    with torch.no_grad():
        assert not answer(leaf, *caches, table, lengths).requires_grad


def test_forward_mode_is_refused():
    rows, offsets, caches, table, lengths, q = _arguments()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            answer(dual, *caches, table, lengths)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            answer(dual, *caches, table, lengths)
        for i in range(2):
            both = list(caches)
            both[i] = forward_ad.make_dual(caches[i], torch.ones_like(caches[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                answer(q, *both, table, lengths)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                append(*rows, offsets, *both, table, lengths)
            moved = list(rows)
            moved[i] = forward_ad.make_dual(rows[i], torch.ones_like(rows[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                append(*moved, offsets, *caches, table, lengths)
