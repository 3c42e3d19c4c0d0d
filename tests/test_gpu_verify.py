"""Draft verification (faq_verify_drafts) against a token-by-token reference with whole-number
sums: the outputs are whole numbers and have to be equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_reference import verify

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _case(b, k, vocab, dtype=torch.float32, drafter=True, seed=0, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(b, k + 1, vocab, generator=g) * sharp
    target = torch.softmax(logits, -1).to(dtype)
    close = torch.softmax(logits[:, :k] + 0.5 * torch.randn(b, k, vocab, generator=g), -1)
    tokens = torch.multinomial(close.reshape(-1, vocab), 1, generator=g).reshape(b, k) if k else torch.zeros(b, 0, dtype=torch.long)
    return (tokens, target, close.to(dtype) if drafter else None, torch.rand(b, k, generator=g), torch.rand(b, generator=g))


def _check(case, counts=None):
    from faquant_b200 import ops

    tokens, target, drafter, accept_u, sample_u = case
    got, accepted = ops.verify_drafts(tokens.to(DEV), target.to(DEV), None if drafter is None else drafter.to(DEV),
                                      accept_u.to(DEV), sample_u.to(DEV),
                                      num_drafts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV))
    limits = [min(max(c, 0), tokens.shape[1]) for c in counts] if counts is not None else [tokens.shape[1]] * tokens.shape[0]
    want, n = verify(tokens.numpy(), target, drafter, accept_u.numpy(), sample_u.numpy(), limits)
    assert got.dtype == torch.int64 and accepted.dtype == torch.int32
    np.testing.assert_array_equal(accepted.cpu().numpy(), n)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    return want, n


@pytest.mark.parametrize("drafter", [True, False], ids=["drafter", "lookup"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 5), (16, 4, 127), (9, 7, 1003), (5, 1, 4096), (2, 5, 33333)],
                         ids=lambda s: "x".join(map(str, s)))
def test_matches_the_reference(shape, dtype, drafter) -> None:
    for seed in range(3):
        _check(_case(*shape, dtype=dtype, drafter=drafter, seed=seed))


def test_ragged_counts_and_none() -> None:
    case = _case(8, 4, 600, seed=4)
    _check(case, [0, 1, 2, 3, 4, 4, 9, -1])
    _check(_case(4, 0, 600, seed=5))  # no drafts: a plain sample


def test_all_accepted_none_accepted() -> None:
    tokens, target, drafter, accept_u, sample_u = _case(6, 3, 300, seed=6)
    _, n = _check((tokens, target, drafter, torch.zeros_like(accept_u), sample_u))
    assert (n == 3).all()
    _, n = _check((tokens, target, drafter, torch.full_like(accept_u, 1e30), sample_u))
    assert (n == 0).all()


def test_random_numbers_at_the_ends() -> None:
    tokens, target, drafter, accept_u, _ = _case(5, 2, 1000, seed=7)
    for u in (0.0, 1.0 - 2.0**-24, 1.0, 2.0, -1.0):
        _check((tokens, target, drafter, accept_u, torch.full((5,), u)))
    target[:, :, :900] = 0  # the first and last entries have no weight
    target[:, :, 950:] = 0
    want, _ = _check((tokens % 900, target, None, accept_u, torch.zeros(5)))
    assert (want[:, 0] >= 900).all()


def test_rows_with_nothing_left() -> None:
    """p == q leaves no residual: p itself is sampled; a row without mass gives -1."""
    tokens, target, drafter, accept_u, sample_u = _case(4, 2, 700, seed=8)
    drafter = target[:, :2].clone()
    accept_u.fill_(3.0)  # rejects
    _check((tokens, target, drafter, accept_u, sample_u))
    target[1] = 0
    want, n = _check((tokens, target, drafter, accept_u, sample_u))
    assert want[1, 0] == -1 and n[1] == 0
    one = torch.zeros(1, 2, 50)
    one[:, :, 7] = 1.0
    want, n = _check((torch.tensor([[7]]), one, None, torch.tensor([[0.5]]), torch.tensor([0.9])))
    assert want.tolist() == [[7, 7]]


def test_drafts_outside_the_vocabulary_are_rejected() -> None:
    tokens, target, drafter, accept_u, sample_u = _case(4, 3, 200, seed=9)
    tokens[0, 0], tokens[1, 1], tokens[2, 0] = -1, 200, 2**40
    accept_u.fill_(0.0)
    for d in (drafter, None):
        _, n = _check((tokens, target, d, accept_u, sample_u))
        assert n.tolist() == [0, 1, 0, 3]


def test_not_a_number_weighs_nothing() -> None:
    from faquant_b200 import ops

    target = torch.full((1, 1, 64), float("nan"))
    target[0, 0, 40] = 0.5
    empty = torch.zeros(1, 0)
    got, _ = ops.verify_drafts(empty.long().to(DEV), target.to(DEV), None, empty.to(DEV), torch.tensor([0.3], device=DEV))
    assert got.tolist() == [[40]]


def test_strides_and_large_vocabulary() -> None:
    from faquant_b200 import ops

    tokens, target, drafter, accept_u, sample_u = _case(3, 2, 151936, seed=10)
    base = [t.to(DEV) for t in (tokens, target, drafter, accept_u, sample_u)]
    want = ops.verify_drafts(*base)
    wide_t = torch.empty(3, 3, 151936 + 5, device=DEV)[..., 2:-3]  # rows not 16-byte aligned
    wide_t.copy_(target)
    wide_d = torch.empty(2, 3, 151936, device=DEV).transpose(0, 1)
    wide_d.copy_(drafter)
    got = ops.verify_drafts(base[0], wide_t, wide_d, base[3].t().contiguous().t(), base[4])
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    _check((tokens, target, drafter, accept_u, sample_u))


def test_the_samples_follow_the_target() -> None:
    """Over many draws the emitted first token is distributed as the target, whatever the
    drafter: the check's defining property (chi-square with 7 degrees of freedom; 40 is
    beyond the 1 - 1e-6 quantile, 38.6 at 1e-6 being 7 + 31.6)."""
    from faquant_b200 import ops

    b, vocab = 20000, 8
    g = torch.Generator().manual_seed(11)
    p = torch.softmax(torch.randn(vocab, generator=g), 0)
    q = torch.softmax(torch.randn(vocab, generator=g), 0)
    tokens = torch.multinomial(q.expand(b, vocab), 1, generator=g)
    got, _ = ops.verify_drafts(tokens.to(DEV), p.expand(b, 2, vocab).contiguous().to(DEV),
                               q.expand(b, 1, vocab).contiguous().to(DEV), torch.rand(b, 1, generator=g).to(DEV),
                               torch.rand(b, generator=g).to(DEV))
    seen = torch.bincount(got[:, 0].cpu(), minlength=vocab).double()
    assert float(((seen - b * p.double()) ** 2 / (b * p.double())).sum()) < 40.0


def test_refusals() -> None:
    from faquant_b200 import ops

    tokens, target, drafter, accept_u, sample_u = (t.to(DEV) for t in _case(2, 2, 50, seed=12))
    with pytest.raises(ValueError):
        ops.verify_drafts(tokens[:, :1], target, drafter, accept_u, sample_u)
    with pytest.raises(ValueError):
        ops.verify_drafts(tokens, target, drafter[:, :1], accept_u, sample_u)
    with pytest.raises(ValueError):
        ops.verify_drafts(tokens, target, drafter.bfloat16(), accept_u, sample_u)
    with pytest.raises(TypeError):
        ops.verify_drafts(tokens.int(), target, drafter, accept_u, sample_u)
    with pytest.raises(TypeError):
        ops.verify_drafts(tokens, target.half(), None, accept_u, sample_u)
    with pytest.raises(ValueError):
        ops.verify_drafts(tokens, target, drafter, accept_u, sample_u, num_drafts=torch.tensor([1, 1], device=DEV))
    with pytest.raises(RuntimeError):
        ops.verify_drafts(tokens.cpu(), target, drafter, accept_u, sample_u)
