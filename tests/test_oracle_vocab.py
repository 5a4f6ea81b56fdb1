"""The 64-bit restatement of the vocabulary operators against independent ways to the same numbers (CPU)."""
import math

import pytest
import torch

from oracle import vocab as O


def _case(seed, N=3, V=23, K=5, tail=True, cap=4.0, T=1.7):
    g = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(N, V, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)])
    ids[1, 2] = -1
    ids[2, 3] = ids[2, 0]          # a token named twice
    teacher = torch.randn(N, V, generator=g, dtype=torch.float64)
    values = teacher.gather(1, ids.clamp(min=0))
    lse = torch.logsumexp(teacher / T, -1) if tail else None
    return x, values, ids, dict(cap=cap, T=T, lse=lse)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("cap", [None, 4.0])
def test_gradient_formula_against_autograd_and_differences(tail, cap):
    x, values, ids, kw = _case(11, tail=tail, cap=cap)
    if tail:
        values[2, 3] -= 2.0        # (its two entries together stay below the whole)
    leaf = x.clone().requires_grad_()
    O.distill(leaf, values, ids, **kw).sum().backward()
    formula = O.distill_grad(x, values, ids, **kw)
    torch.testing.assert_close(formula, leaf.grad, rtol=1e-10, atol=1e-12)
    h = 1e-5   # central differences: truncation h^2 ~ 1e-10, rounding 1e-16 / h ~ 1e-11
    for r, j in ((0, 0), (1, 7), (2, int(ids[2, 0])), (0, int(ids[0, 1]))):
        e = torch.zeros_like(x)
        e[r, j] = h
        d = (O.distill(x + e, values, ids, **kw).sum() - O.distill(x - e, values, ids, **kw).sum()) / (2 * h)
        assert abs(float(d) - float(formula[r, j])) < 1e-8


def test_distillation_from_the_whole_vocabulary_is_the_kl_divergence():
    g = torch.Generator().manual_seed(3)
    x, t = torch.randn(2, 9, generator=g, dtype=torch.float64), torch.randn(2, 9, generator=g, dtype=torch.float64)
    ids = torch.arange(9).expand(2, 9)
    kl = (torch.softmax(t, -1) * (torch.log_softmax(t, -1) - torch.log_softmax(x, -1))).sum(-1)
    torch.testing.assert_close(O.distill(x, t, ids), kl)
    torch.testing.assert_close(O.distill(x, t, ids, lse=torch.logsumexp(t, -1)), kl)


def test_sampling_frequencies_are_the_filtered_softmax():
    x = torch.tensor([0.3, 2.0, -1.0, 2.0, 1.0, -math.inf, math.nan])
    n = 4000
    got = torch.zeros(7)
    for i in range(n):
        got[O.sample_row(x, None, (i + 0.5) / n, T=0.9, k=4)[0]] += 1
    keep = torch.tensor([0, 1, 3, 4])
    want = torch.zeros(7)
    want[keep] = torch.softmax(x[keep] / 0.9, 0)
    assert (got / n - want).abs().max() <= 1.0 / n + 1e-6   # one step of u at each border


def test_sampling_filters():
    x = torch.log(torch.tensor([0.1, 0.4, 0.3, 0.2]))
    assert O.sample_row(x, None, 0.0)[0] == 1
    assert O.sample_row(x, None, 0.9999)[0] == 0
    assert O.sample_row(x, None, 0.9999, k=2)[0] == 2
    assert O.sample_row(x, None, 0.9999, p=0.5)[0] == 2       # 0.4 in front of the second token is below 0.5
    assert O.sample_row(x, None, 0.9999, p=0.0)[0] == 1
    assert O.sample_row(x, None, 0.9999, mp=0.6)[0] == 2
    assert O.sample_row(x, None, 0.9999, mp=1.0)[0] == 1
    assert O.sample_row(torch.full((3,), -math.inf), None, 0.5)[0] == 0
    assert O.sample_row(torch.zeros(4), None, 0.5)[0] == 2    # equal logits: by index
