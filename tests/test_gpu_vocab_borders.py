"""Operators along the vocabulary axis at the borders of their definitions, against the 64-bit oracle; tolerances as in test_gpu_vocab.py."""
import math

import pytest
import torch

from oracle import vocab as O
from test_gpu_vocab import DT, E24, _check_distill, _check_sample, _logits, _rel, _teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 100, 300])   # slices of an eighth and a quarter of a row, whole rows
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_with_a_few_logits_near_the_cap(tag, rows, tail):
    """Single lanes of a warp meet logits beyond three quarters of the cap (22.5 of 30) in slices long enough for batched loads; the
    first row has none, the second some in every slice, the third one alone."""
    g = torch.Generator().manual_seed(rows)
    V, K = 50304, 32
    x = _logits(g, rows, V, DT[tag])
    x.clamp_(-20.0, 20.0)
    x[1, torch.randint(0, V, (40,), generator=g)] = 27.0
    x[2, 40001] = -45.0
    values, ids, lse = _teacher(g, x[:4], K, 30.0, 1.0, tail, holes=False)
    values, ids, lse = (None if t is None else torch.cat([t, t[-1:].expand(rows - t.shape[0], *t.shape[1:])]) if rows > t.shape[0] else t for t in (values, ids, lse))
    _check_distill(x, values, ids, 30.0, 1.0, lse, torch.rand(rows, generator=g), only=slice(0, 4))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [501, 70003, 131072])
def test_sample_rows_without_a_token(tag, V):
    """Nothing but NaN, nothing but -inf, both: token 0 is drawn, on every way through the row (short ones, and beyond what 16 bits count)."""
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(V)
    x = torch.empty(5, V, dtype=dt)
    x[0] = math.nan
    x[1] = -math.inf
    x[2], x[2, ::2] = math.nan, -math.inf
    x[3], x[3, :7] = -math.inf, math.nan
    x[4] = _logits(g, 1, V, dt)[0]
    u = torch.tensor([0.9, 0.5, 0.999, 0.3, 0.5])
    for cap in (30.0, None):
        for kw in ({}, dict(p=0.95, T=0.8), dict(k=300), dict(k=1000, p=0.9, mp=0.01), dict(mp=0.1), dict(k=50), dict(k=1)):
            got = xlstm_b200.softcap_sample(x.cuda(), cap, u.cuda(), kw.get("T", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("mp", 0.0))
            assert got[:4].tolist() == [0, 0, 0, 0], kw
            assert int(got[4]) == O.sample_row(x[4], cap, u[4], **kw)[0]
        # temperature 0 is the greedy head's token: NaN is passed over, and -inf (under a cap: the value -cap) is a value like any other
        got = xlstm_b200.softcap_sample(x.cuda(), cap, u.cuda(), 0.0)
        assert got[:4].tolist() == [0, 0, 0, 7]
        if cap:
            assert torch.equal(got, xlstm_b200.softcap_argmax(x.cuda(), cap))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [40, 3001, 70003])
def test_sample_by_numbers_outside_the_unit_interval(tag, V):
    """u is clamped to [0, 1], NaN counts as 0.  Logits within [-4, 4]: every token weighs more than e^-16, so the last one kept is the
    same in any arithmetic."""
    import xlstm_b200
    g = torch.Generator().manual_seed(V)
    u = torch.tensor([math.inf, 1e30, 2.0 ** 64, 2.0 ** 21, 2.0, 1.0, math.nan, 0.0, -1e-30, -1.0, -1e30, -math.inf])
    x = (8 * torch.rand(len(u), V, generator=g) - 4).to(DT[tag])
    x[1] = 1.0
    v = u.nan_to_num(0.0, 1.0, 0.0).clamp(0.0, 1.0)
    for cap, kw in ((30.0, {}), (None, dict(T=0.5, p=0.9)), (30.0, dict(k=7)), (None, dict(k=300, p=0.8)), (30.0, dict(mp=0.3)), (None, dict(k=1)),
                    (30.0, dict(T=torch.full((len(u),), 0.7), k=torch.arange(len(u), dtype=torch.int32) * 40))):
        dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
        got = xlstm_b200.softcap_sample(x.cuda(), cap, u.cuda(), dev.get("T", 1.0), dev.get("k", 0), dev.get("p", 1.0), dev.get("mp", 0.0))
        _check_sample(x, cap, v, got=got, **kw)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [2000, 70003])
def test_sample_infinite_logits(tag, V):
    """Under a cap +inf stands at the cap like any other saturated logit; without one the +inf tokens share the row.  On every way."""
    g = torch.Generator().manual_seed(V + 1)
    x = _logits(g, 6, V, DT[tag])
    x[0], x[0, 7] = 25.0, math.inf                       # y = 20.5 for all but one of 30
    x[1, 11], x[1, 500], x[1, 900] = math.inf, 500.0, 40.0
    x[2, ::2], x[2, 3] = 1000.0, math.inf                # half of the row saturated
    x[3, 5:] = -math.inf
    x[3, :5] = torch.tensor([math.inf, 500.0, 0.0, 29.0, math.inf])
    x[4, ::3], x[4, 1] = math.nan, math.inf
    x[5, 100], x[5, 200] = math.inf, -math.inf
    u = torch.tensor([0.9, 0.6, 0.77, 0.9, 0.9999, 0.99995])
    for cap, kw in ((30.0, {}), (30.0, dict(T=8.0)), (30.0, dict(T=3.0, p=0.99)), (30.0, dict(k=40, T=20.0)), (30.0, dict(k=400, T=10.0)), (30.0, dict(mp=0.05, T=4.0)), (1.0, dict(T=0.3)),
                    (None, {}), (None, dict(k=40)), (None, dict(p=0.5)), (None, dict(mp=0.1))):
        _check_sample(x, cap, u, **kw)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [300, 20011])
def test_topk_sums_of_rows_with_nan_and_infinities(tag, V):
    """A NaN anywhere makes the log-sum-exp NaN, also in a row without a number or with +inf; without one it is -inf, +inf or a number."""
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(V)
    x = _logits(g, 7, V, dt)
    x[0] = math.nan
    x[1], x[1, 5] = -math.inf, math.nan
    x[2, 8], x[2, 9] = math.inf, math.nan
    x[3] = -math.inf
    x[4, 3] = math.inf
    x[5], x[5, 250] = math.nan, 1.0
    x[6, 2] = -math.inf
    for cap, T in ((None, 1.0), (None, 0.1), (30.0, 1.0), (30.0, 0.1)):
        values, ids, lse = xlstm_b200.softcap_topk(x.cuda(), cap, 3, T)
        for r in range(7):
            y, idx, l = O.topk_row(x[r], cap, 3, T)
            assert ids[r].tolist() == idx
            torch.testing.assert_close(values[r].cpu().double(), y, rtol=8 * E24, atol=0, equal_nan=True)
            zmax = float((y[torch.isfinite(y)].abs() / T).max()) if bool(torch.isfinite(y).any()) else 0.0   # (the terms that count)
            torch.testing.assert_close(lse[r].cpu().double(), l, rtol=E24, atol=_rel(zmax) + 64 * E24, equal_nan=True)


def test_rows_beyond_32_bits_are_refused():
    """A row length is not cut to 32 bits on its way to the kernel (2^32 + 8 tokens are not 8)."""
    import xlstm_b200
    from xlstm_b200._lib import XlError
    values, ids = torch.zeros(1, 3).cuda(), torch.zeros(1, 3, dtype=torch.int32).cuda()
    for V in (2 ** 31, 2 ** 32 + 8):
        x = torch.zeros(1, V, dtype=torch.bfloat16, device="cuda")
        for call in (lambda: xlstm_b200.softcap_sample(x, 30.0, torch.zeros(1).cuda()), lambda: xlstm_b200.softcap_topk(x, None, 3),
                     lambda: xlstm_b200.distill_topk(x, values, ids), lambda: xlstm_b200.distill_topk_grad(x, values, ids)):
            with pytest.raises(XlError, match="capacity"):
                call()
        del x


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("T", [0.3, 1.0])
def test_distill_masked_sides_under_a_cap(tag, T):
    """Under a cap -inf is -cap: a tail, or named tokens, of nothing but -inf have the mass that this says (T = 0.3: down to e^-200 of the rest)."""
    g = torch.Generator().manual_seed(3)
    for V in (40, 10007):
        x = _logits(g, 5, V, DT[tag]).clamp(-20, 20)
        values, ids, lse = _teacher(g, x, 6, 30.0, T, True, holes=False)
        named = torch.zeros(5, V, dtype=torch.bool).scatter_(1, ids.long(), True)
        x[0] = x[0].masked_fill(~named[0], -math.inf)
        x[1] = x[1].masked_fill(named[1], -math.inf)
        x[2] = -math.inf
        x[3] = x[3].masked_fill(~named[3], torch.finfo(DT[tag]).min)
        x[4] = x[4].masked_fill(~named[4], math.inf)
        _check_distill(x, values, ids, 30.0, T, lse + 0.1, None)
        _check_distill(x, values, ids, 30.0, T, None, None)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_distill_named_tokens_of_the_lowest_value(tag):
    """Without a cap: the student masks a token (the type's lowest value) that the teacher gives e^-88 / T.  p log q is a number there
    (6e-39 * 3.4e38 at T = 1), and the loss with it."""
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(4)
    x = _logits(g, 4, 700, dt, 1.0)
    ids = torch.tensor([[1, 2, 3], [5, 3, 2], [3, 3, 9], [3, 600, 601]], dtype=torch.int32)
    values = torch.tensor([[0.0, -1.0, -88.0], [1.0, -87.0, 0.0], [-88.0, -89.0, 0.0], [-100.0, 2.0, 1.0]])
    x[:, 3] = torch.finfo(dt).min
    for T in (1.0, 0.8, 1.3):
        keep = (values.double() / T - (values.double() / T).amax(-1, keepdim=True)).amin(-1) > -690.0
        assert bool(keep.all())
        for lse in (None, torch.logsumexp(values / T, -1) + 0.2):
            # (the operator's temperature is a 32-bit number; 1.3 as one is off by 2e-8, and e^(-88 / T) by 68 times that)
            T32 = float(torch.tensor(T, dtype=torch.float32))
            want, dz = O.distill(x.double(), values, ids, None, T32, lse), O.distill_grad(x.double(), values, ids, None, T32, lse)
            assert bool(torch.isfinite(want).all())
            zmax = float((x.double().masked_fill(x < -1e30, 0.0) / T).abs().max()) + 2.0 / T
            tol = T * T * (2 * (_rel(zmax) + 64 * E24) + 4 * E24 * zmax) + E24 * want.abs()
            leaf = x.cuda().requires_grad_()
            loss = xlstm_b200.distill_topk(leaf, values.cuda(), ids.cuda(), None, T, None if lse is None else lse.cuda())
            assert ((loss.detach().cpu().double() - want).abs() <= tol).all()
            loss.sum().backward()
            grad = xlstm_b200.distill_topk_grad(x.cuda(), values.cuda(), ids.cuda(), None, None, T, None if lse is None else lse.cuda())
            assert ((grad[0].cpu().double() - want).abs() <= tol).all()   # (other threads, another order of the sums)
            # (the two launches scale e_k differently, so their last bits differ: each within the gradient's tolerance, q + p + tail <= 3)
            tol = 3 * T * (2 * _rel(zmax) + 144 * E24) + (torch.finfo(dt).eps / 2 + 2 ** -23) * dz.abs()
            for got in (grad[1], leaf.grad):
                assert ((got.cpu().double() - dz).abs() <= tol).all()


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [40, 10007])
@pytest.mark.parametrize("T", [1.0, 1.8155349493026733, 4.0, 30.0])
def test_distill_tails_of_the_lowest_value(tag, V, T):
    """Without a cap: every token that is not named, or every one that is, is masked by the type's lowest value.  The masked side's own softmax is
    flat (steps of fp32 there are 2e31), its loss a number wherever 3.4e38 times its share is one."""
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(V)
    x = _logits(g, 5, V, dt, 1.0)
    ids = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(5)]).to(torch.int32)
    values = torch.randn(5, 6, generator=g)
    named = torch.zeros(5, V, dtype=torch.bool).scatter_(1, ids.long(), True)
    low = torch.finfo(dt).min
    x[0] = x[0].masked_fill(~named[0], low)                  # the tail
    x[1] = x[1].masked_fill(~named[1], low / 2)
    x[1, (~named[1]).nonzero()[::3, 0]] = low
    x[2] = x[2].masked_fill(named[2], low)                   # the named ones
    x[3] = low                                               # everything
    x[4] = x[4].masked_fill(~named[4], low)
    ids[4, 2:] = -1                                          # (some of the tail are not masked)
    T32 = float(torch.tensor(T, dtype=torch.float32))
    for lse in (None, torch.logsumexp(values / T, -1), torch.logsumexp(values / T, -1) + 0.2):
        if lse is not None:
            lse = lse.clamp(min=torch.logsumexp(values.double() / T32, -1) + 1e-6).float()   # (the entries hold a little less than everything)
        want, dz = O.distill(x.double(), values, ids, None, T32, lse), O.distill_grad(x.double(), values, ids, None, T32, lse)
        zmax = float((x.double().masked_fill(x < -1e30, 0.0) / T).abs().max()) + 4.0 / T
        # p are off by 3e-13 of themselves, and a tail of 1 - sum p = 9e-7 (1e-6 and lse's rounding, 1.2e-7) by 4e-7 of itself
        tol = T * T * (2 * (_rel(zmax) + 64 * E24) + 4 * E24 * zmax) + (4 * E24 + 4e-7) * want.abs()
        tol_grad = 3 * T * (2 * _rel(zmax) + 144 * E24) + (torch.finfo(dt).eps / 2 + 2 ** -23 + 4e-7) * dz.abs()
        dev = None if lse is None else lse.cuda()
        leaf = x.cuda().requires_grad_()
        loss = xlstm_b200.distill_topk(leaf, values.cuda(), ids.cuda(), None, T, dev)
        loss.sum().backward()
        both = xlstm_b200.distill_topk_grad(x.cuda(), values.cuda(), ids.cuda(), None, None, T, dev)
        for l, d in ((loss.detach(), leaf.grad), both):
            l, d = l.cpu().double(), d.cpu().double()
            fits = want.abs() < 3.4e38
            assert (((l - want).abs() <= tol) | (~fits & (l == math.inf))).all(), (l, want)
            assert ((d - dz).abs() <= tol_grad).all()
