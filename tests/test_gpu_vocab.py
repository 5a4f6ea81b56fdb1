"""Operators along the vocabulary axis -- softcap_sample, softcap_topk, distill_topk -- against the 64-bit oracle.

Tokens and ids are whole numbers and have to be equal.  Tolerances of the others, with e = 2^-24 (half a step of fp32):
  y = cap * tanh(x / cap): quotient and product half a step each, tanh within two steps (4 e): |dy| <= 8 e |y| with room for a
      tanh of a few steps;
  z = y / T: |dz| <= 12 e |z| (two more roundings);
  an exponential of z - c: relative error E = 2 (12 e zmax) + 4 e zmax + 16 e, the argument's roundings and the function's;
  a log-sum-exp: E + 64 e for the sum of up to 2^19 terms in blocks + e |lse|;
  a loss: T^2 W (2 (E + 64 e) + 4 e zmax);
  a gradient: weight T [ (q + p) (2 E + 128 e) s + (q + p) 16 e ] with the cap's slope s = 1 - tanh^2 <= 1 and its error, and half
      a step of the output's type.
"""
import math

import pytest
import torch

from oracle import vocab as O

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
E24 = 2.0 ** -24


def _rel(zmax):
    return 24 * E24 * zmax + 4 * E24 * zmax + 16 * E24


def _logits(g, rows, V, dt, scale=3.0):
    x = scale * torch.randn(rows, V, generator=g)
    x[:, :: max(1, V // 7)] += 5.0
    return x.to(dt)


def _check_sample(x, cap, u, T=1.0, k=0, p=1.0, mp=0.0, got=None):
    import xlstm_b200

    def dev(v):
        return v.cuda() if torch.is_tensor(v) else v

    def at(v, r):
        return float(v.reshape(-1)[r]) if torch.is_tensor(v) else v
    if got is None:
        got = xlstm_b200.softcap_sample(x.cuda(), cap, u.cuda(), temperature=dev(T), top_k=dev(k), top_p=dev(p), min_p=dev(mp))
    assert got.dtype == torch.int64 and got.shape == x.shape[:-1]
    rows, uu = x.reshape(-1, x.shape[-1]), u.reshape(-1)
    for r in range(rows.shape[0]):
        want, margin = O.sample_row(rows[r], cap, uu[r], at(T, r), int(at(k, r)), at(p, r), at(mp, r))
        assert int(got.reshape(-1)[r]) == want, (r, margin)


# ------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 2), (3, 31), (5, 257), (3, 2049), (2, 50304), (1, 70001), (300, 64)])
def test_sample_matches_oracle(tag, rows, V):
    g = torch.Generator().manual_seed(rows * 7919 + V)
    x = _logits(g, rows, V, DT[tag])
    u = torch.rand(rows, generator=g)
    for cap, kw in ((30.0, {}), (None, dict(T=0.7, k=5)), (30.0, dict(T=1.3, p=0.8)), (None, dict(mp=0.05)),
                    (10.0, dict(T=0.9, k=40, p=0.9, mp=0.01)), (30.0, dict(k=V, p=0.3)), (None, dict(k=V + 5, T=3.0))):
        _check_sample(x, cap, u, **kw)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_sample_settings_per_row(tag):
    import xlstm_b200
    g = torch.Generator().manual_seed(5)
    rows, V = 64, 4099
    x = _logits(g, rows, V, DT[tag])
    u = torch.rand(rows, generator=g)
    T = 0.3 + 1.5 * torch.rand(rows, generator=g)
    k = torch.randint(-1, 300, (rows,), generator=g, dtype=torch.int32)
    k[::5] = 0
    p, mp = 1.2 * torch.rand(rows, generator=g), 0.2 * torch.rand(rows, generator=g)
    mp[::3] = 0.0
    _check_sample(x, 30.0, u, T, k, p, mp)
    _check_sample(x.reshape(4, 16, V), 30.0, u.reshape(4, 16), T.reshape(4, 16), k.long(), p, mp.double())   # other shapes and types of the settings
    # rows with temperature 0 take the greedy head's token, whose ties are those of the rounded cap
    T0 = T.clone()
    T0[::2] = 0.0
    got = xlstm_b200.softcap_sample(x.cuda() * 12, 30.0, u.cuda(), temperature=T0.cuda())
    greedy = xlstm_b200.softcap_argmax(x.cuda() * 12, 30.0)
    assert torch.equal(got[::2], greedy[::2])
    assert torch.equal(xlstm_b200.softcap_sample(x.cuda() * 12, 30.0, u.cuda(), temperature=0.0), greedy)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_sample_ties_and_borders(tag):
    """Whole-number logits and all-equal rows: ranks inside equals, u at exact borders, the ends of u."""
    g = torch.Generator().manual_seed(8)
    dt = DT[tag]
    x = torch.randint(-3, 4, (6, 1000), generator=g).to(dt)
    x[1] = 0.0
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0
    u = torch.tensor([0.999, 0.5, 0.25, 0.0, 1.0 - 2.0 ** -24, 0.123])
    for kw in ({}, dict(k=7), dict(k=333, p=0.77), dict(p=0.01), dict(mp=1.0), dict(p=0.0), dict(T=1e-3), dict(T=50.0)):
        _check_sample(x, None, u, **kw)
        _check_sample(x, 30.0, u, **kw)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_sample_long_rows_of_every_kind(tag):
    """Rows that fill lists, counters and the table of values: ties by the thousand, more tokens kept than a list holds, many
    distinct values, equal logits beyond 16 bits of count, masks and NaN among them -- few rows (cut over blocks) and several."""
    g = torch.Generator().manual_seed(14)
    dt = DT[tag]
    V = 70003
    x = _logits(g, 8, V, dt)
    x[1] = 2.5                                                   # 70 003 equal logits
    x[2] = torch.randint(-2, 3, (V,), generator=g).to(dt)        # five values
    x[3] = torch.randint(0, 2 ** 15, (V,), generator=g).to(torch.int16).view(torch.bfloat16).nan_to_num(0.0, 0.0, 0.0).clamp(max=50.0).to(dt)   # thousands of values
    x[4, 3:] = -math.inf
    x[5, ::2] = math.nan
    x[6] = 0.01 * torch.randn(V, generator=g)                    # nearly flat
    x[7, 40000:] = torch.finfo(dt).min
    u = torch.rand(8, generator=g)
    for cap, kw in ((30.0, dict(k=50)), (None, dict(k=50, p=0.9)), (30.0, dict(k=400)), (None, dict(k=5000, p=0.7, mp=0.001)), (30.0, dict(mp=0.9)), (None, dict(mp=1e-6)),
                    (30.0, dict(p=0.95, T=0.6)), (None, {}), (30.0, dict(k=1)), (30.0, dict(k=256)), (30.0, dict(k=257))):
        _check_sample(x, cap, u, **kw)
        _check_sample(x[:2], cap, u[:2], **kw)
    _check_sample(x[:, :20011], 30.0, u, torch.full((8,), 0.9), torch.tensor([50, 50, 0, 0, 300, 7, 0, 1000]), torch.tensor([1.0, 0.9, 1.0, 0.5, 1.0, 1.0, 0.3, 0.8]),
                  torch.tensor([0.0, 0.0, 0.5, 0.0, 0.0, 0.1, 0.0, 0.2]))


def test_rows_beyond_the_grid_and_elements_beyond_32_bits():
    import xlstm_b200
    g = torch.Generator().manual_seed(15)
    rows = 70001
    x = torch.randn(rows, 12, generator=g)
    u = torch.rand(rows, generator=g)
    pick = [0, 65535, 65536, 70000]
    got = xlstm_b200.softcap_sample(x.cuda(), None, u.cuda(), top_k=5)
    _check_sample(x[pick], None, u[pick], k=5, got=got[pick])
    values, ids, lse = xlstm_b200.softcap_topk(x.cuda(), None, 3)
    for r in pick:
        assert ids[r].tolist() == O.topk_row(x[r], None, 3)[1]
    loss, grad = xlstm_b200.distill_topk_grad(x.cuda(), values, ids)
    torch.testing.assert_close(loss[pick].cpu().double(), O.distill(x[pick].double(), values[pick].cpu(), ids[pick].cpu()), rtol=1e-5, atol=1e-6)
    del x, got, grad
    big = torch.zeros(42800, 50304, dtype=torch.bfloat16, device="cuda")     # 2.15e9 elements
    tail = _logits(g, 2, 50304, torch.bfloat16)
    big[-2:] = tail.cuda()
    values, ids, lse = xlstm_b200.softcap_topk(big, 30.0, 8)
    alone = xlstm_b200.softcap_topk(tail.cuda(), 30.0, 8)
    assert torch.equal(ids[-2:], alone[1]) and torch.equal(values[-2:], alone[0]) and ids[0].tolist() == list(range(8))
    loss, grad = xlstm_b200.distill_topk_grad(big, values, ids, None, 30.0, 1.0, lse)
    one, want = xlstm_b200.distill_topk_grad(tail.cuda(), *alone[:2], None, 30.0, 1.0, alone[2])
    torch.testing.assert_close(loss[-2:], one, rtol=1e-4, atol=1e-6)
    torch.testing.assert_close(grad[-2:].float(), want.float(), rtol=2 ** -6, atol=1e-7)   # (another cut of the row: a bf16 step here and there)
    u = torch.full((42800,), 0.5, device="cuda")
    assert torch.equal(xlstm_b200.softcap_sample(big, 30.0, u, 0.9, 40)[-2:], xlstm_b200.softcap_sample(tail.cuda(), 30.0, u[:2], 0.9, 40))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_sample_masked_rows(tag):
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(9)
    x = _logits(g, 8, 501, dt)
    low = torch.finfo(dt).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :500] = -math.inf                 # one token left
    x[3, 1:] = low                         # the type's lowest value as a mask
    x[4, ::2] = math.nan
    x[5, 17] = x[5, 400] = math.inf        # two tokens share the row
    x[6] = low
    x[7, 100:] = -math.inf
    u = torch.rand(8, generator=g)
    few = torch.full((3, 30000), -math.inf).to(dt)      # constrained decoding: fewer tokens allowed than top_k
    few[:, ::2999] = _logits(g, 3, 11, dt)
    few[1] = low
    _check_sample(few, 30.0, u[:3], k=50)
    _check_sample(few, None, u[:3], k=12, p=0.9)
    for cap in (None, 30.0):
        for kw in ({}, dict(k=3), dict(p=0.9, T=0.5), dict(mp=0.3), dict(T=math.inf) if cap is None else {}):
            if "T" in kw and kw["T"] == math.inf:   # (as a number it is refused; a tensor's values are not looked at)
                got = xlstm_b200.softcap_sample(x[2:3].cuda(), cap, u[2:3].cuda(), temperature=torch.full((1,), math.inf).cuda())
                assert int(got) == 500
                continue
            _check_sample(x, cap, u, **kw)
    big = xlstm_b200.softcap_sample(x[7:].cuda(), None, torch.tensor([2.0]).cuda())   # u outside [0, 1) is clamped
    assert int(big) == O.sample_row(x[7], None, 1.0)[0]
    assert int(xlstm_b200.softcap_sample(x[7:].cuda(), None, torch.tensor([math.nan]).cuda())) == O.order(x[7])[0]


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_sample_and_topk_read_strided_rows_in_place(tag):
    import xlstm_b200
    g = torch.Generator().manual_seed(10)
    wide = _logits(g, 5, 3 * 1003, DT[tag])
    x = wide[:, 1003:2006]                 # rows that start on odd addresses
    u = torch.rand(5, generator=g)
    dev = wide.cuda()[:, 1003:2006]
    _check_sample(x, 30.0, u, T=0.8, k=100, p=0.95, got=xlstm_b200.softcap_sample(dev, 30.0, u.cuda(), 0.8, 100, 0.95))
    _check_sample(x, 30.0, u, p=0.9, got=xlstm_b200.softcap_sample(dev, 30.0, u.cuda(), top_p=0.9))
    a, b = xlstm_b200.softcap_topk(dev, 30.0, 50), xlstm_b200.softcap_topk(x.contiguous().cuda(), 30.0, 50)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # how a row lies on 16-byte boundaries sets the order of its sum: the same positive terms, each sum of 1003 within
    # 64 e of their exact total (every partial sum rounds by e of at most the total, in chains of at most 1003 / 256 * 4 + 16 < 64
    # additions), and e |lse| for the result's own rounding, on either side
    assert ((a[2] - b[2]).abs() <= 128 * E24 + 2 * E24 * b[2].abs()).all()
    row = dev[:1].expand(4, 1003)
    assert torch.equal(xlstm_b200.softcap_topk(row, None, 3)[1], xlstm_b200.softcap_topk(dev[:1], None, 3)[1].expand(4, 3))
    assert xlstm_b200.softcap_sample(dev[0], None, u[:1].cuda()).shape == ()   # one row without a batch dimension


# ------------------------------------------------------------------------------------------------ top logits
@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 33, 33), (5, 257, 20), (4, 2049, 1024), (2, 50304, 64), (1, 70001, 200), (300, 640, 1)])
def test_topk_matches_oracle(tag, rows, V, k):
    import xlstm_b200
    g = torch.Generator().manual_seed(rows * 31 + V + k)
    x = _logits(g, rows, V, DT[tag])
    for cap, T in ((30.0, 1.0), (None, 2.5)):
        values, ids, lse = xlstm_b200.softcap_topk(x.cuda(), cap, k, T)
        assert values.shape == ids.shape == (rows, k) and lse.shape == (rows,) and ids.dtype == torch.int32
        for r in range(min(rows, 8)):
            y, idx, l = O.topk_row(x[r], cap, k, T)
            assert ids[r].tolist() == idx
            assert ((values[r].cpu().double() - y).abs() <= 8 * E24 * y.abs()).all()
            zmax = float((O.cap64(x[r], cap) / T).abs().max())
            assert abs(float(lse[r]) - float(l)) <= _rel(zmax) + 64 * E24 + E24 * abs(float(l))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_topk_ties_masks_and_crowds(tag):
    """Equal logits (whole rows of them), masked tokens, infinities and NaN, and rows whose largest sit side by side."""
    import xlstm_b200
    dt = DT[tag]
    g = torch.Generator().manual_seed(12)
    V = 20011
    x = _logits(g, 9, V, dt)
    x[0] = 1.5
    x[1] = torch.randint(0, 2, (V,), generator=g).to(dt)
    x[2] = -math.inf
    x[3, 5:] = -math.inf
    x[4, ::3] = math.nan
    x[5] = torch.arange(V).to(dt)
    x[6, 8000:8600] += 100.0
    x[7, 77] = math.inf
    x[8] = torch.finfo(dt).min
    for k in (1, 64, 300, 1000):
        values, ids, lse = xlstm_b200.softcap_topk(x.cuda(), None, k)
        for r in range(9):
            y, idx, l = O.topk_row(x[r], None, k)
            assert ids[r].tolist() == idx, r
            torch.testing.assert_close(values[r].cpu().double(), y, rtol=0, atol=0, equal_nan=True)   # without a cap the logits themselves
            if math.isnan(float(l)):
                assert math.isnan(float(lse[r]))
            elif math.isinf(float(l)):
                assert float(lse[r]) == float(l)
            else:
                zmax = float(y[torch.isfinite(y)].abs().max())   # (the terms that count)
                assert abs(float(lse[r]) - float(l)) <= _rel(zmax) + 64 * E24 + E24 * abs(float(l))


# ------------------------------------------------------------------------------------------------ distillation
def _teacher(g, x, K, cap, T, tail, holes=True):
    """Entries of a teacher near the student: ids, capped values, its log-sum-exp."""
    rows, V = x.shape
    t = O.cap64(x.double() + torch.randn(x.shape, generator=g), cap)
    values, ids = t.topk(K, dim=-1)
    lse = torch.logsumexp(t / T, -1).float() if tail else None
    values, ids = values.float(), ids.to(torch.int32)
    if holes:
        drop = torch.rand(ids.shape, generator=g) < 0.2
        drop[:, 0] = False
        ids = torch.where(drop, -1, ids)
        if rows > 2:
            ids[2] = -1
    return values, ids, lse


def _check_distill(x, values, ids, cap, T, lse, weight, only=None):
    import xlstm_b200
    from xlstm_b200 import ops
    rows, V = x.shape
    r = slice(None) if only is None else only
    dev = [None if t is None else t.cuda() for t in (x, values, ids, lse, weight)]
    xd, vd, idd, ld, wd = dev
    want = O.distill(x[r].double(), values[r], ids[r], cap, T, None if lse is None else lse[r])
    dz = O.distill_grad(x[r].double(), values[r], ids[r], cap, T, None if lse is None else lse[r])
    wr = torch.ones(rows).double()[r] if weight is None else weight.double()[r]
    z = O.cap64(x[r], cap) / T
    zmax = float(z[torch.isfinite(z)].abs().max()) + float((values[r][torch.isfinite(values[r])].abs() / T).max())
    q = torch.softmax(z, -1)
    P = torch.zeros_like(q)
    for i in range(q.shape[0]):
        used = ids[r][i] >= 0
        if bool(used.any()):
            e = values[r][i][used].double() / T
            P[i].index_add_(0, ids[r][i][used].long(), torch.exp(e - (torch.logsumexp(e, 0) if lse is None else float(lse[r][i]))))
    share = q + P
    tail = torch.where(P > 0, 0.0, q)   # p_tail's part of a tail gradient: at most tail / sum(tail)
    share = share + tail / tail.sum(-1, keepdim=True).clamp(min=1e-300)
    E = _rel(zmax)
    tol_loss = T * T * 1.001 * (2 * (E + 64 * E24) + 4 * E24 * zmax)
    half = torch.finfo(x.dtype).eps / 2
    tol_grad = wr[:, None] * T * share * (2 * E + 128 * E24 + 16 * E24) + (half + 2 ** -23) * (wr[:, None] * dz).abs()

    loss = xlstm_b200.distill_topk(xd, vd, idd, cap, T, ld)
    assert loss.shape == (rows,) and loss.dtype == torch.float32
    assert ((loss[r].cpu().double() - want).abs() <= tol_loss + E24 * want.abs()).all()
    loss2, grad = xlstm_b200.distill_topk_grad(xd, vd, idd, wd, cap, T, ld)
    assert ((loss2[r].cpu().double() - want).abs() <= tol_loss + E24 * want.abs()).all()
    assert grad.dtype == x.dtype and grad.shape == x.shape
    assert ((grad[r].cpu().double() - wr[:, None] * dz).abs() <= tol_grad).all()
    leaf = xd.clone().requires_grad_()
    total = ops.distill_topk(leaf, vd, idd, cap, T, ld)
    (total if wd is None else total * wd).sum().backward()
    assert ((leaf.grad[r].cpu().double() - wr[:, None] * dz).abs() <= tol_grad).all()
    xlstm_b200.check_device_status()


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (4, 9, 9), (3, 33, 4), (7, 257, 16), (3, 2049, 200), (5, 10007, 64), (3, 6000, 1024), (300, 70, 3)])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_matches_oracle(tag, rows, V, K, tail):
    g = torch.Generator().manual_seed(rows * 101 + V + K)
    x = _logits(g, rows, V, DT[tag])
    for cap, T, w in ((30.0, 1.0, True), (None, 2.0, False), (8.0, 0.6, True)):
        values, ids, lse = _teacher(g, x, K, cap, T, tail)
        _check_distill(x, values, ids, cap, T, lse, torch.rand(rows, generator=g) if w else None, only=slice(0, 8))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("V", [50304, 50303, 131075])
def test_distill_long_rows(tag, V):
    g = torch.Generator().manual_seed(V)
    x = _logits(g, 3, V, DT[tag])
    values, ids, lse = _teacher(g, x, 64, 30.0, 1.0, True)
    _check_distill(x, values, ids, 30.0, 1.0, lse, torch.rand(3, generator=g))
    _check_distill(x, values, ids, None, 1.0, None, None)


@pytest.mark.parametrize("cap", [0.05, 0.125, 1024.0, 5e4])
def test_caps_of_every_size(cap):
    """Logits below, near and far beyond the cap; caps whose powers leave fp32."""
    import xlstm_b200
    g = torch.Generator().manual_seed(40)
    for scale in (0.1, 0.6, 2.0, 30.0):
        x = cap * scale * torch.randn(4, 3001, generator=g)
        T = max(1e-2, cap * 0.1)          # (weights spread over a few hundred tokens)
        _check_sample(x, cap, torch.rand(4, generator=g), T=T, p=0.9)
        values, ids, lse = _teacher(g, x, 16, cap, T, True)
        _check_distill(x, values, ids, cap, T, lse, None)
        got, at, total = xlstm_b200.softcap_topk(x.cuda(), cap, 20, T)
        for r in range(4):
            y, idx, l = O.topk_row(x[r], cap, 20, T)
            assert at[r].tolist() == idx and ((got[r].cpu().double() - y).abs() <= 8 * E24 * y.abs()).all()
            assert abs(float(total[r]) - float(l)) <= _rel(float((O.cap64(x[r], cap) / T).abs().max())) + 64 * E24 + E24 * abs(float(l))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_distill_extremes(tag):
    """Tokens named twice and often, masked student tokens, entries without mass, far-away tails, all tokens named."""
    g = torch.Generator().manual_seed(21)
    dt = DT[tag]
    x = _logits(g, 8, 40, dt)
    values, ids, lse = _teacher(g, x, 12, None, 1.0, True, holes=False)
    ids[0, 1] = ids[0, 4] = ids[0, 9] = ids[0, 2]
    ids[1] = 7
    lse[0] += 2.0                                # (twice-named entries must not hold more than everything)
    lse[1] += 4.0
    values[2, 5:] = -math.inf
    masked = [j for j in range(40) if j not in ids[3].tolist()]
    x[3, masked[:5]] = -math.inf                 # masked tokens in the student's tail
    x[4, ids[4].long()] += 60.0                  # the named tokens hold all but e^-60 of the student
    lse[4] += 0.5
    x[5] -= 200.0                                # no sum may overflow or underflow
    x[6] += 200.0
    for T, l in ((1.0, lse), (1.0, None), (0.25, None)):
        _check_distill(x, values, ids, None, T, l, None)
    # the same among long rows, whose slices do not all hold the token
    xl, il = torch.cat([x] * 260, 1)[:, :10301], ids.clone()
    il[2:, 3] += 9000
    il[5, 4] = il[5, 3]
    _check_distill(xl, values, il, None, 1.0, None, None)
    # every token named: the tail counts as empty whatever the teacher's sum says
    full = torch.arange(40, dtype=torch.int32).repeat(8, 1)
    _check_distill(x[5:], values.new_zeros(3, 40), full[5:], None, 1.0, torch.full((3,), math.log(40.0) + 0.01), None)
    # int64 ids, half-precision values
    import xlstm_b200
    a = xlstm_b200.distill_topk_grad(x[5:].cuda(), values[5:].bfloat16().cuda(), ids[5:].long().cuda())
    b = xlstm_b200.distill_topk_grad(x[5:].cuda(), values[5:].bfloat16().float().cuda(), ids[5:].cuda())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_distill_rows_of_the_lowest_value(tag):
    """The type's lowest value as a mask: of a whole row (its softmax is flat), of all but a few tokens, of the whole tail."""
    import xlstm_b200
    dt = DT[tag]
    low = torch.finfo(dt).min
    x = torch.full((3, 40), low).to(dt)
    x[1, :10] = 1.0
    x[2, :2] = 0.0
    ids = torch.tensor([[0, 1]] * 3, dtype=torch.int32)
    values = torch.zeros(3, 2)
    for lse, want in ((None, [math.log(20.0), math.log(5.0), 0.0]), (torch.full((3,), math.log(2.0)), [math.log(20.0), math.log(5.0), 0.0])):
        for T in (1.0, 0.5):
            tl = None if lse is None else lse.cuda()
            loss, grad = xlstm_b200.distill_topk_grad(x.cuda(), values.cuda(), ids.cuda(), None, None, T, tl)
            n = 3 if lse is None else 2   # (float32(log 2) leaves 1 - 2 exp(-log 2) = 1.9e-9 to a tail at -3.4e38: the third loss is 6e29 or beyond)
            assert (loss[:n].cpu() / T ** 2 - torch.tensor(want)[:n]).abs().max() < 1e-6
            assert lse is None or float(loss[2]) > 1e29
            flat = torch.zeros(3, 40)
            flat[0], flat[1, :10], flat[2, :2] = 1 / 40, 1 / 10, 1 / 2
            flat[:, :2] -= 0.5
            assert (grad.float().cpu() / T - flat).abs().max() <= 2.0 ** -8 * 0.5
            leaf = x.cuda().requires_grad_()
            xlstm_b200.distill_topk(leaf, values.cuda(), ids.cuda(), None, T, tl).sum().backward()
            assert torch.equal(leaf.grad, grad)


def test_distill_masked_named_token_costs_infinity():
    import xlstm_b200
    x = torch.zeros(2, 8, device="cuda")
    x[:, 3] = -math.inf
    ids = torch.tensor([[3, 1], [3, 1]], dtype=torch.int32, device="cuda")
    values = torch.tensor([[0.0, 0.0], [-math.inf, 0.0]], device="cuda")
    loss, grad = xlstm_b200.distill_topk_grad(x, values, ids)
    assert float(loss[0]) == math.inf                                   # mass where the student has none
    assert abs(float(loss[1]) - math.log(7.0)) < 1e-6                   # no mass there: 0 log 0 = 0
    want = torch.full((8,), 1 / 7.0)
    want[3], want[1] = 0.0, 1 / 7.0 - 1
    assert (grad[1].cpu() - want).abs().max() < 1e-6
    want[3], want[1] = -0.5, 1 / 7.0 - 0.5
    assert (grad[0].cpu() - want).abs().max() < 1e-6


def test_distill_reports_ids_beyond_the_vocabulary():
    import xlstm_b200
    x = torch.randn(2, 50, generator=torch.Generator().manual_seed(1)).cuda()
    values = torch.zeros(2, 3).cuda()
    ids = torch.tensor([[1, 2, 50], [1, 2, 2 ** 30]], dtype=torch.int32).cuda()
    loss, grad = xlstm_b200.distill_topk_grad(x, values, ids)
    with pytest.raises(RuntimeError, match="status 4"):
        xlstm_b200.check_device_status()
    xlstm_b200.check_device_status()
    ok = xlstm_b200.distill_topk_grad(x, values, ids.masked_fill(ids >= 50, -1))
    assert torch.equal(loss, ok[0]) and torch.equal(grad, ok[1])


def test_distill_gradient_against_differences():
    """fp32, V = 24: the loss is good to 64 e ~ 4e-6 absolute, so central differences with h = 1e-2 to 4e-4 + h^2 / 6 * third
    derivative (below 1): 5e-4."""
    import xlstm_b200
    g = torch.Generator().manual_seed(4)
    x = _logits(g, 2, 24, torch.float32, 1.0)
    values, ids, lse = _teacher(g, x, 5, 5.0, 1.5, True, holes=False)
    _, grad = xlstm_b200.distill_topk_grad(x.cuda(), values.cuda(), ids.cuda(), None, 5.0, 1.5, lse.cuda())
    h = 1e-2
    pert = torch.cat([x[:1] + h * torch.eye(24), x[:1] - h * torch.eye(24)])
    l = xlstm_b200.distill_topk(pert.cuda(), values[:1].repeat(48, 1).cuda(), ids[:1].repeat(48, 1).cuda(), 5.0, 1.5, lse[:1].repeat(48).cuda()).cpu()
    assert ((l[:24] - l[24:]) / (2 * h) - grad[0].cpu()).abs().max() < 5e-4


def test_distill_weights_of_every_layout():
    import xlstm_b200
    from xlstm_b200 import ops
    g = torch.Generator().manual_seed(6)
    x = _logits(g, 12, 130, torch.float32)
    values, ids, lse = (t.cuda() for t in _teacher(g, x, 6, 30.0, 1.0, True))
    w = torch.rand(24, generator=g).cuda()
    base = xlstm_b200.distill_topk_grad(x.cuda(), values, ids, w[::2].contiguous(), 30.0, 1.0, lse)
    strided = xlstm_b200.distill_topk_grad(x.cuda(), values, ids, w[::2], 30.0, 1.0, lse)
    assert torch.equal(base[1], strided[1])
    shaped = xlstm_b200.distill_topk_grad(x.cuda().reshape(3, 4, 130), values.reshape(3, 4, 6), ids.reshape(3, 4, 6),
                                          w[::2].reshape(4, 3).t().contiguous().t().reshape(3, 4), 30.0, 1.0, lse.reshape(3, 4))
    assert torch.equal(base[1], shaped[1].reshape(12, 130)) and shaped[0].shape == (3, 4)
    one = xlstm_b200.distill_topk_grad(x.cuda(), values, ids, torch.tensor(0.25).cuda().expand(12), 30.0, 1.0, lse)
    leaf = x.cuda().reshape(3, 4, 130).requires_grad_()
    (0.25 * ops.distill_topk(leaf, values.reshape(3, 4, 6), ids.reshape(3, 4, 6), 30.0, 1.0, lse.reshape(3, 4))).sum().backward()
    torch.testing.assert_close(leaf.grad.reshape(12, 130), one[1], rtol=1e-5, atol=1e-8)
    leaf.grad = None
    ops.distill_topk(leaf, values.reshape(3, 4, 6), ids.reshape(3, 4, 6), 30.0, 1.0, lse.reshape(3, 4)).mean().backward()
    torch.testing.assert_close(leaf.grad.reshape(12, 130) * 3, one[1], rtol=1e-5, atol=1e-8)
    # rows of a wider matrix on odd addresses
    wide = torch.zeros(12, 391).cuda()
    wide[:, 131:261] = x.cuda()
    cut = xlstm_b200.distill_topk_grad(wide[:, 131:261], values, ids, w[::2], 30.0, 1.0, lse)
    torch.testing.assert_close(cut[1], base[1], rtol=1e-4, atol=1e-7)


# ------------------------------------------------------------------------------------------------ streams, graphs, devices, refusals
def test_vocab_operators_on_another_stream_and_in_graphs():
    import xlstm_b200
    from xlstm_b200 import ops
    g = torch.Generator().manual_seed(30)
    x = _logits(g, 6, 5003, torch.bfloat16).cuda()
    y = _logits(g, 6, 5003, torch.bfloat16).cuda()
    u = torch.rand(6, generator=g).cuda()
    vals, ids, lse = xlstm_b200.softcap_topk(y, 30.0, 20)

    def everything(a):
        leaf = a.detach().requires_grad_()
        loss = ops.distill_topk(leaf, vals, ids, 30.0, 1.0, lse)
        return (xlstm_b200.softcap_sample(a, 30.0, u, 0.9, 50, 0.9), xlstm_b200.softcap_sample(a, 30.0, u, 0.9, 0, 0.9),
                *xlstm_b200.softcap_topk(a, 30.0, 20), loss.detach(), *torch.autograd.grad(loss.sum(), leaf),
                *xlstm_b200.distill_topk_grad(a, vals, ids, None, 30.0, 1.0, lse))
    want_x, want_y = everything(x), everything(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want_x))
    buf = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(buf)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):     # two captured graphs, alive at once, replayed side by side
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(everything(buf))
        graphs.append(gr)
    for src, want in ((y, want_y), (x, want_x)):
        buf.copy_(src)
        torch.cuda.synchronize()
        s = [torch.cuda.Stream(), torch.cuda.Stream()]
        for gr, st in zip(graphs, s):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_distill_backward_in_a_graph():
    """Captured behind an eager pass over the same leaf, whose own graph is gone by then (PyTorch ties a leaf's accumulation node to the
    stream it was made on and invalidates a capture that meets an older one)."""
    from xlstm_b200 import ops
    g = torch.Generator().manual_seed(33)
    leaf = _logits(g, 4, 3001, torch.float32).cuda().requires_grad_()
    values, ids, lse = (t.cuda() for t in _teacher(g, leaf.detach().cpu(), 8, 30.0, 1.0, True))
    want, = torch.autograd.grad(ops.distill_topk(leaf, values, ids, 30.0, 1.0, lse).mean(), leaf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ops.distill_topk(leaf, values, ids, 30.0, 1.0, lse).mean(), leaf)
    got.zero_()
    graph.replay()
    assert torch.equal(got, want)
    ops.distill_topk(leaf, values, ids, 30.0, 1.0, lse).mean().backward()   # and eager again
    assert torch.equal(leaf.grad, want)


def test_vocab_operators_give_the_same_bits_again():
    import xlstm_b200
    g = torch.Generator().manual_seed(31)
    x = _logits(g, 40, 9001, torch.float32).cuda()
    u = torch.rand(40, generator=g).cuda()
    vals, ids, lse = xlstm_b200.softcap_topk(x, 30.0, 100)
    ids[:, 3] = ids[:, 0]
    ids[:, 7] = ids[:, 0]
    runs = [(xlstm_b200.softcap_sample(x, 30.0, u, 1.0, 0, 0.95), *xlstm_b200.softcap_topk(x, 30.0, 100),
             *xlstm_b200.distill_topk_grad(x, vals, ids, None, 30.0, 1.0, lse)) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_vocab_operators_on_no_rows():
    import xlstm_b200
    x, u = torch.zeros(0, 10).cuda(), torch.zeros(0).cuda()
    assert xlstm_b200.softcap_sample(x, 30.0, u).shape == (0,)
    values, ids, lse = xlstm_b200.softcap_topk(x, None, 4)
    assert values.shape == ids.shape == (0, 4) and lse.shape == (0,)
    leaf = x.requires_grad_()
    loss = xlstm_b200.distill_topk(leaf, values, ids, None, 1.0, lse)
    loss.sum().backward()
    assert loss.shape == (0,) and leaf.grad.shape == (0, 10)
    assert xlstm_b200.distill_topk_grad(x, values, ids, lse)[1].shape == (0, 10)


def test_vocab_refusals():
    import xlstm_b200
    from xlstm_b200._lib import XlError
    x, u = torch.zeros(2, 16).cuda(), torch.zeros(2).cuda()
    values, ids = torch.zeros(2, 3).cuda(), torch.zeros(2, 3, dtype=torch.int32).cuda()
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.5), dict(top_p=math.nan), dict(min_p=-0.1),
                dict(temperature=u[:1]), dict(top_k=u), dict(top_p=ids[:, 0])):
        with pytest.raises(ValueError):
            xlstm_b200.softcap_sample(x, 30.0, u, **bad)
    for cap in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="cap"):
            xlstm_b200.softcap_sample(x, cap, u)
    for call in (lambda: xlstm_b200.softcap_sample(x.half(), None, u), lambda: xlstm_b200.softcap_sample(x, None, u[:1]), lambda: xlstm_b200.softcap_sample(x, None, u.double()),
                 lambda: xlstm_b200.softcap_sample(x[:, :0], None, u), lambda: xlstm_b200.softcap_sample(x, None, u.cpu()),
                 lambda: xlstm_b200.softcap_topk(x, None, 0), lambda: xlstm_b200.softcap_topk(x, None, 17), lambda: xlstm_b200.softcap_topk(x, None, 3, 0.0),
                 lambda: xlstm_b200.softcap_topk(x.int(), None, 3),
                 lambda: xlstm_b200.distill_topk(x, values, ids.float()), lambda: xlstm_b200.distill_topk(x, values[:1], ids[:1]),
                 lambda: xlstm_b200.distill_topk(x, values, ids[:, :2]), lambda: xlstm_b200.distill_topk(x, values[:, :0], ids[:, :0]),
                 lambda: xlstm_b200.distill_topk(x, values, ids, temperature=0.0), lambda: xlstm_b200.distill_topk(x, values, ids, teacher_lse=u[:1]),
                 lambda: xlstm_b200.distill_topk_grad(x, values, ids, u[:1]), lambda: xlstm_b200.distill_topk(x.half(), values, ids)):
        with pytest.raises(ValueError):
            call()
    wide = torch.zeros(1, 2048).cuda()
    with pytest.raises(XlError, match="capacity"):
        xlstm_b200.softcap_topk(wide, None, 1025)
    with pytest.raises(XlError, match="capacity"):
        xlstm_b200.distill_topk(wide, torch.zeros(1, 1025).cuda(), torch.zeros(1, 1025, dtype=torch.int32).cuda())
    with pytest.raises(XlError, match="capacity"):
        xlstm_b200.softcap_sample(torch.zeros(1, 2 ** 18 + 1).cuda(), None, u[:1])
