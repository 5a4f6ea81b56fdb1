"""Workloads of the operators on a model's vocabulary axis: sampling, top logits, distillation from a teacher's top logits.

`listed()` names the standing cases, `draw(rng)` gives further ones of the same ranges.  A case is a dict of plain values:

  op             entry point
  sample         ops.softcap_sample: tokens from temperature, top-k, top-p, min-p and given uniform numbers
  topk           ops.softcap_topk: the k largest capped logits of every row, their ids, the row's log-sum-exp
  distill        ops.distill_topk: loss of every row
  distill_train  ops.distill_topk and its backward pass through autograd
  distill_grad   ops.distill_topk_grad: losses and the weighted gradient of the logits in one call

Logits ~ N(0, 2.5) with a few tokens per row lifted by up to 14, as a trained head's rows look (most of the mass on tens of
tokens); a teacher's logits are the student's plus N(0, 1).  With `own` the framework's kernels run, without it the same
operators in elementary torch operations.
"""
import math

import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    V = 50304   # vocabulary of the 7B-shaped model
    return [
        # a few interactive streams with one setting for all: latency of one call behind the decode step
        dict(name="sample_8_streams", op="sample", rows=8, V=V, dtype="bf16", cap=30.0, mixed=False, T=0.8, k=0, p=0.95, mp=0.0),
        # the common top-k setting for a middling batch
        dict(name="sample_64_top_k", op="sample", rows=64, V=V, dtype="bf16", cap=30.0, mixed=False, T=0.7, k=50, p=1.0, mp=0.0),
        # a full serving batch, every slot with its own settings
        dict(name="sample_256_slots", op="sample", rows=256, V=V, dtype="bf16", cap=30.0, mixed=True, T=1.0, k=0, p=1.0, mp=0.0),
        # a small fp32 model without a cap, odd vocabulary
        dict(name="sample_fp32_odd", op="sample", rows=5, V=2049, dtype="f32", cap=0.0, mixed=False, T=1.3, k=40, p=0.9, mp=0.02),
        # a teacher's top logits behind single tokens
        dict(name="topk_16_rows", op="topk", rows=16, V=V, dtype="bf16", cap=30.0, k=32, T=1.0),
        # a teacher scoring a prompt of 4096 tokens
        dict(name="topk_4096_tokens", op="topk", rows=4096, V=V, dtype="bf16", cap=30.0, k=64, T=1.0),
        # an fp32 teacher, many entries, odd sizes, softened
        dict(name="topk_fp32_odd", op="topk", rows=301, V=10007, dtype="f32", cap=30.0, k=200, T=2.0),
        # evaluation: losses only, some rows and entries unused
        dict(name="distill_loss_fp32_odd", op="distill", rows=515, V=10007, dtype="f32", cap=0.0, k=50, T=2.0, tail=False, holes=True),
        # evaluation of a bf16 student
        dict(name="distill_loss", op="distill", rows=2048, V=V, dtype="bf16", cap=30.0, k=64, T=1.0, tail=True, holes=False),
        # a training step through autograd
        dict(name="distill_train", op="distill_train", rows=2048, V=V, dtype="bf16", cap=30.0, k=64, T=1.0, tail=True, holes=True),
        # a small micro-batch whose loss weights are known
        dict(name="distill_grad_64", op="distill_grad", rows=64, V=V, dtype="bf16", cap=30.0, k=16, T=2.0, tail=False, holes=False),
        # a training step of 4096 tokens whose loss weights are known
        dict(name="distill_grad_4096", op="distill_grad", rows=4096, V=V, dtype="bf16", cap=30.0, k=64, T=1.0, tail=True, holes=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "sample", "topk", "topk", "distill", "distill_train", "distill_grad", "distill_grad"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    cap = rng.choice([30.0, 30.0, 0.0])
    V = rng.choice([50304, 50304, 2048, _log(rng, 600, 131072), _log(rng, 600, 131072)])
    rows = _log(rng, 1, min(512 if op == "sample" else 4096, 2048 * 50304 // V // (2 if dtype == "f32" else 1)))
    if op == "sample":
        return dict(op=op, rows=rows, V=V, dtype=dtype, cap=cap, mixed=rng.random() < 0.4, T=round(rng.uniform(0.3, 1.5), 2),
                    k=rng.choice([0, 0, _log(rng, 1, 500)]), p=rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
                    mp=rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 3)]))
    k = _log(rng, 1, 256)
    T = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 4.0), 2)])
    if op == "topk":
        return dict(op=op, rows=rows, V=V, dtype=dtype, cap=cap, k=k, T=T)
    return dict(op=op, rows=rows, V=V, dtype=dtype, cap=cap, k=k, T=T, tail=rng.random() < 0.5, holes=rng.random() < 0.5)


def _logits(case, g):
    rows, V = case["rows"], case["V"]
    x = torch.randn(rows, V, generator=g, device=DEV).mul_(2.5)
    at = torch.randint(0, V, (rows, 24), generator=g, device=DEV)
    return x.scatter_reduce_(1, at, 14.0 * torch.rand(rows, 24, generator=g, device=DEV), "amax")   # (a place may be named twice)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[case["dtype"]]
    rows, V, cap = case["rows"], case["V"], case["cap"] or None
    x = _logits(case, g)
    st = dict(op=case["op"], cap=cap)
    if case["op"] == "sample":
        st["u"] = torch.rand(rows, generator=g, device=DEV)
        if case["mixed"]:   # a server's slots: settings lie in vectors on the device; of each setting a third of the rows use none
            third = lambda: torch.randint(0, 3, (rows,), generator=g, device=DEV) == 0   # noqa: E731
            rand = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=DEV)   # noqa: E731
            st["T"] = rand(0.5, 1.4)
            st["k"] = torch.randint(1, 200, (rows,), generator=g, device=DEV, dtype=torch.int32).masked_fill_(third(), 0)
            st["p"] = rand(0.5, 0.99).masked_fill_(third(), 1.0)
            st["mp"] = rand(0.01, 0.1).masked_fill_(third(), 0.0)
        else:
            st.update(T=case["T"], k=case["k"], p=case["p"], mp=case["mp"])
        st["x"] = x.to(dtype)
        return st
    st.update(T=case["T"], k=case["k"])
    if case["op"] == "topk":
        st["x"] = x.to(dtype)
        return st
    st["x"] = x.to(dtype)
    teacher = x.add_(torch.randn(rows, V, generator=g, device=DEV))
    if cap:
        teacher = teacher.div_(cap).tanh_().mul_(cap)
    values, ids = teacher.topk(case["k"], dim=-1)
    ids = ids.to(torch.int32)
    lse = torch.logsumexp(teacher.div_(case["T"]), -1) if case["tail"] else None
    weight = torch.full((rows,), 1.0 / rows, device=DEV)
    if case["holes"]:   # rows of padding, and teachers that gave fewer entries
        n = torch.randint(1, case["k"] + 1, (rows, 1), generator=g, device=DEV)
        n = torch.where(torch.rand(rows, 1, generator=g, device=DEV) < 0.5, case["k"], n)
        n = torch.where(torch.rand(rows, 1, generator=g, device=DEV) < 0.1, 0, n)
        ids = torch.where(torch.arange(case["k"], device=DEV) < n, ids, -1)
        weight = weight * (n[:, 0] > 0)
    st.update(values=values, ids=ids, lse=lse, weight=weight)
    if case["op"] == "distill_train":
        st["x"].requires_grad_()
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    if own:
        from xlstm_b200 import ops
        if st["op"] == "sample":
            return ops.softcap_sample(st["x"], st["cap"], st["u"], temperature=st["T"], top_k=st["k"], top_p=st["p"], min_p=st["mp"])
        if st["op"] == "topk":
            return ops.softcap_topk(st["x"], st["cap"], st["k"], temperature=st["T"])
        if st["op"] == "distill":
            return ops.distill_topk(st["x"], st["values"], st["ids"], st["cap"], temperature=st["T"], teacher_lse=st["lse"])
        if st["op"] == "distill_train":
            loss = ops.distill_topk(st["x"], st["values"], st["ids"], st["cap"], temperature=st["T"], teacher_lse=st["lse"])
            return loss.detach(), torch.autograd.grad(loss, st["x"], st["weight"])[0]
        return ops.distill_topk_grad(st["x"], st["values"], st["ids"], st["weight"], st["cap"], temperature=st["T"], teacher_lse=st["lse"])
    if st["op"] == "sample":
        return _sample(st["x"], st["cap"], st["u"], st["T"], st["k"], st["p"], st["mp"])
    if st["op"] == "topk":
        return _topk(st["x"], st["cap"], st["k"], st["T"])
    x = st["x"].detach()
    if st["op"] == "distill":
        return _distill(x, st["values"], st["ids"], st["cap"], st["T"], st["lse"])
    return _distill(x, st["values"], st["ids"], st["cap"], st["T"], st["lse"], st["weight"])


def _column(v, like):
    return v[:, None] if torch.is_tensor(v) else torch.full((like.shape[0], 1), v, device=like.device)


def _sample(x, cap, u, T, k, p, mp):
    """In 64 bits: a token is a whole number, and which side of a border it falls on is decided by the last digits.  (The
    settings themselves are 32-bit numbers.)"""
    T, k, p, mp = _column(T, x).double(), _column(k, x), _column(p, x).double(), _column(mp, x).double()
    s, idx = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    y = cap * torch.tanh(s / cap) if cap else s
    w = torch.exp((y - y[:, :1]) / T)
    place = torch.arange(x.shape[1], device=x.device)
    w = torch.where((place < k) | (k <= 0), w, 0.0)
    upto = torch.cumsum(w, -1)
    keep = (w > 0) & (((upto - w) < p * upto[:, -1:]) | (p >= 1)) & (w >= mp)
    keep[:, 0] = True
    target = u.double()[:, None] * torch.where(keep, w, 0.0).sum(-1, keepdim=True)
    n = keep.sum(-1, keepdim=True)
    at = torch.minimum((upto <= target).sum(-1, keepdim=True), n - 1)
    return idx.gather(1, at)[:, 0]


def _lse(z):
    m = z.max(-1, keepdim=True).values
    m = torch.where(m > -math.inf, m, 0.0)   # (a row of nothing has the sum zero)
    return (torch.log(torch.exp(z - m).sum(-1, keepdim=True)) + m)


def _topk(x, cap, k, T):
    s, idx = torch.sort(x.float(), dim=-1, descending=True, stable=True)
    y = cap * torch.tanh(s / cap) if cap else s
    return y[:, :k].contiguous(), idx[:, :k].to(torch.int32), _lse(y / T)[:, 0]


def _distill(x, values, ids, cap, T, lse, weight=None):
    y = x.float()
    slope = None
    if cap:
        t = torch.tanh(y / cap)
        y, slope = cap * t, 1 - t * t
    z = y / T
    used = ids >= 0
    at = ids.long().clamp(min=0)
    tz = torch.where(used, values.double() / T, -math.inf)   # (64 bits: 1 - sum(p) is what is left of numbers next to one)
    live = used.any(-1, keepdim=True)
    logp = tz - (_lse(tz) if lse is None else lse.double()[:, None])
    logp = torch.where(used & live, logp, 0.0)
    p = torch.where(used & live, torch.exp(logp), 0.0)
    named = torch.zeros(x.shape, dtype=torch.bool, device=x.device)
    named[torch.arange(x.shape[0], device=x.device)[:, None].expand_as(ids)[used], at[used]] = True
    ptail = torch.zeros_like(live, dtype=torch.float64)
    if lse is not None:
        ptail = torch.where(live & ~named.all(-1, keepdim=True), (1 - p.sum(-1, keepdim=True)).clamp(min=0), 0.0)
    ls = _lse(z)
    lt = _lse(torch.where(named, -math.inf, z))
    zk = z.gather(1, at).double()
    loss = torch.where(p > 0, p * (logp - (zk - ls)), 0.0).sum(-1, keepdim=True)
    loss = loss + torch.where(ptail > 0, ptail * (torch.log(ptail) - (lt - ls)), 0.0)
    loss = (T * T * loss)[:, 0].float()
    if weight is None:
        return loss
    W = (p.sum(-1, keepdim=True) + ptail).float()
    d = W * torch.exp(z - ls) - torch.where(named, 0.0, ptail.float() * torch.exp(z - lt))
    d = d.scatter_add(1, at, -p.float())
    d = weight[:, None] * T * d
    return loss, (d if slope is None else d * slope).to(x.dtype)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    rows, V, s = case["rows"], case["V"], 2 if case["dtype"] == "bf16" else 4
    n = rows * V
    if case["op"] == "sample":   # a cap, an exponential and a sum an element
        return {"bytes": n * s + rows * (4 + (16 if case["mixed"] else 0) + 8), "flops": 4 * n}
    if case["op"] == "topk":
        return {"bytes": n * s + rows * (8 * case["k"] + 4), "flops": 4 * n}
    teacher = rows * (8 * case["k"] + (4 if case["tail"] else 0))
    if case["op"] == "distill":
        return {"bytes": n * s + teacher + 4 * rows, "flops": 4 * n}
    return {"bytes": 2 * n * s + teacher + 8 * rows, "flops": 9 * n}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    rows, V, cap = case["rows"], case["V"], st["cap"]
    x = st["x"].detach()
    piece = max(1, (1 << 25) // V)   # rows at a time
    parts = []
    for r0 in range(0, rows, piece):
        r = slice(r0, min(rows, r0 + piece))
        parts.append(_exact_rows(case["op"], x[r].double(), cap, {k: v[r] if torch.is_tensor(v) else v for k, v in st.items()}))
    if case["op"] == "sample":
        return torch.cat([q[0] for q in parts])
    out = tuple(torch.cat([q[j] for q in parts]) for j in range(len(parts[0])))
    return out[0] if len(out) == 1 else out


def _exact_rows(op, x, cap, st):
    capped = (lambda a: cap * torch.tanh(a / cap)) if cap else (lambda a: a)
    n, V = x.shape
    if op == "sample":
        tokens = []
        for i in range(n):
            # settings are 32-bit numbers, whether they come in vectors or as one for all
            T, k, p, mp = (float(st[c][i] if torch.is_tensor(st[c]) else torch.tensor(st[c], dtype=torch.float32)) for c in ("T", "k", "p", "mp"))
            order = torch.sort(x[i], descending=True, stable=True).indices
            prob = torch.softmax(capped(x[i][order]) / T, -1)
            m = int(k) if k > 0 else V
            cut = prob[:m] / prob[:m].sum()
            before = torch.cat([cut.new_zeros(1), torch.cumsum(cut, 0)[:-1]])
            good = cut >= mp * cut[0]
            if p < 1:
                good &= before < p
            good[0] = True
            cut = cut[good]
            where = torch.searchsorted(torch.cumsum(cut, 0), (st["u"][i].double() * cut.sum()).reshape(1), right=True)
            tokens.append(order[where.clamp(max=cut.numel() - 1)])
        return (torch.cat(tokens),)
    if op == "topk":
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :st["k"]]
        return capped(x.gather(1, order)), order.to(torch.int32), torch.logsumexp(capped(x) / st["T"], -1)
    T, ids, lse = st["T"], st["ids"].long(), st["lse"]
    x = x.requires_grad_(op != "distill")
    logq = torch.log_softmax(capped(x) / T, -1)
    used = ids >= 0
    t = (st["values"].double() / T).masked_fill(~used, -math.inf)
    norm = torch.logsumexp(t, -1) if lse is None else lse.double()
    p = torch.exp(t - torch.where(used.any(-1), norm, 0.0)[:, None])
    at = ids.masked_fill(~used, V)
    named = torch.zeros(n, V + 1, device=x.device).scatter_(1, at, 1.0)[:, :V] > 0
    of_entry = torch.cat([logq, logq.new_zeros(n, 1)], 1).gather(1, at)
    loss = (torch.special.xlogy(p, p) - p * of_entry).sum(-1)
    if lse is not None:
        rest = torch.where(used.any(-1) & ~named.all(-1), (1 - p.sum(-1)).clamp(min=0), 0.0)
        loss = loss + torch.special.xlogy(rest, rest) - rest * torch.logsumexp(logq.masked_fill(named, -1e30), -1)
    loss = T * T * loss
    if op == "distill":
        return (loss,)
    grad, = torch.autograd.grad((loss * st["weight"].double()).sum(), x)
    return loss.detach(), grad
