"""CPU restatement, in 64 bits, of the operators along the vocabulary axis: sampling, top logits, distillation."""
import math

import torch


def cap64(x, cap):
    x = x.double()
    return cap * torch.tanh(x / cap) if cap else x


def order(x):
    """Indices of a row in descending order, lower index first among equals, NaN last."""
    key = [(1, 0.0, j) if math.isnan(v) else (0, -v, j) for j, v in enumerate(x.double().tolist())]
    return [j for _, _, j in sorted(key)]


def sample_row(x, cap, u, T=1.0, k=0, p=1.0, mp=0.0):
    """Token of one row; settings as float32 numbers.  Also the distance of u to the nearest border between two tokens."""
    T, p, mp = (float(torch.tensor(v, dtype=torch.float32)) for v in (T, p, mp))
    idx = order(x)
    y = cap64(x, cap)[idx]
    xs = x.double()[idx]
    if not float(xs[0]) > -math.inf:
        return 0, 1.0
    w = torch.where(xs == xs[0], 1.0, torch.exp((y - y[0]) / T) if math.isfinite(float(y[0])) else 0.0)
    w = torch.where(xs > -math.inf, w, 0.0)   # (NaN compares false)
    if k > 0:
        w = w[:k]
    upto = torch.cumsum(w, 0)
    keep = w >= mp
    if p < 1:
        keep &= (upto - w) < p * upto[-1]
    keep[0] = True
    w = w[keep]
    upto = torch.cumsum(w, 0)
    share = upto / upto[-1]
    j = min(int((share <= min(max(float(u), 0.0), 1.0)).sum()), int((w > 0).sum()) - 1)
    return idx[j], float((share - float(u)).abs().min())


def topk_row(x, cap, k, T=1.0):
    idx = order(x)[:k]
    y = cap64(x, cap)
    return y[idx], idx, torch.logsumexp(y / T, 0)


def distill(x, values, ids, cap=None, T=1.0, lse=None):
    """Losses (N,), differentiable in x (N, V) float64.  Entry by entry, from the definition."""
    N, V = x.shape
    z = (cap * torch.tanh(x / cap) if cap else x) / T
    out = []
    for r in range(N):
        used = [k for k in range(ids.shape[1]) if 0 <= int(ids[r, k]) < V]
        t = [float(values[r, k]) / T for k in used]
        if not used or (lse is None and max(t) == -math.inf):
            out.append((z[r] * 0).nan_to_num(0.0).sum())
            continue
        L = float(torch.logsumexp(torch.tensor(t, dtype=torch.float64), 0)) if lse is None else float(lse[r])
        logq = torch.log_softmax(z[r], 0)
        loss, left = 0.0, 1.0
        for k, tk in zip(used, t):
            p = math.exp(tk - L)
            left -= p
            if p > 0:
                loss = loss + p * (tk - L - logq[int(ids[r, k])])
        rest = sorted(set(range(V)) - {int(ids[r, k]) for k in used})
        if lse is not None and rest and left > 0:
            loss = loss + left * (math.log(left) - torch.logsumexp(logq[rest], 0))
        out.append(T * T * loss if torch.is_tensor(loss) else (z[r] * 0).sum())
    return torch.stack(out)


def distill_grad(x, values, ids, cap=None, T=1.0, lse=None):
    """Gradient of the losses' sum by the closed form, W q - p (named), (W - p_tail / q_tail) q (not named)."""
    N, V = x.shape
    t = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    z = (cap * t if cap else x) / T
    q = torch.softmax(z, -1)
    g = torch.zeros_like(x)
    for r in range(N):
        used = [k for k in range(ids.shape[1]) if 0 <= int(ids[r, k]) < V]
        e = torch.tensor([float(values[r, k]) / T for k in used], dtype=torch.float64)
        if not used or (lse is None and float(e.max()) == -math.inf):
            continue
        p = torch.exp(e - (torch.logsumexp(e, 0) if lse is None else float(lse[r])))
        at = torch.tensor([int(ids[r, k]) for k in used])
        named = torch.zeros(V, dtype=torch.bool)
        named[at] = True
        rest = max(0.0, 1 - float(p.sum())) if lse is not None and not bool(named.all()) else 0.0
        W = float(p.sum()) + rest
        g[r] = W * q[r]
        if rest:
            g[r] -= torch.where(named, 0.0, rest * torch.softmax(z[r].masked_fill(named, -math.inf), 0))
        g[r].index_add_(0, at, -p)
    return T * g * (1 - t * t)
