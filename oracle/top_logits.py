"""Top-logit selection and the distillation loss from their definitions, in float64 on the CPU (test infrastructure).  Classes last: z [R, V]."""
import torch


def top(z, k, T):
    """values, indices (ties: lowest class; NaN above everything), lse."""
    v = z.double()
    nan = torch.isnan(v)
    key = torch.where(nan, torch.full_like(v, float("inf")), v)
    order = torch.sort(key, dim=1, descending=True, stable=True)[1]      # stable: the lower class first
    if bool(nan.any()):                                                  # NaN above +inf: a stable sort by that alone
        order = order.gather(1, torch.sort(nan.gather(1, order).to(torch.int8), dim=1, descending=True, stable=True)[1])
    order = order[:, :k]
    return z.gather(1, order), order, torch.logsumexp(v / T, 1)


def distill(z, idx, val, lse, w, T, reduction, go=None):
    """-> (loss -- "none": w times each row's --, gradient of sum(go * loss) for "none", of go * loss otherwise, error scale of the loss rows)."""
    z, val, idx = z.double(), val.double(), idx.long()
    R, V = z.shape
    w = torch.ones(R, dtype=torch.float64) if w is None else w.double()
    rows, grads, scale = [], [], []
    for r in range(R):
        ok = (idx[r] >= 0) & (idx[r] < V)
        i, t = idx[r][ok], val[r][ok]
        if i.numel() == 0 or lse is None and bool((t == -float("inf")).all()):
            rows.append(torch.zeros((), dtype=torch.float64)); grads.append(torch.zeros(V, dtype=torch.float64)); scale.append(1.0)
            continue
        lq = torch.log_softmax(z[r] / T, 0)
        q = lq.exp()
        lp = t / T - (lse[r].double() if lse is not None else torch.logsumexp(t / T, 0))
        p = lp.exp()
        terms = torch.where(p != 0, p * (lp - lq[i]), torch.zeros_like(p))
        g = q.clone()
        g.index_add_(0, i, -p)
        loss, mag = terms.sum(), terms.abs().sum()
        if lse is not None:
            out = torch.ones(V, dtype=torch.bool)
            out[i] = False
            pr, qr = (1 - p.sum()).clamp(min=0), q[out].sum()
            if float(qr) != 0 and float(pr) != 0:
                lqr = torch.logsumexp(z[r][out] / T, 0) - torch.logsumexp(z[r] / T, 0)
                loss = loss + pr * (pr.log() - lqr)
                mag = mag + (pr * (pr.log() - lqr)).abs()
                g[out] = q[out] - pr * torch.softmax(z[r][out] / T, 0)
        rows.append(T * T * loss); grads.append(T * g); scale.append(float(1 + mag))
    rows, grads = torch.stack(rows), torch.stack(grads)
    live = w != 0
    if reduction == "none":
        go = torch.ones(R, dtype=torch.float64) if go is None else go.double()
        return torch.where(live, w * rows, torch.zeros_like(rows)), torch.where(live[:, None], grads * (go * w)[:, None], torch.zeros_like(grads)), torch.tensor(scale)
    total = (w[live] * rows[live]).sum()
    c = torch.where(live, w, torch.zeros_like(w))
    if reduction == "mean":
        n = w.sum()
        total = total / n if float(n) != 0 else torch.zeros((), dtype=torch.float64)
        c = c / n if float(n) != 0 else torch.zeros_like(c)
    return total, torch.where(live[:, None], grads * c[:, None], torch.zeros_like(grads)) * (1.0 if go is None else float(go)), torch.tensor(scale)
