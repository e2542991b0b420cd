"""The sparse feed-forward operators from their definition in 64 bits, with bounds on what bf16 roundings may change."""
import torch

U = 2.0 ** -8       # half a step of bf16, relative
UH = 2.0 ** -11     # half a step of fp16, relative (the kernels' blocks of 32 keep it down to 2^-28 of the block's largest)
U32 = 2.0 ** -23    # one step of fp32, relative


def route(z, k, sigmoid=False, bias=None, groups=1, top_groups=1, group_top=2, renorm=True, scale=1.0):
    """(weights, experts) in 64 bits, token by token."""
    z = z.detach().double().cpu()
    bias = None if bias is None else bias.detach().double().cpu()
    T, E = z.shape
    W, ids = torch.zeros(T, k, dtype=torch.float64), torch.zeros(T, k, dtype=torch.long)
    size = E // groups
    for t in range(T):
        row = z[t]
        if torch.isnan(row).any() or (not sigmoid and (row == torch.inf).any()):
            W[t], ids[t] = torch.nan, torch.arange(k)
            continue
        if sigmoid:
            s = torch.special.expit(row)
        else:
            e = torch.exp(row - row.max()) if torch.isfinite(row.max()) else torch.zeros_like(row)
            s = e / e.sum() if e.sum() > 0 else e
        c = s if bias is None else s + bias
        c = [-torch.inf if row[i] == -torch.inf else float(c[i]) for i in range(E)]
        score = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top]) for g in range(groups)]
        kept = sorted(sorted(range(groups), key=lambda g: (-score[g], g))[:top_groups])
        allowed = [i for g in kept for i in range(g * size, (g + 1) * size)]
        chosen = sorted(allowed, key=lambda i: (-c[i], i))[:k]
        w = torch.tensor([0.0 if c[i] == -torch.inf else float(s[i]) for i in chosen], dtype=torch.float64)
        if renorm and w.sum() > 0:
            w = w / w.sum()
        W[t], ids[t] = w * scale, torch.tensor(chosen)
    return W, ids


def route_grad(z, ids, dw, sigmoid=False, bias=None, renorm=True, scale=1.0):
    """dlogits in 64 bits by automatic differentiation of the written-out weights of the chosen experts."""
    z, dw = z.detach().double().cpu().requires_grad_(), dw.double().cpu()
    dis = z.detach().gather(1, ids) == -torch.inf
    if bias is not None:
        dis |= bias.double().cpu()[ids] == -torch.inf
    live = (z > -torch.inf).any(1, keepdim=True)
    zz = torch.where(live, z, torch.zeros_like(z))
    s = torch.special.expit(zz) if sigmoid else torch.softmax(zz, -1)
    w = torch.where(dis | ~live, torch.zeros_like(dw), s.gather(1, ids))
    if renorm:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    (w * scale * dw).sum().backward()
    return torch.nan_to_num(z.grad, nan=0.0)


def plan(ids, E, align=16):
    """counts, offsets, slots, rows by a loop over the assignments."""
    flat = ids.reshape(-1).tolist()
    counts = [sum(1 for e in flat if e == x) for x in range(E)]
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + (c + align - 1) // align * align)
    n = len(flat)
    R = (n + (align - 1) * min(n, E) + align - 1) // align * align
    nxt, slots, rows = list(offsets[:E]), [-1] * n, [-1] * R
    for a, e in enumerate(flat):
        if 0 <= e < E:
            slots[a], rows[nxt[e]] = nxt[e], a
            nxt[e] += 1
    return counts, offsets, slots, rows


def experts(x, w, ids, wg, wu, wd, residual=None, dout=None):
    """{"out", "dx", "dw", "dgate", "dup", "ddown"}: (value in 64 bits, elementwise bound) of bf16 kernels that keep sums in
    fp32, round the hidden activations, their gradients and the results to bf16 and each expert's output and input-gradient
    row to fp16, and in the backward pass start from projections that were rounded to fp16 (absolute errors of a block's
    smallest values, 2^-39 of its largest, are far below the fp32 steps of the sums).  Every bound adds half a step per rounding, carried through the following
    product by absolute values, and one fp32 step per summand of a product."""
    dev = x.device
    X, W = x.detach().double(), w.detach().double()
    Wg, Wu, Wd = (v.detach().double() for v in (wg, wu, wd))
    E, F, D = Wg.shape
    out = torch.zeros_like(X) if residual is None else residual.detach().double()
    e_out = torch.zeros_like(X)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    r = {n: [zeros(*s), zeros(*s)] for n, s in (("dx", X.shape), ("dw", W.shape), ("dgate", Wg.shape), ("dup", Wu.shape), ("ddown", Wd.shape))}
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe, we = X[t], W[t, j][:, None]
        g, u = xe @ Wg[e].T, xe @ Wu[e].T
        eg, eu = D * U32 * (xe.abs() @ Wg[e].T.abs()), D * U32 * (xe.abs() @ Wu[e].T.abs())  # of the fp32 sums
        s = torch.sigmoid(g)
        act = g * s
        h = we * act * u
        eh = we * (1.1 * eg * u.abs() + act.abs() * eu) + (U + 16 * U32) * h.abs()
        y = h @ Wd[e].T
        ey = eh @ Wd[e].T.abs() + F * U32 * (h.abs() @ Wd[e].T.abs())
        out.index_add_(0, t, y)
        e_out.index_add_(0, t, ey + UH * (y.abs() + ey))
        if dout is None:
            continue
        do = dout.detach().double()[t]
        dh = do @ Wd[e]
        edh = D * U32 * (do.abs() @ Wd[e].abs())
        eg, eu = eg + UH * (g.abs() + eg), eu + UH * (u.abs() + eu)  # the stored projections
        ds = s + act * (1 - s)  # |silu'| <= 1.1, |silu''| <= 0.5
        dg, du = we * dh * u * ds, we * dh * act
        edg = we * (edh * (u * ds).abs() + dh.abs() * (eu * ds.abs() + (u.abs() + eu) * 0.5 * eg)) + (U + 16 * U32) * dg.abs()
        edu = we * (edh * act.abs() + dh.abs() * 1.1 * eg) + (U + 16 * U32) * du.abs()
        edg, edu = edg * (1 + U), edu * (1 + U)
        r["dw"][0][t, j] = (dh * act * u).sum(1)
        r["dw"][1][t, j] = (edh * (act * u).abs() + dh.abs() * (1.1 * eg * (u.abs() + eu) + act.abs() * eu)).sum(1) + (F + 16) * U32 * (dh * act * u).abs().sum(1)
        rows = dg @ Wg[e] + du @ Wu[e]
        erows = edg @ Wg[e].abs() + edu @ Wu[e].abs() + 2 * F * U32 * (dg.abs() @ Wg[e].abs() + du.abs() @ Wu[e].abs())
        r["dx"][0].index_add_(0, t, rows)
        r["dx"][1].index_add_(0, t, erows + UH * (rows.abs() + erows))
        n = t.numel()
        r["dgate"][0][e], r["dgate"][1][e] = dg.T @ xe, edg.T @ xe.abs() + n * U32 * (dg.abs().T @ xe.abs())
        r["dup"][0][e], r["dup"][1][e] = du.T @ xe, edu.T @ xe.abs() + n * U32 * (du.abs().T @ xe.abs())
        r["ddown"][0][e], r["ddown"][1][e] = do.T @ h, do.abs().T @ eh + n * U32 * (do.abs().T @ h.abs())
    r["out"] = [out, e_out]
    if dout is None:
        r = {"out": r["out"]}
    return r


def outside(got, ref, bound, dtype=torch.bfloat16):
    """How many values are further from ``ref`` than ``bound`` and one rounding to ``dtype`` allow."""
    last = {torch.bfloat16: U, torch.float32: U32}[dtype]
    lim = bound + last * (ref.abs() + bound) + 1e-30
    return int((~((got.double() - ref).abs() <= lim)).sum())
