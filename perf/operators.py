"""The sparse feed-forward operators (routing, grouping by expert, experts' products): the cases on which they are timed,
their plain form in elementary torch operations, and their definition in 64 bits."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ALIGN = 16  # rows: where an expert's segment of the grouped rows may begin


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def _route(name, tokens, experts, k, score="softmax", dtype="bf16", bias=False, groups=1, top_groups=1, group_top=2, renorm=True, scale=1.0,
           masked=False, train=False):
    c = {"op": "route", "tokens": tokens, "experts": experts, "k": k, "score": score, "dtype": dtype, "bias": bias, "groups": groups,
         "top_groups": top_groups, "group_top": group_top, "renorm": renorm, "scale": scale, "masked": masked, "train": train}
    return dict(c, name=name) if name else c


def _plan(name, tokens, experts, k, drop=0.0):
    c = {"op": "plan", "tokens": tokens, "experts": experts, "k": k, "drop": drop}
    return dict(c, name=name) if name else c


def _experts(name, tokens, dim, ffn, experts, k, train=False, drop=0.0, residual=False):
    c = {"op": "experts", "tokens": tokens, "dim": dim, "ffn": ffn, "experts": experts, "k": k, "train": train, "drop": drop, "residual": residual}
    return dict(c, name=name) if name else c


def _layer(name, tokens, dim, ffn, experts, k, score="softmax", bias=False, groups=1, top_groups=1, scale=1.0, train=True):
    c = {"op": "layer", "tokens": tokens, "dim": dim, "ffn": ffn, "experts": experts, "k": k, "score": score, "dtype": "bf16", "bias": bias,
         "groups": groups, "top_groups": top_groups, "group_top": 2, "renorm": True, "scale": scale, "masked": False, "train": train, "drop": 0.0, "residual": True}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of a few sequences: nothing but latency
        _route("route_decode", 4, 16, 2),
        # a training micro-batch of 4 x 2048 tokens through the framework's own rule, gradient included
        _route("route_train_softmax", 8192, 64, 6, train=True),
        # the largest: a router in 32 bits with a bias for balance and limited groups over many experts
        _route("route_train_sigmoid_groups", 32768, 256, 8, score="sigmoid", dtype="fp32", bias=True, groups=8, top_groups=4, scale=2.5, train=True),
        # odd sizes, disabled experts (logits of minus infinity, some rows of nothing else), no renormalisation
        _route("route_odd_masked", 4097, 100, 5, dtype="fp32", renorm=False, masked=True, train=True),
        # grouping a decode batch, padded rows dropped
        _plan("plan_decode", 64, 256, 8, drop=0.1),
        # grouping a long prefill or a large micro-batch
        _plan("plan_large", 32768, 256, 8),
        # a single sequence decodes: a few experts' weights pass through once
        _experts("experts_one_token", 1, 2048, 1408, 16, 4, residual=True),
        # a decode batch of the server, every expert's weights are read
        _experts("experts_decode_batch", 48, 2048, 1408, 64, 6, residual=True),
        # a right-padded prefill batch of uneven prompts
        _experts("experts_prefill", 5003, 2048, 1408, 64, 6, drop=0.07),
        # small odd widths, an uneven batch, every gradient
        _experts("experts_train_odd", 333, 520, 184, 10, 3, train=True, drop=0.05),
        # a training micro-batch of 4 x 2048 tokens: four of sixteen experts, each a quarter of the dense layer's width
        _experts("experts_train", 8192, 2048, 1408, 16, 4, train=True),
        # routing and experts together, as a layer runs them in training
        _layer("layer_train", 4096, 2048, 1408, 32, 4, score="sigmoid", bias=True, groups=4, top_groups=2),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "route", "plan", "experts", "experts", "experts", "layer"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        e = max(2, _log(rng, 8, 256) // groups) * groups
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, e // groups * top_groups))
        score = rng.choice(["softmax", "sigmoid"])
        renorm = rng.random() < 0.7 and k > 1  # one renormalised weight is a constant
        return _route(None, _log(rng, 1, 32768), e, k, score, rng.choice(["bf16", "fp32"]), rng.random() < 0.5, groups, top_groups, rng.choice([1, 2]),
                      renorm, rng.choice([1.0, 2.5]), rng.random() < 0.3, rng.random() < 0.6)
    if op == "plan":
        e = _log(rng, 2, 256)
        return _plan(None, _log(rng, 1, 32768), e, rng.randint(1, min(8, e)), rng.choice([0.0, 0.1]))
    e = _log(rng, 4, 32)
    k = rng.randint(2, min(6, e))
    dim, ffn = 8 * _log(rng, 16, 256), 8 * _log(rng, 8, 176)
    train = rng.random() < 0.5
    tokens = _log(rng, 1, 2048 if train else 4096)
    if op == "experts":
        return _experts(None, tokens, dim, ffn, e, k, train, rng.choice([0.0, 0.1]), rng.random() < 0.5)
    return _layer(None, tokens, dim, ffn, e, k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, train=train)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(c, g):
    """Router logits: some experts are liked more than others, tokens differ."""
    t, e = c["tokens"], c["experts"]
    z = torch.randn(t, e, device="cuda", generator=g) * 1.5 + torch.randn(e, device="cuda", generator=g) * 0.5
    if c.get("masked"):
        z = z.masked_fill(torch.rand(t, e, device="cuda", generator=g) < 0.2, -math.inf)
        z = z.masked_fill(torch.rand(t, 1, device="cuda", generator=g) < 0.01, -math.inf)
    return z.to(DTYPES[c["dtype"]])


def prepare(case, seed):
    c, g = case, _gen(seed)
    t, e, k, op = c["tokens"], c["experts"], c["k"], c["op"]
    s = {"case": c}
    if op in ("route", "layer"):
        s["logits"] = _logits(c, g)
        s["bias"] = torch.randn(e, device="cuda", generator=g) * 0.05 if c["bias"] else None
        if op == "route":
            s["dweights"] = torch.randn(t, k, device="cuda", generator=g).to(DTYPES[c["dtype"]])
    if op in ("plan", "experts"):
        z = torch.randn(t, e, device="cuda", generator=g) * 1.5 + torch.randn(e, device="cuda", generator=g) * 0.5
        w, idx = torch.topk(torch.softmax(z, -1), k, dim=-1)
        live = t - int(t * c["drop"])  # the padded rows at the end of a batch are dropped
        s["ids"] = torch.where(torch.arange(t, device="cuda")[:, None] < live, idx, torch.full_like(idx, -1)).contiguous()
        s["weights"] = (w / w.sum(-1, keepdim=True)).to(torch.bfloat16)
    if op in ("experts", "layer"):
        d, f = c["dim"], c["ffn"]
        rand = lambda *n, scale=1.0: (torch.randn(*n, device="cuda", generator=g) * scale).to(torch.bfloat16)  # noqa: E731
        s["x"] = rand(t, d)
        s["gate"], s["up"], s["down"] = rand(e, f, d, scale=d ** -0.5), rand(e, f, d, scale=d ** -0.5), rand(e, d, f, scale=f ** -0.5)
        s["residual"] = rand(t, d) if c["residual"] else None
        s["dout"] = rand(t, d) if c["train"] else None
        ids = s["ids"] if op == "experts" else _route_plain(s["logits"], s["bias"], c)[1]
        s["cap"] = int(torch.bincount(ids[ids >= 0], minlength=e).max()) if ids.numel() else 0
    return s


# ---------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------
def _select_plain(z, bias, c):
    """The selected experts; in 64 bits, since scores lie next to the border of the k largest."""
    z = z.double()
    s = _scores_plain(z, c["score"])
    s = s if bias is None else s + bias.double()
    s = s.masked_fill(z == -math.inf, -math.inf)  # a disabled expert is chosen only where no other is left
    t, e = s.shape
    n = c["groups"]
    if n > 1:
        of_group = s.view(t, n, e // n).sort(dim=-1, descending=True).values[..., : c["group_top"]].sum(-1)
        best = of_group.sort(dim=-1, descending=True, stable=True).indices[:, : c["top_groups"]]
        keep = torch.zeros(t, n, dtype=torch.bool, device=s.device).scatter(1, best, True).repeat_interleave(e // n, dim=1)
        # what stays comes before what goes, also where both are minus infinity
        s = torch.where(keep, s.clamp(min=-1e30), torch.full_like(s, -math.inf))
    return s.sort(dim=-1, descending=True, stable=True).indices[:, : c["k"]].contiguous()


def _scores_plain(z, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _route_plain(z, bias, c):
    """(weights in 32 bits, experts) of logits in 32 bits."""
    ids = _select_plain(z.detach(), bias, c)
    w = _scores_plain(z.float(), c["score"]).gather(1, ids)
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
    return w * c["scale"], ids


def _plan_plain(ids, e):
    flat = ids.reshape(-1)
    n = flat.numel()
    live = (flat >= 0) & (flat < e)
    key = torch.where(live, flat, torch.full_like(flat, e))
    counts = torch.zeros(e + 1, dtype=torch.long, device=flat.device).index_add_(0, key, torch.ones_like(key))[:e]
    ends = torch.cumsum((counts + ALIGN - 1) // ALIGN * ALIGN, 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    order = key.sort(stable=True).indices
    first = torch.cumsum(counts, 0) - counts
    of = key[order]
    safe = of.clamp(max=e - 1)
    row = offsets[safe] + torch.arange(n, device=flat.device) - first[safe]
    slots = torch.full_like(flat, -1).scatter(0, order, torch.where(of < e, row, torch.full_like(row, -1)))
    room = (n + (ALIGN - 1) * min(e, n) + ALIGN - 1) // ALIGN * ALIGN
    rows = torch.full((room + 1,), -1, dtype=torch.long, device=flat.device)
    rows = rows.scatter(0, torch.where(of < e, row, torch.full_like(row, room)), order)[:room]
    # the dropped ones all went to the place behind the last row
    return [v.to(torch.int32) for v in (counts, offsets, slots.view_as(ids), rows)]


def _experts_plain(x, w, ids, gate, up, down, residual, cap):
    """In 32 bits: the tokens of each expert side by side, padded to the fullest expert's count."""
    t, d = x.shape
    e, k = gate.shape[0], ids.shape[1]
    flat = ids.reshape(-1)
    if cap == 0:  # every assignment is dropped
        return x * 0 if residual is None else residual + x * 0
    key = torch.where(flat >= 0, flat, torch.full_like(flat, e))
    order = key.sort(stable=True).indices
    of = key[order]
    counts = torch.zeros(e + 1, dtype=torch.long, device=x.device).index_add_(0, key, torch.ones_like(key))
    place = torch.arange(flat.numel(), device=x.device) - (torch.cumsum(counts, 0) - counts)[of]
    at = torch.where(of < e, of * cap + place, torch.full_like(of, e * cap))  # the dropped ones share a row behind the last
    rows = torch.zeros(e * cap + 1, d, device=x.device).index_copy(0, at, x[order // k])[: e * cap].view(e, cap, d)
    g, u = rows @ gate.transpose(1, 2), rows @ up.transpose(1, 2)
    y = (g / (1 + torch.exp(-g)) * u) @ down.transpose(1, 2)
    y = torch.cat([y.reshape(e * cap, d), torch.zeros(1, d, device=x.device)])
    back = torch.zeros_like(at).scatter(0, order, at)
    out = (y[back].view(t, k, d) * w.unsqueeze(-1)).sum(1)
    return out if residual is None else out + residual


def _leaf(v):
    return None if v is None else v.detach().requires_grad_(True)


def _leaf32(v):
    return None if v is None else v.detach().float().requires_grad_(True)


def run(state):
    c = state["case"]
    train = c.get("train", False)
    if own:
        return _run_own(state, c, train)
    if c["op"] == "plan":
        return dict(zip(("counts", "offsets", "slots", "rows"), _plan_plain(state["ids"], c["experts"])))
    if c["op"] == "route":
        dt = DTYPES[c["dtype"]]
        with torch.set_grad_enabled(train):
            z = _leaf32(state["logits"])
            w, ids = _route_plain(z, state["bias"], c)
        out = {"weights": w.detach().to(dt), "experts": ids}
        if train:
            out["dlogits"] = _row_grads(z, w, ids, state["dweights"].float(), c).to(dt)
        return out
    keys = ["x", "gate", "up", "down"]
    with torch.set_grad_enabled(train):
        leaves = {n: _leaf32(state[n]) for n in keys}
        if c["op"] == "layer":
            leaves["logits"] = _leaf32(state["logits"])
            w, ids = _route_plain(leaves["logits"], state["bias"], c)
        else:
            leaves["weights"] = _leaf32(state["weights"])
            w, ids = leaves["weights"], state["ids"]
        res = None if state["residual"] is None else state["residual"].float()
        y = _experts_plain(leaves["x"], w, ids, leaves["gate"], leaves["up"], leaves["down"], res, state["cap"])
    out = {"out": y.detach().to(torch.bfloat16)}
    if c["op"] == "layer":
        out["experts"] = ids
    if train:
        if c["op"] == "layer":  # in two steps, as the route's own case
            got = torch.autograd.grad(y, [leaves[n] for n in keys] + [w], state["dout"].float())
            out["dlogits"] = _row_grads(leaves["logits"], w, ids, got[-1], c).to(torch.bfloat16)
            got = got[:-1]
        else:
            got = torch.autograd.grad(y, [leaves[n] for n in keys + ["weights"]], state["dout"].float(), materialize_grads=True)
            out["dweights"] = got[-1].to(torch.bfloat16)
        out.update({"d" + n: v.to(torch.bfloat16) for n, v in zip(keys, got)})
    return out


def _row_grads(z, w, ids, dw, c):
    """Gradient of the logits, from the formulas."""
    z, w = z.detach(), w.detach()
    s, scale = _scores_plain(z, c["score"]), c["scale"]
    picked = s.gather(1, ids)
    mean = (dw * w).sum(-1, keepdim=True) / scale
    if c["score"] == "sigmoid":
        part = w * (1 - picked) * (dw - mean) if c["renorm"] else w * (1 - picked) * dw
        return torch.zeros_like(z).scatter_add(1, ids, part)
    if c["renorm"]:
        return torch.zeros_like(z).scatter_add(1, ids, w * (dw - mean))
    return s * (torch.zeros_like(z).scatter_add(1, ids, dw * scale) - mean * scale)


def _run_own(state, c, train):
    from khaosz_b200 import ops

    if c["op"] == "plan":
        p = ops.moe_plan(state["ids"], c["experts"])
        return {"counts": p.counts, "offsets": p.offsets, "slots": p.slots, "rows": p.rows}
    how = {} if c["op"] == "experts" else dict(score=c["score"], bias=state["bias"], n_groups=c["groups"], topk_groups=c["top_groups"],
                                               group_top=c["group_top"], renormalize=c["renorm"], scale=c["scale"])
    if c["op"] == "route":
        with torch.set_grad_enabled(train):
            z = _leaf(state["logits"]) if train else state["logits"]
            w, ids = ops.moe_route(z, c["k"], **how)
        out = {"weights": w.detach(), "experts": ids}
        if train:
            out["dlogits"], = torch.autograd.grad(w, [z], state["dweights"])
        return out
    keys = ["x", "gate", "up", "down"]
    with torch.set_grad_enabled(train):
        leaves = {n: _leaf(state[n]) if train else state[n] for n in keys}
        if c["op"] == "layer":
            leaves["logits"] = _leaf(state["logits"]) if train else state["logits"]
            w, ids = ops.moe_route(leaves["logits"], c["k"], dtype=torch.float32, **how)
        else:
            leaves["weights"] = _leaf(state["weights"]) if train else state["weights"]
            w, ids = leaves["weights"], state["ids"]
        y = ops.moe_experts(leaves["x"], w, ids, leaves["gate"], leaves["up"], leaves["down"], residual=state["residual"])
    out = {"out": y.detach()}
    if c["op"] == "layer":
        out["experts"] = ids
    if train:
        last = "logits" if c["op"] == "layer" else "weights"
        got = torch.autograd.grad(y, [leaves[n] for n in keys + [last]], state["dout"])
        out.update({"d" + n: v for n, v in zip(keys + [last], got)})
    return out


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    c = case
    t, e, k, op = c["tokens"], c["experts"], c["k"], c["op"]
    n, train = t * k, c.get("train", False)
    nbytes = flops = 0
    if op in ("route", "layer"):
        el = 2 if c["dtype"] == "bf16" else 4
        nbytes += t * e * el + n * (el + 8)
        flops += 8 * t * e
        if train:
            nbytes += n * el + t * e * el
            flops += 6 * t * e
    if op == "plan":
        nbytes += 8 * n + 4 * n + 4 * (2 * e + 1) + 4 * (n + (ALIGN - 1) * min(e, n))
        flops += n
    if op in ("experts", "layer"):
        d, f = c["dim"], c["ffn"]
        live = (t - int(t * c["drop"])) * k
        met = e * (1 - (1 - 1 / e) ** live)  # experts that so many assignments meet, on average
        nbytes += 2 * t * d * (2 + bool(c["residual"])) + 3 * d * f * 2 * met
        nbytes += n * 10 if op == "experts" else 0
        flops += 6 * live * d * f
        if train:
            nbytes += 2 * t * d * 2 + 3 * d * f * 2 * e + (2 * n if op == "experts" else 0)
            flops += 12 * live * d * f
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------
def _route_exact(z, bias, c):
    """(scores, weights, experts): k rounds of taking the largest."""
    z = z.double()
    t, e = z.shape
    if c["score"] == "sigmoid":
        s = torch.special.expit(z)
    else:
        s = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True)).nan_to_num(nan=0.0)
    pick = s.clone() if bias is None else s + bias.double()
    pick[torch.isneginf(z)] = -math.inf
    size = e // c["groups"]
    if c["groups"] > 1:
        score = torch.stack([torch.topk(pick[:, i * size:(i + 1) * size], min(c["group_top"], size), dim=1).values.sum(1) for i in range(c["groups"])], 1)
        open_ = torch.zeros_like(pick, dtype=torch.bool)
        for _ in range(c["top_groups"]):
            g = (score == torch.nan_to_num(score, nan=-math.inf, neginf=-math.inf).max(1, keepdim=True).values).int().argmax(1)
            score[torch.arange(t), g] = math.nan  # taken: it equals nothing any more
            open_ |= (torch.arange(e, device=z.device) // size)[None] == g[:, None]
        pick = pick.clamp(min=-1e6)
        pick[~open_] = -1e7
    ids = []
    for _ in range(c["k"]):
        i = (pick == torch.nan_to_num(pick, nan=-math.inf, neginf=-math.inf).max(1, keepdim=True).values).int().argmax(1)
        pick[torch.arange(t), i] = math.nan  # taken: it equals nothing any more
        ids.append(i)
    ids = torch.stack(ids, 1)
    w = torch.gather(s, 1, ids)
    if c["renorm"]:
        w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
    return s, w * c["scale"], ids


def _dlogits_exact(s, w, ids, dw, c):
    """Through the Jacobians: weights -> selected scores -> logits."""
    picked = torch.gather(s, 1, ids)
    ds = c["scale"] * dw
    if c["renorm"]:
        total = picked.sum(1, keepdim=True)
        ds = torch.nan_to_num((ds - (ds * picked).sum(1, keepdim=True) / total) / total, nan=0.0)
    full = torch.zeros_like(s).scatter_(1, ids, ds)
    if c["score"] == "sigmoid":
        return full * s * (1 - s)
    return s * (full - (full * s).sum(1, keepdim=True))


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None
    state = prepare(c, seed)
    out = {}
    if c["op"] in ("route", "layer"):
        s, w, ids = _route_exact(state["logits"], state["bias"], c)
        out["experts"] = None
        if c["op"] == "route":
            out["weights"] = w
            if c["train"]:
                out["dlogits"] = _dlogits_exact(s, w, ids, state["dweights"].double(), c)
            return out
    else:
        w, ids = state["weights"].double(), state["ids"]
    x = state["x"].double()
    y = torch.zeros_like(x) if state["residual"] is None else state["residual"].double()
    grads = {n: torch.zeros(state[n].shape, dtype=torch.float64, device=x.device) for n in ("x", "gate", "up", "down")} if c["train"] else {}
    dw = torch.zeros_like(w)
    for e in range(c["experts"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        wg, wu, wd, xe, we = state["gate"][e].double(), state["up"][e].double(), state["down"][e].double(), x[t], w[t, j][:, None]
        g, u = xe @ wg.T, xe @ wu.T
        sig = torch.sigmoid(g)
        h = g * sig * u
        y.index_add_(0, t, we * (h @ wd.T))
        if c["train"]:
            do = state["dout"].double()[t]
            grads["down"][e] = (we * do).T @ h
            dh = do @ wd
            dw[t, j] = (dh * h).sum(1)
            dg, du = we * dh * u * sig * (1 + g * (1 - sig)), we * dh * g * sig
            grads["gate"][e], grads["up"][e] = dg.T @ xe, du.T @ xe
            grads["x"].index_add_(0, t, dg @ wg + du @ wu)
    out["out"] = y
    if c["train"]:
        out.update({"d" + n: v for n, v in grads.items()})
        if c["op"] == "layer":
            out["dlogits"] = _dlogits_exact(s, w, ids, dw, c)
        else:
            out["dweights"] = dw
    return out
