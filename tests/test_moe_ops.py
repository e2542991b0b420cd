"""Sparse feed-forward operators on the CPU: the plain forms against the definition, refusals, gradients by differences."""
import pytest
import torch

from khaosz_b200 import ops
from moe_reference import plan as plan_ref
from moe_reference import route as route_ref
from moe_reference import route_grad

ROUTES = [
    dict(), dict(renorm=False), dict(sigmoid=True), dict(sigmoid=True, renorm=False, scale=2.5), dict(bias=True), dict(sigmoid=True, bias=True, groups=4, top_groups=2),
    dict(groups=2, top_groups=1, group_top=1), dict(groups=4, top_groups=3, bias=True, group_top=1, scale=0.5),
]


def _call(z, k, o, dtype=None):
    return ops.moe_route(z, k, score="sigmoid" if o.get("sigmoid") else "softmax", bias=o.get("bias"), n_groups=o.get("groups", 1),
                         topk_groups=o.get("top_groups", 1), group_top=o.get("group_top", 2), renormalize=o.get("renorm", True), scale=o.get("scale", 1.0), dtype=dtype)


@pytest.mark.parametrize("opts", ROUTES)
@pytest.mark.parametrize("masked", [False, True])
def test_route_matches_the_definition(opts, masked):
    torch.manual_seed(3)
    z = torch.randn(37, 24, dtype=torch.float64)
    if masked:
        z[torch.rand(37, 24) < 0.6] = -torch.inf
        z[5] = -torch.inf
    o = dict(opts, bias=torch.randn(24, dtype=torch.float64) * 0.1 if opts.get("bias") else None)
    if masked and o["bias"] is not None:
        o["bias"][3] = -torch.inf
    z.requires_grad_()
    w, ids = _call(z, 5, o)
    rw, rids = route_ref(z, 5, **o)
    if masked and o["bias"] is not None:
        rw = torch.where(o["bias"][rids] == -torch.inf, torch.zeros_like(rw), rw)
        if o.get("renorm", True):
            rw = torch.nan_to_num(rw / rw.sum(1, keepdim=True)) * o.get("scale", 1.0)
    assert torch.equal(ids, rids)
    # fp32 weights where the scores are fp32; these are 64-bit logits
    assert torch.allclose(w, rw, rtol=1e-12, atol=1e-300)
    g = torch.randn_like(w)
    (w * g).sum().backward()
    want = route_grad(z, ids, g, o.get("sigmoid", False), o["bias"], o.get("renorm", True), o.get("scale", 1.0))
    assert torch.allclose(z.grad, want, rtol=1e-9, atol=1e-12)


def test_route_ties_go_to_the_lowest_index_and_nan_rows_show():
    z = torch.zeros(3, 8)
    z[1, 5] = torch.nan
    z[2] = torch.finfo(torch.float32).min
    w, ids = ops.moe_route(z, 3)
    assert ids.tolist() == [[0, 1, 2]] * 3
    assert torch.isnan(w[1]).all() and torch.allclose(w[[0, 2]], torch.full((2, 3), 1 / 3))
    w = ops.moe_route(z, 3, score="sigmoid")[0]
    assert torch.isnan(w[1]).all() and torch.allclose(w[[0, 2]], torch.full((2, 3), 1 / 3))
    tiny = torch.tensor([[-200.0, -201.0, -300.0]])   # the scores are zero in fp32, their ratios are not
    assert torch.allclose(ops.moe_route(tiny, 2, score="sigmoid")[0], torch.softmax(tiny[:, :2], -1))


def test_route_refuses():
    z = torch.randn(4, 12)
    for kw in (dict(k=0), dict(k=13), dict(k=33), dict(k=2, score="tanh"), dict(k=2, n_groups=5), dict(k=2, n_groups=4, topk_groups=5), dict(k=2, n_groups=0),
               dict(k=7, n_groups=4, topk_groups=2), dict(k=2, n_groups=4, group_top=3), dict(k=2, bias=torch.zeros(11)), dict(k=2, bias=torch.zeros(12, dtype=torch.long))):
        with pytest.raises(ValueError):
            ops.moe_route(z, **kw)
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(4, 12, dtype=torch.long), 2)
    with pytest.raises(ValueError):
        ops.moe_route(torch.zeros(1, 1025), 2)
    w, ids = ops.moe_route(torch.zeros(0, 12), 2)
    assert w.shape == ids.shape == (0, 2)


@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (7, 3, 5), (40, 2, 64), (0, 2, 4)])
def test_plan_matches_a_loop(tokens, k, experts):
    torch.manual_seed(1)
    ids = torch.randint(-1, experts + 1, (tokens, k))
    p = ops.moe_plan(ids, experts)
    counts, offsets, slots, rows = plan_ref(ids, experts)
    assert p.counts.tolist() == counts and p.offsets.tolist() == offsets
    assert p.slots.shape == ids.shape and p.slots.reshape(-1).tolist() == slots and p.rows.tolist() == rows
    for got, size in ((p.tiles, 128), (p.pairs, 256)):
        tiles = got[1:1 + int(got[0, 0])].tolist()
        assert [(e, r) for e in range(experts) for r in range(offsets[e], offsets[e + 1], size)] == [(t[0], t[1]) for t in tiles]
        assert all(t[2] == offsets[t[0] + 1] for t in tiles)


def test_plan_refuses():
    for bad in (torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int16)):
        with pytest.raises(ValueError):
            ops.moe_plan(bad, 4)
    for n in (0, 1025):
        with pytest.raises(ValueError):
            ops.moe_plan(torch.zeros(3, 2, dtype=torch.long), n)


def _weights(E, F, D, dtype=torch.float64):
    return [torch.randn(*s, dtype=dtype) * 0.3 for s in ((E, F, D), (E, F, D), (E, D, F))]


def test_experts_match_a_loop_over_tokens_and_differences():
    torch.manual_seed(0)
    E, F, D, T, k = 4, 6, 5, 7, 2
    ws = [w.requires_grad_() for w in _weights(E, F, D)]
    x = torch.randn(T, D, dtype=torch.float64, requires_grad=True)
    w = torch.rand(T, k, dtype=torch.float64, requires_grad=True)
    res = torch.randn(T, D, dtype=torch.float64, requires_grad=True)
    ids = torch.randint(0, E - 1, (T, k))   # the last expert has no token
    ids[2] = ids[2, 0]                      # the same expert twice
    ids[4, 1] = -1                          # dropped
    out = ops.moe_experts(x, w, ids, *ws, residual=res)
    for t in range(T):
        want = res[t].clone()
        for j in range(k):
            e = int(ids[t, j])
            if e >= 0:
                g, u = ws[0][e] @ x[t], ws[1][e] @ x[t]
                want = want + w[t, j] * (ws[2][e] @ (g * torch.sigmoid(g) * u))
        assert torch.allclose(out[t], want)
    assert torch.autograd.gradcheck(lambda *a: ops.moe_experts(a[0], a[1], ids, a[3], a[4], a[5], residual=a[2]), (x, w, res, *ws))
    out.sum().backward()
    assert all(float(v.grad[-1].abs().max()) == 0 for v in ws)


def test_experts_take_sequences_of_matrices():
    torch.manual_seed(0)
    ws = _weights(3, 8, 16, torch.float32)
    x, w, ids = torch.randn(2, 4, 16), torch.rand(2, 4, 2), torch.randint(0, 3, (2, 4, 2))
    assert torch.equal(ops.moe_experts(x, w, ids, *ws), ops.moe_experts(x, w, ids, *(list(v) for v in ws)))


def test_experts_refuse():
    g, u, d = _weights(3, 8, 16, torch.float32)
    x, w, ids = torch.randn(4, 16), torch.rand(4, 2), torch.zeros(4, 2, dtype=torch.long)
    good = dict(x=x, weights=w, experts=ids, w_gate=g, w_up=u, w_down=d)
    ops.moe_experts(**good)
    for bad in (dict(x=torch.randn(4, 8)), dict(x=torch.randn(5, 16)), dict(weights=torch.rand(4, 3)), dict(experts=ids.float()), dict(w_up=u[:2]), dict(w_down=g),
                dict(w_gate=list(g)), dict(w_gate=g[0]), dict(residual=torch.randn(4, 8)), dict(plan=ops.moe_plan(ids[:2], 3)), dict(plan=ops.moe_plan(ids, 4)),
                dict(w_gate=[], w_up=[], w_down=[])):
        with pytest.raises(ValueError):
            ops.moe_experts(**{**good, **bad})
    assert ops.moe_experts(x[:0], w[:0], ids[:0], g, u, d).shape == (0, 16)


def test_route_then_experts_trains_on_the_cpu():
    torch.manual_seed(0)
    ws = [w.requires_grad_() for w in _weights(4, 8, 16, torch.float32)]
    x = torch.randn(9, 16, requires_grad=True)
    router = torch.randn(4, 16, requires_grad=True)
    w, ids = ops.moe_route(x @ router.t(), 2, score="sigmoid", bias=torch.zeros(4))
    ops.moe_experts(x, w, ids, *ws, residual=x).square().sum().backward()
    assert all(t.grad is not None and torch.isfinite(t.grad).all() for t in (x, router, *ws))
