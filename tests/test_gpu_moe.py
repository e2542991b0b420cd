"""Sparse feed-forward operators on the GPU against their definition in 64 bits."""
import pytest
import torch

from khaosz_b200 import ops
from moe_reference import experts as experts_ref
from moe_reference import outside
from moe_reference import plan as plan_ref
from moe_reference import route as route_ref
from moe_reference import route_grad
from test_moe_ops import ROUTES, _call

pytestmark = pytest.mark.gpu


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


# fp32 scores: exp with an argument of at most 30 is off by (30 + 2) steps, the sum and the division by 3 more, in
# numerator and denominator: 2 * 36 * 2^-23 < 1e-5
RTOL = 1e-5


@pytest.mark.parametrize("opts", ROUTES)
@pytest.mark.parametrize("T,E,k,dtype", [(1, 8, 2, torch.bfloat16), (33, 24, 5, torch.float32), (70, 100, 6, torch.bfloat16), (19, 256, 8, torch.float32),
                                         (9, 520, 32, torch.float32), (5, 1024, 3, torch.bfloat16)])
@pytest.mark.parametrize("masked", [False, True])
def test_route(opts, T, E, k, dtype, masked):
    g = _gen(T + E)
    z = (torch.randn(T, E, device="cuda", generator=g) * 2).to(dtype)
    k = min(k, E // opts.get("groups", 1) * opts.get("top_groups", 1))
    o = dict(opts, bias=torch.randn(E, device="cuda", generator=g) * 0.1 if opts.get("bias") else None)
    if masked:
        z[torch.rand(T, E, device="cuda", generator=g) < 0.7] = -torch.inf
        z[0] = -torch.inf
    z.requires_grad_()
    w, ids = _call(z, k, o)
    rw, rids = route_ref(z, k, **o)
    assert w.dtype == dtype and torch.equal(ids.cpu(), rids)
    tol = RTOL + (2.0 ** -8 if dtype == torch.bfloat16 else 0)
    assert ((w.double().cpu() - rw).abs() <= tol * rw).all()
    dw = torch.randn(T, k, device="cuda", generator=g).to(dtype)
    dz, = torch.autograd.grad(w, z, dw)
    want = route_grad(z, rids, dw, o.get("sigmoid", False), o["bias"], o.get("renorm", True), o.get("scale", 1.0))
    # dz is w (or p) times a difference of gradients whose terms are bounded by the largest: the difference is off by RTOL of that bound
    scale = o.get("scale", 1.0)
    unit = rw.sum(1, keepdim=True).clamp_min(1e-30) if o.get("sigmoid") and not o.get("renorm", True) else torch.full((T, 1), float(scale))
    slack = RTOL * 4 * unit * dw.double().cpu().abs().amax(1, keepdim=True)
    lim = slack + (2.0 ** -8 if dtype == torch.bfloat16 else 0) * want.abs()
    assert ((dz.double().cpu() - want).abs() <= lim).all()


def test_route_special_rows_and_layouts():
    z = torch.zeros(6, 40, device="cuda")
    z[1, 7], z[2, 3] = torch.nan, torch.inf
    z[3] = torch.finfo(torch.float32).min
    z[4, ::2] = -0.0
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(40, device="cuda")):
            w, ids = ops.moe_route(z, 4, score=score, bias=bias)
            assert torch.isnan(w[1]).all() and (torch.isnan(w[2]).all() == (score == "softmax"))
            assert ids[[0, 1, 4]].tolist() == [[0, 1, 2, 3]] * 3
            assert torch.allclose(w[[0, 4]], torch.full((2, 4), 0.25, device="cuda"))
    bias = torch.zeros(40, device="cuda")
    bias[:38] = -torch.inf   # two experts are left for four slots
    w, ids = ops.moe_route(z, 4, bias=bias)
    assert ids[0].tolist() == [38, 39, 0, 1] and w[0].tolist() == [0.5, 0.5, 0.0, 0.0]
    # rows of a wider buffer, a transposed one, leading dimensions, a NaN bias
    wide = torch.randn(2, 3, 64, device="cuda")
    a = ops.moe_route(wide[..., :40], 3)
    b = ops.moe_route(wide[..., :40].contiguous(), 3)
    assert a[0].shape == (2, 3, 3) and all(torch.equal(u, v) for u, v in zip(a, b))
    t = torch.randn(40, 6, device="cuda")
    assert torch.equal(ops.moe_route(t.t(), 3)[1], ops.moe_route(t.t().contiguous(), 3)[1])
    bias[0] = torch.nan
    assert torch.isnan(ops.moe_route(z, 4, bias=bias)[0]).all()
    assert ops.moe_route(z[:0], 4)[0].shape == (0, 4)
    assert ops.moe_route(z.bfloat16(), 4, dtype=torch.float32)[0].dtype == torch.float32


def test_route_close_scores_are_told_apart():
    """Scores plus bias that differ by less than fp32 resolves are ordered as 64 bits order them."""
    T, E = 512, 64
    g = _gen(5)
    z = torch.randn(T, E, device="cuda", generator=g)
    bias = -torch.sigmoid(z.double()).mean(0).float()
    near = (torch.randn(T, 1, device="cuda", generator=g) + torch.randn(T, E, device="cuda", generator=g) * 1e-6)
    for score in ("softmax", "sigmoid"):
        for kw in (dict(), dict(n_groups=8, topk_groups=3)):
            w, ids = ops.moe_route(near, 6, score=score, bias=bias * 0, **kw)
            rid = route_ref(near, 6, sigmoid=score == "sigmoid", bias=bias * 0, groups=kw.get("n_groups", 1), top_groups=kw.get("topk_groups", 1))[1]
            assert torch.equal(ids.cpu(), rid)


@pytest.mark.parametrize("T,k,E,dtype", [(1, 1, 1, torch.long), (7, 3, 5, torch.int32), (513, 8, 256, torch.long), (600, 7, 1024, torch.long),
                                         (2048, 2, 3, torch.int32), (4097, 1, 2, torch.long), (5000, 8, 129, torch.long)])
def test_plan(T, k, E, dtype):
    g = _gen(T)
    ids = torch.randint(-1, E + 1, (T, k), device="cuda", generator=g, dtype=dtype)
    p, again = ops.moe_plan(ids, E), ops.moe_plan(ids, E)
    counts, offsets, slots, rows = plan_ref(ids, E)
    assert p.counts.tolist() == counts and p.offsets.tolist() == offsets
    assert p.slots.reshape(-1).tolist() == slots and p.rows.tolist() == rows
    n_tiles = int(p.tiles[0, 0])
    assert n_tiles + 1 <= p.tiles.shape[0]
    want = [[e, r, offsets[e + 1], 0] for e in range(E) for r in range(offsets[e], offsets[e + 1], 128)]
    assert p.tiles[1:1 + n_tiles].tolist() == want
    assert all(torch.equal(a, b) for a, b in zip(p[:4], again[:4]))


def test_plan_drops_everything_and_takes_far_indices():
    ids = torch.full((9, 2), -1, device="cuda")
    ids[3, 0], ids[4, 1] = 2 ** 40 + 1, -2 ** 50
    p = ops.moe_plan(ids, 4)
    assert p.counts.tolist() == [0] * 4 and p.slots.unique().tolist() == [-1] and p.rows.unique().tolist() == [-1] and int(p.tiles[0, 0]) == 0


SIZES = [  # tokens, dim, ffn, experts, k, share dropped
    (1, 64, 64, 4, 2, 0.0), (2, 8, 8, 1, 1, 0.0), (5, 72, 40, 3, 3, 0.2), (130, 136, 200, 5, 2, 0.1), (333, 520, 184, 10, 3, 0.05), (64, 256, 320, 64, 6, 0.0),
    (700, 264, 136, 2, 2, 0.0), (300, 128, 264, 7, 1, 0.5),
]


def _inputs(T, D, F, E, k, drop, seed=0):
    g = _gen(seed)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).bfloat16()  # noqa: E731
    x, res, dout = rnd(T, D), rnd(T, D), rnd(T, D)
    ws = rnd(E, F, D, scale=D ** -0.5), rnd(E, F, D, scale=D ** -0.5), rnd(E, D, F, scale=F ** -0.5)
    w = torch.rand(T, k, device="cuda", generator=g).bfloat16()
    ids = torch.randint(0, E, (T, k), device="cuda", generator=g)
    if E > 2:
        ids[ids == 1] = 0  # an expert without tokens
    ids[torch.rand(T, k, device="cuda", generator=g) < drop] = -1
    return x, w, ids, ws, res, dout


def _check(got, ref, names, dtypes=None):
    for n in names:
        bad = outside(got[n], *ref[n], dtype=(dtypes or {}).get(n, torch.bfloat16))
        assert bad == 0, f"{n}: {bad} of {got[n].numel()} values are further off than the roundings allow"


@pytest.mark.parametrize("T,D,F,E,k,drop", SIZES)
def test_experts_forward(T, D, F, E, k, drop):
    x, w, ids, ws, res, _ = _inputs(T, D, F, E, k, drop)
    ref = experts_ref(x, w, ids, *ws, residual=res)
    out = ops.moe_experts(x, w, ids, *ws, residual=res)
    _check({"out": out}, ref, ["out"])
    plain = ops.moe_experts(x, w.float(), ids.int(), *ws, plan=ops.moe_plan(ids.int(), E))
    _check({"out": plain}, experts_ref(x, w, ids, *ws), ["out"])
    ops.raise_on_device_error()


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D,F,E,k,drop", SIZES)
def test_experts_gradients(T, D, F, E, k, drop, w_dtype):
    x, w, ids, ws, res, dout = _inputs(T, D, F, E, k, drop)
    leaves = [t.detach().requires_grad_() for t in (x, w.to(w_dtype), *ws, res)]
    out = ops.moe_experts(leaves[0], leaves[1], ids, *leaves[2:5], residual=leaves[5])
    grads = torch.autograd.grad(out, leaves, dout)
    got = dict(zip(("dx", "dw", "dgate", "dup", "ddown"), grads), out=out)
    ref = experts_ref(x, w, ids, *ws, residual=res, dout=dout)
    _check(got, ref, list(got), {"dw": w_dtype})
    assert torch.equal(grads[5], dout)
    again = torch.autograd.grad(ops.moe_experts(leaves[0], leaves[1], ids, *leaves[2:5], residual=leaves[5]), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # no order of additions depends on timing
    ops.raise_on_device_error()
