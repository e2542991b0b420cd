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
            assert torch.allclose(w[[0, 3, 4]], torch.full((3, 4), 0.25, device="cuda"))
    tiny = torch.tensor([[-200.0, -201.0, -300.0]], device="cuda")   # the scores are zero in fp32, their ratios are not
    assert torch.allclose(ops.moe_route(tiny, 2, score="sigmoid")[0], torch.softmax(tiny[:, :2], -1), rtol=1e-5)
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
    for tiles, size in ((p.tiles, 128), (p.pairs, 256)):
        n_tiles = int(tiles[0, 0])
        assert n_tiles + 1 <= tiles.shape[0]
        assert tiles[1:1 + n_tiles].tolist() == [[e, r, offsets[e + 1], 0] for e in range(E) for r in range(offsets[e], offsets[e + 1], size)]
    assert all(torch.equal(a, b) for a, b in zip(p[:4], again[:4]))


@pytest.mark.parametrize("T,k,E", [(140000, 4, 1024), (2_500_000, 1, 7), (70000, 8, 200)])
def test_plan_of_many_assignments(T, k, E):
    """Against a stable sort: the loop of the reference is too slow here."""
    ids = torch.randint(-1, E, (T, k), device="cuda", generator=_gen(T))
    p = ops.moe_plan(ids, E)
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=E)
    offsets = torch.cat([counts.new_zeros(1), ((counts + 15) // 16 * 16).cumsum(0)])
    order = torch.argsort(flat, stable=True)[int((flat < 0).sum()):]
    rows = offsets[flat[order]] + torch.arange(order.numel(), device="cuda") - (counts.cumsum(0) - counts)[flat[order]]
    slots = torch.full_like(flat, -1)
    slots[order] = rows
    assert torch.equal(p.counts.long(), counts) and torch.equal(p.offsets.long(), offsets)
    assert torch.equal(p.slots.reshape(-1).long(), slots)
    back = torch.full_like(p.rows, -1)
    back[rows] = order.int()
    assert torch.equal(p.rows, back)


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


@pytest.fixture(params=["one CTA", "pairs"])
def form(request, monkeypatch):
    """Both forms of the grouped products, whatever the rule between them says of the sizes."""
    from khaosz_b200.ops import moe

    monkeypatch.setattr(moe, "_use_pairs", lambda n, E: request.param == "pairs")


def _check(got, ref, names, dtypes=None):
    for n in names:
        bad = outside(got[n], *ref[n], dtype=(dtypes or {}).get(n, torch.bfloat16))
        assert bad == 0, f"{n}: {bad} of {got[n].numel()} values are further off than the roundings allow"


@pytest.mark.parametrize("T,D,F,E,k,drop", SIZES)
def test_experts_forward(T, D, F, E, k, drop, form):
    x, w, ids, ws, res, _ = _inputs(T, D, F, E, k, drop)
    ref = experts_ref(x, w, ids, *ws, residual=res)
    out = ops.moe_experts(x, w, ids, *ws, residual=res)
    _check({"out": out}, ref, ["out"])
    plain = ops.moe_experts(x, w.float(), ids.int(), *ws, plan=ops.moe_plan(ids.int(), E))
    _check({"out": plain}, experts_ref(x, w, ids, *ws), ["out"])
    ops.raise_on_device_error()


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D,F,E,k,drop", SIZES)
def test_experts_gradients(T, D, F, E, k, drop, w_dtype, form):
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


@pytest.mark.parametrize("T,E,k", [(900, 64, 2), (900, 4, 4), (3, 16, 5), (4, 8, 4), (40, 300, 8)])
def test_experts_all_tokens_at_one_expert_or_spread_thin(T, E, k, form):
    x, w, ids, ws, res, dout = _inputs(T, 64, 72, E, k, 0.0)
    ids[:] = E - 1  # the same expert in every slot of every token
    leaves = [t.detach().requires_grad_() for t in (x, w, *ws)]
    out = ops.moe_experts(leaves[0], leaves[1], ids, *leaves[2:])
    got = dict(zip(("dx", "dw", "dgate", "dup", "ddown"), torch.autograd.grad(out, leaves, dout)), out=out)
    _check(got, experts_ref(x, w, ids, *ws, dout=dout), list(got))
    with torch.no_grad():
        _check({"out": ops.moe_experts(x, w, ids, *ws)}, experts_ref(x, w, ids, *ws), ["out"])
    ids[:] = -1
    assert torch.equal(ops.moe_experts(x, w, ids, *ws, residual=res), res)
    out = ops.moe_experts(leaves[0], leaves[1], ids, *leaves[2:])
    assert all(int(v.count_nonzero()) == 0 for v in (out, *torch.autograd.grad(out, leaves, dout)))


@pytest.mark.parametrize("T", [3, 200])
def test_experts_layouts(T):
    """Rows of wider buffers, gate and up as halves of one tensor, transposed and odd-pitched weights, leading dimensions."""
    D, F, E, k = 128, 72, 6, 2
    x, w, ids, ws, res, dout = _inputs(T, D, F, E, k, 0.1)
    want = ops.moe_experts(x, w, ids, *ws, residual=res)
    wide = torch.zeros(T, 3 * D, device="cuda", dtype=torch.bfloat16)
    wide[:, D:2 * D], wide[:, 2 * D:] = x, res
    both = torch.cat(ws[:2], 1).contiguous()
    turned = ws[2].transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(E, F, D + 1, device="cuda", dtype=torch.bfloat16)
    odd[..., 1:] = ws[1]
    for up in (both[:, F:], odd[..., 1:]):
        leaves = [t.detach().requires_grad_() for t in (wide, w, both, up, turned)]
        args = (leaves[0][:, D:2 * D], leaves[1], ids, leaves[2][:, :F], leaves[3], leaves[4])
        with torch.no_grad():
            assert torch.equal(ops.moe_experts(*args, residual=wide[:, 2 * D:]), want)
        out = ops.moe_experts(*(a.unflatten(0, (1, T)) if a.dim() == 2 else a for a in args), residual=leaves[0][:, 2 * D:].unflatten(0, (1, T)))
        assert out.shape == (1, T, D)
        grads = torch.autograd.grad(out, leaves, dout.view(1, T, D).expand(1, T, D))
        ref = experts_ref(x, w, ids, *ws, residual=res, dout=dout)
        got = {"dx": grads[0][:, D:2 * D], "dw": grads[1], "dgate": grads[2][:, :F], "dup": grads[3], "ddown": grads[4]}
        _check(got, ref, list(got))
        assert torch.equal(grads[0][:, 2 * D:], dout) and float(grads[0][:, :D].float().abs().max()) == 0


@pytest.mark.parametrize("T", [1, 2, 60])
def test_experts_leading_dimensions_and_single_rows_run_on_the_kernels(T):
    x, w, ids, ws, res, dout = _inputs(T, 64, 72, 6, 2, 0.0)
    want = ops.moe_experts(x, w.float(), ids, *ws, residual=res)
    before = ops.launch_count()
    lead = lambda t: t.unflatten(0, (1, T))  # noqa: E731
    assert torch.equal(ops.moe_experts(lead(x), lead(w.float()), lead(ids), *ws, residual=lead(res))[0], want)
    assert ops.launch_count() > before
    if T == 1:   # one row of any pitch
        odd = lambda t: t.reshape(-1, 1).clone().t()  # noqa: E731
        assert odd(x).stride() == (1, 1)
        assert torch.equal(ops.moe_experts(odd(x), w.float(), ids, *ws, residual=odd(res)), want)
        leaf = odd(x).detach().requires_grad_()
        out = ops.moe_experts(leaf, w, ids, *ws)
        out.backward(odd(dout))
        _check({"dx": leaf.grad}, experts_ref(x, w, ids, *ws, dout=dout), ["dx"])


def test_second_derivatives_are_refused():
    x, w, ids, ws, res, dout = _inputs(30, 64, 72, 6, 2, 0.0)
    x.requires_grad_()
    z = torch.randn(30, 6, device="cuda", requires_grad=True)
    for f, leaf in ((lambda: ops.moe_experts(x, w, ids, *ws).float().square().sum(), x), (lambda: ops.moe_route(z, 2)[0].square().sum(), z)):
        g, = torch.autograd.grad(f(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_experts_broadcast_gradient_and_frozen_parts():
    x, w, ids, ws, res, dout = _inputs(50, 64, 64, 5, 2, 0.0)
    ref = experts_ref(x, w, ids, *ws, dout=torch.ones_like(dout))
    names = ("dx", "dw", "dgate", "dup", "ddown")
    for wanted in ((0,), (1,), (2,), (4,), (0, 4), (0, 1, 2, 3, 4)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w, *ws))]
        out = ops.moe_experts(leaves[0], leaves[1], ids, *leaves[2:])
        grads = torch.autograd.grad(out.sum(), [leaves[i] for i in wanted])   # a gradient of stride 0
        _check(dict(zip([names[i] for i in wanted], grads)), ref, [names[i] for i in wanted])


def test_experts_bad_values_stay_where_they_are():
    for T in (6, 300):
        x, w, ids, ws, res, dout = _inputs(T, 64, 64, 8, 2, 0.0)
        with torch.no_grad():
            clean = ops.moe_experts(x, w, ids, *ws)
            x[1, 3], x[2, 5] = torch.nan, torch.inf
            out = ops.moe_experts(x, w, ids, *ws)
        keep = torch.ones(T, dtype=torch.bool, device="cuda")
        keep[1:3] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[1]).all() and not torch.isfinite(out[2]).all()


def test_sequences_read_in_place_and_accumulate_into_flat_gradients():
    from khaosz_b200.models.components.ffn import DeepSeekMoE
    from khaosz_b200.utils import FlatParameters

    torch.manual_seed(0)
    moe = DeepSeekMoE(128, 72, n_routed_experts=6, n_shared_experts=1, n_activated_experts=2, topk_method="sigmoid", router_bias=True).cuda().bfloat16()
    x = torch.randn(300, 128, device="cuda").bfloat16()
    plain = moe(x)
    plain.backward(torch.ones_like(plain))
    grads = {n: p.grad.clone() for n, p in moe.named_parameters() if p.grad is not None}
    moe.zero_grad(set_to_none=True)
    flat = FlatParameters(moe)
    packed = moe(x)
    assert torch.equal(packed, plain)
    stacks = moe._expert_weights()
    from khaosz_b200.ops.moe import _uniform

    assert all(_uniform(s) is not None and _uniform(s).data_ptr() == s[0].data_ptr() for s in stacks)
    packed.backward(torch.ones_like(packed))
    for n, p in moe.named_parameters():
        if "routed" in n:
            assert torch.equal(p.main_grad, grads.get(n, torch.zeros_like(p))), n
    first = flat.grad.clone()
    out = moe(x)
    out.backward(torch.ones_like(out))
    for n, p in moe.named_parameters():
        if "routed" in n:   # one more rounding: the second gradient is added in fp32 to the stored first one
            assert torch.equal(p.main_grad, (grads[n].float() * 2).bfloat16()), n
    assert torch.isfinite(first).all()


def _graph_of(f):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


@pytest.mark.parametrize("T", [2, 150])
def test_captured_forward_follows_its_inputs_and_graphs_do_not_share_scratch(T):
    E, k, D, F = 8, 2, 128, 136
    x, w, ids, ws, res, _ = _inputs(T, D, F, E, k, 0.0)
    z = torch.randn(T, E, device="cuda")

    def step():
        with torch.no_grad():
            a, b = ops.moe_route(z, k, score="sigmoid", bias=torch.zeros(E, device="cuda"), dtype=torch.float32)
            return ops.moe_experts(x, a, b, *ws, residual=res)

    g1, o1 = _graph_of(step)
    g2, o2 = _graph_of(step)
    for seed in range(3):
        z.copy_(torch.randn(T, E, device="cuda", generator=_gen(seed)))
        x.copy_(torch.randn(T, D, device="cuda", generator=_gen(seed + 9)))
        want = step()
        for g in (g1, g2, g1):
            g.replay()
        assert torch.equal(o1, want) and torch.equal(o2, want)


def test_captured_training_step():
    x, w, ids, ws, res, dout = _inputs(200, 128, 136, 8, 2, 0.0)
    z = torch.randn(200, 8, device="cuda").bfloat16()
    leaves = [t.detach().requires_grad_() for t in (x, z, *ws)]

    def step():
        a, b = ops.moe_route(leaves[1], 2, dtype=torch.float32)
        out = ops.moe_experts(leaves[0], a, b, *leaves[2:])
        return torch.autograd.grad(out, leaves, dout)

    g, got = _graph_of(step)
    for seed in range(2):
        with torch.no_grad():
            leaves[1].copy_(torch.randn(200, 8, device="cuda", generator=_gen(seed)))
        want = step()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_behind_a_joined_side_stream():
    """The first launch of a call follows two streams at once in the recorded graph."""
    x, w, ids, ws, res, _ = _inputs(150, 128, 136, 8, 2, 0.0)
    side = torch.cuda.Stream()

    def step():
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = w * 2
        a = x * 2
        here.wait_stream(side)
        with torch.no_grad():
            return ops.moe_experts(a, b, ids, *ws, residual=res), ops.moe_experts(a[:3], b[:3], ids[:3], *ws)

    g, got = _graph_of(step)
    x.mul_(0.5)
    want = step()
    g.replay()
    assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_streams_run_side_by_side():
    sets = [_inputs(T, 128, 136, 8, 2, 0.1, seed=T) for T in (5, 120, 260, 333)]
    want = [ops.moe_experts(x, w, ids, *ws, residual=res) for x, w, ids, ws, res, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, (x, w, ids, ws, res, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(ops.moe_experts(x, w, ids, *ws, residual=res))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_other_types_take_the_plain_form():
    x, w, ids, ws, res, _ = _inputs(20, 64, 72, 5, 2, 0.1)
    want = experts_ref(x, w, ids, *ws, residual=res)["out"][0]
    for dt, tol in ((torch.float32, 1e-5), (torch.float16, 2e-3), (torch.float64, 1e-12)):
        got = ops.moe_experts(x.to(dt), w.to(dt), ids, *(v.to(dt) for v in ws), residual=res.to(dt))
        assert got.dtype == dt and ((got.double() - want).norm() <= tol * want.norm())
    narrow = ops.moe_experts(x[:, :60], w, ids, ws[0][..., :60], ws[1][..., :60], ws[2][:, :60])
    assert narrow.shape == (20, 60) and torch.isfinite(narrow).all()
    z = torch.randn(7, 12, device="cuda", dtype=torch.float16)
    assert ops.moe_route(z, 3)[0].dtype == torch.float16


@pytest.mark.parametrize("kind", [dict(topk_method="softmax"), dict(topk_method="sigmoid", router_bias=True, n_expert_groups=4, n_limited_groups=2, router_scale=2.0)])
def test_model_trains_captured_and_serves_captured(kind):
    from khaosz_b200 import AutoRegressiveLM, AutoRegressiveLMConfig
    from khaosz_b200.inference.core.cache import KVCache
    from khaosz_b200.inference.core.executor import Executor
    from khaosz_b200.inference.core.task import Task

    torch.manual_seed(0)
    cfg = AutoRegressiveLMConfig(vocab_size=512, dim=256, n_layers=2, norm_eps=1e-5, dim_ffn=136, tie_weight=True, max_len=128, rope_theta=1e4, n_heads=2,
                                 n_kv_heads=1, ffn_type="moe", n_routed_experts=8, n_shared_experts=1, n_activated_experts=2, **kind)
    model = AutoRegressiveLM(cfg).cuda().bfloat16()
    model.pack_parameters(with_grad=False)
    ids = torch.randint(0, 512, (2, 64), device="cuda")

    def loss():
        return ops.cross_entropy(model(ids)["logits"].reshape(-1, 512), ids.reshape(-1))

    want = torch.autograd.grad(loss(), [p for p in model.parameters()])
    g, got = _graph_of(lambda: torch.autograd.grad(loss(), [p for p in model.parameters()]))
    g.replay()
    for a, b in zip(got, want):  # the embedding's gradient is summed by atomics: not bit-exact
        assert (a.float() - b.float()).norm() <= 1e-2 * b.float().norm() + 1e-6
    # a decode step is recorded and gives what plain launches give
    outs = []
    for graphs in (False, True):
        cache = KVCache(2, 32, 16, 1, 128, torch.device("cuda"), torch.bfloat16)
        ex = Executor(model, None, cache, torch.device("cuda"), torch.bfloat16, max_seq_len=96, cuda_graphs=graphs)
        tasks = [Task(f"t{i}", list(range(5 + i, 25 + i)), max_tokens=8, temperature=1.0, top_k=1, top_p=1.0) for i in range(3)]
        for t in tasks:
            assert cache.task_alloc(t.task_id, t.prompt_ids)
        for t, tok in zip(tasks, ex.execute_prefill(tasks, 20)):
            t.output_ids.append(tok)
            t.input_tokens = 20
        for _ in range(5):
            for t in tasks:
                assert cache.task_extend(t.task_id, t.next_pos - 1)
            for t, tok in zip(tasks, ex.execute_decode(tasks)):
                t.output_ids.append(tok)
        outs.append([t.output_ids for t in tasks])
        assert not graphs or (ex.cuda_graphs and any(s.graph is not None for s in ex._slots.values()))
    assert outs[0] == outs[1]
    ops.raise_on_device_error()


def test_trainer_steps_recorded_and_plain_agree():
    """Optimizer steps of a mixture-of-experts model through an executor: the recorded micro-step (accumulated into the flat
    gradient buffer) against plain launches.  The embedding's gradient is summed by atomics, so the two runs may part by
    roundings; a bf16 loss of the same weights agrees to a few steps."""
    from khaosz_b200 import AutoRegressiveLM, AutoRegressiveLMConfig
    from khaosz_b200.parallel import ExecutorFactory
    from khaosz_b200.trainer import FusedAdamW, StrategyFactory

    def run(cuda_graph):
        torch.manual_seed(0)
        cfg = AutoRegressiveLMConfig(vocab_size=512, dim=256, n_layers=2, norm_eps=1e-5, dim_ffn=136, tie_weight=True, max_len=128, rope_theta=1e4, n_heads=2,
                                     n_kv_heads=1, ffn_type="moe", n_routed_experts=8, n_shared_experts=1, n_activated_experts=2, topk_method="sigmoid",
                                     router_bias=True)
        model = AutoRegressiveLM(cfg).to(device="cuda", dtype=torch.bfloat16)
        ex = ExecutorFactory.create("none", grad_accum_steps=2, cuda_graph=cuda_graph)
        opt = FusedAdamW(model.parameters(), lr=1e-3, betas=(0.9, 0.95), weight_decay=0.01)
        model, opt, _, _ = ex.prepare(model, opt, None, None)
        strategy = StrategyFactory.create("seq", model, "cuda", label_smoothing=0.0)
        losses = []
        for step in range(4):
            for micro in range(2):
                g = _gen(10 * step + micro)
                ids = torch.randint(0, 512, (2, 65), device="cuda", generator=g)
                with ex.accumulate(model):
                    losses.append(float(ex.micro_step(strategy, {"input_ids": ids[:, :-1], "target_ids": ids[:, 1:]})))
                    if ex.sync_gradients:
                        opt.fused_clip(1.0)
                        opt.step()
                        opt.zero_grad()
        recorded = cuda_graph and any("graph" in e for e in ex._graphed.entries.values())
        return losses, recorded

    plain, _ = run(False)
    graphed, recorded = run(True)
    assert recorded
    assert all(abs(a - b) <= 2.0 ** -6 * abs(a) for a, b in zip(plain, graphed)), (plain, graphed)
    ops.raise_on_device_error()
