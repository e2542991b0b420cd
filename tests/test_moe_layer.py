"""The mixture-of-experts layer with the fused routing methods (CPU): against the written-out formula, in a model, in a configuration."""
import pytest
import torch

from conftest import tiny_config
from khaosz_b200 import AutoRegressiveLM, AutoRegressiveLMConfig
from khaosz_b200.models import inject_lora
from khaosz_b200.models.components.ffn import DeepSeekMoE
from moe_reference import route as route_ref

KINDS = [dict(topk_method="softmax"), dict(topk_method="sigmoid", router_scale=2.5),
         dict(topk_method="sigmoid", router_bias=True, n_expert_groups=4, n_limited_groups=2)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shared", [0, 1, 2])
def test_fused_layer_matches_a_per_token_loop(kind, shared):
    torch.manual_seed(4)
    moe = DeepSeekMoE(16, 24, n_routed_experts=8, n_shared_experts=shared, n_activated_experts=3, **kind)
    if moe.router_bias is not None:
        moe.router_bias.copy_(torch.randn(8) * 0.2)
    x, res = torch.randn(2, 6, 16), torch.randn(2, 6, 16)
    flat = x.reshape(-1, 16)
    w, ids = route_ref(moe.router(flat), 3, sigmoid=kind["topk_method"] == "sigmoid", bias=moe.router_bias, groups=kind.get("n_expert_groups", 1),
                       top_groups=kind.get("n_limited_groups", 1), scale=kind.get("router_scale", 1.0))
    want = res.reshape(-1, 16).clone()
    for t in range(12):
        for j in range(3):
            want[t] += w[t, j].float() * moe.routed_experts[int(ids[t, j])](flat[t:t + 1])[0]
        if shared:
            want[t] += sum(e(flat[t:t + 1])[0] for e in moe.shared_experts) / shared
    got = moe(x, residual=res)
    assert torch.allclose(got, want.view(2, 6, 16), atol=1e-5)
    assert torch.allclose(moe(x), got - res, atol=1e-5)
    got.square().sum().backward()
    assert moe.router.weight.grad is not None and any(e.down.weight.grad is not None for e in moe.routed_experts)


def test_greedy_routing_keeps_its_rule_and_refuses_the_new_fields():
    torch.manual_seed(0)
    moe = DeepSeekMoE(16, 24, n_routed_experts=4, n_shared_experts=1, n_activated_experts=2)
    x = torch.randn(5, 16)
    w, ids = moe.route(x)
    probs = torch.softmax(x @ moe.router.weight.t(), -1)
    top = probs.topk(2)
    assert torch.equal(ids, top.indices) and torch.equal(w, top.values / top.values.sum(-1, keepdim=True))
    for kw in (dict(router_bias=True), dict(n_expert_groups=2), dict(n_limited_groups=1), dict(router_scale=2.0)):
        with pytest.raises(ValueError):
            DeepSeekMoE(16, 24, n_routed_experts=4, **kw)


@pytest.mark.parametrize("kind", KINDS)
def test_model_configuration_round_trip_and_training(kind, tmp_path):
    cfg = tiny_config(ffn_type="moe", n_routed_experts=8, n_shared_experts=1, n_activated_experts=2, **kind)
    cfg.to_file(str(tmp_path / "config.json"))
    again = AutoRegressiveLMConfig.from_file(str(tmp_path / "config.json"))
    assert again.to_dict() == cfg.to_dict()
    model = AutoRegressiveLM(again)
    keys = [k for k in model.state_dict() if k.endswith("router_bias")]
    assert bool(keys) == bool(kind.get("router_bias"))
    ids = torch.randint(0, cfg.vocab_size, (2, 12))
    model(ids)["logits"].square().mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)
    assert all(p.grad is not None for n, p in model.named_parameters() if "router" in n or "shared" in n)
    fresh = AutoRegressiveLM(again)
    fresh.load_state_dict(model.state_dict())
    assert torch.equal(fresh(ids)["logits"], model(ids)["logits"])


def test_adapters_on_the_experts_keep_working():
    torch.manual_seed(0)
    model = AutoRegressiveLM(tiny_config(ffn_type="moe", n_routed_experts=4, n_shared_experts=1, n_activated_experts=2, topk_method="sigmoid"))
    ids = torch.randint(0, 100, (1, 7))
    before = model(ids)["logits"]
    inject_lora(model, r=2, alpha=4, target_modules=("down", "gate", "up"))
    assert torch.allclose(model(ids)["logits"], before, atol=1e-5)   # adapters start at zero
