"""Model configurations, dispatched by ``model_type`` (reference:
``astrai/config/model_config.py:9-92``; field names are the on-disk ``config.json`` contract)."""

from __future__ import annotations

import json
from dataclasses import dataclass
from typing import Any, Dict, Optional

from ..factory import BaseFactory
from .base import BaseConfig


class ConfigFactory(BaseFactory[BaseConfig]):
    """``ConfigFactory.load(raw_dict)`` -> the config class registered for ``model_type``."""

    DEFAULT_TYPE = "autoregressive_lm"

    @classmethod
    def load(cls, raw: Dict[str, Any]) -> BaseConfig:
        return cls.get_component_class(raw.get("model_type") or cls.DEFAULT_TYPE).from_dict(raw)


@dataclass
class BaseModelConfig(BaseConfig):
    model_type: Optional[str] = None

    @classmethod
    def from_file(cls, config_path: str):
        with open(config_path, "r") as fh:
            return cls.from_dict(json.load(fh))

    def to_file(self, config_path: str) -> None:
        payload = {k: v for k, v in self.to_dict().items() if v is not None}
        with open(config_path, "w") as fh:
            json.dump(payload, fh, indent=4)


@ConfigFactory.register("autoregressive_lm")
@dataclass
class AutoRegressiveLMConfig(BaseModelConfig):
    # trunk
    vocab_size: Optional[int] = None
    dim: Optional[int] = None
    n_layers: Optional[int] = None
    norm_eps: Optional[float] = None
    dim_ffn: Optional[int] = None
    tie_weight: Optional[bool] = None
    # positions
    max_len: Optional[int] = None
    rope_theta: Optional[float] = None
    rope_scaling: Optional[dict] = None
    # attention
    attn_type: str = "gqa"
    n_heads: Optional[int] = None
    n_kv_heads: Optional[int] = None
    use_qk_norm: Optional[bool] = None
    use_gated_attention: Optional[bool] = None
    # multi-head latent attention
    kv_lora_rank: Optional[int] = None
    qk_nope_head_dim: Optional[int] = None
    qk_rope_head_dim: Optional[int] = None
    # feed-forward
    ffn_type: str = "mlp"
    n_routed_experts: Optional[int] = None
    n_shared_experts: Optional[int] = None
    n_activated_experts: Optional[int] = None
    topk_method: Optional[str] = None        # "softmax" / "sigmoid": fused routing and grouped experts
    n_expert_groups: Optional[int] = None    # the rest with those two methods only
    n_limited_groups: Optional[int] = None
    router_bias: Optional[bool] = None
    router_scale: Optional[float] = None


@ConfigFactory.register("embedding")
@dataclass
class EncoderConfig(BaseModelConfig):
    vocab_size: Optional[int] = None
    dim: Optional[int] = None
    n_layers: Optional[int] = None
    norm_eps: Optional[float] = None
    dim_ffn: Optional[int] = None
    max_len: Optional[int] = None
    rope_theta: Optional[float] = None
    rope_scaling: Optional[dict] = None
    n_heads: Optional[int] = None
    n_kv_heads: Optional[int] = None
    use_qk_norm: Optional[bool] = None
    use_gated_attention: Optional[bool] = None
    pooling_type: Optional[str] = None
    normalize_embeddings: Optional[bool] = None
