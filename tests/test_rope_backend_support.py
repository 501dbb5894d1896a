"""For which models the backend says that it rotates and stores in one call (no GPU; the
engine's current config is a stand-in, vLLM is not importable here)."""
from __future__ import annotations

import sys
from types import ModuleType, SimpleNamespace

import pytest

from backend_cases import make_impl


def engine(monkeypatch, config):
    module = ModuleType("vllm.config")

    def get_current_vllm_config():
        assert config is not None, "no engine"
        return config

    module.get_current_vllm_config = get_current_vllm_config
    monkeypatch.setitem(sys.modules, "vllm.config", module)


@pytest.mark.parametrize("head,hf,supported", [
    (128, {}, True), (256, {}, True), (128, dict(rotary_dim=64), True), (128, dict(rotary_dim=24), False),
    (128, dict(rotary_dim=0), False), (128, dict(partial_rotary_factor=0.5), True), (128, dict(partial_rotary_factor=1.0), True),
    (128, dict(partial_rotary_factor=0.3), False), (256, dict(partial_rotary_factor=0.25), True),
    (128, dict(rotary_pct=0.25), True), (128, dict(rotary_pct=0.2), False), (128, dict(rotary_dim=None), True),
    (128, dict(rope_parameters=dict(rope_type="default", partial_rotary_factor=0.75)), True),
    (128, dict(rope_parameters=dict(rope_type="default", partial_rotary_factor=0.7)), False),
    (128, dict(rope_parameters=dict(full=dict(rope_theta=1e6), sliding=dict(partial_rotary_factor=0.55))), False),
    (128, dict(rope_parameters=None, rope_scaling=dict(partial_rotary_factor=0.5)), True),
])
def test_the_models_rotary_dim(monkeypatch, head, hf, supported):
    engine(monkeypatch, SimpleNamespace(model_config=SimpleNamespace(hf_text_config=SimpleNamespace(**hf))))
    assert make_impl(head=head).fused_rope_kvcache_supported() is supported


@pytest.mark.parametrize("config", [None, SimpleNamespace(), SimpleNamespace(model_config=None),
                                    SimpleNamespace(model_config=SimpleNamespace(hf_config=SimpleNamespace()))])
def test_no_model_to_ask(monkeypatch, config):
    engine(monkeypatch, config)
    assert make_impl().fused_rope_kvcache_supported()


def test_no_engine_at_all():
    assert make_impl().fused_rope_kvcache_supported()
