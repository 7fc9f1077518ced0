"""Projections held as int8 codes, on the host: what a model keeps, saves, loads and hands out.  The quantiser and the product
are restated in plain torch (the kernels have no CPU path)."""
import pytest
import torch

from oracle import kv8_oracle as ko


def _quant_rows(x):
    codes, scale = ko.quantise(x.double()[:, None], 1, "int8")
    return codes[:, 0].to(torch.int8), scale[:, 0].float()


def _linear_w8a8(x8, x_scale, w8, w_scale, *, out_dtype):
    return ko.linear(x8, x_scale, w8, w_scale).to(out_dtype)


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    from omnikv_b200 import ops
    monkeypatch.setattr(ops, "quant_rows", _quant_rows)
    monkeypatch.setattr(ops, "linear_w8a8", _linear_w8a8)


def config(**omni):
    from omnikv_b200.modeling import LlamaCompressorConfig
    cfg = LlamaCompressorConfig(num_hidden_layers=2, hidden_size=256, intermediate_size=512, num_attention_heads=2,
                                num_key_value_heads=1, vocab_size=64, head_dim=128)
    cfg.set_config_of_compressor(model_cls="multi", cache_cls="multi", do_select_layers="1", num_wait_load_layers=0,
                                 real_offload=False, dense_more=True, num_of_selected_tokens=0.25, selector_cls="last",
                                 window_size=16, **omni)
    return cfg


def build(seed=0, dtype=torch.bfloat16, **omni):
    from omnikv_b200.modeling import OmniKVMulLM
    return OmniKVMulLM.from_config(config(**omni), dtype=dtype, device="cpu", seed=seed)


OWNERS = (("self_attn", ("qkv", "o")), ("mlp", ("gate_up", "down")))


def projections(lm):
    return {f"{i}.{part}.{name}": (getattr(getattr(layer, part), name + "_codes"), getattr(getattr(layer, part), name + "_scale"))
            for i, layer in enumerate(lm.model.layers) for part, names in OWNERS for name in names}


def test_state_dict_holds_the_projections():
    a, b = build(1, linear_dtype="int8"), build(2, linear_dtype="int8")
    sd = a.state_dict()
    assert sum(k.endswith("_codes") for k in sd) == sum(k.endswith("_scale") for k in sd) == 8
    assert not all(torch.equal(x[0], y[0]) for x, y in zip(projections(a).values(), projections(b).values()))
    b.load_state_dict(sd)
    for name, (codes, scale) in projections(a).items():
        assert torch.equal(codes, projections(b)[name][0]) and torch.equal(scale, projections(b)[name][1]), name


@pytest.mark.parametrize("kinds", [(None, "int8"), ("int8", None)])
def test_a_state_dict_of_the_other_kind_is_refused(kinds):
    saved, target = (build(1, linear_dtype=kind) for kind in kinds)
    with pytest.raises(RuntimeError, match="qkv_codes"):
        target.load_state_dict(saved.state_dict())


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double().to(torch.bfloat16),
                                  lambda m: m.to("cpu", torch.float16)])
def test_scales_stay_fp32_when_the_model_is_cast(cast):
    lm = build(1, linear_dtype="int8")
    before = {name: (c.clone(), s.clone()) for name, (c, s) in projections(lm).items()}
    assert cast(lm) is lm
    for name, (codes, scale) in projections(lm).items():
        assert codes.dtype is torch.int8 and scale.dtype is torch.float32, name
        assert torch.equal(codes, before[name][0]) and torch.equal(scale, before[name][1]), name


@pytest.mark.parametrize("kind", [None, "int8"])
def test_projection_views_multiply_with_what_is_held(kind):
    from omnikv_b200.modeling.omnikv import _project
    lm = build(3, linear_dtype=kind)
    x = torch.randn(2, 5, 256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    act = torch.randn(2, 5, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    for layer in lm.model.layers:
        a, mlp = layer.self_attn, layer.mlp
        assert torch.equal(torch.cat([a.q_proj(x), a.k_proj(x), a.v_proj(x)], -1), _project(x, a, "qkv"))
        assert torch.equal(torch.cat([mlp.gate_proj(x), mlp.up_proj(x)], -1), _project(x, mlp, "gate_up"))
        assert torch.equal(a.o_proj(x), _project(x, a, "o")) and torch.equal(mlp.down_proj(act), _project(act, mlp, "down"))
        for view in (a.q_proj, a.k_proj, a.v_proj, a.o_proj, mlp.gate_proj, mlp.up_proj, mlp.down_proj):
            if kind is None:
                assert view.weight.dtype is torch.bfloat16
                continue
            with pytest.raises(RuntimeError, match="int8 codes"):
                view.weight


def test_weights_loaded_later_are_quantised_as_the_config_says():
    source, lm = build(4), build(seed=None, linear_dtype="int8")
    lm.load_hf_state_dict(source.hf_state_dict())
    want = projections(source.quantize_weights_())
    for name, (codes, scale) in projections(lm).items():
        assert torch.equal(codes, want[name][0]) and torch.equal(scale, want[name][1]), name
    bad = build(seed=None, linear_dtype="int4")
    with pytest.raises(NotImplementedError, match="linear_dtype"):
        bad.load_hf_state_dict(build(4).hf_state_dict())


def test_a_refused_quantisation_leaves_the_weights(monkeypatch):
    from omnikv_b200 import ops
    lm = build(5)
    want = {k: v.clone() for k, v in lm.state_dict().items()}
    calls = []

    def refuse_the_third(w):
        calls.append(w)
        if len(calls) == 3:
            raise ops.abi.OmniKVError("refused")
        return _quant_rows(w)

    monkeypatch.setattr(ops, "quant_rows", refuse_the_third)
    with pytest.raises(ops.abi.OmniKVError):
        lm.quantize_weights_()
    first = lm.model.layers[0]
    assert torch.equal(first.mlp.gate_up_weight, want["model.layers.0.mlp.gate_up_weight"])
    assert first.mlp.gate_proj(torch.zeros(1, 256, dtype=torch.bfloat16)).shape == (1, 512)
    assert torch.equal(lm.model.layers[1].self_attn.qkv_weight, want["model.layers.1.self_attn.qkv_weight"])
    monkeypatch.setattr(ops, "quant_rows", _quant_rows)
    for name, (codes, scale) in projections(lm.quantize_weights_()).items():
        assert torch.equal(codes, projections(build(5).quantize_weights_())[name][0]), name


def test_quantising_one_model_leaves_the_config_and_others_alone():
    from omnikv_b200.modeling import OmniKVMulLM
    cfg = config()
    a = OmniKVMulLM.from_config(cfg, device="cpu", seed=1).quantize_weights_()
    assert cfg.get("linear_dtype", None) is None
    b = OmniKVMulLM.from_config(cfg, device="cpu", seed=1)
    assert "model.layers.0.mlp.down_codes" in a.state_dict() and "model.layers.0.mlp.down_weight" in b.state_dict()
    for model, held in ((a, True), (b, False)):  # the fused kernels are kept from layers by what those hold
        assert all(layer.holds_codes is held for layer in model.model.layers)


def test_a_16_bit_projection_asks_for_no_missing_attribute():
    """A module's lookup of a name that it does not have costs a microsecond (an exception inside), four times per layer and
    step: whether there are codes is read from the buffers."""
    from omnikv_b200.modeling.omnikv import _project

    class Owner(torch.nn.Module):
        missed = 0

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                Owner.missed += 1
                raise

    owner = Owner()
    owner.qkv_weight = torch.nn.Parameter(torch.randn(8, 4))
    x = torch.randn(3, 4)
    Owner.missed = 0  # setting a parameter looks its name up once
    assert torch.equal(_project(x, owner, "qkv"), torch.nn.functional.linear(x, owner.qkv_weight)) and Owner.missed == 0


@pytest.mark.parametrize("kind", [None, "int8"])
def test_rotary_frequencies_stay_fp32_when_the_model_is_cast(kind):
    lm = build(1, linear_dtype=kind)
    before = lm.model.rotary_emb.inv_freq.clone()
    for dtype in (torch.bfloat16, torch.float16, torch.float64):
        lm.to(dtype)
        for rotary in [lm.model.rotary_emb] + [layer.self_attn.rotary_emb for layer in lm.model.layers]:
            assert rotary.inv_freq.dtype is torch.float32 and torch.equal(rotary.inv_freq, before), dtype
