"""The 8-bit KV cache and the 8-bit projections inside the model: config keys ``kv_cache_dtype``, ``linear_dtype``.

The comparisons are made at every call inside the model, on the very inputs that the kernel got, against the definition in
64 bits: two free-running models would part for good where a rounding flips an 8-bit code.  Tolerances as derived in
test_kv8_gpu.py (attention, scores) and test_linear_w8a8_gpu.py (products).
"""
import pytest
import torch

from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu


def config(**omni):
    from omnikv_b200.modeling import LlamaCompressorConfig
    cfg = LlamaCompressorConfig(num_hidden_layers=6, hidden_size=512, intermediate_size=1024, num_attention_heads=4,
                                num_key_value_heads=1, vocab_size=1000, rope_theta=500000.0, head_dim=128)
    d = dict(model_cls="multi", cache_cls="multi", do_select_layers="1,3", num_wait_load_layers=1, real_offload=False,
             dense_more=True, num_of_selected_tokens=0.25, selector_cls="last", window_size=16)
    d.update(omni)
    cfg.set_config_of_compressor(**d)
    return cfg


def build(dtype=torch.bfloat16, **omni):
    from omnikv_b200.modeling import OmniKVMulLM
    return OmniKVMulLM.from_config(config(**omni), dtype=dtype, device="cuda", seed=0)


def tokens(B, n, seed):
    return torch.randint(0, 1000, (B, n), generator=torch.Generator().manual_seed(seed)).cuda()


HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def checked_attend(real, calls):
    """``attend`` that compares an 8-bit layer's result (and scores) with the definition over its codes."""

    def attend(cache, q, layer_idx, out=None, score_out=None, score_len=None):
        got = real(cache, q, layer_idx, out=out, score_out=score_out, score_len=score_len)
        if not cache.is_kv8(layer_idx):
            return got
        k8, v8, ks, vs = cache._kv8[layer_idx]
        k, v = (ko.values(c.float().double(), s.double(), cache.kv_block) for c, s in ((k8, ks), (v8, vs)))
        for b in range(q.shape[0]):
            P, n = int(cache.prefill_len_dev[b]), int(cache.cur_len_dev[b])
            rows = list(range(n))
            if cache.is_sparse(layer_idx):
                idx, count = cache._idx[cache.layer_state[layer_idx][1]]
                rows = idx[b, :int(count[b])].tolist() + list(range(P, n))
            o, mass, logits, size = ko.attention(q[b].double(), k[b], v[b], rows)
            tol = HALF[q.dtype] * o.abs() + (2.0 ** -11 + 2.0 ** -16 + 2.0 ** -16 * size) * mass + 1e-30
            assert ((got[b].double() - o).abs() <= tol).all(), layer_idx
            if score_out is not None:
                m = int(score_len[b])
                best = logits.view(k.shape[1], -1, n)[:, :, :m].amax(1)
                assert ((score_out[:, b, :m].double() - best).abs() <= 2.0 ** -17 * size).all(), layer_idx
        calls.append((layer_idx, score_out is not None))
        return got

    return attend


@pytest.mark.parametrize("kind", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("dtype,omni,B", [
    (torch.bfloat16, {}, 1), (torch.float16, dict(kv_cache_block=16), 1), (torch.bfloat16, dict(fused_decode=False), 1),
    (torch.bfloat16, dict(cache_cls="lazy", skip_threshold=0.5), 1), (torch.bfloat16, dict(chained_decode=True), 1),
    (torch.bfloat16, dict(selector_cls="exp"), 1), (torch.float16, {}, 3), (torch.bfloat16, dict(linear_dtype="int8"), 2)])
def test_attention_of_every_layer(kind, dtype, omni, B, monkeypatch):
    from omnikv_b200.modeling import OmniKVMultiStageCache
    lm = build(dtype, kv_cache_dtype=kind, **omni)
    ids, forced, calls = tokens(B, 333, 1), tokens(B, 10, 2), []
    monkeypatch.setattr(OmniKVMultiStageCache, "attend", checked_attend(OmniKVMultiStageCache.attend, calls))
    cache = lm(input_ids=ids).past_key_values
    cache.stage = "decoding"
    for t in range(forced.shape[1]):
        logits, _ = lm._decode_step(forced[:, t:t + 1], cache)
        assert torch.isfinite(logits).all()
    kept = [1, 3] if omni.get("selector_cls") == "exp" else []
    assert sorted(cache._kv8) == [i for i in range(6) if i not in kept]
    assert sorted(set(calls)) == [(i, not kept and i in (1, 3)) for i in range(6) if i not in kept]
    assert len(calls) == 10 * (6 - len(kept))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B", [1, 5])
def test_int8_projections(dtype, B, monkeypatch):
    from omnikv_b200 import ops
    lm = build(dtype, linear_dtype="int8")
    for layer in lm.model.layers:  # the 16-bit matrices are gone
        assert not layer.self_attn._parameters and layer.mlp.gate_up_codes.dtype is torch.int8
    ids, forced, calls = tokens(B, 200, 3), tokens(B, 4, 4), []
    real_quant, real_linear = ops.quant_rows, ops.linear_w8a8

    def quant(x):
        codes, scale = real_quant(x)
        want, scales = ko.quantise(x.double()[:, None], 1, "int8")
        assert torch.equal(codes.double(), want[:, 0])
        assert ((scale.double() - scales[:, 0]).abs() <= 2.0 ** -24 * scales[:, 0]).all()
        return codes, scale

    def linear(x8, sx, w8, sw, *, out_dtype):
        y, want = real_linear(x8, sx, w8, sw, out_dtype=out_dtype), ko.linear(x8, sx, w8, sw)
        tol = (HALF[out_dtype] + 2.0 ** -22) * want.abs() + 2.0 ** -25
        assert ((y.double() - want).abs() <= tol).all()
        calls.append(tuple(w8.shape))
        return y

    monkeypatch.setattr(ops, "quant_rows", quant)
    monkeypatch.setattr(ops, "linear_w8a8", linear)
    out = lm(input_ids=ids)
    for t in range(forced.shape[1]):
        out = lm(input_ids=forced[:, t:t + 1], past_key_values=out.past_key_values)
    assert len(calls) == 6 * 4 * 5 and torch.isfinite(out.logits).all()


def test_int8_projections_stay_near_the_16_bit_model():
    """Per product the 8-bit operands are off by at most half a step of their row's maximum; over a row that is a few
    percent of the result's size (127 steps, 4 sigma maxima, two operands), so the logits keep their direction."""
    a, b = build(), build(linear_dtype="int8")
    ids = tokens(1, 300, 5)
    x, y = a(input_ids=ids).logits.flatten().double(), b(input_ids=ids).logits.flatten().double()
    assert torch.dot(x, y) / (x.norm() * y.norm()) > 0.98


@pytest.mark.parametrize("omni,B", [
    (dict(kv_cache_dtype="int8"), 1), (dict(kv_cache_dtype="fp8_e4m3", selector_cls="uniform"), 1),
    (dict(kv_cache_dtype="int8", linear_dtype="int8"), 3), (dict(linear_dtype="int8"), 1),
    (dict(kv_cache_dtype="fp8_e4m3", cache_cls="lazy"), 1)])
def test_graph_decoding_equals_eager(omni, B):
    lm = build(**omni)
    ids = tokens(B, 400, 6)
    eager = lm.generate_greedy(ids, 24, use_cuda_graph=False)
    graph = lm.generate_greedy(ids, 24, use_cuda_graph=True)
    assert eager.shape == (B, 24) and torch.equal(eager, graph)


@pytest.mark.parametrize("kind,codes", [("int8", torch.int8), ("fp8_e4m3", torch.float8_e4m3fn)])
def test_cache_through_the_reference_api(kind, codes):
    """update() of an 8-bit cache: the prompt's fresh rows, then the rows as the codes read, selected rows and tail."""
    from omnikv_b200.modeling import OmniKVMultiStageCache
    B, KVH, P, d, block = 2, 2, 150, 128, 32
    cache = OmniKVMultiStageCache([0, 4], 4, 1, False, kv_dtype=codes, kv_block=block)
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = [[torch.randn(B, KVH, P, d, generator=g, device="cuda").to(torch.float16) for _ in range(2)] for _ in range(4)]
    for i, (k, v) in enumerate(rows):
        got = cache.update(k, v, i)
        assert got[0] is k and got[1] is v
    idx = torch.stack([torch.randperm(P, generator=torch.Generator().manual_seed(b))[:20].sort().values for b in range(B)]).cuda()
    cache.set_idx_on_gpu(idx, 0)
    for step in range(3):
        for i in range(4):
            new = [torch.randn(B, KVH, 1, d, generator=g, device="cuda").to(torch.float16) * (step + 1) for _ in range(2)]
            got = cache.update(*new, i)
            k8, v8, ks, vs = cache._kv8[i]
            for x, code, scale in zip(got, (k8, v8), (ks, vs)):
                full = ko.values(code.float().double(), scale.double(), block)
                n = P + step + 1
                want = full[:, :, :n]
                if cache.is_sparse(i):
                    want = torch.stack([torch.cat([full[b, :, idx[b]], full[b, :, P:n]], 1) for b in range(B)])
                assert x.shape == want.shape
                assert ((x.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -11) * want.abs() + 2.0 ** -25).all()
            # the new row is among them: half a step of its block
            err = (got[0][:, :, -1].double() - new[0][:, :, 0].double()).abs()
            step_size = cache._kv8[i][2][:, :, (P + step) // block].double()[..., None]
            lim = 0.5 * step_size if kind == "int8" else 2.0 ** -4 * new[0][:, :, 0].double().abs() + 2.0 ** -10 * step_size
            assert (err <= lim * 1.001 + 2.0 ** -11 * new[0][:, :, 0].double().abs()).all()
    assert cache.get_seq_length() == P + 3


def test_a_prompt_of_any_layout_is_taken_over():
    from omnikv_b200.modeling import OmniKVMultiStageCache
    k, v = (torch.randn(1, 2, 70, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    odd = torch.zeros(2 * 70 * 129 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(1, 2, 70, 129)[..., :128]
    odd.copy_(v)
    got = []
    for keys, values in ((k, v), (k.transpose(2, 3).contiguous().transpose(2, 3), odd)):
        cache = OmniKVMultiStageCache([0, 2], 2, 0, False, kv_dtype=torch.int8, kv_block=16)
        for i in range(2):
            cache.update(keys, values, i)
        got.append([t for i in range(2) for t in cache.kv8_rows(i, rows=70)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_synthetic_ragged_cache():
    from omnikv_b200.modeling import OmniKVMultiStageCache
    cache = OmniKVMultiStageCache([0, 3], 3, 0, False, kv_dtype=torch.int8, kv_block=16)
    cache.init_synthetic(3, 2, 128, [70, 5, 33], torch.bfloat16, "cuda", reserve=20)
    for i in range(3):
        k, v = cache.kv8_rows(i)
        for b, n in enumerate([70, 5, 33]):
            assert (k[b, :, n:] == 0).all() and 0.9 < v[b, :, :n].float().std().item() < 1.1


def test_refusals():
    from omnikv_b200.modeling import OmniKVMulLM, select_tokens_by_attn_universal
    lm = build(kv_cache_dtype="int8")
    out = lm(input_ids=tokens(1, 40, 0))
    attn = lm.model.layers[1].self_attn
    with pytest.raises(NotImplementedError, match="8-bit"):
        select_tokens_by_attn_universal(attn, torch.zeros(1, 1, 512, device="cuda", dtype=torch.bfloat16),
                                        torch.zeros(1, 1, device="cuda"), out.past_key_values, 4, 40)
    with pytest.raises(NotImplementedError, match="keep_layers"):
        lm.model.layers[1]._select(torch.zeros(1, 1, 512, device="cuda", dtype=torch.bfloat16), None, out.past_key_values)
    with pytest.raises(NotImplementedError, match="kv_cache_dtype"):
        build(kv_cache_dtype="int4")(input_ids=tokens(1, 40, 0))
    with pytest.raises(NotImplementedError, match="real_offload"):
        build(kv_cache_dtype="int8", real_offload=True)(input_ids=tokens(1, 40, 0))
    with pytest.raises(NotImplementedError, match="linear_dtype"):
        build(linear_dtype="int4")
    q = build(linear_dtype="int8")
    for call in (q.hf_state_dict, lambda: q.load_hf_state_dict({})):
        with pytest.raises(RuntimeError, match="int8 codes"):
            call()
    from omnikv_b200.abi import OmniKVError
    with pytest.raises(OmniKVError, match="bfloat16 or float16"):
        build(torch.float32, kv_cache_dtype="int8")(input_ids=tokens(1, 40, 0))


@pytest.mark.parametrize("selector", ["last", "exp"])
def test_the_selector_function_reads_int8_projections(selector, monkeypatch):
    """``select_tokens_by_attn_universal`` on a model with int8 projections and a 16-bit cache: the queries are those of the
    8-bit product."""
    from omnikv_b200.modeling import omnikv, select_tokens_by_attn_universal
    lm = build(linear_dtype="int8", selector_cls=selector)
    cache = lm(input_ids=tokens(1, 300, 8)).past_key_values
    attn = lm.model.layers[1].self_attn
    hs = torch.randn(1, 1 if selector == "last" else 16, 512, generator=torch.Generator().manual_seed(9)).cuda().to(torch.bfloat16)
    pos = torch.full((1, 1), 300, device="cuda")
    got = select_tokens_by_attn_universal(attn, hs, pos, cache, 40, 300, selector_cls=selector)
    q = omnikv._project(hs, attn, "qkv")[..., :512]
    monkeypatch.setattr(attn, "q_proj", lambda x: q)
    assert got.shape == (1, 40) and torch.equal(got, select_tokens_by_attn_universal(attn, hs, pos, cache, 40, 300, selector_cls=selector))


@pytest.mark.parametrize("part", [0, 5, 24])
def test_a_model_quantised_in_part_decodes_as_its_modules_do(part, monkeypatch):
    """Where the quantiser refuses a matrix the ones before it are codes and the rest 16-bit: batch-1 decoding then runs
    through the modules for every layer (the fused kernels hand the residual stream on in another way)."""
    from omnikv_b200 import ops
    real = ops.quant_rows
    ids, got = tokens(1, 200, 11), []
    for fused in (True, False):
        lm, calls = build(fused_decode=fused), []

        def quant(w):
            calls.append(w)
            if len(calls) > part:
                raise ops.abi.OmniKVError("refused")
            return real(w)

        with monkeypatch.context() as m:
            m.setattr(ops, "quant_rows", quant)
            if part == 24:
                lm.quantize_weights_()
            else:
                with pytest.raises(ops.abi.OmniKVError):
                    lm.quantize_weights_()
        cache = lm(input_ids=ids).past_key_values
        cache.stage = "decoding"
        got.append(torch.stack([lm._decode_step(tokens(1, 1, 20 + t), cache)[0].clone() for t in range(6)]))
        assert lm.model.layers[5].holds_codes is (part > 0)
    if part:
        assert torch.equal(*got)
    else:  # nothing was changed: the fused kernels decode, whose sums run in another order
        assert torch.nn.functional.cosine_similarity(got[0].flatten().double(), got[1].flatten().double(), 0) > 0.99


def test_a_saved_quantised_model_decodes_as_it_did(tmp_path):
    """Through a file, into a model whose projections are others; then cast to the other 16-bit type, which leaves codes and scales."""
    a = build(linear_dtype="int8")
    ids = tokens(1, 150, 13)
    want = a.generate_greedy(ids, 12)
    torch.save(a.state_dict(), tmp_path / "model.pt")
    c = build(linear_dtype="int8")
    for layer in c.model.layers:
        layer.mlp.down_codes.zero_()
    c.load_state_dict(torch.load(tmp_path / "model.pt"))
    assert torch.equal(c.generate_greedy(ids, 12), want)
    half = c.to(torch.float16)
    out = half(input_ids=ids)
    logits, _ = half._decode_step(tokens(1, 1, 14), out.past_key_values)
    assert torch.isfinite(logits).all()
    for x, y in zip(half.model.layers, a.model.layers):
        assert torch.equal(x.self_attn.qkv_scale, y.self_attn.qkv_scale) and torch.equal(x.mlp.gate_up_codes, y.mlp.gate_up_codes)
