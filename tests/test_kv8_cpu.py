"""Host-side refusals of the 8-bit entry points (validation comes before any launch, so no GPU is needed) and the
64-bit definitions against one another."""
import ctypes

import pytest
import torch

from oracle import kv8_oracle as ko


def _cache(abi):
    return abi.Kv8Cache(abi.KV8_INT8, 64, 1, 8, 128, 1000, 256, 4096, 8 * 1000 * 256, 1000 * 256, 256, 256, 512, 128, 16)


def test_cache_descriptions_are_checked():
    from omnikv_b200 import abi
    lib = abi.lib()

    def store(dtype=abi.BF16, k=256, start=0, n=10, stride=128, **change):
        c = _cache(abi)
        for name, v in change.items():
            setattr(c, name, v)
        return lib.omnikv_kv8_store(ctypes.byref(c), dtype, k, 0, 0, stride, 256, 0, 0, 128, start, n, None, None)

    for change in (dict(k=8), dict(k=None), dict(start=32), dict(start=-64), dict(n=0), dict(n=1001), dict(start=960, n=41),
                   dict(start=64, n=2 ** 31 - 1), dict(stride=4), dict(rows=0), dict(stride_row=64), dict(stride_row=136),
                   dict(stride_h=8), dict(k_scale=None), dict(B=0)):
        assert store(**change) == -1, change
    for change in (dict(dtype=abi.F32), dict(format=2), dict(block=48), dict(block=0), dict(block=512), dict(head_dim=64),
                   dict(KVH=40000), dict(B=70000)):
        assert store(**change) == -2, change
    # two sequences, or two heads, in the same memory: not to be written
    for name in ("stride_b", "stride_h", "scale_stride_b", "scale_stride_h"):
        assert store(B=2, **{name: 0}) == -1, name
    assert lib.omnikv_kv8_store(None, 1, 256, 0, 0, 128, 256, 0, 0, 128, 0, 1, None, None) == -1
    c = _cache(abi)
    assert lib.omnikv_kv8_append(ctypes.byref(c), abi.BF16, 256, 256, 0, 128, None, None) == -1
    assert lib.omnikv_kv8_append(ctypes.byref(c), abi.BF16, 256, 256, 0, 4, 256, None) == -1
    assert lib.omnikv_kv8_append(ctypes.byref(c), abi.F32, 256, 256, 0, 128, 256, None) == -2
    assert lib.omnikv_kv8_load(ctypes.byref(c), abi.F32, 0, 10, None, 0, 256, 256, 0, 0, 128, None) == -2
    assert lib.omnikv_kv8_load(ctypes.byref(c), abi.BF16, 5, 10, 256, 10, 256, 256, 0, 0, 128, None) == -1
    assert lib.omnikv_kv8_load(ctypes.byref(c), abi.BF16, 0, 10, None, 0, 256, 256, 0, 0, 64, None) == -1


def test_attention_arguments_are_checked():
    from omnikv_b200 import abi
    lib = abi.lib()

    def call(**change):
        p = abi.Kv8AttnParams()
        p.cache, p.dtype, p.H, p.scale = _cache(abi), abi.BF16, 32, 0.1
        p.q = p.out = p.len = p.workspace = 256
        p.q_stride_b, p.q_stride_h, p.n_ctas = 4096, 128, 4
        p.out_stride_b, p.out_stride_h = 4096, 128
        p.workspace_bytes = lib.omnikv_kv8_attn_workspace_bytes(1, 32, 8, 4)
        for name, v in change.items():
            setattr(p, name, v)
        return lib.omnikv_kv8_decode_attn(ctypes.byref(p), None)

    for change in (dict(q=None), dict(q=8), dict(len=None), dict(H=30), dict(n_ctas=0), dict(q_stride_h=4), dict(idx=256),
                   dict(tail_len=256), dict(score_out=256), dict(score_out=256, score_len=256, score_stride=8, idx=256, idx_cap=4),
                   dict(workspace=264), dict(out_stride_h=4), dict(out_stride_h=0), dict(out=None)):
        assert call(**change) == -1, change
    for change in (dict(dtype=abi.F32), dict(H=136), dict(n_ctas=32769)):
        assert call(**change) == -2, change
    assert call(workspace_bytes=16384) == -3 and call(workspace=None) == -3
    assert lib.omnikv_kv8_decode_attn(None, None) == -1


def test_workspace_sizes():
    from omnikv_b200 import abi
    lib = abi.lib()
    # counters, then a partial (128 sums and four numbers) per head of every (CTA, segment) pair
    assert lib.omnikv_kv8_attn_workspace_bytes(3, 16, 2, 700) == 16384 + (700 + 6) * 8 * 528
    assert lib.omnikv_kv8_attn_workspace_bytes(1, 30, 8, 4) == 0
    assert lib.omnikv_linear_w8a8_workspace_bytes(16, 512, 14336) == 0  # a stream of the weights
    assert lib.omnikv_linear_w8a8_workspace_bytes(17, 512, 14336) == 0  # a cluster per tile
    assert lib.omnikv_linear_w8a8_workspace_bytes(17, 28672, 4096) > 0  # CTAs share what is left behind whole tiles
    assert lib.omnikv_linear_w8a8_workspace_bytes(200, 512, 14336) == 0


def test_the_extension_is_built_and_checks_its_arguments():
    from omnikv_b200 import ops
    bind = ops._bind()
    assert bind.launches() == 0 or torch.cuda.is_available()
    with pytest.raises(TypeError):
        bind.quant_rows()
    with pytest.raises(ops.abi.OmniKVError, match="must be a tensor"):
        ops.quant_rows([1.0])


def test_linear_arguments_are_checked():
    from omnikv_b200 import abi
    lib = abi.lib()

    def call(**change):
        p = abi.LinearW8A8Params(4, 32, 64, 256, 64, 256, 256, 64, 256, abi.BF16, None, 0, 256, 32, None, 0, None)
        for name, v in change.items():
            setattr(p, name, v)
        return lib.omnikv_linear_w8a8(ctypes.byref(p), None)

    for change in (dict(n_tokens=0), dict(channels=-1), dict(K=40), dict(x=None), dict(x=8), dict(w=8), dict(x_scale=None),
                   dict(w_stride_row=72), dict(x_stride_row=48), dict(out=None), dict(out_stride_row=31),
                   dict(residual=256, residual_stride_row=8)):
        assert call(**change) == -1, change
    for change in (dict(out_dtype=5), dict(K=32784, x_stride_row=32784, w_stride_row=32784)):
        assert call(**change) == -2, change
    assert lib.omnikv_linear_w8a8(None, None) == -1
    assert lib.omnikv_quant_rows(abi.F32, 256, 64, 1, 64, 256, 64, 256, None) == -2
    assert lib.omnikv_quant_rows(abi.BF16, 256, 64, 1, 40, 256, 64, 256, None) == -1
    assert lib.omnikv_quant_rows(abi.BF16, 256, 64, 1, 64, 256, 48, 256, None) == -1
    assert lib.omnikv_quant_rows(abi.BF16, 256, 65, 1, 64, 256, 64, 256, None) == -1


def test_ops_refuse_cpu_tensors():
    from omnikv_b200 import abi, ops
    cache = ops.kv8_alloc(1, 2, 32, block=16, dtype=torch.int8, device="cpu")
    k = torch.zeros(1, 2, 32, 128, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.kv8_store(k, k, *cache, block=16), lambda: ops.kv8_append(k[:, :, 0], k[:, :, 0], *cache, n, block=16),
                 lambda: ops.kv8_load(*cache, block=16, dtype=torch.bfloat16), lambda: ops.kv8_decode_attn(k[:, :, 0], *cache, n, block=16),
                 lambda: ops.quant_rows(k[0, 0]), lambda: ops.linear_w8a8(cache[0][0, 0], n.float(), cache[0][0, 0], n.float())):
        with pytest.raises(abi.OmniKVError):
            call()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_nearest_is_the_formats_rounding(fmt):
    y = torch.cat([torch.linspace(-127, 127, 4001), torch.randn(2000)]).double()
    want = torch.round(y) if fmt == "int8" else y.float().to(torch.float8_e4m3fn).double()
    assert torch.equal(ko.nearest(y.float().double(), fmt), want)
    assert ((ko.nearest(y, fmt) - y).abs() <= ko.half_step(y, fmt) * (1 + 1e-12)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_appending_rows_in_falling_order_equals_storing_them(fmt):
    """When a block's first row is its largest no scale grows, and both ways give the same codes."""
    x = torch.randn(40, 128, generator=torch.Generator().manual_seed(0)).double()
    x = x[x.abs().amax(1).argsort(descending=True)]
    codes, scales = torch.zeros_like(x), torch.zeros(5, dtype=torch.float64)
    for p in range(40):
        codes, scales, _ = ko.append(codes, scales, x[p], p, 8, fmt)
    want, ws = ko.quantise(x, 8, fmt)
    assert torch.allclose(scales, ws, rtol=1e-15)
    assert ((codes - want).abs() <= 1e-9).float().mean() > 0.999  # a tie may fall to either side of the last bit


def test_cache_options_are_checked():
    from omnikv_b200.modeling import OmniKVLazyCache, OmniKVMultiStageCache, WOPackCache
    for cls in (OmniKVMultiStageCache, WOPackCache, OmniKVLazyCache):
        c = cls.from_dynamic_cache(None, [0, 1, 4], 4, 1, False, kv_dtype=torch.int8, kv_block=32, keep_layers=[1])
        assert [c.is_kv8(i) for i in range(4)] == [True, False, True, True] and c.kv_block == 32
        assert not any(cls.from_dynamic_cache(None, [0, 1, 4], 4, 1, False).is_kv8(i) for i in range(4))
        with pytest.raises(NotImplementedError):
            cls.from_dynamic_cache(None, [0, 1, 4], 4, 1, True, kv_dtype=torch.int8)
        with pytest.raises(ValueError):
            cls.from_dynamic_cache(None, [0, 1, 4], 4, 1, False, kv_dtype=torch.uint8)
        for block in (0, 48, 512):
            with pytest.raises(ValueError):
                cls.from_dynamic_cache(None, [0, 1, 4], 4, 1, False, kv_dtype=torch.int8, kv_block=block)


def test_allocation_checks_its_block():
    from omnikv_b200 import abi, ops
    for block in (0, 48, 512, -1):
        with pytest.raises(abi.OmniKVError):
            ops.kv8_alloc(1, 1, 64, block=block, dtype=torch.int8, device="cpu")


def test_every_status_of_a_bounded_wait_is_named(monkeypatch):
    from omnikv_b200 import ops
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(ops, "status_word", lambda device: word)
    ops.check_status("cuda")
    for code in range(1, 8):
        word.fill_(code)
        with pytest.raises(ops.abi.OmniKVError, match=f"status {code}") as e:
            ops.check_status("cuda")
        assert "unknown" not in str(e.value) and int(word) == 0


def test_rows_that_32_bits_do_not_count_are_refused():
    """Listed rows and the tail together pass 2^31: refused before anything is planned."""
    from omnikv_b200 import abi
    lib = abi.lib()
    p = abi.Kv8AttnParams()
    p.cache, p.dtype, p.H, p.scale = _cache(abi), abi.BF16, 32, 0.1
    p.cache.KVH, p.H = 1, 4
    p.q = p.out = p.len = p.workspace = p.idx = p.tail_start = p.tail_len = 256
    p.q_stride_b, p.q_stride_h, p.out_stride_b, p.out_stride_h, p.n_ctas = 512, 128, 512, 128, 4
    p.workspace_bytes = lib.omnikv_kv8_attn_workspace_bytes(1, 4, 1, 4)
    for cap in (2 ** 31 - 1, 2 ** 31 - 1000):
        p.idx_cap = p.idx_stride = cap
        assert lib.omnikv_kv8_decode_attn(ctypes.byref(p), None) == -2, cap


def test_tokens_and_channels_that_32_bits_do_not_count_are_refused():
    """Rounded up to a tile they pass 2^31: refused before anything is planned."""
    from omnikv_b200 import abi
    lib = abi.lib()
    for n, channels in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 100), (2 ** 31 - 1, 16), (2 ** 31 - 50, 300)):
        assert lib.omnikv_linear_w8a8_workspace_bytes(n, channels, 16) == 0
        q = abi.LinearW8A8Params(n, channels, 16, 256, 16, 256, 256, 16, 256, abi.BF16, None, 0, 256, channels, None, 0, None)
        assert lib.omnikv_linear_w8a8(ctypes.byref(q), None) == -2, (n, channels)
