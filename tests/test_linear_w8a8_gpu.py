"""The row quantiser and the 8-bit integer product against their definition in 64 bits.

Tolerances: codes are exact; a scale is one fp32 division (2^-24).  The integer sum is exact; its conversion to fp32, two
products and one addition are each off by at most 2^-24 of their value, the result by half a step of its type.
"""
import pytest
import torch

from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def ops():
    from omnikv_b200 import ops as _ops
    return _ops


def operands(n, N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x8 = torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    w8 = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    sx, sw = (torch.rand(m, generator=g, device="cuda") * 1e-3 + 1e-5 for m in (n, N))
    return x8, sx, w8, sw


def check(y, x8, sx, w8, sw, residual=None):
    prod = ko.linear(x8, sx, w8, sw)
    want = prod if residual is None else prod + residual.double()
    tol = HALF[y.dtype] * want.abs() + 3 * 2.0 ** -24 * prod.abs() + 2.0 ** -24 * want.abs()
    tol = tol * (1 + 2.0 ** -8) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)  # fp16 subnormals have a fixed step
    off = (y.double() - want).abs()
    assert (off <= tol).all(), (off / tol.clamp(min=1e-300)).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,K", [(1, 16), (1, 4096), (3, 1040), (17, 14336), (2, 32768), (300, 512), (5, 8208)])
def test_quant_rows(dtype, n, K):
    g = torch.Generator(device="cuda").manual_seed(K + n)
    wide = torch.randn(n, K + 40, generator=g, device="cuda").to(dtype)
    x = wide[:, 8:8 + K] if (K + 40) % 8 == 0 else wide[:, :K].contiguous()
    codes, scale = ops().quant_rows(x)
    want, scales = ko.quantise(x.double()[:, None], 1, "int8")
    assert torch.equal(codes.double(), want[:, 0])
    assert ((scale.double() - scales[:, 0]).abs() <= 2.0 ** -24 * scales[:, 0]).all()


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 11)])
def test_quant_rows_of_every_maximum(dtype, bits):
    """All mantissas of the row's maximum against values that hit the middles between two codes: odd multiples of a / 254
    where those are numbers of the type, a / 2, and their neighbours."""
    lo = 1 << (bits - 1)
    a = torch.arange(lo, 2 * lo, dtype=torch.float64, device="cuda")[:, None]
    mids = (torch.arange(0, 127, dtype=torch.float64, device="cuda")[None] + 0.5) * a / 127
    near = mids.to(dtype)
    step = torch.tensor([1], dtype=torch.int16, device="cuda")
    below, above = ((near.view(torch.int16) + d * step).view(dtype) for d in (-1, 1))
    x = torch.cat([a.to(dtype), near, -near, below, above, (a / 2).to(dtype), torch.zeros(len(a), 2, dtype=dtype, device="cuda")], 1)
    assert x.shape[1] == 512
    for scale in (1.0, 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -100):
        xs = x * scale
        codes, _ = ops().quant_rows(xs)
        want, _ = ko.quantise(xs.double()[:, None], 1, "int8")
        assert torch.equal(codes.double(), want[:, 0])


def test_quant_rows_of_extreme_values():
    x = torch.randn(7, 64, device="cuda").to(torch.bfloat16)
    x[0] = 0
    x[1, 5] = 3.3895e38
    x[2], x[2, 9] = 0, 9.2e-41
    x[3, 1] = float("nan")
    x[4, 1] = float("inf")
    x[5, ::2] = x[5, 0].abs() / 2  # exactly half of the maximum: a tie
    x[5, 1::2] = x[5, 0].abs() * 2
    codes, scale = ops().quant_rows(x)
    want, _ = ko.quantise(x.double()[:, None], 1, "int8")
    assert torch.equal(codes.double(), want[:, 0])
    assert scale[0] == 0 and scale[2] > 0 and torch.isnan(scale[3]) and torch.isinf(scale[4])
    y = ops().linear_w8a8(codes, scale, codes, scale, out_dtype=torch.float32)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[0, 2, 5, 6]][:, [0, 2, 5, 6]]).all()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,N,K", [
    (1, 1, 16), (1, 6144, 4096), (2, 1000, 32), (7, 129, 4096), (8, 256, 128), (9, 64, 272), (16, 4096, 1040), (17, 33, 14336),
    (33, 700, 96), (64, 512, 512), (65, 1001, 2064), (77, 1001, 1040), (128, 256, 4096), (129, 257, 144), (200, 3000, 64),
    (513, 640, 1024), (1000, 1024, 4096), (1, 16411, 4112), (16, 16411, 4112), (40, 19000, 1040), (100, 37900, 144),
    (24, 500, 4096), (31, 3000, 8192), (64, 1024, 8192), (90, 2048, 2064), (128, 4096, 4096), (130, 130, 8208), (200, 1001, 1040),
    (256, 1024, 8192), (300, 4000, 14336), (500, 300, 4096), (16, 4096, 14336), (1, 4096, 14336), (5, 13, 32768), (100, 10241, 1040)])
def test_linear(out_dtype, n, N, K):
    ops_ = operands(n, N, K, seed=n + N + K)
    check(ops().linear_w8a8(*ops_, out_dtype=out_dtype), *ops_)
    g = torch.Generator(device="cuda").manual_seed(1)
    res = torch.randn(n, N, generator=g, device="cuda").to(out_dtype)
    keep = res.clone()
    check(ops().linear_w8a8(*ops_, residual=res), *ops_, residual=keep)
    assert torch.equal(res, keep)
    out = ops().linear_w8a8(*ops_, residual=res, out=res)  # in place
    assert out.data_ptr() == res.data_ptr()
    check(out, *ops_, residual=keep)


@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_largest_sums(n):
    """Every product 127 x 127 or -128 x 127 over the longest rows: sums near 2^29."""
    K, N = 32768, 130
    x8 = torch.full((n, K), 127, dtype=torch.int8, device="cuda")
    w8 = torch.full((N, K), 127, dtype=torch.int8, device="cuda")
    w8[1::2] = -128
    s = torch.ones(max(n, N), device="cuda")
    y = ops().linear_w8a8(x8, s[:n].contiguous(), w8, s[:N].contiguous(), out_dtype=torch.float32)
    want = torch.tensor([127.0 * 127 * K, -128.0 * 127 * K], dtype=torch.float64, device="cuda").repeat(N // 2)
    assert ((y.double() - want).abs() <= 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("n", [1, 12, 130])
def test_strided_operands_and_rows_left_alone(n):
    N, K = 200, 160
    x8, sx, w8, sw = operands(n, N, K)
    xw = torch.zeros(n, K + 48, dtype=torch.int8, device="cuda")
    ww = torch.zeros(N, K + 16, dtype=torch.int8, device="cuda")
    xw[:, 16:16 + K], ww[:, :K] = x8, w8
    xw[:, :16], xw[:, 16 + K:], ww[:, K:] = 99, 99, 99
    big = torch.full((n + 2, N + 13), 5.0, dtype=torch.bfloat16, device="cuda")
    ops().linear_w8a8(xw[:, 16:16 + K], sx, ww[:, :K], sw, out=big[1:1 + n, 3:3 + N])
    check(big[1:1 + n, 3:3 + N], x8, sx, w8, sw)
    big[1:1 + n, 3:3 + N] = 5.0
    assert (big == 5.0).all()


@pytest.mark.parametrize("n", [1, 16, 200])
def test_repeated_and_captured_calls_agree(n):
    N, K = 1024, 2048
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(n, K, generator=g, device="cuda").to(torch.bfloat16)
    w8, sw = ops().quant_rows(torch.randn(N, K, generator=g, device="cuda").to(torch.bfloat16))

    def call():
        return ops().linear_w8a8(*ops().quant_rows(x), w8, sw)

    want = call()
    for _ in range(5):
        assert torch.equal(call(), want)
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        graphs.append((graph, got))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for _, got in graphs)


@pytest.mark.parametrize("N,K", [(1024, 8192), (18944 + 300, 1040)])  # a cluster per tile; tiles that CTAs share next to whole ones
def test_shared_tiles_on_two_streams_and_in_graphs(N, K):
    n = 40
    x8, sx, w8, sw = operands(n, N, K)
    want = ops().linear_w8a8(x8, sx, w8, sw)
    check(want, x8, sx, w8, sw)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops().linear_w8a8(x8, sx, w8, sw))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(ops().linear_w8a8(x8, sx, w8, sw))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(10):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        got.append(ops().linear_w8a8(x8, sx, w8, sw))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


@pytest.mark.parametrize("n,N,K", [(1, 72, 64), (16, 500, 512), (40, 1024, 8192), (130, 300, 96)])
def test_residual_in_place_and_one_row_for_all(n, N, K):
    x8, sx, w8, sw = operands(n, N, K)
    res = torch.randn(n, N, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    want = ops().linear_w8a8(x8, sx, w8, sw, residual=res)
    check(want, x8, sx, w8, sw, res)
    own = res.clone()
    assert ops().linear_w8a8(x8, sx, w8, sw, residual=own, out=own).data_ptr() == own.data_ptr()
    assert torch.equal(own, want)
    bias = res[:1].expand(n, N)
    assert torch.equal(ops().linear_w8a8(x8, sx, w8, sw, residual=bias), ops().linear_w8a8(x8, sx, w8, sw, residual=bias.contiguous()))


def test_strides_of_a_single_row_do_not_matter():
    x8, sx, w8, sw = operands(1, 200, 160)
    want = ops().linear_w8a8(x8, sx, w8, sw)
    out = torch.empty(200, dtype=torch.bfloat16, device="cuda").as_strided((1, 200), (1, 1))
    assert torch.equal(ops().linear_w8a8(x8.as_strided(x8.shape, (7, 1)), sx, w8, sw, out=out), want)
    x = torch.randn(1, 160, device="cuda").to(torch.bfloat16)
    for a, b in zip(ops().quant_rows(x.as_strided(x.shape, (5, 1))), ops().quant_rows(x)):
        assert torch.equal(a, b)


def test_refusals():
    from omnikv_b200.abi import OmniKVError
    o = ops()
    x8, sx, w8, sw = operands(4, 32, 64)
    x = torch.randn(4, 64, device="cuda").to(torch.bfloat16)
    bad = [
        lambda: o.quant_rows(x.float()), lambda: o.quant_rows(x[:, :40]), lambda: o.quant_rows(x.t()), lambda: o.quant_rows(x.cpu()),
        lambda: o.quant_rows(torch.zeros(1, 32784, dtype=torch.bfloat16, device="cuda")),
        lambda: o.quant_rows(torch.zeros(4, 65, dtype=torch.bfloat16, device="cuda")[:, 1:]),
        lambda: o.linear_w8a8(x8.int(), sx, w8, sw), lambda: o.linear_w8a8(x8[:, :48], sx, w8, sw),
        lambda: o.linear_w8a8(x8[:, :40], sx, w8[:, :40], sw), lambda: o.linear_w8a8(x8, sx[:3], w8, sw),
        lambda: o.linear_w8a8(x8, sx.double(), w8, sw), lambda: o.linear_w8a8(x8, sx, w8.cpu(), sw),
        lambda: o.linear_w8a8(x8, sx, w8, sw, residual=torch.zeros(4, 31, device="cuda")),
        lambda: o.linear_w8a8(x8, sx, w8, sw, residual=torch.zeros(4, 32, device="cuda"), out_dtype=torch.bfloat16),
        lambda: o.linear_w8a8(x8, sx, w8, sw, out_dtype=torch.float64),
        lambda: o.linear_w8a8(torch.zeros(4, 65, dtype=torch.int8, device="cuda")[:, 1:], sx, w8, sw),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(OmniKVError):
            call()
            raise AssertionError(f"call {i} was not refused")
    assert o.linear_w8a8(x8[:0], sx[:0], w8, sw).shape == (0, 32)


def test_codes_and_scales_have_memory_of_their_own(tmp_path):
    """Results of a call can be saved together, and one of them does not hold the other's memory."""
    codes, scale = ops().quant_rows(torch.randn(48, 640, device="cuda").to(torch.bfloat16))
    assert codes.untyped_storage().nbytes() == 48 * 640 and scale.untyped_storage().nbytes() == 48 * 4
    torch.save((codes, scale), tmp_path / "w.pt")
    for a, b in zip(torch.load(tmp_path / "w.pt"), (codes, scale)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,N,K", [(1, 500, 512), (40, 1024, 8192), (24, 19000, 1040), (300, 300, 1040)])  # every kernel
def test_activations_of_extreme_size(out_dtype, n, N, K):
    """Results in the range of normal numbers (2^-33 2^-92 at least, as the scales are at least 10^-5) whose integer sum times
    the token's scale leaves fp32 (about 2^17 to 2^20 times 2^112)."""
    x8, sx, w8, sw = operands(n, N, K, seed=7)
    for e in (122, -92):
        check(ops().linear_w8a8(x8, sx * 2.0 ** e, w8, sw, out_dtype=out_dtype), x8, sx * 2.0 ** e, w8, sw)
