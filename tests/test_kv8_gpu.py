"""The 8-bit KV cache's kernels against their definition in 64 bits.

Tolerances.  eps(t)/2 is half a step of type t relative to a value (bf16 2^-8, fp16 2^-11, fp32 2^-24).
* scales: one fp32 division, 2^-24.
* codes of a store: exact (16-bit inputs: an fp32 quotient cannot cross the middle between two codes).
* codes of an append: the re-coded value and the new row's come from at most two fp32 roundings, so a code is a nearest
  one up to |y| 2^-22.
* rows read back: one fp32 product, one rounding: |v| (2^-24 + eps/2).
* attention: a weight is off by its rounding to 11 bits (2^-11), by the logit's error (128 fp32 additions of terms whose
  absolute sum is `size`: 2^-17 size, counted twice for numerator and denominator) and by a few fp32 operations
  (2^-16); the result is rounded once: eps/2 |out|.
"""
import math

import pytest
import torch

from oracle import kv8_oracle as ko

pytestmark = pytest.mark.gpu

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
D = 128


def ops():
    from omnikv_b200 import ops as _ops
    return _ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def draw(shape, dtype, seed, outliers=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    if outliers:
        x[..., 3::37] *= 5.0
    return x.to(dtype)


def filled(B, KVH, rows, fmt, dtype, block, seed, tokens_first=False):
    """(cache tuple, float64 K, float64 V as they read) with the kernels' own store."""
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=CODES[fmt], device="cuda", tokens_first=tokens_first)
    k, v = draw((B, KVH, rows, D), dtype, seed), draw((B, KVH, rows, D), dtype, seed + 1)
    ops().kv8_store(k, v, *cache, block=block)
    return cache, *as_read(cache, block)


def as_read(cache, block):
    k8, v8, ks, vs = cache
    return ko.values(k8.float().double(), ks.double(), block), ko.values(v8.float().double(), vs.double(), block)


def check_attention(out, q, k, v, row_lists):
    half = HALF[out.dtype]
    for b, rows in enumerate(row_lists):
        want, mass, logits, size = ko.attention(q[b].double(), k[b], v[b], rows)
        tol = half * want.abs() + (2.0 ** -11 + 2.0 ** -16 + 2 * 2.0 ** -17 * size) * mass + 1e-30
        off = (out[b].double() - want).abs()
        assert torch.isfinite(out[b]).all(), (b, len(rows))
        assert (off <= tol).all(), (b, len(rows), (off / tol).max().item())


# ---------------------------------------------------------------------------------------------- store, load
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,KVH,rows,block,tokens_first", [
    (1, 8, 300, 64, False), (2, 3, 129, 32, True), (1, 1, 1, 16, False), (3, 2, 77, 1, False), (1, 2, 1000, 256, True),
    (1, 2, 257, 128, False), (2, 1, 64, 8, True)])
def test_store_and_load(dtype, fmt, B, KVH, rows, block, tokens_first):
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=CODES[fmt], device="cuda", tokens_first=tokens_first)
    # keys and values as views of one fused projection: other strides than the cache's
    kv = draw((B, rows, 2, KVH, D), dtype, 5)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    ops().kv8_store(k, v, *cache, block=block)
    back = ops().kv8_load(*cache, block=block, dtype=dtype)
    for x, code, scale, got in ((k, cache[0], cache[2], back[0]), (v, cache[1], cache[3], back[1])):
        codes, scales = ko.quantise(x.double(), block, fmt)
        assert torch.equal(code.float().double(), codes)
        assert ((scale.double() - scales).abs() <= 2.0 ** -24 * scales).all()
        want = ko.values(codes, scale.double(), block)
        assert ((got.double() - want).abs() <= (2.0 ** -24 + HALF[dtype]) * want.abs() + 2.0 ** -25).all()
        # the distance to the stored value: half a code step of the block
        step = ko.values(torch.ones_like(codes), scales, block)
        lim = ko.half_step(codes.abs() + 1, fmt) * step
        assert ((want - x.double()).abs() <= lim + 2.0 ** -20 * x.double().abs()).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_store_of_a_padded_batch_touches_only_what_exists(fmt):
    B, KVH, rows, block = 4, 2, 200, 32
    lens = [200, 0, 33, 1]
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=CODES[fmt], device="cuda")
    for t in cache[:2]:
        t.view(torch.int8).fill_(7)
    for t in cache[2:]:
        t.fill_(-3.0)
    k, v = draw((B, KVH, rows, D), torch.bfloat16, 1), draw((B, KVH, rows, D), torch.bfloat16, 2)
    for b, n in enumerate(lens):  # what lies behind a sequence is never looked at
        k[b, :, n:], v[b, :, n:] = float("nan"), float("inf")
    ops().kv8_store(k, v, *cache, block=block, lens=i32(lens))
    for x, code, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        for b, n in enumerate(lens):
            nb = -(-n // block)
            assert (code[b, :, n:].view(torch.int8) == 7).all() and (scale[b, :, nb:] == -3.0).all()
            if n:
                codes, scales = ko.quantise(x[b, :, :n].double(), block, fmt)
                assert torch.equal(code[b, :, :n].float().double(), codes)
                assert ((scale[b, :, :nb].double() - scales).abs() <= 2.0 ** -24 * scales).all()


def test_store_in_chunks_equals_one_store():
    B, KVH, rows, block = 1, 4, 300, 64
    k, v = draw((B, KVH, rows, D), torch.float16, 3), draw((B, KVH, rows, D), torch.float16, 4)
    one, two = (ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda") for _ in range(2))
    ops().kv8_store(k, v, *one, block=block)
    for lo, hi in ((0, 128), (128, 192), (192, 300)):
        ops().kv8_store(k[:, :, lo:hi], v[:, :, lo:hi], *two, block=block, start=lo)
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_store_of_extreme_values(fmt):
    """Zeros, the largest and smallest 16-bit numbers, infinities and NaN: each confined to its block and head."""
    block, rows = 16, 96
    x = draw((1, 2, rows, D), torch.bfloat16, 9)
    x[:, :, 0:16] = 0
    x[0, 0, 16:32, 5] = 3.3895e38
    x[0, 0, 32:48] = 0
    x[0, 0, 40, 7] = 9.2e-41  # the smallest subnormal
    x[0, 0, 50, 0] = float("nan")
    x[0, 0, 70, 127] = float("-inf")
    cache = ops().kv8_alloc(1, 2, rows, block=block, dtype=CODES[fmt], device="cuda")
    ops().kv8_store(x, x, *cache, block=block)
    k, _ = ops().kv8_load(*cache, block=block, dtype=torch.bfloat16)
    codes, scales = ko.quantise(x.double(), block, fmt)
    assert torch.equal(cache[0].float().double(), codes)
    bad = torch.zeros(1, 2, rows, dtype=torch.bool, device="cuda")
    bad[0, 0, 48:80] = True
    assert torch.isnan(k[bad]).all() and torch.isfinite(k[~bad]).all()
    assert (k[:, :, :16] == 0).all() and k[0, 0, 40, 7] != 0
    assert math.isinf(cache[2][0, 0, 4].item()) and math.isnan(cache[2][0, 0, 3].item())


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 11)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_store_of_every_maximum(dtype, bits, fmt):
    """All mantissas of a block's maximum against values in the middle between two codes, and their neighbours."""
    lo = 1 << (bits - 1)
    a = torch.arange(lo, 2 * lo, dtype=torch.float64, device="cuda")[:, None]
    half = torch.arange(126, dtype=torch.float64, device="cuda")[None] + 0.5
    if fmt == "e4m3":  # (16 + j) / 32 2^e: the middles of every binade, and those of the subnormals
        j = torch.arange(1, 16, 2, dtype=torch.float64, device="cuda")
        half = torch.cat([(16 + j) * 2.0 ** e for e in range(-11, 4)] + [j * 2.0 ** -10])[None, :126]
    top = ko.TOP[fmt]
    near = (half * a / top).to(dtype)
    step = torch.tensor([1], dtype=torch.int16, device="cuda")
    for other in (near, (near.view(torch.int16) + step).view(dtype), -(near.view(torch.int16) - step).view(dtype)):
        x = torch.cat([a.to(dtype), other, (a / 2).to(dtype)], 1)[None, None]
        cache = ops().kv8_alloc(1, 1, lo, block=1, dtype=CODES[fmt], device="cuda")
        ops().kv8_store(x, x, *cache, block=1)
        assert torch.equal(cache[0].float().double(), ko.quantise(x.double(), 1, fmt)[0])


def test_load_by_index():
    B, KVH, rows, block = 2, 3, 150, 16
    cache, k, v = filled(B, KVH, rows, "int8", torch.float16, block, 11, tokens_first=True)
    idx = i32([[0, 149, 149, -1, 7, 150, 2 ** 31 - 1], [5, 4, 3, 2, 1, 0, -2 ** 31]])
    got_k, got_v = ops().kv8_load(*cache, block=block, dtype=torch.float16, idx=idx)
    for got, x in ((got_k, k), (got_v, v)):
        for b in range(B):
            for i, r in enumerate(idx[b].tolist()):
                want = x[b, :, r] if 0 <= r < rows else torch.zeros(KVH, D, dtype=torch.float64, device="cuda")
                assert ((got[b, :, i].double() - want).abs() <= (2.0 ** -24 + 2.0 ** -11) * want.abs() + 2.0 ** -25).all()
    some_k, _ = ops().kv8_load(*cache, block=block, dtype=torch.float16, start=33, rows=50)
    all_k, _ = ops().kv8_load(*cache, block=block, dtype=torch.float16)
    assert torch.equal(some_k, all_k[:, :, 33:83])


def test_loaded_keys_and_values_have_memory_of_their_own():
    cache, _, _ = filled(1, 2, 40, "int8", torch.bfloat16, 16, 13)
    for pair in (ops().kv8_load(*cache, block=16, dtype=torch.bfloat16), ops().kv8_load(*cache, block=16, dtype=torch.bfloat16, rows=0),
                 ops().kv8_load(*cache, block=16, dtype=torch.float16, idx=i32([[3, 1, 4]]))):
        for t in pair:
            assert t.is_contiguous() and t.untyped_storage().nbytes() == t.numel() * 2


# ---------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [1, 8, 64, 256])
def test_append_row_by_row(dtype, fmt, block):
    """Rows of very different size: scales that grow, stay, and start afresh at every block; three sequences at
    positions of their own, one of them skipped."""
    B, KVH, rows = 3, 2, 300
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=CODES[fmt], device="cuda", tokens_first=True)
    for t in cache[2:]:
        t.fill_(1e9)  # what an earlier sequence left
    steps = 70
    size = torch.exp2(torch.randint(-6, 7, (steps, B, 1, 1), generator=torch.Generator().manual_seed(1)).float()).cuda()
    start = [0, 200, -1000]
    for t in range(steps):
        k, v = (draw((B, KVH, D), dtype, 100 + 2 * t + i) * size[t].to(dtype) for i in (0, 1))
        if t == 20:
            k[0] = 0
        before = [x.clone() for x in cache]
        pos = [p + t for p in start]
        ops().kv8_append(k, v, *cache, i32(pos), block=block)
        for new, code0, code1, s0, s1 in ((k, before[0], cache[0], before[2], cache[2]), (v, before[1], cache[1], before[3], cache[3])):
            assert torch.equal(code0[2].view(torch.int8), code1[2].view(torch.int8)) and torch.equal(s0[2], s1[2])
            for b in (0, 1):
                for h in range(KVH):
                    p, first = pos[b], pos[b] // block * block
                    _, scales, raw = ko.append(code0[b, h].float().double(), s0[b, h].double(), new[b, h].double(), p, block, fmt)
                    got = code1[b, h].float().double()
                    assert ((s1[b, h].double() - scales).abs() <= 2.0 ** -24 * scales).all()
                    assert ((got[first:p + 1] - raw).abs() <= ko.half_step(raw, fmt) + raw.abs() * 2.0 ** -22).all()
                    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
                    keep[first:p + 1] = False
                    assert torch.equal(got[keep], code0[b, h].float().double()[keep])
        again = [x.clone() for x in cache]
        ops().kv8_append(k, v, *cache, i32(pos), block=block)
        assert all(torch.equal(a.view(torch.int8), c.view(torch.int8)) for a, c in zip(again, cache))


def test_append_outside_the_cache_is_skipped():
    cache = ops().kv8_alloc(2, 1, 40, block=16, dtype=torch.int8, device="cuda")
    k = draw((2, 1, D), torch.bfloat16, 0)
    ops().kv8_append(k, k, *cache, i32([40, 2 ** 31 - 1]), block=16)
    assert all((t.float() == 0).all() for t in cache)
    ops().kv8_append(k, k, *cache, i32([39, -1]), block=16)
    assert (cache[0][0, 0, 39] != 0).any() and (cache[0][1].float() == 0).all()


def test_append_of_a_row_that_is_not_finite():
    cache = ops().kv8_alloc(1, 1, 32, block=16, dtype=torch.int8, device="cuda")
    for p in range(4):
        ops().kv8_append(*[draw((1, 1, D), torch.bfloat16, p)] * 2, *cache, i32([p]), block=16)
    bad = draw((1, 1, D), torch.bfloat16, 9)
    bad[0, 0, 3] = float("nan")
    ops().kv8_append(bad, bad, *cache, i32([4]), block=16)
    fine = draw((1, 1, D), torch.bfloat16, 10)
    ops().kv8_append(fine, fine, *cache, i32([5]), block=16)
    ops().kv8_append(fine, fine, *cache, i32([16]), block=16)
    k, _ = ops().kv8_load(*cache, block=16, dtype=torch.bfloat16)
    assert torch.isnan(k[0, 0, :6]).all() and torch.isfinite(k[0, 0, 16]).all()


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("H,KVH,block,lens,splits", [
    (32, 8, 64, [777], None), (32, 8, 64, [1], None), (8, 8, 1, [65, 0, 33], 1), (5, 1, 16, [64, 63], 3), (8, 1, 128, [5000], 41),
    (12, 1, 32, [300, 2], 5), (16, 1, 256, [1029], 2), (32, 2, 64, [31, 32, 129, 0, 96], None), (2, 2, 64, [200], 512)])
def test_dense_attention_and_scores(dtype, fmt, H, KVH, block, lens, splits):
    B, rows = len(lens), max(lens) + 3
    cache, k, v = filled(B, KVH, rows, fmt, dtype, block, 21)
    q = draw((B, H, D), dtype, 3, outliers=False) * 2
    slen = [max(0, n - 1) for n in lens]
    score = torch.full((KVH, B, rows + 5), 123.0, device="cuda")
    out = ops().kv8_decode_attn(q, *cache, i32(lens), block=block, score_out=score, score_len=i32(slen), n_splits=splits)
    check_attention(out, q, k, v, [list(range(n)) for n in lens])
    plain = ops().kv8_decode_attn(q, *cache, i32(lens), block=block, n_splits=splits)
    assert torch.equal(out, plain)
    for b in range(B):
        _, _, logits, size = ko.attention(q[b].double(), k[b], v[b], list(range(slen[b])))
        want = logits.view(KVH, H // KVH, -1).amax(1) if slen[b] else logits.new_zeros(KVH, 0)
        assert ((score[:, b, :slen[b]].double() - want).abs() <= 2.0 ** -17 * size).all()
        assert (score[:, b, slen[b]:] == 123.0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("tokens_first", [False, True])
@pytest.mark.parametrize("H,KVH,P,counts,tails,splits", [
    (32, 8, 2000, [137], [5], None), (4, 1, 500, [1, 0, 33, 500], [0, 0, 40, 64], None), (8, 2, 900, [64, 65], [1, 31], 7),
    (16, 1, 300, [0], [3], 2), (32, 8, 5000, [2048], [100], 1)])
def test_selected_rows_and_tail(fmt, tokens_first, H, KVH, P, counts, tails, splits):
    B, dtype, block = len(counts), torch.bfloat16, 32
    cache, k, v = filled(B, KVH, P + 70 + max(tails), fmt, dtype, block, 31, tokens_first)
    q = draw((B, H, D), dtype, 4, outliers=False) * 2
    g = torch.Generator().manual_seed(2)
    lists = [torch.randperm(P, generator=g)[:n].sort().values.tolist() for n in counts]
    cap = max(counts) + 9
    idx = i32([r + [0] * (cap - len(r)) for r in lists])
    starts = [P + 2 * b for b in range(B)]
    out = ops().kv8_decode_attn(q, *cache, i32(counts), block=block, idx=idx, tail_start=i32(starts), tail_len=i32(tails),
                                n_splits=splits, max_rows=cap + 64)
    check_attention(out, q, k, v, [r + list(range(s, s + t)) for r, s, t in zip(lists, starts, tails)])
    no_tail = ops().kv8_decode_attn(q, *cache, i32(counts), block=block, idx=idx, n_splits=splits)
    check_attention(no_tail, q, k, v, lists)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("splits", [2, 3, 5, 7, 8, 9, 10, 13, 16, None])
def test_one_to_sixteen_ctas_per_head(fmt, splits):
    """A cluster of `splits` CTAs per (sequence, KV head) merges its partials, however many rows each of them gets."""
    for B, KVH, G, lens in ((1, 1, 8, [1537]), (1, 1, 16, [1537]), (2, 1, 11, [1537, 600]), (2, 1, 3, [70, 1500]), (1, 2, 5, [33]), (3, 1, 1, [0, 1, 1537]), (1, 7, 7, [1100])):
        H, rows = KVH * G, 1537
        cache, k, v = filled(B, KVH, rows, fmt, torch.float16, 64, 31)
        q = draw((B, H, D), torch.float16, 32, outliers=False) * 2
        score = torch.full((KVH, B, rows), 123.0, device="cuda")
        out = ops().kv8_decode_attn(q, *cache, i32(lens), block=64, n_splits=splits, score_out=score, score_len=i32(lens))
        check_attention(out, q, k, v, [list(range(n)) for n in lens])
        for b in range(B):
            _, _, logits, size = ko.attention(q[b].double(), k[b], v[b], list(range(lens[b])))
            want = logits.view(KVH, G, -1).amax(1) if lens[b] else logits.new_zeros(KVH, 0)
            assert ((score[:, b, :lens[b]].double() - want).abs() <= 2.0 ** -17 * size).all()
            assert (score[:, b, lens[b]:] == 123.0).all()
        idx = torch.randperm(rows, device="cuda")[:1200].int().expand(B, -1)
        counts, tails = [min(n, 1200) for n in lens], [n % 50 for n in lens]
        got = ops().kv8_decode_attn(q, *cache, i32(counts), block=64, n_splits=splits, idx=idx, tail_start=i32([100] * B), tail_len=i32(tails))
        rows_of = [idx[0, :c].tolist() + list(range(100, 100 + t)) for c, t in zip(counts, tails)]
        check_attention(got, q, k, v, rows_of)
        assert torch.equal(got, ops().kv8_decode_attn(q, *cache, i32(counts), block=64, n_splits=splits, idx=idx,
                                                       tail_start=i32([100] * B), tail_len=i32(tails)))


def test_rows_outside_the_cache_count_as_none():
    """An index list with entries outside the cache, lengths and tails that reach past it: the rows that exist are used."""
    B, H, KVH, rows, block = 2, 8, 2, 100, 16
    cache, k, v = filled(B, KVH, rows, "int8", torch.float16, block, 41)
    q = draw((B, H, D), torch.float16, 4, outliers=False)
    idx = i32([[3, -1, 100, 50, 2 ** 31 - 1], [-5, -4, 200, 100, -2 ** 31]])
    out = ops().kv8_decode_attn(q, *cache, i32([99, 5]), block=block, idx=idx, tail_start=i32([98, 400]), tail_len=i32([7, 3]))
    check_attention(out, q, k, v, [[3, 50, 98, 99], []])
    assert (out[1] == 0).all()
    out = ops().kv8_decode_attn(q, *cache, i32([1000, -3]), block=block)
    check_attention(out, q, k, v, [list(range(rows)), []])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_lies_behind_a_sequence_does_not_matter(fmt):
    B, H, KVH, rows, block, n = 1, 8, 1, 200, 16, 70
    x = draw((B, KVH, rows, D), torch.bfloat16, 51)
    cache, k, v = filled(B, KVH, rows, fmt, torch.bfloat16, block, 51)
    q = draw((B, H, D), torch.bfloat16, 4, outliers=False)
    want = ops().kv8_decode_attn(q, *cache, i32([n]), block=block)
    for t in cache[2:]:
        t[:, :, 5:] = float("nan")  # blocks behind row 80
    for t in cache[:2]:
        t[:, :, n:].copy_(x[:, :, n:].to(CODES[fmt]) if fmt == "e4m3" else torch.full_like(t[:, :, n:], -128))
        t.view(torch.int8)[:, :, n:, ::3] = 127  # a NaN code in e4m3
    assert torch.equal(ops().kv8_decode_attn(q, *cache, i32([n]), block=block), want)
    cache[1].view(torch.int8)[:, :, 32:48], cache[3][:, :, 2] = 0, float("inf")  # a block inside it that reads as NaN
    assert torch.isnan(ops().kv8_decode_attn(q, *cache, i32([n]), block=block)).all()


def test_values_of_very_different_size():
    """Scales from 2^-90 to 2^90 among the rows of one call: rows with small values still carry their weight."""
    B, H, KVH, rows, block = 1, 4, 1, 640, 16
    k = draw((B, KVH, rows, D), torch.bfloat16, 61) * 0.1
    v = draw((B, KVH, rows, D), torch.bfloat16, 62)
    q = draw((B, H, D), torch.bfloat16, 5, outliers=False)
    for case, factor in (("tiny", 2.0 ** -90), ("huge", 2.0 ** 90)):
        x = v.clone()
        x[:, :, 0:320] *= factor
        cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda")
        ops().kv8_store(k, x, *cache, block=block)
        out = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block)
        check_attention(out, q, *as_read(cache, block), [list(range(rows))])
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda")
    ops().kv8_store(k, torch.zeros_like(v), *cache, block=block)
    assert (ops().kv8_decode_attn(q, *cache, i32([rows]), block=block) == 0).all()


def test_one_strong_row_among_many_weak_ones():
    """Weights far below the largest still add up: 40000 rows of weight 2^-18 of the strongest."""
    B, H, KVH, rows, block = 1, 4, 1, 40000, 64
    k = torch.zeros(B, KVH, rows, D, dtype=torch.float16, device="cuda")
    k[..., 0] = 1.0
    k[:, :, 0:64, 0] = 0.0
    k[:, :, 17, 0] = 2.0
    q = torch.zeros(B, H, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 18 * math.log(2) * math.sqrt(D)
    v = draw((B, KVH, rows, D), torch.float16, 71)
    v[..., 64:] = v[..., 64:].abs()
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda")
    ops().kv8_store(k, v, *cache, block=block)
    out = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block)
    check_attention(out, q, *as_read(cache, block), [list(range(rows))])


def test_large_queries():
    """bf16 queries far outside fp16's range (with keys small enough for ordinary logits)."""
    B, H, KVH, rows, block = 1, 4, 1, 300, 32
    q = draw((B, H, D), torch.bfloat16, 5, outliers=False) * 2.0 ** 30
    k = draw((B, KVH, rows, D), torch.bfloat16, 6) * 2.0 ** -31
    v = draw((B, KVH, rows, D), torch.bfloat16, 7)
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda")
    ops().kv8_store(k, v, *cache, block=block)
    check_attention(ops().kv8_decode_attn(q, *cache, i32([rows]), block=block), q, *as_read(cache, block), [list(range(rows))])
    q = q * 2.0 ** -60
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=torch.int8, device="cuda")
    ops().kv8_store(k * 2.0 ** 61, v, *cache, block=block)
    check_attention(ops().kv8_decode_attn(q, *cache, i32([rows]), block=block), q, *as_read(cache, block), [list(range(rows))])
    q[0, 1, 0] = float("nan")
    out = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block)
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, [0, 2, 3]]).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_keys_and_queries_of_extreme_size(fmt):
    """Products of a key's scale and its codes that leave fp32's range although the logits are in it."""
    B, H, KVH, rows, block = 1, 4, 1, 300, 16
    q = draw((B, H, D), torch.bfloat16, 15, outliers=False)
    k, v = draw((B, KVH, rows, D), torch.bfloat16, 16), draw((B, KVH, rows, D), torch.bfloat16, 17)
    tiny = q * 2.0 ** -120
    cache = ops().kv8_alloc(B, KVH, rows, block=block, dtype=CODES[fmt], device="cuda")
    ops().kv8_store(k * 2.0 ** 118, v, *cache, block=block)
    check_attention(ops().kv8_decode_attn(tiny, *cache, i32([rows]), block=block), tiny, *as_read(cache, block), [list(range(rows))])
    k[0, 0, 37, 5], q[0, :, 5] = 3e38, torch.tensor([0.5, -0.5, 0.25, 0.0], dtype=torch.bfloat16, device="cuda")
    ops().kv8_store(k, v, *cache, block=block)
    score = torch.zeros(KVH, B, rows, device="cuda")
    out = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block, score_out=score, score_len=i32([rows]))
    kk, vv = as_read(cache, block)
    # two heads see nothing but row 37, one everything else, one all rows (its products with that row are zero)
    rest = [r for r in range(rows) if r != 37]
    check_attention(out[:, :1], q[:, :1], kk, vv, [[37]])
    check_attention(out[:, 2:3], q[:, 2:3], kk, vv, [[37]])
    check_attention(out[:, 1:2], q[:, 1:2], kk, vv, [rest])
    check_attention(out[:, 3:], q[:, 3:], kk, vv, [list(range(rows))])
    want = kk[0, 0, 37, 5].item() * 0.5 / math.sqrt(D)
    assert abs(score[0, 0, 37].item() - want) <= 2.0 ** -17 * want


def test_offsets_past_32_bits():
    """A cache of more than 2^31 codes per sequence, read at its end."""
    KVH, rows, block = 8, 1_100_000, 64
    kv = torch.zeros(1, rows, KVH, 2, D, dtype=torch.int8, device="cuda")  # 2.25 GB
    k8, v8 = kv[:, :, :, 0].permute(0, 2, 1, 3), kv[:, :, :, 1].permute(0, 2, 1, 3)
    scales = torch.zeros(2, 1, KVH, -(-rows // block), device="cuda")
    cache = (k8, v8, scales[0], scales[1])
    k, v = draw((1, KVH, 64, D), torch.bfloat16, 1), draw((1, KVH, 64, D), torch.bfloat16, 2)
    last = rows // block * block - block
    ops().kv8_store(k, v, *cache, block=block, start=last)
    ops().kv8_append(k[:, :, 0], v[:, :, 0], *cache, i32([rows - 1]), block=block)
    got, _ = ops().kv8_load(*cache, block=block, dtype=torch.bfloat16, start=last, rows=64)
    codes, s = ko.quantise(k.double(), block, "int8")
    want = ko.values(codes, s, block)
    assert ((got.double() - want).abs() <= (2.0 ** -23 + 2.0 ** -8) * want.abs()).all()
    q = draw((1, 32, D), torch.bfloat16, 5, outliers=False)
    idx = torch.arange(last, last + 64, device="cuda", dtype=torch.int32)[None]
    out = ops().kv8_decode_attn(q, *cache, i32([64]), block=block, idx=idx, tail_start=i32([rows - 1]), tail_len=i32([1]))
    sub = [last + i for i in range(64)] + [rows - 1]
    kk = torch.stack([k8[0, :, r].double() * scales[0][0, :, r // block, None].double() for r in sub], 1)
    vv = torch.stack([v8[0, :, r].double() * scales[1][0, :, r // block, None].double() for r in sub], 1)
    check_attention(out, q, kk[None], vv[None], [list(range(65))])
    dense = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block)
    assert torch.isfinite(dense).all()


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_prompt_then_steps_in_a_graph(fmt):
    """A prompt enters the cache; then steps (append, dense attention with scores, top-k, attention over the selection and
    the tail) run eagerly and as a replayed graph, on a stream of their own, with equal results."""
    o = ops()
    B, H, KVH, P, block, steps, k_sel = 2, 8, 2, 130, 32, 40, 24
    k, v = draw((B, KVH, P, D), torch.bfloat16, 1), draw((B, KVH, P, D), torch.bfloat16, 2)
    new = [draw((steps, B, n, D), torch.bfloat16, 3 + i, outliers=i < 2) for i, n in enumerate((KVH, KVH, H))]

    def build():
        cache = o.kv8_alloc(B, KVH, P + steps, block=block, dtype=CODES[fmt], device="cuda")
        o.kv8_store(k, v, *cache, block=block)
        st = dict(cache=cache, pos=i32([P - 1] * B), cur=i32([P] * B), tail=i32([0] * B), P=i32([P] * B), k=i32([k_sel] * B),
                  score=torch.zeros(KVH, B, P, device="cuda"), kn=new[0][0].clone(), vn=new[1][0].clone(), q=new[2][0].clone())
        return st

    def step(st):
        for t in (st["pos"], st["cur"], st["tail"]):
            t.add_(1)
        o.kv8_append(st["kn"], st["vn"], *st["cache"], st["pos"], block=block)
        dense = o.kv8_decode_attn(st["q"], *st["cache"], st["cur"], block=block, score_out=st["score"], score_len=st["P"])
        idx, count = o.topk(st["score"], st["P"], st["k"])
        sparse = o.kv8_decode_attn(st["q"], *st["cache"], count, block=block, idx=idx, tail_start=st["P"], tail_len=st["tail"])
        return dense, sparse, idx

    eager, want = build(), []
    for t in range(steps):
        for name, n in (("kn", 0), ("vn", 1), ("q", 2)):
            eager[name].copy_(new[n][t])
        want.append([x.clone() for x in step(eager)])
        if t % 13 == 0:
            kk, vv = as_read(eager["cache"], block)
            check_attention(want[-1][0], eager["q"], kk, vv, [list(range(P + t + 1))] * B)
            check_attention(want[-1][1], eager["q"], kk, vv,
                            [want[-1][2][b, :k_sel].tolist() + list(range(P, P + t + 1)) for b in range(B)])
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):  # two graphs of their own state, replayed side by side
        st = build()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(st)
        graphs.append((st, g, res))
    torch.cuda.synchronize()
    for t in range(steps):
        for i, (st, g, res) in enumerate(graphs):
            with torch.cuda.stream(side if i else torch.cuda.current_stream()):
                for name, n in (("kn", 0), ("vn", 1), ("q", 2)):
                    st[name].copy_(new[n][t])
                g.replay()
        torch.cuda.synchronize()
        for st, g, res in graphs:
            for a, b in zip(res[:2], want[t][:2]):
                assert torch.equal(a, b), t
            assert torch.equal(res[2][:, :k_sel], want[t][2][:, :k_sel])


def test_a_destroyed_graph_gives_its_workspace_back():
    cache, _, _ = filled(2, 2, 9000, "int8", torch.bfloat16, 64, 79)
    q, n = draw((2, 16, D), torch.bfloat16, 80, outliers=False), i32([9000, 5000])
    ws = torch.zeros(ops().abi.lib().omnikv_kv8_attn_workspace_bytes(2, 16, 2, 148), dtype=torch.uint8, device="cuda")
    want = ops().kv8_decode_attn(q, *cache, n, block=64, n_splits=37, ws=ws)
    used = []
    for _ in range(24):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops().kv8_decode_attn(q, *cache, n, block=64, n_splits=37)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del graph, out
        used.append(torch.cuda.memory_allocated())
    assert max(used[4:]) - used[3] < 8 * (1 << 20), used  # not one of 1 MiB and more for each graph


def test_graphs_that_share_a_memory_pool():
    """A graph's workspace lies in its pool, where another graph's temporaries may have been: it is zeroed by the graph itself,
    whatever ran in between."""
    cache, k, v = filled(2, 2, 9000, "int8", torch.bfloat16, 64, 179)
    q, n = draw((2, 16, D), torch.bfloat16, 180, outliers=False), i32([9000, 5000])
    w8, sw = ops().quant_rows(draw((19000, 1040), torch.bfloat16, 181))
    x8, sx = ops().quant_rows(draw((40, 1040), torch.bfloat16, 182))

    def call():
        a, b = ops().kv8_decode_attn(q, *cache, n, block=64, n_splits=37), ops().linear_w8a8(x8, sx, w8, sw)
        for size in (1 << 18, 1 << 20, 1 << 22, 1 << 24):  # temporaries, given back to the pool
            torch.full((size,), -1, dtype=torch.int32, device="cuda")
        return a, b

    want = [t.clone() for t in call()]
    check_attention(want[0], q, k, v, [list(range(9000)), list(range(5000))])
    graphs, pool = [], None
    for _ in range(3):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            got = call()
        pool = graph.pool()
        graphs.append((graph, got))
    for i in (0, 1, 2, 2, 0, 1, 0, 2, 1):
        graphs[i][0].replay()
        torch.cuda.synchronize()
        for a, b in zip(graphs[i][1], want):
            assert torch.equal(a, b), i
        assert torch.equal(call()[0], want[0])


def test_two_streams_at_once():
    B, H, KVH, rows, block = 1, 32, 8, 20000, 64
    cache, _, _ = filled(B, KVH, rows, "int8", torch.bfloat16, block, 81)
    qs = [draw((B, H, D), torch.bfloat16, 90 + i, outliers=False) for i in range(2)]
    want = [ops().kv8_decode_attn(q, *cache, i32([rows]), block=block) for q in qs]
    torch.cuda.synchronize()
    streams, got, n = [torch.cuda.Stream() for _ in range(2)], [[], []], i32([rows])
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops().kv8_decode_attn(qs[i], *cache, n, block=block))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_sequences_that_share_a_cache_and_a_query():
    """Strides of 0, which reading allows: a shared prompt, one query for all sequences."""
    B, H, KVH, rows, block = 3, 16, 4, 700, 32
    cache, k, v = filled(1, KVH, rows, "int8", torch.bfloat16, block, 83)
    q = draw((1, H, D), torch.bfloat16, 84, outliers=False)
    lens = [700, 0, 401]
    wide = [t.expand(B, *t.shape[1:]) for t in cache]
    out = ops().kv8_decode_attn(q.expand(B, H, D), *wide, i32(lens), block=block)
    check_attention(out, q.expand(B, H, D), k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), [list(range(n)) for n in lens])
    assert torch.equal(out, ops().kv8_decode_attn(q.repeat(B, 1, 1), *[t.repeat(B, *[1] * (t.dim() - 1)) for t in cache], i32(lens), block=block))
    idx = torch.randperm(rows, device="cuda")[:300].int().expand(B, -1)
    sel = ops().kv8_decode_attn(q.expand(B, H, D), *wide, i32([300, 7, 0]), block=block, idx=idx)
    check_attention(sel, q.expand(B, H, D), k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), [idx[0, :n].tolist() for n in (300, 7, 0)])
    kk, _ = ops().kv8_load(*wide, block=block, dtype=torch.bfloat16)
    assert torch.equal(kk[1], kk[0]) and torch.equal(kk[:1], ops().kv8_load(*cache, block=block, dtype=torch.bfloat16)[0])


def test_results_in_place_and_in_strided_memory():
    B, H, KVH, rows, block = 2, 24, 2, 3000, 64
    cache, k, v = filled(B, KVH, rows, "e4m3", torch.float16, block, 85)
    q = draw((B, H, D), torch.float16, 86, outliers=False)
    lens = [rows, 0]
    want = ops().kv8_decode_attn(q, *cache, i32(lens), block=block)
    check_attention(want, q, k, v, [list(range(n)) for n in lens])
    wide = torch.full((H + 2, B, D + 8), 7.0, dtype=torch.float16, device="cuda")
    place = wide.permute(1, 0, 2)[:, 1:-1, :D]
    assert ops().kv8_decode_attn(q, *cache, i32(lens), block=block, out=place).data_ptr() == place.data_ptr()
    assert torch.equal(place, want)
    place.fill_(7.0)
    assert (wide == 7.0).all()
    same = q.clone()
    ops().kv8_decode_attn(same, *cache, i32(lens), block=block, out=same)
    assert torch.equal(same, want)


def test_scores_end_where_their_memory_ends():
    B, H, KVH, rows, stride = 2, 8, 2, 500, 300
    cache, _, _ = filled(B, KVH, rows, "int8", torch.bfloat16, 64, 87)
    q = draw((B, H, D), torch.bfloat16, 88, outliers=False)
    full = torch.zeros(KVH, B, rows, device="cuda")
    ops().kv8_decode_attn(q, *cache, i32([rows, 250]), block=64, score_out=full, score_len=i32([rows, rows]))
    flat = torch.full((KVH * B * stride + 1000,), 5.0, device="cuda")
    narrow = flat[:KVH * B * stride].view(KVH, B, stride)
    ops().kv8_decode_attn(q, *cache, i32([rows, 250]), block=64, score_out=narrow, score_len=i32([rows, rows]))
    assert torch.equal(narrow[:, 0], full[:, 0, :stride]) and torch.equal(narrow[:, 1, :250], full[:, 1, :250])
    assert (narrow[:, 1, 250:] == 5.0).all() and (flat[KVH * B * stride:] == 5.0).all()


@pytest.mark.parametrize("B,KVH,H,splits", [(70, 1, 3, None), (70, 2, 8, 3), (200, 8, 32, None)])
def test_many_sequences(B, KVH, H, splits):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    lens[3], lens[33], lens[B - 1] = 1500, 0, 0
    cache, k, v = filled(B, KVH, 1500, "int8", torch.bfloat16, 16, 89)
    q = draw((B, H, D), torch.bfloat16, 90, outliers=False)
    out = ops().kv8_decode_attn(q, *cache, i32(lens), block=16, n_splits=splits)
    check_attention(out, q, k, v, [list(range(n)) for n in lens])


@pytest.mark.parametrize("B,KVH,G,lens", [(4, 2, 4, [700, 300, 0, 1000]), (40, 3, 2, None), (5, 1, 16, [1, 0, 33, 900, 64])])
def test_few_rows_of_different_numbers_in_a_large_cache(B, KVH, G, lens):
    lens = lens or torch.randint(0, 900, (B,), generator=torch.Generator().manual_seed(7)).tolist()
    cap, top = 40000, 1024
    cache = ops().kv8_alloc(B, KVH, cap, block=64, dtype=torch.int8, device="cuda")
    ops().kv8_store(draw((B, KVH, top, D), torch.bfloat16, 95), draw((B, KVH, top, D), torch.bfloat16, 96), *cache, block=64)
    k, v = as_read(tuple(t[:, :, :top] for t in cache[:2]) + tuple(t[:, :, :top // 64] for t in cache[2:]), 64)
    q = draw((B, KVH * G, D), torch.bfloat16, 97, outliers=False)
    out = ops().kv8_decode_attn(q, *cache, i32(lens), block=64)
    check_attention(out, q, k, v, [list(range(n)) for n in lens])
    for n_splits in (1, 2, 9):
        check_attention(ops().kv8_decode_attn(q, *cache, i32(lens), block=64, n_splits=n_splits), q, k, v, [list(range(n)) for n in lens])


def test_strides_of_single_entries_do_not_matter():
    cache, _, _ = filled(1, 1, 60, "int8", torch.bfloat16, 64, 91)
    q = draw((1, 4, D), torch.bfloat16, 92, outliers=False)
    want = ops().kv8_decode_attn(q, *cache, i32([60]), block=64)
    k8, v8, ks, vs = cache
    odd = [t.as_strided(t.shape, (3, 5, t.stride(2), 1)) for t in (k8, v8)] + [ks.as_strided((1, 1, 1), (7, 11, 5)), vs.as_strided((1, 1, 1), (2, 9, 3))]
    qo = q.as_strided(q.shape, (9, D, 1))
    assert torch.equal(ops().kv8_decode_attn(qo, *odd, i32([60]), block=64), want)
    row = draw((1, 1, D), torch.bfloat16, 93)
    ops().kv8_append(row.as_strided(row.shape, (3, 1, 1)), row, *odd, i32([59]), block=64)
    ops().kv8_append(row, row, *cache, i32([59]), block=64)  # the same row again changes nothing
    got = [t.clone() for t in cache]
    k = draw((1, 1, 60, D), torch.bfloat16, 91)
    ops().kv8_store(k, draw((1, 1, 60, D), torch.bfloat16, 92), *odd, block=64)
    ops().kv8_append(row, row, *odd, i32([59]), block=64)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(cache, got))


# ---------------------------------------------------------------------------------------------- refusals
def test_refusals():
    from omnikv_b200.abi import OmniKVError
    o = ops()
    cache = k8, v8, ks, vs = o.kv8_alloc(2, 2, 64, block=16, dtype=torch.int8, device="cuda")
    k = draw((2, 2, 64, D), torch.bfloat16, 1)
    n = i32([64, 64])
    q = draw((2, 4, D), torch.bfloat16, 1)
    bad = [
        lambda: o.kv8_store(k.float(), k.float(), *cache, block=16),
        lambda: o.kv8_store(k, k, *cache, block=24),
        lambda: o.kv8_store(k, k, *cache, block=512),
        lambda: o.kv8_store(k, k, *cache, block=8),                      # fewer scales than blocks
        lambda: o.kv8_store(k[:, :, :16], k[:, :, :16], *cache, block=16, start=8),
        lambda: o.kv8_store(k, k, *cache, block=16, start=16),           # past the cache
        lambda: o.kv8_store(k[:1], k[:1], *cache, block=16),
        lambda: o.kv8_store(k, k[:, :, :3], *cache, block=16),
        lambda: o.kv8_store(k, k, *cache, block=16, lens=n.long()),
        lambda: o.kv8_store(k, k, k8, v8.float(), ks, vs, block=16),
        lambda: o.kv8_store(k.cpu(), k, *cache, block=16),
        lambda: o.kv8_store(k, k, k8, v8, ks.double(), vs, block=16),
        lambda: o.kv8_append(k[:, :, 0].float(), k[:, :, 0].float(), *cache, n, block=16),
        lambda: o.kv8_append(k[:, :, 0], k[:, :, 0], *cache, i32([1]), block=16),
        lambda: o.kv8_append(k[:, :, 0, :64], k[:, :, 0, :64], *cache, n, block=16),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.float32),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.bfloat16, start=1, rows=64),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.bfloat16, idx=n),
        lambda: o.kv8_decode_attn(q.float(), *cache, n, block=16),
        lambda: o.kv8_decode_attn(q[:, :3], *cache, n, block=16),
        lambda: o.kv8_decode_attn(q, *cache, n.long(), block=16),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, tail_len=n),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, score_out=torch.zeros(2, 2, 64, device="cuda")),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, out=torch.empty(2, 4, D, device="cuda")),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, n_splits=20000),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, n_splits=2 ** 62),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, n_splits=0),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, out=q[:1].expand(2, 4, D)),  # sequences in the same memory
        lambda: o.kv8_store(k, k, *[t[:1].expand(2, *t.shape[1:]) for t in cache], block=16),
        lambda: o.kv8_append(k[:, :, 0], k[:, :, 0], *[t[:, :1].expand(2, 2, *t.shape[2:]) for t in cache], n, block=16),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.bfloat16, start=-2 ** 62),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.bfloat16, rows=-1),
        lambda: o.kv8_load(*cache, block=16, dtype=torch.bfloat16, rows=2 ** 40),
        lambda: o.kv8_decode_attn(q, *cache, n, block=16, ws=torch.zeros(64, dtype=torch.uint8, device="cuda")),
        lambda: o.kv8_decode_attn(torch.zeros(2, 34, D, dtype=torch.bfloat16, device="cuda"), *cache, n, block=16),
        lambda: o.kv8_alloc(1, 1, 16, block=16, dtype=torch.uint8, device="cuda"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(OmniKVError):
            call()
            raise AssertionError(f"call {i} was not refused")
    assert all((t.float() == 0).all() for t in cache)
    with pytest.raises(OmniKVError):  # rows of codes that are not 16-byte aligned
        wide = torch.zeros(2, 2, 64, 2 * D + 1, dtype=torch.int8, device="cuda")
        o.kv8_load(wide[..., :D], wide[..., D:2 * D], ks, vs, block=16, dtype=torch.bfloat16)


def test_a_workspace_that_is_not_one_piece_of_memory_is_refused():
    from omnikv_b200.abi import OmniKVError
    cache, k, v = filled(1, 2, 500, "int8", torch.bfloat16, 64, 101)
    q, n = draw((1, 8, D), torch.bfloat16, 102, outliers=False), i32([500])
    need = ops().abi.lib().omnikv_kv8_attn_workspace_bytes(1, 8, 2, 148)
    whole = torch.zeros(2 * need, dtype=torch.uint8, device="cuda")
    for ws in (whole[:1].expand(need), whole[::2], whole.view(2, -1).t()):
        assert ws.numel() >= need
        with pytest.raises(OmniKVError, match="contiguous"):
            ops().kv8_decode_attn(q, *cache, n, block=64, ws=ws)
    assert (whole == 0).all()
    check_attention(ops().kv8_decode_attn(q, *cache, n, block=64, ws=whole), q, k, v, [list(range(500))])


def test_the_most_pairs_of_sequence_and_head():
    """4096 pairs run, one more is refused by name."""
    from omnikv_b200.abi import OmniKVError
    cache, k, v = filled(1, 1, 40, "int8", torch.bfloat16, 16, 103)
    q, lens = draw((4097, 2, D), torch.bfloat16, 104, outliers=False), torch.arange(4097, device="cuda").remainder(41).int()
    wide = lambda B: [t.expand(B, *t.shape[1:]) for t in cache]  # noqa: E731
    out = ops().kv8_decode_attn(q[:4096], *wide(4096), lens[:4096], block=16)
    for b in (0, 40, 41, 2049, 4095):
        check_attention(out[b:b + 1], q[b:b + 1], k, v, [list(range(b % 41))])
    with pytest.raises(OmniKVError, match="4096"):
        ops().kv8_decode_attn(q, *wide(4097), lens, block=16)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,KVH,G,rows,splits", [(1, 8, 4, 900, None), (3, 2, 5, 333, 3), (2, 1, 12, 2500, 40)])
def test_codes_of_k_and_v_in_separate_buffers(fmt, B, KVH, G, rows, splits):
    """Two code tensors with nothing between them but their layout: every entry point, and rows of both fetched apart."""
    dtype, block = torch.float16, 32
    k8, v8 = (torch.zeros(B, KVH, rows, D, dtype=torch.int8, device="cuda").view(CODES[fmt]) for _ in range(2))
    ks, vs = (torch.zeros(B, KVH, -(-rows // block), device="cuda") for _ in range(2))
    cache = (k8, v8, ks, vs)
    xk, xv = draw((B, KVH, rows, D), dtype, 201), draw((B, KVH, rows, D), dtype, 202)
    ops().kv8_store(xk, xv, *cache, block=block)
    ops().kv8_append(xk[:, :, 7].contiguous(), xv[:, :, 9].contiguous(), *cache, i32([rows - 1 - b for b in range(B)]), block=block)
    k, v = as_read(cache, block)
    back = ops().kv8_load(*cache, block=block, dtype=dtype)
    for got, want in zip(back, (k, v)):
        assert ((got.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -11) * want.abs() + 2.0 ** -25).all()
    q = draw((B, KVH * G, D), dtype, 203, outliers=False)
    lens = [rows - 11 * b for b in range(B)]
    score = torch.full((KVH, B, rows), 123.0, device="cuda")
    out = ops().kv8_decode_attn(q, *cache, i32(lens), block=block, n_splits=splits, score_out=score, score_len=i32(lens))
    check_attention(out, q, k, v, [list(range(n)) for n in lens])
    for b in range(B):
        _, _, logits, size = ko.attention(q[b].double(), k[b], v[b], list(range(lens[b])))
        assert ((score[:, b, :lens[b]].double() - logits.view(KVH, G, -1).amax(1)).abs() <= 2.0 ** -17 * size).all()
    g = torch.Generator().manual_seed(5)
    lists = [torch.randperm(rows - 40, generator=g)[:rows // 3 + b].tolist() for b in range(B)]
    idx, counts = i32([r + [-1] * (rows // 3 + B - len(r)) for r in lists]), i32([len(r) for r in lists])
    starts, tails = i32([rows - 40] * B), [40 - 13 * b for b in range(B)]
    out = ops().kv8_decode_attn(q, *cache, counts, block=block, n_splits=splits, idx=idx, tail_start=starts, tail_len=i32(tails))
    check_attention(out, q, k, v, [r + list(range(rows - 40, rows - 40 + t)) for r, t in zip(lists, tails)])
    heads = [100 + b for b in range(B)]  # a tail behind the first rows
    out = ops().kv8_decode_attn(q, *cache, i32(heads), block=block, n_splits=splits, tail_start=starts, tail_len=i32(tails))
    check_attention(out, q, k, v, [list(range(n)) + list(range(rows - 40, rows - 40 + t)) for n, t in zip(heads, tails)])


@pytest.mark.parametrize("tokens_first", [False, True])
def test_all_rows_of_a_cache_past_32_bits(tokens_first):
    """1.1 million rows of 8 heads (2.25 GB of codes), of which the last ones hold something.  The others have scales of
    zero: a logit of 0 and a value of 0 each, so the definition is a sum over the rows that do.  Tolerance: as above, and
    2^-13 for the sum of the weights of one (a thread adds 1240 of them up in fp32, 2^-24 each)."""
    KVH, H, rows, block = 8, 32, 1_100_000, 64
    cache = ops().kv8_alloc(1, KVH, rows, block=block, dtype=torch.int8, device="cuda", tokens_first=tokens_first)
    last = rows // block * block - block
    k, v = draw((1, KVH, 64, D), torch.bfloat16, 1), draw((1, KVH, 64, D), torch.bfloat16, 2)
    ops().kv8_store(k, v, *cache, block=block, start=last)
    ops().kv8_append(k[:, :, 3], v[:, :, 5], *cache, i32([rows - 1]), block=block)
    q = draw((1, H, D), torch.bfloat16, 5, outliers=False) * 4
    score = torch.zeros(KVH, 1, rows, device="cuda")
    out = ops().kv8_decode_attn(q, *cache, i32([rows]), block=block, score_out=score, score_len=i32([rows]))[0].double()
    at = list(range(last, last + 64)) + [rows - 1]
    blocks = torch.tensor([r // block for r in at], device="cuda")
    kk, vv = (c[0][:, at].double() * s[0][:, blocks].double()[..., None] for c, s in (cache[0::2], cache[1::2]))
    logits = torch.einsum("hgd,hnd->hgn", q[0].double().view(KVH, H // KVH, D), kk) / math.sqrt(D)
    size = (torch.einsum("hgd,hnd->hgn", q[0].double().view(KVH, H // KVH, D).abs(), kk.abs()) / math.sqrt(D)).max().item()
    top = logits.amax(2, keepdim=True).clamp(min=0)
    p = torch.exp(logits - top)
    p = p / (p.sum(2, keepdim=True) + (rows - len(at)) * torch.exp(-top))
    assert (p.sum(2) > 0.01).float().mean() > 0.5  # what was stored matters
    want, mass = (torch.einsum("hgn,hnd->hgd", p, x).reshape(H, D) for x in (vv, vv.abs()))
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -16 + 2 * 2.0 ** -17 * size + 2.0 ** -13) * mass + 1e-30
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max().item()
    best = logits.amax(1)
    assert ((score[:, 0, at].double() - best).abs() <= 2.0 ** -17 * size).all()
    score[:, 0, at] = 0
    assert (score == 0).all()
