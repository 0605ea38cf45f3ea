"""Norms, rows in 8 bits, their products and the choice of a token (``mlc.ops``) against
their definitions in 64 bits (``decoder_reference``), at the sizes, strides and values where
kernels go wrong."""

from __future__ import annotations

import gc
import math

import pytest
import torch

import decoder_reference as ref
import mlc
from mlc import ops
from mlc.runtime import hip_runtime
from mlc.runtime.executor import ExecutionError
from operators_reference import F

gpu = pytest.mark.gpu
HALF, BF, FULL = torch.float16, torch.bfloat16, torch.float32
TYPES = (HALF, BF, FULL)
E4M3 = torch.float8_e4m3fn
INF, NAN = float("inf"), float("nan")


def normal(*shape, dtype=HALF, seed=0, spread=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * spread).to(dtype).to(device)


def strided(x, how):
    """``x`` with other strides: a slice of wider rows, an odd place in memory, tokens in
    front of the batch, one row for all."""
    if how == "wide":
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 48), NAN, device=x.device).to(x.dtype)
        wide[..., 16:16 + x.shape[-1]] = x
        return wide[..., 16:16 + x.shape[-1]]
    if how == "odd":
        flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=x.device)
        flat[1:] = x.flatten()
        return flat[1:].view(x.shape)
    if how == "turned":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "one":
        return x[:1, :1].expand(x.shape)
    return x


# --------------------------------------------------------------------------
# norms and rows in 8 bits
# --------------------------------------------------------------------------

# In fp32's norm of the fp32 sum, what it does to the root, and the norm's own rounding. 16-bit values': 2 of the
# sum, 4 of eight squares added in fp32 under the root, 1 of the mean, 2 of the reciprocal root, 2 products.
NORM_SLACK = {t: (4 if t == FULL else 12) * F for t in TYPES}


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,how", [
    ((1, 1, 768), ""), ((3, 5, 7), ""), ((2, 1), ""), ((5, 16), "odd"), ((2, 3, 1000), "turned"),
    ((2, 9, 2048), "wide"), ((1, 3, 4096), "odd"), ((2, 2, 5120), "one"), ((3, 8200), ""),
    ((1, 2, 20001), "turned"), ((2, 32768), ""), ((0, 4, 64), "")])
@pytest.mark.parametrize("with_residual", (False, True))
@pytest.mark.parametrize("wide_weight", (False, True))
def test_rms_norm(dtype, shape, how, with_residual, wide_weight):
    x = strided(normal(*shape, dtype=dtype, spread=3.0), how)
    r = strided(normal(*shape, dtype=dtype, seed=1), "wide" if how else "") if with_residual else None
    w = normal(shape[-1], dtype=FULL if wide_weight else dtype, seed=2) + 1
    y, h = ref.norm(x, w, r, 1e-5)
    got = ops.rms_norm(x, w, r, eps=1e-5)
    if with_residual:
        got, total = got
        ref.check_values(total, h, dtype, F)
    ref.check_values(got, y, dtype, NORM_SLACK[dtype])
    if shape[-1] % 16 == 0:
        codes, scales, *rest = ops.rms_norm(x, w, r, eps=1e-5, quantized=True)
        ref.check_eight(codes, scales, y, NORM_SLACK[dtype])
        assert len(rest) == with_residual and all(torch.equal(z, total) for z in rest)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_norms_of_the_largest_and_smallest_values(dtype):
    """Squares beyond fp32, and rows whose mean is far below eps; one row does not reach another."""
    big, small = torch.finfo(dtype).max / 4, torch.finfo(dtype).tiny
    x = normal(5, 64, dtype=FULL).clamp(-3, 3)
    x[0] *= big / 3
    x[1] *= small
    x[2], x[3, 5], x[4, 6] = 0.0, NAN, INF
    x, w = x.to(dtype), torch.ones(64, dtype=dtype, device="cuda")
    y, _ = ref.norm(x, w)
    got = ops.rms_norm(x, w)
    ref.check_values(got[:3], y[:3], dtype, NORM_SLACK[dtype])
    assert got[3].isnan().all() and got[4, 6].isnan() and not got[4].nan_to_num().any()
    codes, scales = ops.rms_norm(x, w, quantized=True)
    ref.check_eight(codes[:3], scales[:3], y[:3], NORM_SLACK[dtype])
    assert codes[3].float().isnan().all() and scales[3, 0] == 2.0 ** -126


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,how", [
    ((1, 1, 16), ""), ((3, 128), "odd"), ((2, 3, 144), "wide"), ((4, 2, 4096), ""), ((2, 37, 1008), "turned"),
    ((1, 3, 12288), "odd"), ((5, 400), "wide"), ((0, 64), ""), ((3, 2, 48), "one")])
@pytest.mark.parametrize("gated", (False, True))
def test_quantize(dtype, shape, how, gated):
    x = strided(normal(*shape, dtype=dtype, spread=2.0), how)
    g = strided(normal(*shape, dtype=dtype, seed=1, spread=3.0), "wide" if how else "") if gated else None
    y, slack = ref.quantized(x, g)
    ref.check_eight(*ops.quantize(x, g), y, slack if gated else 0.0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_of_zeros_extremes_and_what_is_not_finite(dtype):
    x = normal(4, 400, dtype=dtype)
    x[0, :128], x[0, 128:256] = 0.0, torch.finfo(dtype).tiny
    x[1, 5], x[1, 130], x[1, 256], x[1, 399] = NAN, INF, -INF, torch.finfo(dtype).max
    x[2] = NAN
    x[3, :128] = torch.finfo(dtype).max
    x[3, 128:256:2] *= 2.0 ** -9  # below e4m3's normal numbers
    codes, scales = ops.quantize(x)
    ref.check_eight(codes, scales, x.cpu().double(), 0.0)
    assert (scales[2] == 2.0 ** -126).all() and codes[2].float().isnan().all()
    # gates far to both sides: 1 and 0 times x
    g = torch.full_like(x, 80.0)
    g[:, ::2] = -1000.0
    codes, scales = ops.quantize(x[3:], g[3:].clamp(max=1.0))
    y, slack = ref.quantized(x[3:], g[3:].clamp(max=1.0))
    ref.check_eight(codes, scales, y, slack)


@gpu
def test_gates_whose_sigmoid_is_no_normal_number():
    g = torch.linspace(-95.0, -80.0, 128, device="cuda")[None].repeat(2, 1)
    x = torch.full((2, 128), 1e36, device="cuda")
    x[1] = 1e-3
    codes, scales = ops.quantize(x, g)
    y, _ = ref.quantized(x, g)
    got = codes.float().cpu().double() * scales.cpu().double()
    fine = (g[0] > -88).cpu()  # beyond, e^88.7 is an infinity in fp32
    assert ((got[0] - y[0]).abs() <= 2.0 ** -4 * 1.01 * y[0].abs() + scales[0].item() * 2.0 ** -9)[fine].all()


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------

def coded(n, k, rows, seed=0, spread=1.0):
    """Codes and scales of random values, scales of very different sizes."""
    codes = (normal(n, k, dtype=FULL, seed=seed, spread=100.0 * spread).clamp(-448, 448)).to(E4M3)
    scales = normal(-(-n // rows), ref.blocks_of(k), dtype=FULL, seed=seed + 1).exp2() * 0.01
    return codes, scales


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 16), (1, 16, 128), (3, 17, 144), (15, 40, 256), (16, 128, 4096), (17, 130, 400), (32, 256, 1280),
    (33, 100, 1152), (48, 33, 1024), (64, 300, 2304), (65, 129, 272), (100, 7, 160), (128, 128, 2048),
    (130, 257, 1008), (200, 1024, 128), (300, 256, 4112), (513, 640, 640), (1, 5, 12304),
    (3, 100, 4240), (8, 48, 8208), (16, 4100, 272), (9, 4100, 144)])
@pytest.mark.parametrize("biased", (False, True))
def test_scaled_product(dtype, rows, n, k, biased):
    a, a_scales = coded(rows, k, 1)
    b, b_scales = coded(n, k, 128, seed=7)
    bias = normal(n, dtype=dtype if n % 2 else FULL, seed=5, spread=50.0) if biased else None
    got = ops.scaled_product(a, a_scales, b, b_scales, bias, dtype=dtype)
    ref.check_product(got, *ref.product(a, a_scales, b, b_scales, bias), dtype)


@gpu
@pytest.mark.parametrize("batch,tokens,n,k", [(2, 3, 40, 272), (3, 50, 200, 400), (0, 4, 16, 128), (2, 2, 0, 128)])
def test_products_of_rows_that_lie_apart(batch, tokens, n, k):
    """Slices of wider rows, tokens in front of the batch: what lies beside is not read as values."""
    a, a_scales = coded(batch * tokens, k, 1)
    a, a_scales = a.view(batch, tokens, k), a_scales.view(batch, tokens, ref.blocks_of(k))
    b, b_scales = coded(n, k, 128, seed=7)
    want = ref.product(a, a_scales, b, b_scales)
    for x, s in ((strided(a.float(), "wide").to(E4M3), a_scales), (a, strided(a_scales, "wide")),
                 (strided(a, "turned"), strided(a_scales, "turned"))):
        wide = torch.full((n, k + 32), 127, dtype=torch.uint8, device="cuda").view(E4M3)
        wide[:, 16:16 + k] = b
        ref.check_product(ops.scaled_product(x, s, wide[:, 16:16 + k], b_scales, dtype=FULL), *want, FULL)
        flipped = b_scales.t().contiguous().t()
        ref.check_product(ops.scaled_product(x, s, b, flipped, dtype=BF), *want, BF)
    one = a[:, :1].expand(a.shape)
    ref.check_product(ops.scaled_product(one, a_scales, b, b_scales, dtype=HALF),
                      *ref.product(one, a_scales, b, b_scales), HALF)


@gpu
@pytest.mark.parametrize("rows", (5, 80))
def test_products_behind_nan_and_scales_of_any_size(rows):
    a, a_scales = coded(rows, 400, 1)
    b, b_scales = coded(150, 400, 128, seed=3)
    a_scales[1], a_scales[2], b_scales[0, 1], b_scales[1] = 0.0, -3.0, 1e-30, 1e20
    clean = ops.scaled_product(a, a_scales, b, b_scales, dtype=FULL)
    ref.check_product(clean, *ref.product(a, a_scales, b, b_scales), FULL)
    a.view(torch.uint8)[3, 399] = 127
    b.view(torch.uint8)[140, 2] = 255
    got = ops.scaled_product(a, a_scales, b, b_scales, dtype=FULL)
    assert got[3].isnan().all() and got[:, 140].isnan().all()
    rest = torch.arange(rows) != 3
    assert torch.equal(got[rest][:, :140], clean[rest][:, :140])


@gpu
def test_a_quantized_layer_is_near_its_weight():
    torch.manual_seed(0)
    linear = torch.nn.Linear(400, 300, dtype=BF, device="cuda")
    layer = ops.ScaledLinear.from_linear(linear)
    x = normal(2, 9, 400, dtype=BF)
    codes, scales = ops.quantize(x)
    with torch.no_grad():
        got = layer(x)
        assert torch.equal(got, layer(codes, scales)) and got.dtype == BF
        want = torch.nn.functional.linear(x.double(), linear.weight.double(), linear.bias.double())
        size = torch.nn.functional.linear(x.double().abs(), linear.weight.double().abs())
    # both operands are off by 2^-4 of themselves, or 2^-10 of a scale that is 1/448 of a block's largest
    assert ((got - want).abs() <= 2.1 * 2.0 ** -4 * size + 2.0 ** -8 * want.abs() + 0.05).all()
    y, slack = ref.quantized(linear.weight)
    assert layer.codes.shape == (300, 400) and layer.scales.shape == (3, 4)
    off = (layer.codes.cpu().double() * layer.scales.cpu().double().repeat_interleave(128, 0)[:300]
           .repeat_interleave(128, 1)[:, :400] - y).abs()
    assert (off <= 2.0 ** -4 * 1.001 * y.abs() + 2.0 ** -10 * layer.scales.max().item()).all()


# --------------------------------------------------------------------------
# the choice of a token
# --------------------------------------------------------------------------

def options_of(batch, **given):
    made = {}
    for name, value in given.items():
        if value is not None:
            value = value if isinstance(value, (list, tuple)) else [value] * batch
            made[name] = torch.tensor(value, dtype=torch.int32 if name == "top_k" else FULL, device="cuda")
    return made


#: a weight is off by 2^-22 of itself and half a step of 2^-40: sums of 2^17 of them and the
#: borders they are compared with by less than this share
NEAR = 2.0 ** -20


def check_sample(logits, uniform, options, fewest=0.95):
    got = ops.sample(logits, uniform, **options).cpu()
    assert got.dtype == torch.int64 and got.shape == (len(logits),)
    rows, told = logits.double().cpu().numpy(), 0
    for b, row in enumerate(rows):
        token, margin = ref.drawn(row, float(uniform[b]), **{n: x[b].item() for n, x in options.items()})
        if margin > NEAR:
            told += 1
            assert got[b] == token, (b, got[b], token, margin)
    assert told >= fewest * len(rows)
    return got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,size,how", [(3, 1, ""), (5, 7, ""), (4, 513, "wide"), (17, 5000, "odd"),
                                            (3, 50257, ""), (2, 131072, "wide")])
@pytest.mark.parametrize("given", [
    {}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05},
    {"temperature": 1.3, "top_k": 300, "top_p": 0.8}, {"temperature": 0.8, "top_p": 0.5, "min_p": 0.2},
    {"temperature": 2.0, "top_k": 1000, "top_p": 0.99, "min_p": 1e-3}], ids=lambda o: "-".join(o))
def test_sample(dtype, batch, size, how, given):
    logits = strided(normal(batch, size, dtype=dtype, spread=3.0), how)
    g = torch.Generator().manual_seed(size)
    uniform = torch.rand(batch, generator=g).cuda()
    check_sample(logits, uniform, options_of(batch, **given), fewest=0.6)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_have_options_of_their_own(dtype):
    batch = 24
    logits = normal(batch, 3001, dtype=dtype, spread=4.0)
    uniform = torch.rand(batch, generator=torch.Generator().manual_seed(1)).cuda()
    options = options_of(
        batch, temperature=[0.0, 1e-38, 0.3, 1.0, 1.7, 1e30] * 4, top_k=[-1, 0, 5, 2999, 3001, 2 ** 31 - 1] * 4,
        top_p=[1.0, 0.3, 0.0, 0.95] * 6, min_p=[0.0, 0.0, 1.0, 1e-3, 0.3, 0.0, 0.5, 0.0] * 3)
    got = check_sample(logits, uniform, options, fewest=0.9)
    assert torch.equal(got[::6], logits[::6].float().argmax(-1).cpu())
    wide = {n: torch.stack([x, x * 0], 1)[:, 0] for n, x in options.items()}  # strided options
    assert torch.equal(ops.sample(logits, torch.stack([uniform, uniform], 1)[:, 1], **wide).cpu(), got)


@gpu
def test_tokens_that_are_equal_go_by_their_index():
    """Borders inside a run of equal logits, -0 and 0 among them, over more of a row than any list of a
    workgroup holds."""
    for size in (50, 3000, 40000):
        x = torch.zeros(6, size, device="cuda")
        x[:, 1::2] = -0.0
        x[:, size // 2] = 1.0
        uniform = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.9999, 0.999999], device="cuda")
        for given in ({"top_k": 10}, {"top_p": 0.5}, {"top_k": size // 2, "top_p": 0.7}, {"min_p": 0.9}, {}):
            check_sample(x, uniform, options_of(6, **given), fewest=0.6)
        first = ops.sample(x, uniform, **options_of(6, temperature=0.0)).cpu()
        assert (first == size // 2).all()
        assert (ops.sample(x * 0, uniform, **options_of(6, top_k=1)) == 0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ("even", "steps", "masked", "far", "cliff", "one"))
def test_borders_in_rows_of_many_kinds(dtype, kind):
    """As a model's, few different logits, few that are not masked, all but one far below the largest, some so and
    some near, and one alone: with fewer tokens than top_k asks for, lists too short for what lies at a border, or
    nothing there."""
    size = 60000
    x = normal(4, size, dtype=dtype, spread=1.0)
    if kind == "even":
        x *= 2.5
    elif kind == "steps":
        x = (x * 4).round() / 4
    elif kind == "masked":
        x[x < 2.5] = -INF
    elif kind == "far":
        x[:, 777] = 60.0
    elif kind == "cliff":
        x[:, ::7] += 40.0
    else:
        x[:] = -INF
        x[:, 59999] = -3.0
    uniform = torch.tensor([0.02, 0.5, 0.93, 0.9999], device="cuda")
    for given in ({"top_k": 60}, {"top_k": 1500}, {"top_p": 0.9}, {"top_p": 0.995}, {"min_p": 0.3},
                  {"top_k": 30000, "top_p": 0.95},
                  {"temperature": 0.01, "top_p": 0.6}, {"temperature": 30.0, "top_k": 20000, "top_p": 0.5}):
        check_sample(x, uniform, options_of(4, **given), fewest=0.5)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logits_that_are_masked(dtype):
    """Infinities and the type's lowest value are never taken beside others; a row of the lowest value
    alone is an even choice, one of -infinity has none."""
    low = torch.finfo(dtype).min
    x = torch.full((6, 999), -INF, dtype=dtype, device="cuda")
    x[1, 500] = low
    x[2] = low
    x[3, 10:20], x[4, ::3], x[5, 998] = 2.0, low, -5.0
    x[4, 6], x[4, 900] = 1.0, 1.5
    uniform = torch.tensor([0.5, 0.99, 0.5, 0.95, 0.3, 0.0], device="cuda")
    for given in ({}, {"top_p": 0.97}, {"top_k": 700}, {"temperature": 0.5, "min_p": 0.01}):
        got = ops.sample(x, uniform, **options_of(6, **given)).tolist()
        assert got[0] == -1 and got[1] == 500 and got[3] == 19 and got[5] == 998
        # the lesser of two has 1 / (1 + e^0.5) = 0.38 of their weight, at half the temperature 0.27
        assert got[4] == (900 if "temperature" in given else 6)
        n = int(ref.kept(torch.zeros(999), **given)[0][-1]) + 1
        assert got[2] == int(0.5 * n)
    ops.check_errors()


@gpu
def test_rows_that_are_invalid_are_told_and_left_at_none():
    batch = 12
    x = normal(batch, 300, dtype=BF)
    x[0, 7], x[1, 299] = NAN, INF
    uniform = torch.full((batch,), 0.5, device="cuda")
    uniform[2], uniform[3], uniform[4] = 1.0, -0.1, NAN
    options = options_of(batch, temperature=[1, 1, 1, 1, 1, -1, NAN, 1, 1, 1, 1, 1], top_p=[1] * 7 + [1.5, NAN, 1, 1, 1],
                         min_p=[0] * 9 + [2, -1, 0])
    got = ops.sample(x, uniform, **options)
    with pytest.raises(ExecutionError, match="sample"):
        ops.check_errors()
    assert (got[:11] == -1).all() and got[11] >= 0
    for which in range(11):
        one = slice(which, which + 1)
        ops.sample(x[one], uniform[one], **{n: o[one] for n, o in options.items()})
        with pytest.raises(ExecutionError, match="sample"):
            ops.check_errors()
    assert ops.sample(x[:0], uniform[:0]).shape == (0,)
    ops.check_errors()


@gpu
def test_shares_of_drawn_tokens():
    """Even random numbers give every kept token its share of them."""
    n, x = 4096, torch.tensor([[0.0, 1.0, -INF, 2.0, 3.0, -1.0]], device="cuda")
    uniform = (torch.arange(n, device="cuda") + 0.5) / n
    got = ops.sample(x.expand(n, 6), uniform, **options_of(n, temperature=0.9, top_p=0.99))
    at, w = ref.kept(x[0].cpu(), temperature=0.9, top_p=0.99)
    counts = torch.bincount(got.cpu(), minlength=6)
    assert counts.sum() == n and abs(counts[at].numpy() - n * w / w.sum()).max() <= 1


# --------------------------------------------------------------------------
# offsets past 32 bits
# --------------------------------------------------------------------------

@gpu
def test_rows_past_32_bits():
    n = 2 ** 17 + 5  # times 32768 values of 16 bits: 8 GB
    x = torch.zeros(n, 1, 32768, dtype=BF, device="cuda")
    x[-3:] = normal(3, 1, 32768, dtype=BF)
    w = torch.ones(32768, dtype=BF, device="cuda")
    want = ops.rms_norm(x[-3:], w)
    assert torch.equal(ops.rms_norm(x, w)[-3:], want)
    codes, scales = ops.quantize(x)
    few, few_scales = ops.quantize(x[-3:].contiguous())
    assert torch.equal(codes[-3:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scales[-3:], few_scales)
    del x
    # a, and then the result, past 2^31 values
    b, b_scales = coded(128, 32768, 128)
    got = ops.scaled_product(codes, scales, b, b_scales)
    assert torch.equal(got[-3:], ops.scaled_product(codes[-200:], scales[-200:], b, b_scales)[-3:])
    assert not got[:-3].any()
    b, b_scales = coded(2 ** 14 + 3, 128, 128)
    got = ops.scaled_product(codes[..., -128:], scales[..., -1:], b, b_scales)
    want = ops.scaled_product(codes[-200:, :, -128:], scales[-200:, :, -1:], b, b_scales)
    assert torch.equal(got[-3:], want[-3:]) and not got[:-3].any()


@gpu
def test_a_weight_and_logits_past_32_bits():
    n, k = 2 ** 17 + 70, 32768
    b = torch.zeros(n, k, dtype=torch.uint8, device="cuda").view(E4M3)
    b[-90:], some = coded(90, k, 128)
    b_scales = torch.ones(ref.blocks_of(n), ref.blocks_of(k), device="cuda")
    for rows in (2, 70):
        a, a_scales = coded(rows, k, 1, seed=3)
        got = ops.scaled_product(a, a_scales, b, b_scales, dtype=FULL)
        want = ops.scaled_product(a, a_scales, b[-90:], b_scales[:1], dtype=FULL)
        # another place in a tile of rows, and in the order of parts
        assert (got[:, -90:] - want).abs().max() <= 1e-4 * want.abs().max() and not got[:, :-90].any()
    del b
    x = torch.full((2 ** 12 + 3, 2 ** 20), -INF, dtype=HALF, device="cuda")
    x[-1, 7], x[-1, -1], x[0, 5] = 1.0, 1.0, 0.0
    uniform = torch.full((len(x),), 0.6, device="cuda")
    got = ops.sample(x, uniform)
    assert got[-1] == 2 ** 20 - 1 and got[0] == 5 and (got[1:-1] == -1).all()


# --------------------------------------------------------------------------
# a decoder's step: streams, graphs, compiled
# --------------------------------------------------------------------------

class Step(torch.nn.Module):
    """One layer of a decoder in 8 bits around its cache, and the choice of the next token."""

    def __init__(self, width=256, heads=4, kv=2, hidden=400, vocabulary=517, batch=2, capacity=1024, dtype=BF):
        super().__init__()
        torch.manual_seed(0)
        self.heads, self.kv, self.dim, dim = heads, kv, width // heads, width // heads
        linear = lambda i, o, **more: ops.ScaledLinear.from_linear(torch.nn.Linear(i, o, **more), dtype)  # noqa: E731
        self.embed = torch.nn.Embedding(vocabulary, width, dtype=dtype)
        self.qkv, self.out = linear(width, (heads + 2 * kv) * dim), linear(heads * dim, width, bias=False)
        self.gate, self.up = linear(width, hidden, bias=False), linear(width, hidden, bias=False)
        self.down = linear(hidden, width, bias=False)
        self.head = ops.ScaledLinear.from_linear(torch.nn.Linear(width, vocabulary, bias=False), FULL)
        for i in range(3):
            self.register_parameter(f"norm{i}", torch.nn.Parameter(torch.ones(width, dtype=dtype) + 0.1 * i, False))
        self.cache = ops.KeyValueCache(batch, kv, capacity, dim)
        self.register_buffer("frequencies", ops.rotary_frequencies(dim)[0])
        self.requires_grad_(False)

    def forward(self, tokens, start, uniform, temperature, top_k, top_p, min_p):
        x = self.embed(tokens)
        b, t, width = x.shape
        codes, scales = ops.rms_norm(x, self.norm0, quantized=True)
        y = self.qkv(codes, scales).view(b, t, self.heads + 2 * self.kv, self.dim)
        q, k, v = y.split([self.heads, self.kv, self.kv], 2)
        at = start.unsqueeze(1) + torch.arange(t, device=start.device, dtype=torch.int32)
        q, k = ops.rotary(q, k, at, self.frequencies)
        self.cache.append(k, v, start)
        a = self.cache.attend(q, start)
        codes, scales, x = ops.rms_norm(self.out(a.view(b, t, width)), self.norm1, x, quantized=True)
        y = self.down(*ops.quantize(self.up(codes, scales), self.gate(codes, scales)))
        y, x = ops.rms_norm(y, self.norm2, x)
        logits = self.head(y)[:, -1]
        return ops.sample(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p), logits, x


def step_inputs(batch=2, tokens=1, seed=0, start=(5, 600)):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 517, (batch, tokens), generator=g).cuda()
    uniform = torch.rand(batch, generator=g).cuda()
    options = options_of(batch, temperature=[0.8, 1.2][:batch], top_k=[50, 0][:batch], top_p=[1.0, 0.9][:batch],
                         min_p=[0.0, 0.01][:batch])
    return ids, torch.tensor(start[:batch], dtype=torch.int32, device="cuda"), uniform, *options.values()


@gpu
@pytest.mark.parametrize("tokens", (1, 5, 70))
@pytest.mark.parametrize("config", [{}, {"memory_planning": False}, {"cuda_graphs": False}],
                         ids=("graph", "unplanned", "planned"))
def test_a_compiled_step_is_the_step_to_the_bit(tokens, config):
    model, other = Step().cuda(), Step().cuda()
    compiled = mlc.compile(model, step_inputs(tokens=tokens), mlc.Config(**config))
    for i in range(4):
        args = step_inputs(tokens=tokens, seed=i, start=(5 + i, 900 - 70 * i))
        got = [x.clone() for x in compiled(*args)]
        with torch.no_grad():
            want = other(*args)
        for x, y in zip(got, want):
            assert x.dtype == y.dtype and torch.equal(x, y)
    compiled.check_errors()
    assert sum("mlc." in k.summary() for k in compiled.schedule) == 3 + 3 + 3 + 6 + 1
    args = list(step_inputs(tokens=tokens))
    args[2] = args[2] + 2
    assert (compiled(*args)[0] == -1).all()
    with pytest.raises(ExecutionError, match="sample"):
        compiled.check_errors()


@gpu
def test_steps_captured_into_graphs_and_replayed_in_turn():
    """Two graphs, each with memory of its own, eager steps and waits between their replays."""
    model, eager = Step().cuda(), Step().cuda()
    inputs = [step_inputs(tokens=1, seed=3), step_inputs(tokens=80, seed=4)]
    for args in inputs:
        model(*args)
    graphs, outs = [], []
    for args in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(model(*args))
        graphs.append(g)
    eager.cache.load_state_dict(model.cache.state_dict(), strict=False)
    for name, x in model.cache.named_buffers():
        dict(eager.cache.named_buffers())[name].copy_(x)
    for i in range(4):
        for args, g, out in zip(inputs, graphs, outs):
            fresh = step_inputs(tokens=args[0].shape[1], seed=10 + i, start=(7 + i, 300 + 90 * i))
            for x, y in zip(args, fresh):
                x.copy_(y)
            g.replay()
            want = eager(*fresh)
            for x, y in zip(out, want):
                assert torch.equal(x, y)
    ops.check_errors()


@gpu
def test_a_compiled_step_that_is_collected_while_a_graph_is_captured():
    model, args = Step().cuda(), step_inputs(tokens=3)
    compiled = mlc.compile(model, args)
    compiled(*args)
    want = model(*args)
    g = torch.cuda.CUDAGraph()
    gc.collect()
    with torch.cuda.graph(g):
        del compiled
        gc.collect()
        got = model(*args)
    assert hip_runtime._late
    g.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    again = mlc.compile(model, args)
    assert not hip_runtime._late and torch.equal(again(*args)[0], want[0])


def test_runtimes_that_are_collected_late(monkeypatch):
    closed, capturing = [], [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(hip_runtime.HipRuntime, "close", lambda self: closed.append(self.name))
    for name in ("first", "second"):
        r = hip_runtime.HipRuntime.__new__(hip_runtime.HipRuntime)
        r.name = name
        del r
        assert closed == []
    capturing[0] = False
    r = hip_runtime.HipRuntime.__new__(hip_runtime.HipRuntime)
    r.name = "third"
    del r
    assert sorted(closed) == ["first", "second", "third"] and not hip_runtime._late


@gpu
def test_operators_on_several_streams_have_memory_of_their_own():
    a, a_scales = coded(100, 4096, 1)  # few tiles: the sum is split and joined
    weights = [coded(256, 4096, 128, seed=i) for i in (3, 5)]
    x = normal(2, 40000, dtype=HALF, spread=3.0)
    uniform = torch.tensor([0.2, 0.7], device="cuda")
    options = options_of(2, top_p=0.9)
    wants = [ops.scaled_product(a, a_scales, *w, dtype=FULL) for w in weights]
    tokens = ops.sample(x, uniform, **options)
    streams, got = [torch.cuda.Stream() for _ in weights], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.scaled_product(a, a_scales, *weights[i], dtype=FULL),
                               ops.sample(x, uniform, **options)))
    torch.cuda.synchronize()
    for outs, want in zip(got, wants):
        for y, t in outs:
            assert torch.equal(y, want) and torch.equal(t, tokens)


@gpu
def test_calls_that_something_looks_on():
    """A dispatch mode, a tracer and a function transform see the operators; results are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, w, r = normal(3, 256), normal(256, seed=1), normal(3, 256, seed=2)
    layer = ops.ScaledLinear.from_linear(torch.nn.Linear(256, 99, bias=False, dtype=HALF, device="cuda"))
    uniform = torch.tensor([0.1, 0.5, 0.9], device="cuda")

    def f(x):
        codes, scales, total = ops.rms_norm(x, w, r, quantized=True)
        y, _ = ops.rms_norm(x, w, r)
        z = layer(codes, scales) + layer(*ops.quantize(ops.rms_norm(y, w), total))
        return ops.sample(z, uniform, top_p=uniform), *ops.rms_norm(y, w, quantized=True)

    want, seen = f(x), []
    with Log():
        got = f(x)
    for name in ("rms_norm", "add_rms_norm", "rms_norm_quantized", "add_rms_norm_quantized", "quantize",
                 "scaled_product", "sample"):
        assert f"mlc.{name}.default" in seen, name
    traced = torch.jit.trace(lambda x: f(x)[0], (x,), check_trace=False)
    kinds = [n.kind() for n in traced.graph.nodes()]
    assert "mlc::sample" in kinds and "mlc::scaled_product" in kinds
    assert torch.equal(traced(x), want[0])
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with torch.profiler.profile() as p:
        f(x)
    names = {e.key for e in p.key_averages()}
    assert {"mlc::sample", "mlc::scaled_product", "mlc::add_rms_norm_quantized"} <= names


# --------------------------------------------------------------------------
# what is refused, and what needs no GPU
# --------------------------------------------------------------------------

def host(*shape, dtype=HALF):
    return torch.zeros(*shape, dtype=dtype)


def _refused(call, match):
    with pytest.raises((ops.OperatorError, ExecutionError), match=match):
        call()


def test_what_norms_refuse():
    x, w = host(2, 3, 64), host(64)
    for args, why in (((x[0, 0], w), "rows, dim"), ((x.double(), w), "expected, got"), ((x, w[:32]), "weight"),
                      ((x, w.to(BF)), "weight"), ((x, host(128)[::2]), "weight"), ((x, w, x[:1]), "differ"),
                      ((x, w, x.float()), "differ"), ((x.transpose(1, 2), host(3)), "stride"),
                      ((x, w, host(2, 64, 3).transpose(1, 2)), "stride"), ((host(2, 0), host(0)), "dim of 1"),
                      ((host(1, 32769), host(32769)), "32768"), ((x, w), "ROCm GPU")):
        _refused(lambda: ops.rms_norm(*args), why)
    _refused(lambda: ops.rms_norm(host(2, 24), host(24), quantized=True), "multiple of 16")
    for eps in (0.0, -1.0, INF, NAN, 1e300):
        _refused(lambda: ops.rms_norm(x, w, eps=eps), "eps")


def test_what_quantize_refuses():
    x = host(2, 64)
    for args, why in (((host(2, 24),), "multiple of 16"), ((x.double(),), "expected, got"), ((x, x[:1]), "differ"),
                      ((x, x.float()), "differ"), ((host(64, 32).t(),), "stride"), ((x[0],), "rows, dim"),
                      ((x,), "ROCm GPU")):
        _refused(lambda: ops.quantize(*args), why)
    for bad in (host(3), torch.zeros(4, 4, dtype=torch.int32), host(4, 24), host(4, 0)):
        _refused(lambda: ops.quantize_weight(bad), "weight")


def test_what_scaled_product_refuses():
    codes = lambda *shape: torch.zeros(*shape, dtype=torch.uint8).view(E4M3)  # noqa: E731
    a, s, b, t = codes(2, 3, 272), torch.ones(2, 3, 3), codes(40, 272), torch.ones(1, 3)
    for args, why in (((a.float(), s, b, t), "expected, got"), ((a, s, b.float(), t), "expected, got"),
                      ((a, s[..., :2], b, t), "a_scales"), ((a, s.half(), b, t), "a_scales"),
                      ((a, s, b, t[:, :1]), "b_scales"), ((a, s, b[:, :256], t), "outputs, 272"),
                      ((a, s, codes(1, 40, 272), t), "outputs, 272"), ((codes(2, 24), s, codes(4, 24), t), "multiple"),
                      ((a, s, codes(40, 280)[:, :272], t), "16 bytes"), ((codes(2, 3, 280)[..., :272], s, b, t), "16 bytes"),
                      ((a, s, b, t, host(39)), "bias"), ((a, s, b, t, host(40)), "bias"),
                      ((a, s, codes(272, 40).t(), t), "stride"), ((a, s, b, t), "ROCm GPU")):
        _refused(lambda: ops.scaled_product(*args), why)
    for dtype in (torch.float64, E4M3, torch.int32):
        _refused(lambda: ops.scaled_product(a, s, b, t, dtype=dtype), "dtype")
    _refused(lambda: ops.ScaledLinear(24, 8), "multiple of 16")
    _refused(lambda: ops.ScaledLinear(32, 8, dtype=torch.float64), "dtype")


def test_what_sample_refuses():
    x, u, k = host(3, 9), torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    for call, why in ((lambda: ops.sample(x[0], u), "batch, tokens"), (lambda: ops.sample(x, u[:2]), "uniform"),
                      (lambda: ops.sample(x, u.double()), "uniform"), (lambda: ops.sample(x, u, temperature=u[:1]), "temperature"),
                      (lambda: ops.sample(x, u, top_k=u), "top_k"), (lambda: ops.sample(x, u, top_p=k), "top_p"),
                      (lambda: ops.sample(x, u, min_p=u.half()), "min_p"), (lambda: ops.sample(host(3, 0), u), "dim of 1"),
                      (lambda: ops.sample(host(9, 3).t(), u), "stride"), (lambda: ops.sample(x.long(), u), "expected, got"),
                      (lambda: ops.sample(torch.empty(1, 2 ** 22 + 1, device="meta"), u[:1].to("meta")), "4194304"),
                      (lambda: ops.sample(x, u, top_k=k), "ROCm GPU")):
        _refused(call, why)


def test_gradients_are_refused():
    x = host(2, 64).requires_grad_()
    _refused(lambda: ops.rms_norm(x, x[0].detach()), "gradient")
    _refused(lambda: ops.rms_norm(x.detach(), x[0], x.detach(), quantized=True), "gradient")
    _refused(lambda: ops.quantize(x), "gradient")
    _refused(lambda: ops.sample(x, torch.zeros(2)), "gradient")
    with torch.no_grad():
        _refused(lambda: ops.quantize(x), "ROCm GPU")


def test_a_weights_scales_and_codes():
    w = normal(130, 272, dtype=FULL, device="cpu")
    w[0, 0], w[128:, 256:], w[129, 3] = INF, 0.0, NAN
    codes, scales = ops.quantize_weight(w)
    assert codes.shape == (130, 272) and codes.is_contiguous() and scales.shape == (2, 3)
    assert codes[0, 0].float().isnan() and codes[129, 3].float().isnan() and scales[1, 2] == 2.0 ** -126
    assert not codes[128:, 256:].float().any()
    for i in range(2):
        for j in range(3):
            part = w[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            top = part[part.isfinite()].abs().max()
            assert abs(scales[i, j] - max(top / 448, 2.0 ** -126)) <= 2 * F * scales[i, j]
            got = codes[128 * i:128 * i + 128, 128 * j:128 * j + 128].float() * scales[i, j]
            assert ((got - part).abs() <= 2.0 ** -4 * 1.001 * part.abs() + 2.0 ** -10 * scales[i, j])[part.isfinite()].all()


def test_a_layer_keeps_its_types_and_its_state():
    m = torch.nn.Sequential(ops.ScaledLinear(64, 40, bias=True))
    m.half()
    assert m[0].codes.dtype == E4M3 and m[0].scales.dtype == FULL and m[0].bias.dtype == FULL
    assert m.to("meta")[0].codes.device.type == "meta"
    one = ops.ScaledLinear.from_linear(torch.nn.Linear(64, 40))
    two = ops.ScaledLinear(64, 40, bias=True, dtype=FULL)
    two.load_state_dict(one.state_dict())
    assert torch.equal(two.codes.view(torch.uint8), one.codes.view(torch.uint8)) and torch.equal(two.bias, one.bias)


def test_a_captured_step_keeps_its_operators():
    from mlc.api import build_pipeline
    from mlc.ir.capture import capture

    args = (torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.ones(2),
            torch.ones(2, dtype=torch.int32), torch.ones(2), torch.zeros(2))
    graph = capture(Step(), args)
    for cfg in (mlc.Config(), mlc.Config(merge_parallel_gemms=True, gemm_epilogue=True, layout_selection=True,
                                         fused_attention=True)):
        schedule = build_pipeline(capture(Step(), args), cfg)
        order = [k.node.op.split(".")[1] for k in schedule if hasattr(k, "node") and k.node.op.startswith("mlc.")]
        assert order.index("rms_norm_quantized") < order.index("cache_append") < order.index("cache_attention")
        assert sorted(order) == sorted(["rms_norm_quantized", "add_rms_norm_quantized", "add_rms_norm", "rotary",
                                        "cache_append", "cache_attention", "sample"] + 6 * ["scaled_product"]
                                       + 3 * ["quantize"])
    assert [tuple(v.shape) for v in graph.outputs] == [(2,), (2, 517), (2, 1, 256)]


def test_every_kernel_a_plan_asks_for_is_built_beforehand():
    import random

    from mlc.codegen import hip_decoder as plans
    from mlc.codegen.hip_operators import Operand

    def dense(*shape, dtype=HALF, aligned=True):
        strides = [1]
        for n in shape[:0:-1]:
            strides.insert(0, strides[0] * n)
        return Operand(shape, tuple(strides), dtype, aligned=aligned)

    known = {kernel for _, kernel in plans.all_kernels()}
    random.seed(1)
    seen = set()
    for _ in range(30000):
        if seen == known:
            break
        dtype, aligned = random.choice(TYPES), random.random() < 0.5
        rows, dim = round(2 ** random.uniform(0, 14)), round(2 ** random.uniform(0, 11)) * 16
        x, w = dense(rows, dim, dtype=dtype, aligned=aligned), dense(dim, dtype=dtype)
        other = x if random.random() < 0.5 else None
        n = round(2 ** random.uniform(0, 16))
        codes, weight = dense(rows, dim, dtype=E4M3), dense(n, dim, dtype=E4M3)
        scales, by = dense(rows, -(-dim // 128), dtype=FULL), dense(-(-n // 128), -(-dim // 128), dtype=FULL)
        option = lambda t=FULL: dense(rows, dtype=t) if random.random() < 0.5 else None  # noqa: E731
        found = [plans.plan_norm(x, w, other, 1e-6, random.random() < 0.5), plans.plan_quantize(x, other),
                 plans.plan_product(codes, scales, weight, by, None, dtype),
                 plans.plan_sample(dense(rows, n, dtype=dtype, aligned=aligned), dense(rows, dtype=FULL), option(),
                                   option(torch.int32), option(), option())]
        seen |= {launch.kernel for p in found for launch in p.launches}
    assert seen <= known, seen - known
    assert known <= seen, known - seen


def test_plans_refuse_codes_off_their_pieces_and_launches_too_large():
    from mlc.codegen import hip_decoder as plans
    from mlc.codegen.hip_operators import Operand

    a, s = Operand((4, 256), (256, 1), E4M3, 8, aligned=False), Operand((4, 2), (2, 1), FULL)
    b, t = Operand((64, 256), (256, 1), E4M3), Operand((1, 2), (2, 1), FULL)
    _refused(lambda: plans.plan_product(a, s, b, t, None, BF), "a: rows of codes")
    _refused(lambda: plans.plan_product(b, Operand((64, 2), (2, 1), FULL), a, t, None, BF), "b: rows of codes")
    x = Operand((2 ** 31 - 256, 1, 4096), (4096, 4096, 1), HALF)
    _refused(lambda: plans.plan_quantize(x, None), "split the batch")


def test_limits_that_kernels_and_plans_share():
    """Written in both: a limit of one that the other does not know would be a read past its end."""
    from mlc.codegen import hip_decoder as plans
    from mlc.codegen.hip_operators import SOURCES

    text = {n: (SOURCES / f"{n}.hip").read_text() for n in ("rows", "scaled_product", "sample")}
    assert f"QUANTIZE_BLOCK = {plans.QUANTIZE_THREADS}, QUANTIZE_PACKS = {plans.QUANTIZE_PACKS};" in text["rows"]
    assert f"JOIN_BLOCK = {plans.JOIN_THREADS};" in text["scaled_product"]
    assert f"SAMPLE_THREADS = {plans.SAMPLE_THREADS}," in text["sample"]
    assert plans.MOST_TOKENS <= 2 ** 22 and math.log2(plans.MOST_TOKENS) + 40 < 63
