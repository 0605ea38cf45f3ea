"""Where ``mlc.ops`` decides between neighbours: which tokens a row of logits keeps, and which of
two codes a quotient goes to. Rows and blocks whose borders lie where a kernel can miss them,
against the definitions in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import decoder_reference as ref
from mlc import ops
from test_decoder_operators import NEAR, TYPES, normal, options_of

gpu = pytest.mark.gpu
FULL = torch.float32
INF = float("inf")


# --------------------------------------------------------------------------
# the tokens that a row keeps
# --------------------------------------------------------------------------

def check_shares(row, n, **given):
    """``n`` random numbers, evenly over [0, 1), for one row: that the tokens are the right ones
    says which are kept and with which shares, as one draw does not."""
    uniform = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float()
    got = ops.sample(row.expand(n, -1), uniform.cuda(), **options_of(n, **given)).cpu().numpy()
    at, w = ref.kept(row.double().cpu().numpy(), **given)
    sums, u = np.cumsum(w), uniform.double().numpy()
    place = np.searchsorted(sums, u * sums[-1], side="right").clip(max=len(at) - 1)
    edges = np.concatenate([[-1.0], sums[:-1] / sums[-1], [2.0]])
    margin = np.minimum(u - edges[place], edges[place + 1] - u)
    wrong = (got != at[place]) & (margin > NEAR)
    assert not wrong.any(), (int(wrong.sum()), n, got[wrong][:5], at[place][wrong][:5], margin[wrong][:5])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", (1025, 1031, 2044, 4099, 8193, 8199, 50256, 50257, 50260, 50263, 50265))
def test_rows_whose_likely_tokens_lie_behind_the_last_whole_pack(dtype, size):
    """A token of the row's end, where it is no multiple of eight, at a border or in front of it: an
    end of text that is likely."""
    for rank in (1, 2, 5, 20, 50):
        x = normal(size, dtype=dtype, seed=rank, spread=3.0)
        other = x.float().argsort(descending=True, stable=True)[rank - 1].item()
        last = size - 1 - rank % max(1, size % 8)
        x[[last, other]] = x[[other, last]]
        for top_k in (2, 50, 512):
            for given in ({}, {"top_p": 0.9}, {"min_p": 0.01}, {"temperature": 0.8, "top_p": 0.95, "min_p": 0.002}):
                check_shares(x, 257, top_k=top_k, **given)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_tokens_take_nothing_of_their_neighbours(dtype):
    """A weight of 2^-41, half a step, beside masked tokens, at the random number 0."""
    x = torch.full((1, 3000), -INF, dtype=dtype, device="cuda")
    x[0, 8], x[0, 2992] = -41.0, 0.0
    for given in ({}, {"top_k": 2000}, {"top_k": 600, "min_p": 0.0}):
        # the temperature is log2 e, so that the weight is 2^-41
        options = options_of(1, temperature=1.4426950408889634, **given)
        assert ops.sample(x, torch.zeros(1, device="cuda"), **options).item() in (8, 2992)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_small_weights_beside_a_large_one(dtype):
    """Eight tokens that a pass over the row adds in fp32, of which seven have 2^-18 of the first: a random number in
    the middle of a token's share, 2^-19 from both ends, draws it."""
    x = torch.full((1, 3000), -INF, dtype=dtype, device="cuda")
    x[0, 64], x[0, 65:72] = 0.0, -18.0
    uniform = torch.tensor([(1 + (i + 0.5) * 2.0 ** -18) / (1 + 7 * 2.0 ** -18) for i in range(7)]).cuda()
    for given in ({}, {"top_p": 0.9999999}, {"top_k": 600}, {"min_p": 2.0 ** -20}):
        options = options_of(7, temperature=1.4426950408889634, **given)  # weights of 2^x
        assert ops.sample(x.expand(7, -1), uniform, **options).tolist() == list(range(65, 72))


# --------------------------------------------------------------------------
# the code that a quotient goes to
# --------------------------------------------------------------------------

F = 2.0 ** -24
LADDER = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
MIDDLES = (LADDER[1:] + LADDER[:-1]) / 2


def nearest(q):
    """``(code, distance)``: of each magnitude the nearest code, the even one of two, and how far, in
    shares of it, the nearest middle of two codes is."""
    q, middles = q.abs().clamp(max=448.0), MIDDLES.to(q.device)
    code = torch.searchsorted(middles, q.contiguous())
    above, below = middles[code.clamp(max=125)], middles[(code - 1).clamp(min=0)]
    distance = torch.minimum((above - q).abs(), (q - below).abs()) / q.clamp(min=2.0 ** -20)
    return code + ((q == above) & (code % 2 == 1)), distance


def check_codes(codes, y, bound):
    """Codes of ``y`` [rows, dim] are the nearest ones, but for those whose quotient is within ``bound`` of
    itself of a middle, and in it if ``bound`` is not zero."""
    y = y.cpu().double()
    codes = codes.view(torch.uint8).cpu()
    for i in range(0, y.shape[-1], 128):
        part, got = y[:, i:i + 128], codes[:, i:i + 128]
        q = part * 448 / part.abs().amax(-1, keepdim=True)  # exact in the middle of two codes
        want, distance = nearest(q)
        wrong = (got & 127) != want
        assert not (wrong & ((distance > bound) | (bound == 0))).any(), \
            (int(wrong.sum()), distance[wrong].max().log2(), q[wrong][:4], got[wrong][:4])
        assert ((got >> 7 == 1) == (part < 0))[want > 0].all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_of_rows_as_they_are(dtype):
    """Two operands of 16 bits have quotients in the middle of two codes, where the even one is right; of
    fp32 a quotient is rounded to fp32 once."""
    x = normal(2048, 512, dtype=dtype, seed=4)
    x[:, 1::7] *= 2.0 ** -9  # below e4m3's normal numbers
    x[::2, :128] = (x[::2, :128] * 8).round() / 8  # many quotients in the middle
    codes, _ = ops.quantize(x)
    check_codes(codes, x, 0.0 if dtype != FULL else 2 * F)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_residual", (False, True))
def test_every_code_of_norms(dtype, with_residual):
    """What all values of a row have in common does not count for its codes. A sum's rounding, the weight's
    product, the same for the largest, and the quotient's: 5 F."""
    x, w = normal(1024, 1024, dtype=dtype, seed=5), normal(1024, dtype=dtype, seed=6) + 1
    x[:, 3::5] *= 2.0 ** -8
    r = normal(1024, 1024, dtype=dtype, seed=7) if with_residual else None
    codes, *_ = ops.rms_norm(x, w, r, quantized=True)
    y, _ = ref.norm(x, w, r)
    check_codes(codes, y, 6 * F)


def gated(x, g):
    return x.double() * g.double() * torch.special.expit(g.double())


def near_middles(dtype, gates, small, rows=256, tries=1 << 17):
    """``(x, gate)``: rows of a block of 128, the largest value first and behind it values whose quotients lie
    within 2^-21 of the middle of two codes, but not within 2^-23. small: below e4m3's normal numbers."""
    r = torch.Generator(device="cuda").manual_seed(rows + small)
    uniform = lambda lo, hi, *shape: lo + (hi - lo) * torch.rand(*shape, generator=r, device="cuda")  # noqa: E731
    g = uniform(*gates, rows, tries).to(dtype)
    size = 60000.0 if gates[1] < 0 else 64.0
    x = (size * uniform(0.5, 1.0, rows, tries)).to(dtype)
    g[:, :1] = uniform(gates[1] - 4.0, gates[1], rows, 1).to(dtype)
    top = gated(x[:, :1], g[:, :1]).abs()
    q = uniform(*((-9.9, -6.01) if small else (-6.0, 8.6)), rows, tries).double().exp2()
    x[:, 1:] = (q * top / 448 / gated(torch.ones_like(g), g)).to(dtype)[:, 1:]
    y = gated(x, g)
    q = 448 * y / top
    _, distance = nearest(q)
    fine = (distance > 2.0 ** -23) & (distance < 2.0 ** -21) & (y.abs() < top) & (x.abs() > 2.0 ** -13)
    fine &= x.isfinite()
    fine[:, 0] = False
    order = fine.float().argsort(dim=1, descending=True, stable=True)[:, :127]
    keep = fine.gather(1, order)
    take = lambda t: torch.cat([t[:, :1], torch.where(keep, t.gather(1, order), 0.0)], 1)  # noqa: E731
    assert keep.sum() > 20
    return take(x), take(g)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("small", (False, True))
@pytest.mark.parametrize("gates", ((-4.0, 6.0), (-42.0, -36.0)), ids=("near", "far"))
def test_every_code_of_gated_rows(dtype, small, gates):
    """In 64 bits where fp32 does not tell: the gate is within 2^-28 of itself, and so is the
    largest value; a quotient is rounded to fp32."""
    x, g = near_middles(dtype, gates, small)
    check_codes(ops.quantize(x, g)[0], gated(x, g), 2 * F)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_of_gated_rows_of_many(dtype):
    x, g = normal(4096, 1024, dtype=dtype, seed=8), normal(4096, 1024, dtype=dtype, seed=9, spread=3.0)
    x[:, ::3] *= 2.0 ** -7
    x[:, 5] *= 30
    check_codes(ops.quantize(x, g)[0], gated(x, g), 2 * F)


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, FULL))
def test_every_code_of_values_and_gates_far_apart(dtype):
    """Products of both that fp32 holds where one of them or their product alone is beside its normal numbers."""
    x, g = normal(512, 256, dtype=FULL, seed=10), normal(512, 256, dtype=FULL, seed=11)
    for more, gates in ((2.0 ** 120, 2.0 ** -130), (2.0 ** -120, 2.0 ** 100), (2.0 ** 126, 1.0), (2.0 ** 70, 30.0)):
        a, b = (x * more).to(dtype), (g * gates).to(dtype)
        fine = gated(a, b).abs().view(512, 2, 128).amax(-1).repeat_interleave(128, 1) < 2.0 ** 127
        a = torch.where(fine, a, 1.0)  # of what is beyond fp32 the codes are NaN
        check_codes(ops.quantize(a, b)[0], gated(a, b), 2 * F)


# --------------------------------------------------------------------------
# sums whose large terms cancel
# --------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", (4, 40, 300))
def test_products_whose_large_terms_cancel(dtype, rows):
    """What is left of pairs of opposite terms shows how products are added: whole in fp32 and for few rows, else each
    cut at 2^-13 of the largest of eight (``groups``)."""
    n, k = 200, 1024
    a = normal(rows, k, dtype=FULL, seed=12).clamp(-3, 3)
    a[:, ::4] *= 100.0
    a[:, 1::4] = a[:, ::4]
    b = normal(n, k, dtype=FULL, seed=13).clamp(-3, 3)
    b[:, ::4] *= 100.0
    b[:, 1::4] = -b[:, ::4]
    a, b = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    a_scales, b_scales = torch.ones(rows, 8, device="cuda"), torch.ones(2, 8, device="cuda")
    want, *bounds = ref.product(a, a_scales, b, b_scales)
    got = ops.scaled_product(a, a_scales, b, b_scales, dtype=dtype)
    ref.check_product(got, want, *bounds, dtype)


# --------------------------------------------------------------------------
# norms near the end of fp32
# --------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_norms_near_the_largest_values(dtype):
    """Weights near fp32's largest: a norm that fp32 holds has codes and a scale, whatever the row's root is."""
    for size in (0.6, 0.7, 0.8, 1.0, 1.3, 1.5, 3.0, 1000.0):
        sign = normal(4, 256, dtype=FULL, seed=14).sign()
        x = (size * sign).to(dtype)
        w = torch.full((256,), 3.0e38, device="cuda")
        w[::3] = 1.0e38
        w[130:] = 1.0
        codes, scales = ops.rms_norm(x, w, quantized=True)
        y, _ = ref.norm(x, w)
        # a rounding of the weight's product, of the largest's and of the quotient
        check_codes(codes, y, 6 * F)
        want = y.abs().view(4, 2, 128).amax(-1) / 448
        assert ((scales.cpu().double() - want).abs() <= 16 * F * want).all()
