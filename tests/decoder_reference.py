"""Norms, rows in 8 bits, their products and the choice of a token from their definitions,
in 64 bits on the CPU, and how far a kernel may be from them (``U``, ``F`` and ``LEAST`` of
``operators_reference``)."""

from __future__ import annotations

import math

import numpy as np
import torch

from mlc.codegen.hip_decoder import is_exact
from operators_reference import F, LEAST, U

E4M3 = torch.float8_e4m3fn
BLOCK = 128
LEAST_SCALE = 2.0 ** -126


def _host(x):
    return None if x is None else x.detach().cpu().double()


def blocks_of(n):
    return -(-n // BLOCK)


def norm(x, weight, residual=None, eps=1e-6):
    """``(y, sum)``. The sum of x and the residual is rounded to fp32 once (F of it, and F at most
    of the mean's root with it), the norm once more to fp32."""
    h = _host(x) if residual is None else _host(x) + _host(residual)
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * _host(weight), h


def check_values(got, want, dtype, slack):
    """``got`` is ``want`` rounded to ``dtype`` from something that is ``slack`` of it off."""
    assert got.dtype == dtype and got.is_contiguous() and got.shape == want.shape
    bound = (U[dtype] * (1 + slack) + slack) * want.abs() + LEAST[dtype]
    off = (_host(got) - want).abs()
    fine = want.isfinite() & (want.abs() <= torch.finfo(dtype).max)
    assert (off <= bound)[fine].all(), (off / bound)[fine].max()
    assert not _host(got)[want.isnan()].isfinite().any()


def check_eight(codes, scales, y, slack):
    """``codes`` and ``scales`` are those of ``y``, that the kernel has within ``slack`` of it.

    A scale is off by that, and a division's rounding. A quotient is off by twice that and two
    roundings, and a code by half a step of e4m3: 2^-4 of the quotient, and below the smallest
    normal number 2^-6 2^-10.
    """
    n = y.shape[-1]
    assert codes.dtype == E4M3 and codes.is_contiguous() and codes.shape == y.shape
    assert scales.dtype == torch.float32 and scales.shape == (*y.shape[:-1], blocks_of(n))
    codes, scales = _host(codes.float()), _host(scales)
    for i in range(blocks_of(n)):
        part = y[..., i * BLOCK:(i + 1) * BLOCK]
        top = torch.where(part.isfinite(), part.abs(), 0.0).amax(-1)
        want = (top / 448).clamp(min=LEAST_SCALE)
        assert ((scales[..., i] - want).abs() <= (slack + 2 * F) * want).all()
        got = codes[..., i * BLOCK:(i + 1) * BLOCK]
        q = part * (448 / top).clamp(max=1 / LEAST_SCALE)[..., None]  # exact in the middle of two codes
        fine = part.isfinite()
        bound = (2.0 ** -4 + 2 * slack + 6 * F) * q.abs() + 2.0 ** -10
        assert ((got - q).abs() <= bound)[fine].all()
        # rounded, not cut: most are the nearest code
        near = (q.clamp(-448, 448).float().to(E4M3).double() == got)[fine]
        assert near.numel() < 64 or near.double().mean() > 0.99
        assert got[~fine].isnan().all()


def quantized(x, gate=None):
    """What :func:`check_eight` takes. fp32: in 64 bits, with a polynomial of 2^-28, within 2 F. 16-bit values': e^(-|g| / 2), twice, has an
    exponent that is 0.6 |g| F off, by the product's rounding and its factor's 0.22 F, and a unit of 2 F; with a sum,
    a reciprocal and four products that is within (16 + 1.25 |g|) F, until |g| = 175 leaves nothing."""
    y, slack = _host(x), 2 * F
    if gate is not None:
        g = _host(gate)
        y = y * (g * torch.special.expit(g))
        if gate.dtype != torch.float32:
            slack = (16 + 1.25 * g.abs().clamp(max=175).nan_to_num().max().item()) * F if g.numel() else 0.0
    return y, slack


def product(a, a_scales, b, b_scales, bias=None):
    """``(want, bound, groups, k)`` without the result's rounding. Within a block 128 products, exact in
    fp32, are added in any order: 128 F of their magnitudes' sum; a factor of two roundings, an
    addition for every block, of parts of them and of the bias.

    ``groups`` is what the 8-bit instruction adds to that: of eight neighbouring products each is
    cut to a multiple of 2^-13 of the group's largest power of two, so that eight are off by less than
    2^-10 of the largest."""
    k, n = a.shape[-1], b.shape[0]
    def wide(x, dim, size):
        return _host(x).repeat_interleave(BLOCK, dim).narrow(dim, 0, size)

    x = _host(a.float()) * wide(a_scales, -1, k)
    w = _host(b.float()) * wide(wide(b_scales, 0, n), 1, k)
    want = x @ w.t()
    bound = (BLOCK + blocks_of(k) + 8) * F * (x.abs() @ w.abs().t())
    # the largest product of a group is at most that of both sides' largest factors
    x, w = (torch.nn.functional.pad(z.abs(), (0, -k % 8)).unflatten(-1, (-1, 8)).amax(-1) for z in (x, w))
    groups = 2.0 ** -10 * (x @ w.t())
    if bias is not None:
        want = want + _host(bias)
        bound = bound + 2 * F * want.abs()
    return want, bound, groups, k


def check_product(got, want, bound, groups, k, dtype):
    assert got.dtype == dtype and got.is_contiguous() and got.shape == want.shape
    if not is_exact(math.prod(want.shape[:-1]), want.shape[-1], k, dtype):
        bound = bound + groups
    bound = bound * (1 + U[dtype]) + U[dtype] * want.abs() + LEAST[dtype]
    off = (_host(got) - want).abs()
    assert (off <= bound).all(), (off / bound).max()


def kept(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(indexes, weights)`` of what a row keeps, by index, from sorted sums in 64 bits."""
    x = np.asarray(row, dtype=np.float64)
    order = np.argsort(-x, kind="stable")
    if temperature < 2.0 ** -100:
        return order[:1], np.ones(1)
    w = np.exp((x[order] - x[order[0]]) / temperature)
    n = len(x)
    if 0 < top_k < n:
        n = top_k
    sums = np.cumsum(w[:n])
    n = min(n, max(1, int(np.count_nonzero(sums - w[:n] < top_p * sums[-1]))))
    n = min(n, int(np.count_nonzero(w >= min_p)))
    back = np.sort(order[:n])
    return back, np.exp((x[back] - x[order[0]]) / temperature)


def drawn(row, uniform, **options):
    """``(token, margin)``: how far, in shares of the kept weight, the next border is that a token
    was drawn by."""
    at, w = kept(row, **options)
    sums = np.cumsum(w)
    i = min(int(np.searchsorted(sums, uniform * sums[-1], side="right")), len(at) - 1)
    edges = np.abs(np.concatenate([[0.0], sums[:-1]]) / sums[-1] - uniform)
    return int(at[i]), float(edges[1:].min()) if len(edges) > 1 else 1.0
