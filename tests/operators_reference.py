"""The operators of ``mlc.ops`` from their definitions, in 64 bits on the CPU, and how
far a kernel may be from them: a rounding to a type is off by half a step, ``U[type]``
relative to the value, and fp32 arithmetic by ``F`` an operation.
"""

from __future__ import annotations

import math

import numpy as np
import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}
F = 2.0 ** -24
#: below the smallest normal number the step no longer shrinks with the value: fp16's
#: is 2^-24 there (numbers are multiples of it), so a rounding is off by up to 2^-25
#: whatever the value; bf16 2^-133, fp32 2^-149
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def _cpu(x):
    return None if x is None else x.detach().cpu()


def rotary(q, k, positions, frequencies, interleaved=False, magnitude=1.0):
    """``[(want, bound), (want, bound)]`` of queries and keys.

    Bound: the result's rounding, and of a cos - b sin the roundings of the cosine
    and sine (within 2 fp32 steps each, one more for the magnitude), two products and
    a sum: at most 8 F (|a| + |b|) * magnitude.
    """
    out = []
    n = 2 * frequencies.numel()
    p = _cpu(positions).double()
    p = p.expand(q.shape[0], -1) if p.dim() == 1 else p
    angle = (p[..., None] * _cpu(frequencies)).unsqueeze(2)
    for x in (q, k):
        y = _cpu(x).double().clone()
        bound = y.abs() * 0.0
        one = slice(0, n, 2) if interleaved else slice(0, n // 2)
        two = slice(1, n, 2) if interleaved else slice(n // 2, n)
        a, b = y[..., one].clone(), y[..., two].clone()
        y[..., one] = (a * angle.cos() - b * angle.sin()) * magnitude
        y[..., two] = (a * angle.sin() + b * angle.cos()) * magnitude
        slack = 8 * F * (a.abs() + b.abs()) * abs(magnitude)
        bound[..., one] = bound[..., two] = slack
        bound[..., :n] += U[x.dtype] * y[..., :n].abs() + LEAST[x.dtype]
        out.append((y, bound))
    return out


def _attend(q, k, v, seen, distance, scale, cap, slope, out_type, p_type):
    """One head: q [t, d], k and v [n, d], seen [t, n] -> (want, bound).

    The kernel's scores are off by delta: d products summed in fp32, the factor, the
    exponent's rounding (relative to the score), a cap evaluated within 2^-21 of cap.
    exp(s + delta) is off by delta relatively, in a weight and in their sum; weights
    are rounded to ``p_type`` and in fp16 lose what is below 2^-25.
    """
    s = q @ k.T * scale
    delta = (q.abs() @ k.abs().T) * scale * (q.shape[1] + 8) * F + s.abs() * 8 * F
    if cap:
        s = cap * torch.tanh(s / cap)
        delta = delta + cap * 2.0 ** -21
    if slope:
        s = s - slope * distance.abs()
        delta = delta + slope * distance.abs() * 8 * F
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    w = torch.where(seen, (s - top.nan_to_num(neginf=0.0)).exp(), torch.zeros_like(s))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    # only what is seen counts: 0 * inf is left out
    used = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    finite = used.nan_to_num(0.0, 0.0, 0.0)
    want = w @ finite
    for j in (~used.isfinite()).any(1).nonzero().flatten().tolist():
        hit = seen[:, j] & (w[:, j] > 0)
        want[hit] += (w[hit, j][:, None] * used[j]) - w[hit, j][:, None] * finite[j]
    d = torch.where(seen, delta, torch.zeros_like(delta)).amax(-1, keepdim=True) if s.shape[1] \
        else torch.zeros_like(top)
    bound = LEAST[out_type] + U[out_type] * want.abs() + (w @ finite.abs()) * (U[p_type] + 2 * d + 16 * F)
    if p_type == torch.float16:
        bound = bound + 2.0 ** -24 * (seen.double() @ finite.abs())
    return want, bound


def attention(q, k, v, *, scale=None, causal=False, cap=0.0, slopes=None, documents=None,
              prefix=None):
    b, tq, h, d = q.shape
    tk, group = k.shape[1], h // k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    kind = q.dtype
    q, k, v, slopes, documents, prefix = map(_cpu, (q, k, v, slopes, documents, prefix))
    want = torch.zeros(b, tq, h, d, dtype=torch.float64)
    bound = torch.zeros_like(want)
    at = torch.arange(tq)[:, None] + (tk - tq)
    key = torch.arange(tk)[None]
    for i in range(b):
        seen = torch.ones(tq, tk, dtype=torch.bool)
        if causal:
            seen = key <= at
            if prefix is not None:
                seen = seen | (key < prefix[i])
        if documents is not None:
            mine = documents[i][tk - tq:][:, None]
            seen = seen & (mine == documents[i][None]) & (mine >= 0)
        for j in range(h):
            want[i, :, j], bound[i, :, j] = _attend(
                q[i, :, j].double(), k[i, :, j // group].double(), v[i, :, j // group].double(), seen,
                (key - at).double(), scale, cap, 0.0 if slopes is None else float(slopes[j]), kind,
                kind)
    return want, bound


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count=None, *, scale=None,
                    cap=0.0, slopes=None):
    b, t, h, d = q.shape
    kv, capacity = k_cache.shape[1:3]
    block, group = capacity // k_scale.shape[2], h // kv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    kind = q.dtype
    q, start, slopes = _cpu(q), _cpu(start), _cpu(slopes)
    counts = [t] * b if count is None else _cpu(count).tolist()
    want = torch.zeros(b, t, h, d, dtype=torch.float64)
    bound = torch.zeros_like(want)
    for i in range(b):
        first, n = int(start[i]), counts[i]
        if first < 0 or n <= 0 or n > t or first + n > capacity:
            continue
        at = first + torch.arange(n)[:, None]
        key = torch.arange(first + n)[None]
        for j in range(h):
            kk, vv = (_cpu(c)[i, j // group].double()[:first + n]
                      * _cpu(s)[i, j // group].double().repeat_interleave(block)[:first + n, None]
                      for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
            want[i, :n, j], bound[i, :n, j] = _attend(
                q[i, :n, j].double(), kk, vv, key <= at, (key - at).double(), scale, cap,
                0.0 if slopes is None else float(slopes[j]), kind, torch.float16)
    return want, bound


# --------------------------------------------------------------------------
# the cache
# --------------------------------------------------------------------------

_GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()  # 0 .. 448


def e4m3(x: np.ndarray) -> np.ndarray:
    """Codes of ``x`` to the nearest value, a tie to the even code; what is not finite
    is NaN."""
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(_GRID, a), 1, 126)
    below, above = a - _GRID[hi - 1], _GRID[hi] - a
    code = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)
    code = code + 128 * np.signbit(x)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def exponent(amax: float) -> int:
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def values(codes: np.ndarray) -> np.ndarray:
    return torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()


def cache_append(cache, scales, fresh, start, count=None):
    """``(codes, scales)`` of one cache, keys or values, after the append: uint8 codes
    (NaN always 127) and float64 scales."""
    codes = cache.detach().cpu().view(torch.uint8).numpy().copy()
    codes[(codes & 127) == 127] = 127
    scales = scales.detach().cpu().double().numpy().copy()
    x = fresh.detach().cpu().double().numpy()
    batch, heads, capacity, _ = codes.shape
    block = capacity // scales.shape[2]
    for b in range(batch):
        first = int(start[b])
        n = x.shape[1] if count is None else int(count[b])
        if first < 0 or n < 0 or n > x.shape[1] or first + n > capacity:
            continue
        for at in range(first // block, -(-(first + n) // block)):
            lo, hi = max(first, at * block), min(first + n, (at + 1) * block)
            for h in range(heads):
                new = x[b, lo - first:hi - first, h]
                amax = np.abs(new[np.isfinite(new)]).max(initial=0.0)
                scale = 2.0 ** exponent(float(amax))
                if lo > at * block:
                    before = scales[b, h, at]
                    if before >= scale:
                        scale = before
                    else:
                        old = codes[b, h, at * block:lo]
                        codes[b, h, at * block:lo] = e4m3(values(old) * (before / scale))
                codes[b, h, lo:hi] = e4m3(new / scale)
                scales[b, h, at] = scale
    return codes, scales


def close(got, want, bound) -> None:
    """``got`` within ``bound`` of ``want`` everywhere; NaN and infinities alike."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    odd = ~want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[odd & ~want.isnan()], want[odd & ~want.isnan()])
    off = ((got - want).abs() - bound).masked_fill(odd, -math.inf)
    worst = off.argmax() if off.numel() else 0
    assert not off.numel() or off.max() <= 0, (
        f"{int((off > 0).sum())} of {off.numel()} values off; worst {got.flatten()[worst]:.6g} for "
        f"{want.flatten()[worst]:.6g}, bound {bound.flatten()[worst]:.3g}")
