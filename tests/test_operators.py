"""Operators of ``mlc.ops`` against their definitions in 64 bits
(``operators_reference``), at the sizes, strides and masks where kernels go wrong."""

from __future__ import annotations

import pytest
import torch

import mlc
import operators_reference as ref
from mlc import ops
from mlc.runtime.executor import ExecutionError

gpu = pytest.mark.gpu
HALF, BF, FULL = torch.float16, torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn


def normal(*shape, dtype=HALF, seed=0, spread=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=g) * spread).to(dtype).to(device)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def strided(x, how):
    """``x`` with other strides: heads in front of tokens, a slice of wider rows, or
    an odd place in memory."""
    if how == "heads":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "wide":
        wide = torch.zeros(*x.shape[:3], x.shape[3] + 24, dtype=x.dtype, device=x.device)
        wide[..., 8:8 + x.shape[3]] = x
        return wide[..., 8:8 + x.shape[3]]
    if how == "odd":
        flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=x.device)
        flat[1:] = x.flatten()
        return flat[1:].view(x.shape)
    if how == "qkv":  # one part of a merged projection
        both = torch.zeros(*x.shape[:2], 3, *x.shape[2:], dtype=x.dtype, device=x.device)
        both[:, :, 1] = x
        return both[:, :, 1]
    return x


# --------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", (HALF, BF, FULL))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,turned,far,how", [
    (1, 1, 12, 12, 64, 64, 0, ""),
    (2, 7, 4, 2, 128, 128, 1000000, "qkv"),
    (3, 5, 3, 1, 80, 32, 100000, "heads"),
    (1, 33, 2, 2, 6, 2, 5, ""),
    (2, 3, 5, 5, 96, 96, 7, "odd"),
    (2, 4, 2, 1, 72, 24, 2**31 - 9, "wide"),
    (1, 2, 2, 2, 64, 0, 3, ""),
    (1, 1500, 2, 1, 256, 256, 12345, ""),
])
def test_rotary(dtype, interleaved, batch, tokens, heads, kv, dim, turned, far, how):
    q = strided(normal(batch, tokens, heads, dim, dtype=dtype), how)
    k = strided(normal(batch, tokens, kv, dim, dtype=dtype, seed=1), how)
    f, magnitude = ops.rotary_frequencies(turned, scaling="bands", factor=4.0, original=512,
                                          device="cuda")
    p = (torch.arange(tokens, dtype=torch.int64) + far)[None] - torch.arange(batch)[:, None] * 2
    p = p.clamp(max=2**31 - 1).to("cuda").to(torch.int32 if tokens % 2 else torch.int64)
    for at in (p, p[0].contiguous()):
        got = ops.rotary(q, k, at, f, interleaved=interleaved, magnitude=magnitude)
        for x, (want, bound) in zip(got, ref.rotary(q, k, at, f, interleaved, magnitude)):
            assert x.dtype == dtype and x.is_contiguous()
            ref.close(x, want, bound)


@gpu
def test_rotary_positions_may_be_negative_and_frequencies_strided():
    q = normal(1, 4, 2, 64)
    f, _ = ops.rotary_frequencies(128, device="cuda")
    p = ints([-3, -2, 0, 1])
    got = ops.rotary(q, q, p, f[::2])
    for x, (want, bound) in zip(got, ref.rotary(q, q, p, f[::2])):
        ref.close(x, want, bound)


def test_rotary_frequencies_scalings():
    plain, one = ops.rotary_frequencies(64, 10000.0)
    assert one == 1.0 and plain[0] == 1.0 and plain.dtype == torch.float64
    assert torch.equal(ops.rotary_frequencies(64, scaling="linear", factor=4.0)[0], plain / 4)
    based, _ = ops.rotary_frequencies(64, scaling="base", factor=4.0)
    assert based[0] == 1.0 and abs(based[-1] / plain[-1] - 0.25) < 1e-12
    banded, mag = ops.rotary_frequencies(64, scaling="bands", factor=4.0, original=4096)
    assert banded[0] == 1.0 and banded[-1] == plain[-1] / 4 and abs(mag - 1.1386294) < 1e-6
    with pytest.raises(ops.OperatorError, match="even number"):
        ops.rotary_frequencies(7)
    with pytest.raises(ops.OperatorError, match="scaling"):
        ops.rotary_frequencies(8, scaling="other")


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def _heads(batch, tq, tk, heads, kv, dim, dtype, seed=0):
    return (normal(batch, tq, heads, dim, dtype=dtype, seed=seed, spread=2.0),
            normal(batch, tk, kv, dim, dtype=dtype, seed=seed + 1),
            normal(batch, tk, kv, dim, dtype=dtype, seed=seed + 2))


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("batch,tq,tk,heads,kv,dim,causal,how", [
    (1, 1, 1, 1, 1, 64, True, ""),
    (1, 128, 128, 12, 12, 64, True, ""),
    (2, 65, 65, 4, 2, 96, True, "qkv"),
    (1, 1, 300, 8, 1, 128, True, ""),
    (1, 257, 130, 2, 1, 64, True, ""),       # queries in front of every key: empty rows
    (2, 33, 129, 6, 2, 80, False, "heads"),
    (1, 64, 64, 2, 2, 256, False, "wide"),
    (3, 17, 200, 3, 3, 8, True, ""),
    (1, 190, 190, 7, 1, 128, True, "odd"),
    (8, 40, 40, 2, 1, 128, False, "qkv"),
    (1, 5, 0, 2, 2, 64, False, ""),
    (2, 3, 64, 64, 1, 64, True, ""),
])
def test_attention(dtype, batch, tq, tk, heads, kv, dim, causal, how):
    q, k, v = (strided(x, how) for x in _heads(batch, tq, tk, heads, kv, dim, dtype))
    got = ops.attention(q, k, v, causal=causal)
    assert got.is_contiguous() and got.dtype == dtype
    ref.close(got, *ref.attention(q, k, v, causal=causal))


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("tq,tk,dim", [(70, 70, 64), (33, 161, 128), (1, 97, 256), (200, 200, 96)])
@pytest.mark.parametrize("options", [
    {"cap": 5.0}, {"slopes": True}, {"documents": True}, {"prefix": True, "causal": True},
    {"cap": 3.0, "slopes": True, "documents": True, "prefix": True, "causal": True, "scale": 0.3},
    {"documents": True, "causal": True}, {"slopes": True, "causal": True}],
    ids=lambda o: "-".join(o))
def test_attention_masks_and_biases(dtype, tq, tk, dim, options):
    q, k, v = _heads(2, tq, tk, 4, 2, dim, dtype, seed=5)
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.tensor([0.5, 0.1, 0.0, 0.02], device="cuda")
    if "documents" in options:
        ids = torch.arange(tk) * 3 // tk
        other = torch.randint(-1, 3, (tk,), generator=torch.Generator().manual_seed(3))
        options["documents"] = torch.stack([ids, other]).to(torch.int32).to("cuda")
    if "prefix" in options:
        options["prefix"] = ints([tk // 2, tk + 7])
    ref.close(ops.attention(q, k, v, **options), *ref.attention(q, k, v, **options))


@gpu
@pytest.mark.parametrize("batch,tq,tk,heads,kv,dim", [
    (2, 1200, 1200, 2, 2, 64), (2, 700, 900, 4, 1, 128), (2, 600, 640, 2, 1, 256), (2, 2, 5000, 2, 1, 96),
    (2, 500, 700, 1, 1, 80), (8, 300, 333, 24, 24, 64), (2, 260, 700, 32, 32, 128), (2, 700, 700, 16, 16, 80)])
@pytest.mark.parametrize("causal", (False, True))
def test_attention_over_documents_of_many_tiles(batch, tq, tk, heads, kv, dim, causal):
    """In order, out of order with gaps, and few large ones with padding, where workgroups share
    tiles of keys and where their waves take them apart."""
    q, k, v = _heads(batch, tq, tk, heads, kv, dim, BF, seed=11)
    g = torch.Generator().manual_seed(5)
    at = torch.arange(tk)
    ordered = at * 9 // tk
    mixed = torch.randint(-1, 4, (tk // 50 + 1,), generator=g).repeat_interleave(50)[:tk]
    padded = torch.where(at < tk * 7 // 8, at // (tk // 2), -1)
    documents = torch.stack([(ordered, mixed, padded)[i % 3] for i in range(batch)]).to(torch.int32).cuda()
    if batch == 2:
        documents[0] = padded.to(torch.int32)
    ref.close(ops.attention(q, k, v, documents=documents, causal=causal),
              *ref.attention(q, k, v, documents=documents, causal=causal))


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("dim", (64, 128))
def test_attention_is_not_touched_by_what_it_does_not_see(dtype, dim):
    """NaN, infinities and the type's lowest value at keys that rows do not see, in
    tiles that other rows see part of."""
    q, k, v = _heads(1, 150, 150, 2, 1, dim, dtype, seed=9)
    documents = torch.cat([torch.zeros(75), torch.ones(60), -torch.ones(15)])[None].to(torch.int32).cuda()
    low = torch.finfo(dtype).min
    for at, kk, vv in ((149, float("nan"), float("inf")), (140, low, float("nan")),
                       (74, float("inf"), -float("inf")), (100, 0.5, float("inf"))):
        k[0, at], v[0, at] = kk, vv
    ref.close(ops.attention(q, k, v, documents=documents, causal=True),
              *ref.attention(q, k, v, documents=documents, causal=True))
    k[0, 74], v[0, 74] = 0.5, 2.0
    ref.close(ops.attention(q[:, :100], k[:, :100], v[:, :100], causal=True),
              *ref.attention(q[:, :100], k[:, :100], v[:, :100], causal=True))
    clean = ops.attention(q[:, :120], k[:, :120], v[:, :120], causal=True)
    assert clean[0, :100].isfinite().all() and not clean[0, 100:].isfinite().any()


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("bad", (float("nan"), float("inf")))
def test_a_key_of_hardly_any_weight_is_still_seen(dtype, bad):
    """A weight of e^-100 is below what its type holds, and times infinity it is not zero."""
    q, k, v = _heads(1, 40, 100, 1, 1, 64, dtype, seed=4)
    k[0, 7], v[0, 7, 0, 5] = -1.0, bad
    q.fill_(10.0)
    k[0, 8:] = 0.25
    got = ops.attention(q, k, v)
    ref.close(got, *ref.attention(q, k, v))
    assert not got[..., 5].isfinite().any() and got[..., 6:].isfinite().all()


@gpu
def test_prefixes_of_any_value():
    q, k, v = _heads(4, 70, 70, 2, 1, 64, HALF, seed=4)
    prefix = ints([-2 ** 31, 2 ** 31 - 1, -1, 1])
    ref.close(ops.attention(q, k, v, causal=True, prefix=prefix),
              *ref.attention(q, k, v, causal=True, prefix=prefix))


@gpu
def test_attention_over_a_long_row_and_its_last_tokens():
    q, k, v = _heads(1, 3, 5000, 4, 2, 64, HALF, seed=2)
    ref.close(ops.attention(q, k, v, causal=True), *ref.attention(q, k, v, causal=True))
    slopes = torch.tensor([0.3, 0.01, 0.001, 0.0], device="cuda")
    ref.close(ops.attention(q, k, v, causal=True, slopes=slopes, cap=4.0),
              *ref.attention(q, k, v, causal=True, slopes=slopes, cap=4.0))


@gpu
def test_attention_of_scores_that_are_far_apart():
    """A later key far above the earlier ones, and far below: the running maximum
    grows by more than an exponent holds."""
    q, k, v = _heads(1, 200, 200, 1, 1, 64, BF, seed=3)
    k[0, 130:] *= 60
    ref.close(ops.attention(q, k, v), *ref.attention(q, k, v))
    ref.close(ops.attention(q, k.flip(1), v), *ref.attention(q, k.flip(1), v))


# --------------------------------------------------------------------------
# the cache
# --------------------------------------------------------------------------

def filled(batch, kv, capacity, dim, block=64, seed=0):
    cache = ops.KeyValueCache(batch, kv, capacity, dim, block=block, device="cuda")
    for name, at in (("key", seed), ("value", seed + 1)):
        x = normal(batch, kv, capacity // block, block * dim, dtype=FULL, seed=at)
        x = x * normal(1, 1, capacity // block, 1, dtype=FULL, seed=at + 7).exp2()
        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1) / 448)))
        getattr(cache, f"{name}_scales").copy_(scale)
        getattr(cache, f"{name}s").copy_((x / scale[..., None]).to(E4M3).view(batch, kv, capacity, dim))
    return cache


def parts(cache):
    return cache.keys, cache.values, cache.key_scales, cache.value_scales


def check_append(cache, k, v, start, count=None):
    wants = [ref.cache_append(c, s, x, start, count)
             for c, s, x in ((cache.keys, cache.key_scales, k), (cache.values, cache.value_scales, v))]
    cache.append(k, v, start, count)
    for _ in range(2):  # a second time changes nothing
        torch.cuda.synchronize()
        for (codes, scales), c, s in zip(wants, (cache.keys, cache.values),
                                         (cache.key_scales, cache.value_scales)):
            got = c.cpu().view(torch.uint8).numpy().copy()
            got[(got & 127) == 127] = 127
            assert (got == codes).all()
            assert (s.double().cpu().numpy() == scales).all()
        cache.append(k, v, start, count)


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF, FULL))
@pytest.mark.parametrize("batch,tokens,kv,dim,capacity,block,start,count,how", [
    (1, 1, 1, 64, 64, 64, [0], None, ""),
    (3, 1, 2, 128, 256, 64, [63, 64, 255], None, "qkv"),
    (2, 5, 2, 16, 128, 32, [30, 0], [5, 3], "heads"),
    (2, 200, 1, 256, 512, 128, [100, 312], None, ""),
    (4, 70, 3, 96, 256, 64, [0, 1, 127, 186], [70, 0, 65, 70], "wide"),
    (2, 9, 2, 80, 96, 32, [40, 87], [9, 9], "odd"),
])
def test_cache_append(dtype, batch, tokens, kv, dim, capacity, block, start, count, how):
    cache = filled(batch, kv, capacity, dim, block)
    k = strided(normal(batch, tokens, kv, dim, dtype=dtype, seed=3, spread=3.0), how)
    v = strided(normal(batch, tokens, kv, dim, dtype=dtype, seed=4, spread=0.01), how)
    check_append(cache, k, v, ints(start), None if count is None else ints(count))
    # larger ones behind: the scale grows and the codes in front are rounded to it
    room = capacity - max(start) - tokens
    if room:
        check_append(cache, k[:, :1] * 100, v[:, :1] * 100,
                     ints([s + (tokens if count is None else c) for s, c in
                           zip(start, count or start)]))


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF, FULL))
def test_cache_append_of_zeros_and_of_what_is_not_finite(dtype):
    cache = filled(1, 1, 64, 16)
    x = torch.zeros(1, 6, 1, 16, dtype=dtype, device="cuda")
    check_append(cache, x, x, ints([0]))
    y = x.clone()
    y[0, 1, 0, 3], y[0, 2, 0, 4], y[0, 3, 0, 5] = float("nan"), float("inf"), -float("inf")
    y[0, 4, 0, :] = torch.finfo(dtype).max
    y[0, 5, 0, :] = torch.finfo(dtype).tiny
    check_append(cache, y, y * 0.5, ints([2]))
    check_append(cache, y[:, 5:], y[:, 4:5], ints([0]))


@gpu
def test_sequences_outside_of_their_cache_are_left_alone_and_told():
    cache = filled(4, 2, 128, 64)
    before = [x.clone().view(torch.uint8) if x.dtype == E4M3 else x.clone() for x in parts(cache)]
    x = normal(4, 2, 2, 64)
    cache.append(x, x, ints([-1, 127, 2**31 - 1, 5]), ints([2, 2, 2, 3]))
    with pytest.raises(ExecutionError, match="outside its cache"):
        ops.check_errors()
    for a, b in zip(before, parts(cache)):
        assert torch.equal(a, b.view(torch.uint8) if b.dtype == E4M3 else b)
    got = cache.attend(normal(4, 2, 4, 64), ints([-1, 127, 5, 6]), ints([2, 2, -1, 2]))
    torch.cuda.synchronize()
    assert not got[:3].any() and got[3].any()
    with pytest.raises(ExecutionError, match="outside its cache"):
        cache.append(x, x, ints([0, 0, 0, 0]))
    cache.append(x, x, ints([0, 0, 0, 0]))
    ops.check_errors()


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,capacity,block,start,count", [
    (1, 1, 12, 12, 64, 1024, 64, [0], None),
    (1, 1, 12, 12, 64, 1024, 64, [1023], None),
    (3, 1, 8, 2, 128, 2048, 64, [5, 2000, 640], None),
    (2, 1, 16, 1, 256, 512, 32, [511, 33], None),
    (2, 3, 4, 4, 96, 256, 128, [100, 0], [3, 1]),
    (2, 9, 8, 2, 128, 384, 64, [60, 375], None),
    (1, 70, 6, 2, 64, 192, 32, [100], [66]),
    (4, 1, 2, 1, 16, 128, 32, [0, 31, 32, 127], [1, 1, 0, 1]),
    (2, 40, 4, 1, 256, 128, 64, [88, 1], None),
    (1, 1, 4, 2, 80, 8192, 64, [8191], None),
    (70, 1, 2, 1, 64, 2048, 64, [i * 29 for i in range(70)], None),
])
@pytest.mark.parametrize("options", ({}, {"cap": 4.0, "slopes": True, "scale": 0.2}), ids=("", "all"))
def test_cache_attention(dtype, batch, tokens, heads, kv, dim, capacity, block, start, count, options):
    cache = filled(batch, kv, capacity, dim, block, seed=2)
    q = normal(batch, tokens, heads, dim, dtype=dtype, seed=6)
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = torch.linspace(0, 0.3, heads, device="cuda")
    start, count = ints(start), None if count is None else ints(count)
    for at in (q, strided(q, "wide")):
        ref.close(cache.attend(at, start, count, **options),
                  *ref.cache_attention(q, *parts(cache), start, count, **options))


@gpu
@pytest.mark.parametrize("dtype", (HALF, BF))
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,capacity,block,start,count", [
    (1, 64, 4, 2, 64, 512, 64, [300], None),
    (2, 33, 8, 2, 128, 256, 32, [0, 223], [33, 20]),
    (3, 40, 4, 1, 96, 128, 128, [0, 88, 5], [40, 40, 0]),
    (1, 150, 1, 1, 256, 384, 64, [100], [149]),
    (2, 20, 16, 2, 16, 96, 32, [76, 1], None),
    (1, 128, 2, 2, 128, 4096, 64, [3900], None),
])
@pytest.mark.parametrize("options", ({}, {"cap": 4.0, "slopes": True, "scale": 0.2}), ids=("", "all"))
def test_cache_attention_of_many_rows(monkeypatch, dtype, batch, tokens, heads, kv, dim, capacity, block,
                                      start, count, options):
    """By tiles of codes, which are for more products than a test has."""
    from mlc.codegen import hip_operators

    monkeypatch.setattr(hip_operators, "MANY_PRODUCTS", 0)
    monkeypatch.setattr(hip_operators, "MANY_ROWS", 1)
    ops._plans.clear()
    try:
        cache = filled(batch, kv, capacity, dim, block, seed=2)
        q = normal(batch, tokens, heads, dim, dtype=dtype, seed=6)
        options = dict(options)
        if "slopes" in options:
            options["slopes"] = torch.linspace(0, 0.3, heads, device="cuda")
        start, count = ints(start), None if count is None else ints(count)
        for at in (q, strided(q, "wide")):
            ref.close(cache.attend(at, start, count, **options),
                      *ref.cache_attention(q, *parts(cache), start, count, **options))
        # NaN behind the last key, and at a key that the first rows do not see
        codes = cache.values.view(torch.uint8)
        end = int(start[0]) + (tokens if count is None else int(count[0]))
        codes[0, :, end:] = 127
        codes[0, 0, end - 1, 3] = 255
        ref.close(cache.attend(q, start, count, **options),
                  *ref.cache_attention(q, *parts(cache), start, count, **options))
        assert any("attention_" in x.symbol and "codes" in x.symbol for plan in ops._plans.values()
                   for x in plan.launches)
    finally:
        ops._plans.clear()


@gpu
def test_cache_attention_of_a_piece_of_a_prompt():
    """As many rows and keys as go through tiles of codes by themselves."""
    cache = filled(1, 2, 16384, 128)
    q, start = normal(1, 192, 8, 128, seed=1, dtype=BF), ints([16000])
    got = cache.attend(q, start)
    for t in (0, 100, 191):
        one = ops.cache_attention(q[:, t:t + 1], *parts(cache), start + t)
        ref.close(one, *ref.cache_attention(q[:, t:t + 1], *parts(cache), start + t))
        ref.close(got[:, t:t + 1], *ref.cache_attention(q[:, t:t + 1], *parts(cache), start + t))


@gpu
def test_cache_attention_does_not_read_behind_a_sequence():
    """NaN behind the last key and, among several new tokens, at keys that only the
    later ones see."""
    cache = filled(2, 1, 256, 64)
    codes = cache.values.view(torch.uint8), cache.keys.view(torch.uint8)
    codes[0][0, :, 150:], codes[1][0, :, 150:] = 127, 255
    codes[0][0, :, 147, 5] = 255
    start, q = ints([145, 20]), normal(2, 5, 4, 64)
    got = cache.attend(q, start)
    ref.close(got, *ref.cache_attention(q, *parts(cache), start))
    assert got[0, :2].isfinite().all() and got[0, 2:, :, 5].isnan().all()
    assert got[0, :, :, 6:].isfinite().all() and got[1].isfinite().all()


@gpu
def test_cache_attention_over_blocks_of_very_different_scales():
    cache = filled(1, 1, 512, 64)
    cache.value_scales[0, 0] = torch.exp2(torch.tensor([-120., 0, 60, -60, 10, -10, 90, -126]))
    cache.key_scales[0, 0, 2] = 0.0
    q = normal(1, 1, 2, 64, dtype=BF)
    ref.close(cache.attend(q, ints([400])), *ref.cache_attention(q, *parts(cache), ints([400])))


@pytest.fixture(params=("rows", "tiles"))
def way(request, monkeypatch):
    """Both ways that rows go over the cache, whatever their number."""
    from mlc.codegen import hip_operators

    if request.param == "tiles":
        monkeypatch.setattr(hip_operators, "MANY_PRODUCTS", 0)
        monkeypatch.setattr(hip_operators, "MANY_ROWS", 1)
    ops._plans.clear()
    yield request.param
    ops._plans.clear()


@gpu
@pytest.mark.parametrize("dim,capacity", [(64, 256), (128, 8192)])
def test_cache_attention_of_the_largest_values(way, dim, capacity):
    """As many keys of bf16's largest values as there are: the sum of weights and values
    stays finite."""
    cache = ops.KeyValueCache(1, 1, capacity, dim, device="cuda")
    cache.keys.fill_(0.0)
    cache.values.fill_(1.75)
    cache.value_scales.fill_(2.0 ** 127)
    q = normal(1, 3, 2, dim, dtype=BF)
    ref.close(cache.attend(q, ints([capacity - 3])),
              *ref.cache_attention(q, *parts(cache), ints([capacity - 3])))


@gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf")))
def test_scales_of_blocks_that_a_row_does_not_see(way, bad):
    cache = filled(1, 1, 256, 64)
    cache.key_scales[0, 0, 2:], cache.value_scales[0, 0, 2:] = bad, bad
    q, start = normal(1, 40, 2, 64), ints([100])  # 28 rows see two blocks, 12 a third
    got = cache.attend(q, start)
    assert got[:, 28:].isnan().all()
    ref.close(got[:, :28], *ref.cache_attention(q[:, :28], *parts(cache), start))


# --------------------------------------------------------------------------
# offsets past 32 bits
# --------------------------------------------------------------------------

@gpu
def test_rotary_past_32_bits():
    n = 2 ** 17 + 3  # times 128 heads of 128
    q = torch.zeros(1, n, 128, 128, dtype=HALF, device="cuda")
    q[0, -3:] = normal(3, 128, 128)
    k = q[:, :, :1]
    positions = torch.arange(n, device="cuda", dtype=torch.int32)
    f, _ = ops.rotary_frequencies(128, device="cuda")
    got = ops.rotary(q, k, positions, f)
    want = ops.rotary(q[:, -3:], k[:, -3:], positions[-3:], f)
    for x, y in zip(got, want):
        assert torch.equal(x[:, -3:], y)


@gpu
@pytest.mark.parametrize("documents", (False, True))
def test_attention_past_32_bits(documents):
    """Keys of zeros, and the last ones so large that they alone have weight: the same as
    over them alone."""
    n, near = 2 ** 24 + 130, 100
    k, v = (torch.zeros(1, n, 1, 128, dtype=BF, device="cuda") for _ in range(2))
    q, k[:, -9:], v[:, -9:] = normal(1, 2, 2, 128, dtype=BF) + 8, normal(1, 9, 1, 128, dtype=BF) + 8, 1.0
    v[0, -9:, 0] += normal(9, 128, dtype=BF)
    ids = torch.zeros(1, n, dtype=torch.int32, device="cuda") if documents else None
    got = ops.attention(q, k, v, causal=True, documents=ids)
    ref.close(got, *ref.attention(q, k[:, -near:], v[:, -near:], causal=True))


@gpu
def test_the_cache_past_32_bits(way):
    """The same where a sequence's codes, and a second sequence, begin past 2^31 bytes."""
    capacity, dim = 2 ** 24 + 128, 128
    long, short = (ops.KeyValueCache(2, 1, n, dim, device="cuda") for n in (capacity, 256))
    k, v = (normal(2, 3, 1, dim, dtype=BF, seed=i) + 8 for i in range(2))
    q, at = normal(2, 3, 2, dim, dtype=BF, seed=4) + 8, ints([125, 70])
    far = at + (capacity - 128)
    long.append(k, v, far)
    short.append(k, v, at)
    for x, y in zip(parts(long), parts(short)):
        m = y.shape[2] // 2
        assert torch.equal(x[:, :, -m:].view(torch.uint8), y[:, :, :m].view(torch.uint8))
    ref.close(long.attend(q, far), *ref.cache_attention(q, *parts(short), at))
    ops.check_errors()


# --------------------------------------------------------------------------
# streams, graphs, devices
# --------------------------------------------------------------------------

@gpu
def test_operands_that_are_not_plain_tensors():
    """Parameters are; a subclass goes through torch's dispatcher, where a mode sees the call,
    and so does a batched tensor."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Subclass(torch.Tensor):
        pass

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    seen = []
    q, k, v = _heads(1, 5, 70, 2, 1, 64, HALF)
    want = ops.attention(q, k, v)
    assert torch.equal(ops.attention(q, torch.nn.Parameter(k, requires_grad=False), v), want)
    assert torch.equal(ops.attention(q, k.as_subclass(Subclass), v), want)
    with Log():
        assert torch.equal(ops.attention(q, k, v), want)
    assert "mlc.attention.default" in seen
    assert torch.equal(torch.vmap(lambda x: ops.attention(x, k, v))(q[None])[0], want)


@gpu
def test_calls_of_several_threads():
    import concurrent.futures

    cache = filled(2, 2, 8192, 64)

    def calls(i):
        q, start = normal(2, 1 + i % 2, 4, 64, seed=i), ints([8000 - i, 17 * i])
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            outs = [cache.attend(q, start) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return q, start, outs

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        results = list(pool.map(calls, range(8)))
    for q, start, outs in results:
        ref.close(outs[0], *ref.cache_attention(q, *parts(cache), start))
        assert all(torch.equal(x, outs[0]) for x in outs)


@gpu
def test_operators_run_on_the_current_stream_with_memory_of_their_own():
    """Two streams at once over a cache that is cut into items: the shared memory of
    one call is not another's."""
    cache = filled(1, 2, 16384, 128)
    qs = [normal(1, 1, 8, 128, seed=i) for i in range(2)]
    start = ints([16383])
    wants = [ref.cache_attention(q, *parts(cache), start) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attend(qs[i], start))
    torch.cuda.synchronize()
    for outs, want in zip(got, wants):
        for x in outs:
            ref.close(x, *want)


@gpu
def test_two_captured_graphs_replayed_in_turn():
    cache = filled(1, 2, 16384, 64)
    q = [normal(1, 1, 4, 64, seed=i, dtype=BF) for i in range(2)]
    k = normal(1, 1, 2, 64, dtype=BF, seed=8)
    start = ints([9000])
    f, _ = ops.rotary_frequencies(64, device="cuda")

    def step(x):
        a, b = ops.rotary(x, k, start, f)
        cache.append(b, b, start)
        return cache.attend(a, start), ops.attention(x, b, b)

    for x in q:
        step(x)
    graphs, outs = [], []
    for x in q:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for at in (9000, 70, 16383, 9001):
        start.fill_(at)
        for g in graphs:
            g.replay()
        eager = [step(x) for x in q]
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            for x, y in zip(a, b):
                assert torch.equal(x, y)
    ops.check_errors()


@gpu
def test_results_do_not_change_from_call_to_call():
    cache = filled(5, 2, 4096, 128)
    q, start = normal(5, 1, 8, 128, seed=1), ints([4000, 1, 77, 2047, 3000])
    first = cache.attend(q, start)
    a = [normal(2, 300, 4, 128, seed=i) for i in range(3)]
    want = ops.attention(*a, causal=True)
    for _ in range(5):
        assert torch.equal(cache.attend(q, start), first)
        assert torch.equal(ops.attention(*a, causal=True), want)


# --------------------------------------------------------------------------
# in compiled models
# --------------------------------------------------------------------------

class Block(torch.nn.Module):
    """A decoder's attention, for a prompt (over its own keys) or for new tokens
    (over the cache)."""

    def __init__(self, width, heads, kv, batch, capacity, prompt, dtype):
        super().__init__()
        self.heads, self.kv, self.dim, self.prompt = heads, kv, width // heads, prompt
        self.norm = torch.nn.LayerNorm(width)
        self.qkv = torch.nn.Linear(width, (heads + 2 * kv) * self.dim)
        self.out = torch.nn.Linear(width, width)
        self.to(dtype)
        self.cache = ops.KeyValueCache(batch, kv, capacity, self.dim)
        f, self.magnitude = ops.rotary_frequencies(self.dim, scaling="bands", factor=2.0, original=256)
        self.register_buffer("frequencies", f)
        self.register_buffer("slopes", torch.linspace(0.01, 0.1, heads))

    def forward(self, x, positions, start, count):
        b, t, _ = x.shape
        y = self.qkv(self.norm(x)).view(b, t, self.heads + 2 * self.kv, self.dim)
        q, k, v = y.split([self.heads, self.kv, self.kv], 2)
        q, k = ops.rotary(q, k, positions, self.frequencies, magnitude=self.magnitude)
        self.cache.append(k, v, start, count)
        if self.prompt:
            a = ops.attention(q, k, v, causal=True, cap=20.0, slopes=self.slopes)
        else:
            a = self.cache.attend(q, start, count, cap=20.0, slopes=self.slopes)
        return x + self.out(a.reshape(b, t, -1))


def _block(prompt, tokens, capacity=4096, batch=2, dtype=HALF):
    torch.manual_seed(0)
    m = Block(256, 4, 2, batch, capacity, prompt, dtype).cuda().eval()
    x = normal(batch, tokens, 256, dtype=dtype, seed=11)
    return m, x


def _inputs(x, starts, counts):
    t = x.shape[1]
    return (x, (ints(starts)[:, None] + torch.arange(t, device="cuda")).to(torch.int32),
            ints(starts), ints(counts))


@gpu
@pytest.mark.parametrize("prompt,tokens", [(True, 37), (False, 1), (False, 5)])
@pytest.mark.parametrize("config", [{}, {"memory_planning": False}, {"cuda_graphs": False},
                                    {"merge_parallel_gemms": True, "gemm_epilogue": True,
                                     "layout_selection": True, "fused_attention": True}],
                         ids=("graph", "unplanned", "planned", "variants"))
def test_a_compiled_block_is_the_block(prompt, tokens, config):
    m, x = _block(prompt, tokens)
    other, _ = _block(prompt, tokens)
    starts, counts = [(0, 700), (500, 3), (4096 - tokens, 64)], (tokens, tokens - tokens // 2)
    compiled = mlc.compile(m, _inputs(x, starts[0], counts), mlc.Config(**config))
    with torch.no_grad():
        for at, n in zip(starts, (counts, counts[::-1], counts)):
            args = _inputs(x * 1.5, at, n)
            got = compiled(*args).clone()
            want = other(*args)
            torch.cuda.synchronize()
            # the products round in another order: fp16 steps of values of size 4
            assert (got - want).abs().max() <= 2 ** -6
            # a code near the middle of two may differ by a step of e4m3
            for a, b, sa, sb in ((m.cache.keys, other.cache.keys, m.cache.key_scales, other.cache.key_scales),
                                 (m.cache.values, other.cache.values, m.cache.value_scales,
                                  other.cache.value_scales)):
                a = a.float() * sa.repeat_interleave(64, -1)[..., None]
                b = b.float() * sb.repeat_interleave(64, -1)[..., None]
                assert ((a - b).abs() <= 2 ** -3 * b.abs() + 2 ** -8 * sb.amax()).all()
                m_off = (a != b).float().mean()
                assert m_off < 0.02
    compiled.check_errors()
    assert sum("mlc." in k.summary() for k in compiled.schedule) == 3


@gpu
@pytest.mark.parametrize("many", (False, True))
def test_a_compiled_operator_is_the_direct_call_to_the_bit(many):
    """As launches of their own on the caller's inputs, and (many) in a graph."""

    class Step(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = filled(2, 2, 8192, 128)
            f, _ = ops.rotary_frequencies(128, device="cuda")
            self.register_buffer("f", f)

        def forward(self, q, k, v, start):
            for _ in range(12 if many else 1):
                a, b = ops.rotary(q, k, start.unsqueeze(1), self.f, interleaved=True)
                self.cache.append(b, v, start)
                a = self.cache.attend(a, start)
            return a, ops.attention(q, b, v)

    m = Step()
    args = [normal(2, 1, 8, 128, dtype=BF), normal(2, 1, 2, 128, dtype=BF, seed=1),
            normal(2, 1, 2, 128, dtype=BF, seed=2), ints([5, 6000])]
    compiled = mlc.compile(m, args)
    for i in range(4):
        args = [x * (1 + i) if x.dtype == BF else x + 64 * i + 1 for x in args]
        # an input that is a slice of something wider is copied first
        wide = torch.cat([args[0], args[0]], -1)
        got = [x.clone() for x in compiled(wide[..., :128], *args[1:])]
        held = [x.clone().view(torch.uint8) for x in (m.cache.keys, m.cache.values)]
        with torch.no_grad():
            want = m(*args)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(held[0], m.cache.keys.view(torch.uint8))
        assert torch.equal(held[1], m.cache.values.view(torch.uint8))
    compiled(args[0], args[1], args[2], ints([9000, 1]))
    with pytest.raises(ExecutionError, match="outside its cache"):
        compiled.check_errors()


@gpu
def test_a_buffer_that_would_be_copied_is_refused():
    m, x = _block(False, 1)
    inputs = _inputs(x, (0, 0), (1, 1))
    with pytest.raises(ops.OperatorError, match="k_cache is on cpu"):
        held, m.cache.keys = m.cache.keys, m.cache.keys.cpu()
        mlc.compile(m, inputs)
    m.cache.keys = held
    with pytest.raises(ExecutionError, match="changed in place"):
        mlc.compile(m.cpu(), [t.cpu() for t in inputs], device="cuda")


@gpu
def test_operands_of_a_compiled_operator_that_lie_otherwise_are_copied():
    """A pointwise result keeps a permuted order in torch and not in a compiled model, where
    its rows of heads then lie apart."""

    class Turned(torch.nn.Module):
        def __init__(self):
            super().__init__()
            f, _ = ops.rotary_frequencies(64, device="cuda")
            self.register_buffer("f", f)

        def forward(self, q, positions):
            y = (q.permute(0, 3, 1, 2) * 2.0).permute(0, 2, 3, 1)  # [batch, tokens, heads, dim]
            a, b = ops.rotary(y, y, positions, self.f)
            return ops.attention(a, b, y, causal=True)

    m, q = Turned(), normal(2, 9, 3, 64)
    args = (q, torch.arange(9, device="cuda", dtype=torch.int32))
    compiled = mlc.compile(m, args)
    with torch.no_grad():
        assert torch.equal(compiled(*args), m(*args))


@gpu
def test_unplanned_calls_leave_no_memory_behind():
    class Step(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = filled(1, 1, 8192, 64)

        def forward(self, q, start):
            return self.cache.attend(q, start) * 2.0

    m, args = Step(), (normal(1, 1, 2, 64), ints([8000]))
    compiled = mlc.compile(m, args, mlc.Config(memory_planning=False))
    for _ in range(3):
        compiled(*args)
    held = torch.cuda.memory_allocated()
    for _ in range(5):
        compiled(*args)
    assert torch.cuda.memory_allocated() == held


@gpu
def test_a_cache_given_for_both_keys_and_values_is_refused():
    c = filled(1, 1, 64, 64)
    k = normal(1, 1, 1, 64)
    _refused(lambda: ops.cache_append(c.keys, c.keys, c.key_scales, c.value_scales, k, k, ints([0])), "share")
    _refused(lambda: ops.cache_append(c.keys, c.values, c.key_scales, c.key_scales, k, k, ints([0])), "share")


# --------------------------------------------------------------------------
# what is refused
# --------------------------------------------------------------------------

def host(*shape, dtype=HALF):
    return torch.zeros(*shape, dtype=dtype)


def _refused(call, match):
    with pytest.raises((ops.OperatorError, ExecutionError), match=match):
        call()


def test_what_rotary_refuses():
    q, k, f = host(2, 3, 4, 64), host(2, 3, 2, 64), torch.ones(32, dtype=torch.float64)
    p = torch.arange(3, dtype=torch.int32)
    for args, why in (((q[0], k, p, f), "batch, tokens, heads"), ((q.double(), k, p, f), "expected, got"),
                      ((q, k.float(), p, f), "expected, got"), ((q, k[:, :2], p, f), "differ"),
                      ((q, k, p.float(), f), "integers"), ((q, k, p[:2], f), "positions"),
                      ((q, k, p, f.float()), "float64"), ((q, k, p, torch.cat([f, f])), "do not fit"),
                      ((q.transpose(2, 3), k.transpose(2, 3), p, f), "stride"),
                      ((q, k, p, f), "ROCm GPU")):
        _refused(lambda: ops.rotary(*args), why)
    for magnitude in (float("inf"), 1e300, float("nan")):
        _refused(lambda: ops.rotary(q, k, p, f, magnitude=magnitude), "magnitude")


def test_what_attention_refuses():
    q, k = host(2, 3, 4, 64), host(2, 5, 2, 64)
    doc = torch.zeros(2, 5, dtype=torch.int32)
    for call, why in ((lambda: ops.attention(q.float(), k.float(), k.float()), "expected, got"),
                      (lambda: ops.attention(q, k, k[:, :4]), "differ in shape"),
                      (lambda: ops.attention(q, k[:1], k[:1]), "differ in batch"),
                      (lambda: ops.attention(q[:, :, :3], k, k), "multiple"),
                      (lambda: ops.attention(q[:, :, :0], k[:, :, :0], k[:, :, :0]), "multiple"),
                      (lambda: ops.attention(q[..., :60], k[..., :60], k[..., :60]), "multiple of 8"),
                      (lambda: ops.attention(host(1, 1, 1, 264), host(1, 1, 1, 264),
                                             host(1, 1, 1, 264)), "up to 256"),
                      (lambda: ops.attention(q, k, k, scale=0.0), "scale"),
                      (lambda: ops.attention(q, k, k, scale=float("nan")), "scale"),
                      (lambda: ops.attention(q, k, k, cap=-1.0), "cap"),
                      (lambda: ops.attention(q, k, k, slopes=torch.ones(3)), "slopes"),
                      (lambda: ops.attention(q, k, k, documents=doc.long()), "documents"),
                      (lambda: ops.attention(q, k[:, :2], k[:, :2], documents=doc[:, :2]), "last of the keys"),
                      (lambda: ops.attention(q, k, k, prefix=doc[:, 0]), "causal"),
                      (lambda: ops.attention(q, k, k, causal=True, prefix=doc[0]), "prefix"),
                      (lambda: ops.attention(q, k, k), "ROCm GPU")):
        _refused(call, why)


def test_what_the_cache_refuses():
    c = ops.KeyValueCache(2, 2, 128, 64)
    k, start = host(2, 3, 2, 64), torch.zeros(2, dtype=torch.int32)
    p = parts(c)
    for call, why in ((lambda: c.append(k[:1], k[:1], start), "does not fit"),
                      (lambda: c.append(k, k[:, :2], start), "differ in shape"),
                      (lambda: c.append(k, k, start.long()), "start"),
                      (lambda: c.append(k, k, start, start[:1]), "count"),
                      (lambda: ops.cache_append(p[0].half(), *p[1:], k, k, start), "float8"),
                      (lambda: ops.cache_append(*p[:2], p[2][..., :1], p[3][..., :1], k, k, start),
                       "contiguous"),
                      (lambda: ops.cache_append(*p[:2], p[2].half(), p[3], k, k, start), "float32"),
                      (lambda: ops.cache_append(p[0][:, :, ::2], p[1][:, :, ::2], p[2][..., :1],
                                                p[3][..., :1], k, k, start), "contiguous"),
                      (lambda: ops.cache_append(p[0][:, :, :96], p[1][:, :, :96], p[2], p[3], k, k, start),
                       "blocks of 32"),
                      (lambda: c.attend(host(2, 1, 3, 64), start), "multiple"),
                      (lambda: c.attend(host(2, 1, 2, 64, dtype=FULL), start), "expected, got"),
                      (lambda: c.attend(host(2, 1, 2, 48), start), "does not fit"),
                      (lambda: c.attend(host(2, 1, 2, 64), start, cap=float("inf")), "cap"),
                      (lambda: c.attend(host(2, 1, 2, 64), start, slopes=torch.ones(3)), "slopes"),
                      (lambda: c.attend(host(2, 1, 2, 64), start), "ROCm GPU")):
        _refused(call, why)
    for bad in ((2, 2, 100, 64), (2, 2, 96, 64)):
        _refused(lambda: ops.KeyValueCache(*bad), "capacity")
    _refused(lambda: ops.KeyValueCache(1, 1, 64, 64, block=16), "capacity")
    odd = ops.KeyValueCache(1, 1, 64, 24)
    _refused(lambda: odd.attend(host(1, 1, 1, 24), start[:1]), "multiple of 16")


@pytest.mark.parametrize("option,value", [("scale", 1e300), ("scale", 0.0), ("scale", -1.0), ("cap", 1e-300),
                                          ("cap", 2000.0), ("cap", -1.0), ("cap", float("nan")),
                                          ("scale", float("inf"))])
def test_options_that_fp32_or_the_cap_do_not_hold_are_refused(option, value):
    q = host(1, 1, 2, 64)
    cache, start = ops.KeyValueCache(1, 2, 64, 64), torch.zeros(1, dtype=torch.int32)
    _refused(lambda: ops.attention(q, q, q, **{option: value}), option)
    _refused(lambda: cache.attend(q, start, **{option: value}), option)


def test_sizes_beyond_the_kernels_indexes_are_refused():
    shape = lambda *s, dtype=HALF: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    _refused(lambda: ops.attention(shape(1, 1, 1, 8), *[shape(1, 2 ** 30 + 1, 1, 8)] * 2), "too many tokens")
    _refused(lambda: ops.rotary(*[shape(1, 1, 2 ** 19 + 1, 2)] * 2, shape(1, dtype=torch.int32),
                                shape(1, dtype=torch.float64)), "too many heads")
    cache = ops.KeyValueCache(1, 1, 2 ** 30 + 64, 16, device="meta")
    _refused(lambda: cache.attend(shape(1, 1, 1, 16), shape(1, dtype=torch.int32)), "too large")


def test_a_cache_keeps_its_types_when_a_model_changes_its_own():
    m = torch.nn.Sequential(torch.nn.Linear(4, 4))
    m.cache = ops.KeyValueCache(1, 1, 64, 16)
    m.half()
    assert m[0].weight.dtype == HALF
    assert m.cache.keys.dtype == E4M3 and m.cache.key_scales.dtype == FULL
    assert m.to("meta").cache.values.device.type == "meta"


def test_what_the_module_of_calls_refuses():
    from mlc.runtime import native

    calls, x = native.load_calls(), torch.ones(2)
    for args in ((0, (3,), (), 1, None, True), (0, (), (), 0, None, True), (0, (x,), (), 2, None, True),
                 (0, (x,) * 17, (), 1, None, True), (0, [x], (), 1, None, True), (0, (x,), ()), (0, (x, "k"), (), 1, None, 1)):
        with pytest.raises(TypeError):
            calls.call(*args)
    assert calls.call(0, (x,), (), 1, None, True) is None
    for launch in ((7, 1, 2, b"\x00\x05", b"tail"), (7, 1, 2, b"\x00", b"x" * 2000), (0, 1, 2, b"\x00", b"")):
        with pytest.raises(ValueError, match="fit"):
            calls.add(b"not a signature", 5, 0, 1, (launch,), 0, 0, 0, 0)


def test_operands_that_ask_for_gradients_are_refused():
    q = host(1, 1, 2, 64).requires_grad_()
    _refused(lambda: ops.attention(q, q, q), "gradient")
    with torch.no_grad():
        _refused(lambda: ops.attention(q, q, q), "ROCm GPU")


def test_models_that_cannot_keep_a_cache_are_refused():
    from mlc.ir.capture import CaptureError, capture

    class Reads(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = ops.KeyValueCache(2, 2, 128, 64)

        def forward(self, k, start):
            a = self.cache.attend(k, start)
            self.cache.append(k, k, start)
            return a

    class Given(torch.nn.Module):
        def forward(self, kc, vc, ks, vs, k, start):
            ops.cache_append(kc, vc, ks, vs, k, k, start)
            return ops.cache_attention(k, kc, vc, ks, vs, start)

    class Part(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = ops.KeyValueCache(4, 2, 128, 64)

        def forward(self, k, start):
            ops.cache_append(*(x[:2] for x in parts(self.cache)), k, k, start)
            return k + 1

    k, start = host(2, 1, 2, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(CaptureError, match="read by another operator"):
        capture(Reads(), (k, start))
    with pytest.raises(CaptureError, match="buffer of the module"):
        capture(Given(), (*parts(ops.KeyValueCache(2, 2, 128, 64)), k, start))
    with pytest.raises(CaptureError, match="buffer of the module"):
        capture(Part(), (k, start))


def test_a_captured_block_keeps_its_operators_in_order():
    from mlc.api import build_pipeline
    from mlc.ir.capture import capture

    m = Block(256, 4, 2, 2, 128, False, HALF)
    x = host(2, 1, 256)
    start = torch.zeros(2, dtype=torch.int32)
    for cfg in (mlc.Config(), mlc.Config(merge_parallel_gemms=True, gemm_epilogue=True,
                                         layout_selection=True, fused_attention=True)):
        g = capture(m, (x, start[:, None] + 0, start, start + 1))
        schedule = build_pipeline(g, cfg)
        order = [k.node.op for k in schedule if hasattr(k, "node") and k.node.op.startswith("mlc.")]
        assert order == ["mlc.rotary.default", "mlc.cache_append.default", "mlc.cache_attention.default"]
        assert not [v for v in g.outputs if v.buffer.kind == "param"]


def test_every_kernel_a_plan_asks_for_is_built_beforehand():
    import random

    from mlc.codegen import hip_operators as plans
    from mlc.codegen.hip_operators import Operand

    def dense(*shape, dtype=HALF):
        strides = [1]
        for n in shape[:0:-1]:
            strides.insert(0, strides[0] * n)
        return Operand(shape, tuple(strides), dtype, aligned=random.random() < 0.7)

    known = {kernel for _, kernel in plans.all_kernels()}
    random.seed(1)
    seen = set()
    for _ in range(100000):
        if seen == known:
            break
        dtype, kv, group = random.choice((HALF, BF, FULL)), random.choice((1, 2, 8)), random.choice((1, 4, 16))
        b, t = random.choice((1, 2, 40, 300)), random.choice((1, 2, 3, 5, 31, 50, 200, 5000))
        dim, block = random.choice((16, 64, 80, 96, 128, 256)), random.choice((32, 64, 128))
        q, k = dense(b, t, kv * group, dim, dtype=dtype), dense(b, t, kv, dim, dtype=dtype)
        blocks = random.choice((8, 64))
        cache = dense(b, kv, blocks * block, dim, dtype=E4M3)
        scale, start = dense(b, kv, blocks, dtype=FULL), dense(b, dtype=torch.int32)
        slopes = dense(kv * group, dtype=FULL) if random.random() < 0.5 else None
        pairs = dim // 2 - random.choice((0, 1, 2, 4))
        found = [plans.plan_rotary(q, k, dense(t, dtype=torch.int32), dense(pairs, dtype=torch.float64),
                                   random.random() < 0.5, 1.0),
                 plans.plan_cache_append(cache, cache, scale, scale, k, k, start, None)]
        if dtype != FULL:
            documents = dense(b, t, dtype=torch.int32) if random.random() < 0.3 else None
            keys = dense(b, t + random.choice((0, 10, 900)), kv, dim, dtype=dtype)
            found += [plans.plan_attention(q, keys, keys, slopes, documents, None, 0.1, True, 0.0),
                      plans.plan_cache_attention(q, cache, cache, scale, scale, start, None, slopes, 0.1, 0.0)]
        seen |= {launch.kernel for p in found for launch in p.launches}
    assert seen <= known, seen - known
    assert len(known - seen) == 0, known - seen
