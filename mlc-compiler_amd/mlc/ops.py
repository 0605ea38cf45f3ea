"""Operators of decoders, as functions on GPU tensors: positions turned into
queries and keys, attention whose masks are made from indices, a cache of keys and
values in 8 bits and the attention over it.

    q, k = mlc.ops.rotary(q, k, positions, frequencies)
    out = mlc.ops.attention(q, k, v, causal=True)            # a prompt
    cache = mlc.ops.KeyValueCache(batch, kv_heads, capacity, dim, device="cuda")
    cache.append(k, v, start)                                # then, token by token
    out = cache.attend(q, start)

Tensors are token-major, ``[batch, tokens, heads, dim]``, as a linear layer's output
is viewed, with any strides whose last is 1; results are contiguous. ``heads`` of the
queries is a multiple of ``kv_heads`` of keys and values: query head ``h`` reads
key head ``h // (heads // kv_heads)``.

Called with GPU tensors, each launches this build's kernels on the current stream.
Used in a module given to ``mlc.compile`` they become launches of the compiled
schedule; ``cache_append`` then changes the module's own buffers. They are for
inference: a tensor that asks for a gradient is refused. Softmax statistics and
sums are held in fp32, the angles of ``rotary`` in 64 bits.
"""

from __future__ import annotations

import math

import torch

from .codegen import hip_operators as plans
from .codegen.hip_operators import Operand, OperatorError

__all__ = ["rotary", "rotary_frequencies", "attention", "cache_append", "cache_attention",
           "KeyValueCache", "check_errors", "OperatorError"]

_HALF = (torch.float16, torch.bfloat16)
_FLOATS = (*_HALF, torch.float32)
_INTS = (torch.int32, torch.int64)
_E4M3 = torch.float8_e4m3fn
_MAX = 2 ** 31 - 256


# --------------------------------------------------------------------------
# checks: on shapes, types and strides, so that they also run while a module is
# exported
# --------------------------------------------------------------------------

def _require(ok, what: str) -> None:
    if not ok:
        raise OperatorError(what)


def _rows(name: str, x, dtypes) -> None:
    _require(x.dim() == 4, f"{name}: [batch, tokens, heads, dim] expected, got {tuple(x.shape)}")
    _require(x.dtype in dtypes, f"{name}: one of {[str(d) for d in dtypes]} expected, got {x.dtype}")
    _require(x.shape[3] <= 1 or x.stride(3) == 1, f"{name}: the last dimension's stride is "
             f"{x.stride(3)}, and 1 is expected")


def _vector(name: str, x, dtype, size: int) -> None:
    _require(tuple(x.shape) == (size,) and x.dtype == dtype,
             f"{name}: {dtype}[{size}] expected, got {x.dtype}{list(x.shape)}")


def _same(first, others) -> None:
    for name, x in others.items():
        _require(x.device == first.device, f"{name} is on {x.device}, other operands on "
                 f"{first.device}")


def _scale(scale, dim: int) -> float:
    value = plans.score_scale(scale, dim)
    _require(0.0 < value < math.inf, f"scale: a positive number expected, got {scale}")
    return value


def _cap(cap) -> float:
    value = float(cap)
    _require(0.0 <= value < math.inf, f"cap: a positive number, or 0 for none, expected, got {cap}")
    return value


def _check_rotary(q, k, positions, frequencies, interleaved, magnitude) -> None:
    _rows("q", q, _FLOATS)
    _rows("k", k, (q.dtype,))
    _require(q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3],
             f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, tokens or dim")
    _require(positions.dtype in _INTS, f"positions: integers expected, got {positions.dtype}")
    _require(tuple(positions.shape) in (tuple(q.shape[1:2]), tuple(q.shape[:2])),
             f"positions: [tokens] or [batch, tokens] expected, got {tuple(positions.shape)} for q "
             f"{tuple(q.shape)}")
    _require(frequencies.dim() == 1 and frequencies.dtype == torch.float64,
             f"frequencies: float64[pairs] expected, got {frequencies.dtype}"
             f"{list(frequencies.shape)}")
    _require(2 * frequencies.shape[0] <= min(q.shape[3], 2 * plans.ROTARY_PAIRS),
             f"{frequencies.shape[0]} pairs do not fit a dim of {q.shape[3]}")
    _require(math.isfinite(magnitude), f"magnitude: a finite number expected, got {magnitude}")
    _require(q.shape[0] * q.shape[1] <= _MAX, "rotary: too many tokens for one call")
    _same(q, {"k": k, "positions": positions, "frequencies": frequencies})


def _check_attention(q, k, v, scale, causal, cap, slopes, documents, prefix) -> None:
    _rows("q", q, _HALF)
    _rows("k", k, (q.dtype,))
    _rows("v", v, (q.dtype,))
    batch, queries, heads, dim = q.shape
    _require(k.shape == v.shape, f"k {tuple(k.shape)} and v {tuple(v.shape)} differ in shape")
    _require(k.shape[0] == batch and k.shape[3] == dim,
             f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or dim")
    keys, kv_heads = k.shape[1], k.shape[2]
    _require(kv_heads > 0 and heads % kv_heads == 0,
             f"{heads} query heads are not a multiple of {kv_heads} key heads")
    _require(dim % 8 == 0 and dim <= plans.ATTENTION_DIMS[-1],
             f"dim {dim}: a multiple of 8 up to {plans.ATTENTION_DIMS[-1]} expected")
    _require(keys <= _MAX and queries * (heads // kv_heads) <= _MAX,
             "attention: too many tokens for one call")
    _scale(scale, dim)
    _cap(cap)
    others = {"k": k, "v": v}
    if slopes is not None:
        _vector("slopes", slopes, torch.float32, heads)
        others["slopes"] = slopes
    if documents is not None:
        _require(tuple(documents.shape) == (batch, keys) and documents.dtype == torch.int32,
                 f"documents: int32[{batch}, {keys}] expected, got {documents.dtype}"
                 f"{list(documents.shape)}")
        _require(queries <= keys, "documents: the queries are the last of the keys' tokens, and "
                 f"there are {queries} of them for {keys} keys")
        others["documents"] = documents
    if prefix is not None:
        _require(causal, "prefix: it widens a causal mask, so causal=True is expected")
        _vector("prefix", prefix, torch.int32, batch)
        others["prefix"] = prefix
    _same(q, others)


def _check_cache(k_cache, v_cache, k_scale, v_scale) -> None:
    _require(k_cache.dim() == 4 and k_cache.shape == v_cache.shape,
             f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)}: "
             "[batch, kv_heads, capacity, dim] expected of both")
    batch, heads, capacity, dim = k_cache.shape
    _require(k_scale.shape == v_scale.shape and k_scale.dim() == 3
             and tuple(k_scale.shape[:2]) == (batch, heads),
             f"k_scale {tuple(k_scale.shape)} and v_scale {tuple(v_scale.shape)}: "
             f"[{batch}, {heads}, capacity / block] expected of both")
    blocks = k_scale.shape[2]
    _require(blocks > 0 and capacity % blocks == 0 and capacity // blocks in (32, 64, 128),
             f"a capacity of {capacity} in {blocks} blocks: blocks of 32, 64 or 128 tokens expected")
    _require(dim % 16 == 0 and 16 <= dim <= plans.CACHED_DIMS[-1],
             f"dim {dim}: a multiple of 16 up to {plans.CACHED_DIMS[-1]} expected")
    _require(capacity <= _MAX, "the cache's capacity is too large")
    for name, x, dtype in (("k_cache", k_cache, _E4M3), ("v_cache", v_cache, _E4M3),
                           ("k_scale", k_scale, torch.float32), ("v_scale", v_scale, torch.float32)):
        _require(x.dtype == dtype and x.is_contiguous(),
                 f"{name}: contiguous {dtype} expected, got {x.dtype} with strides {x.stride()}")


def _check_places(tokens: int, batch: int, start, count) -> None:
    _vector("start", start, torch.int32, batch)
    if count is not None:
        _vector("count", count, torch.int32, batch)


def _check_cache_append(k_cache, v_cache, k_scale, v_scale, k, v, start, count) -> None:
    _check_cache(k_cache, v_cache, k_scale, v_scale)
    batch, heads, capacity, dim = k_cache.shape
    _rows("k", k, _FLOATS)
    _rows("v", v, (k.dtype,))
    _require(k.shape == v.shape, f"k {tuple(k.shape)} and v {tuple(v.shape)} differ in shape")
    _require((k.shape[0], k.shape[2], k.shape[3]) == (batch, heads, dim),
             f"k {tuple(k.shape)} does not fit a cache {tuple(k_cache.shape)}")
    _check_places(k.shape[1], batch, start, count)
    _same(k, {"k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
              "v": v, "start": start, **({"count": count} if count is not None else {})})


def _check_cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count, scale, cap,
                           slopes) -> None:
    _check_cache(k_cache, v_cache, k_scale, v_scale)
    batch, kv_heads, capacity, dim = k_cache.shape
    _rows("q", q, _HALF)
    _require(q.shape[0] == batch and q.shape[3] == dim,
             f"q {tuple(q.shape)} does not fit a cache {tuple(k_cache.shape)}")
    heads = q.shape[2]
    _require(kv_heads > 0 and heads % kv_heads == 0,
             f"{heads} query heads are not a multiple of {kv_heads} key heads")
    _require(q.shape[1] * (heads // kv_heads) <= _MAX, "cache_attention: too many tokens")
    _check_places(q.shape[1], batch, start, count)
    _scale(scale, dim)
    _cap(cap)
    others = {"k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
              "start": start}
    if count is not None:
        others["count"] = count
    if slopes is not None:
        _vector("slopes", slopes, torch.float32, heads)
        others["slopes"] = slopes
    _same(q, others)


# --------------------------------------------------------------------------
# direct calls
# --------------------------------------------------------------------------

#: (operator, shapes, strides, types, options) -> plan
_plans: dict = {}
#: plans kept: calls of ever new sizes start again
_MOST_PLANS = 4096


def _direct(*tensors) -> bool:
    """Whether the operands are plain GPU tensors outside of any tracing. One
    that asks for a gradient is refused."""
    if torch.compiler.is_compiling():
        return False
    plain = True
    for x in tensors:
        if x is None:
            continue
        if x.requires_grad and torch.is_grad_enabled():
            raise OperatorError("an operand asks for a gradient, and the operators of mlc.ops are "
                                "for inference: call them under torch.no_grad()")
        plain = plain and type(x) is torch.Tensor and x.is_cuda
    return plain


def _operand(x, at: int | None = None) -> Operand | None:
    if x is None:
        return None
    return Operand(tuple(x.shape), x.stride(), x.dtype,
                   aligned=(x.data_ptr() if at is None else at) % 16 == 0)


def _signature(*tensors):
    return [None if x is None else (x.dtype, x.shape, x.stride(), x.device.index,
                                    x.data_ptr() % 16) for x in tensors]


def _run(plan, device: torch.device, pointers: dict[str, int]) -> None:
    from .runtime import operators

    modules = operators.device_modules(device.index)
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            return _run(plan, device, pointers)
    flags = any("error" in launch.pointers for launch in plan.launches)
    if flags:
        pointers["error"] = modules.error_word()
        if modules.pending() and not torch.cuda.is_current_stream_capturing():
            _raise(modules)
    if plan.workspace:
        space = torch.empty(plan.workspace, dtype=torch.uint8, device=device)
        pointers["workspace"] = space.data_ptr()
    modules.run(plan, pointers, torch.cuda.current_stream(device).cuda_stream)


def _raise(modules) -> None:
    from .runtime.executor import ExecutionError
    from .runtime.operators import INVALID

    code = modules.pending()
    modules.clear()
    raise ExecutionError(INVALID.get(code, f"an operator flagged an invalid input ({code})"))


def check_errors() -> None:
    """Wait for the device and raise ``ExecutionError`` if an operator called so far
    met an invalid ``start`` or ``count``. Without it the next call of an operator
    that can meet one raises, once the call that met it is done."""
    from .runtime import operators

    for index, modules in list(operators._devices.items()):
        torch.cuda.synchronize(index)
        if modules.pending():
            _raise(modules)


def _planned(op: str, tensors: dict, options: tuple, check, build):
    """The plan of a call, checked the first time its signature comes."""
    key = (op, options, tuple(_signature(*tensors.values())))
    found = _plans.get(key)
    if found is None:
        check(*tensors.values(), *options)
        first = next(iter(tensors.values()))
        for name, x in tensors.items():
            if name.endswith("cache") or name.endswith("_scale"):
                _require(x.data_ptr() % 16 == 0, f"{name}: not on 16 bytes")
        found = build({n: _operand(x) for n, x in tensors.items()}, *options)
        if len(_plans) >= _MOST_PLANS:
            _plans.clear()
        _plans[key] = found
    return found


def _pointers(tensors: dict) -> dict[str, int]:
    return {n: x.data_ptr() for n, x in tensors.items() if x is not None}


def _rotary_now(q, k, positions, frequencies, interleaved, magnitude):
    tensors = {"q": q, "k": k, "positions": positions, "frequencies": frequencies}
    plan = _planned("rotary", tensors, (interleaved, magnitude), _check_rotary,
                    lambda t, *o: plans.plan_rotary(t["q"], t["k"], t["positions"],
                                                    t["frequencies"], *o))
    out = (torch.empty(q.shape, dtype=q.dtype, device=q.device),
           torch.empty(k.shape, dtype=k.dtype, device=k.device))
    _run(plan, q.device, {**_pointers(tensors), "out0": out[0].data_ptr(), "out1": out[1].data_ptr()})
    return out


def _attention_now(q, k, v, scale, causal, cap, slopes, documents, prefix):
    tensors = {"q": q, "k": k, "v": v, "slopes": slopes, "documents": documents, "prefix": prefix}

    def check(q, k, v, slopes, documents, prefix, scale, causal, cap):
        _check_attention(q, k, v, scale, causal, cap, slopes, documents, prefix)

    plan = _planned("attention", tensors, (scale, causal, cap), check,
                    lambda t, s, c, p: plans.plan_attention(*t.values(), _scale(s, q.shape[3]),
                                                            c, _cap(p)))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _run(plan, q.device, {**_pointers(tensors), "out0": out.data_ptr()})
    return out


def _cache_append_now(k_cache, v_cache, k_scale, v_scale, k, v, start, count):
    tensors = {"k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
               "k": k, "v": v, "start": start, "count": count}
    plan = _planned("cache_append", tensors, (), _check_cache_append,
                    lambda t: plans.plan_cache_append(*t.values()))
    _run(plan, k.device, _pointers(tensors))


def _cache_attention_now(q, k_cache, v_cache, k_scale, v_scale, start, count, scale, cap, slopes):
    tensors = {"q": q, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale,
               "v_scale": v_scale, "start": start, "count": count, "slopes": slopes}

    def check(q, kc, vc, ks, vs, start, count, slopes, scale, cap):
        _check_cache_attention(q, kc, vc, ks, vs, start, count, scale, cap, slopes)

    plan = _planned("cache_attention", tensors, (scale, cap), check,
                    lambda t, s, p: plans.plan_cache_attention(*t.values(), _scale(s, q.shape[3]),
                                                               _cap(p)))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _run(plan, q.device, {**_pointers(tensors), "out0": out.data_ptr()})
    return out


# --------------------------------------------------------------------------
# the same as torch operators, for modules that are exported
# --------------------------------------------------------------------------

_lib = torch.library.Library("mlc", "DEF")
_lib.define("rotary(Tensor q, Tensor k, Tensor positions, Tensor frequencies, bool interleaved, "
            "float magnitude) -> (Tensor, Tensor)")
_lib.define("attention(Tensor q, Tensor k, Tensor v, float? scale, bool causal, float cap, "
            "Tensor? slopes, Tensor? documents, Tensor? prefix) -> Tensor")
_lib.define("cache_append(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
            "Tensor(d!) v_scale, Tensor k, Tensor v, Tensor start, Tensor? count) -> ()")
_lib.define("cache_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, "
            "Tensor v_scale, Tensor start, Tensor? count, float? scale, float cap, "
            "Tensor? slopes) -> Tensor")


def _like(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _fake_rotary(q, k, positions, frequencies, interleaved, magnitude):
    _check_rotary(q, k, positions, frequencies, interleaved, magnitude)
    return _like(q), _like(k)


def _fake_attention(q, *rest):
    _check_attention(q, *rest)
    return _like(q)


def _fake_cache_append(*args):
    _check_cache_append(*args)


def _fake_cache_attention(q, *rest):
    _check_cache_attention(q, *rest)
    return _like(q)


def _refuse_host(check):
    def refuse(*args):
        from .runtime.executor import ExecutionError

        check(*args)
        raise ExecutionError("the operators of mlc.ops run on a ROCm GPU (torch device 'cuda'), "
                             "not on the CPU")

    return refuse


for _name, _now, _fake in (("rotary", _rotary_now, _fake_rotary),
                           ("attention", _attention_now, _fake_attention),
                           ("cache_append", _cache_append_now, _fake_cache_append),
                           ("cache_attention", _cache_attention_now, _fake_cache_attention)):
    _lib.impl(_name, _now, "CUDA")
    _lib.impl(_name, _refuse_host(_fake), "CPU")
    torch.library.register_fake(f"mlc::{_name}", _fake, lib=_lib)


# --------------------------------------------------------------------------
# the public functions
# --------------------------------------------------------------------------

def rotary(q, k, positions, frequencies, *, interleaved: bool = False, magnitude: float = 1.0):
    """Queries ``[batch, tokens, heads, dim]`` and keys ``[batch, tokens, kv_heads,
    dim]`` (fp16, bf16 or fp32) turned by their positions.

    ``positions``: int32 or int64, ``[tokens]`` or ``[batch, tokens]``.
    ``frequencies``: float64 radians per position, one for each pair of values
    (:func:`rotary_frequencies`); the first ``2 * len(frequencies)`` values of a head
    are turned, the rest is copied. A pair is values ``(i, i + len(frequencies))``, or
    ``(2 i, 2 i + 1)`` if ``interleaved``. ``magnitude`` multiplies what is turned.
    """
    if _direct(q, k, positions, frequencies):
        return _rotary_now(q, k, positions, frequencies, interleaved, magnitude)
    return torch.ops.mlc.rotary(q, k, positions, frequencies, interleaved, magnitude)


def rotary_frequencies(turned: int, base: float = 10000.0, *, scaling: str = "none",
                       factor: float = 1.0, original: int = 0, low: float = 1.0,
                       high: float = 32.0, device=None):
    """``(frequencies, magnitude)`` for :func:`rotary` over ``turned`` values a head.

    Pair ``i`` turns by ``base ** (-2 i / turned)`` a position. ``scaling`` stretches
    a context of ``original`` positions by ``factor``: "linear" slows every pair by
    it; "base" raises the base so that the slowest pair is slowed by it and the
    fastest not at all; "bands" slows pairs that turn fewer than ``low`` times within
    ``original`` positions by it, leaves those that turn more than ``high`` times and
    blends between, with the magnitude ``0.1 ln(factor) + 1`` for the flatter scores.
    """
    _require(turned >= 0 and turned % 2 == 0, f"an even number of values turns, not {turned}")
    _require(base > 0 and factor > 0, "base and factor are positive")
    half = turned // 2
    step = torch.arange(half, dtype=torch.float64, device=device)
    f = float(base) ** (-step / max(half, 1))
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "base":
        return f * float(factor) ** (-step / max(half - 1, 1)), 1.0
    if scaling == "bands":
        _require(original > 0 and high > low, "bands: original, and low below high, expected")
        turns = original * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(max(factor, 1.0)) + 1.0
    raise OperatorError(f"scaling {scaling!r}: none, linear, base or bands expected")


def attention(q, k, v, *, scale: float | None = None, causal: bool = False, cap: float = 0.0,
              slopes=None, documents=None, prefix=None):
    """``softmax(scores) v`` of queries ``[batch, queries, heads, dim]`` over keys and
    values ``[batch, keys, kv_heads, dim]`` in fp16 or bf16, ``dim`` a multiple of 8 up
    to 256.

    A score is ``q . k * scale`` (``1 / sqrt(dim)``); with ``cap`` it becomes
    ``cap * tanh(score / cap)``; with ``slopes`` (float32[heads]) ``slope * |i - j|`` is
    taken off for query position ``i`` and key position ``j``. Queries stand at the last
    positions of the keys: query ``t`` at ``t + keys - queries``. What it sees:

    * ``causal``: keys up to its own position, and with ``prefix`` (int32[batch]) also
      keys below ``prefix``;
    * ``documents`` (int32[batch, keys]): of those the keys of its own document; a token
      of a negative document sees nothing and is seen by none.

    A query that sees nothing gets zeros. What is not seen has no influence, NaN and
    infinities included.
    """
    if _direct(q, k, v, slopes, documents, prefix):
        return _attention_now(q, k, v, scale, causal, cap, slopes, documents, prefix)
    return torch.ops.mlc.attention(q, k, v, scale, causal, cap, slopes, documents, prefix)


def cache_append(k_cache, v_cache, k_scale, v_scale, k, v, start, count=None) -> None:
    """New keys and values ``[batch, tokens, kv_heads, dim]`` (fp16, bf16 or fp32) into
    the cache, in place.

    The cache is ``float8_e4m3fn [batch, kv_heads, capacity, dim]``, contiguous, with
    ``dim`` a multiple of 16 up to 256; scales are ``float32 [batch, kv_heads, capacity /
    block]`` with blocks of 32, 64 or 128 tokens. Sequence ``b``'s first ``count[b]`` new
    tokens (all, without ``count``) go to positions ``start[b]``, .... A value is code
    times the scale of its block, the smallest power of two that brings the block's
    largest value to 448 or less: where new tokens raise it, the codes in front of them
    are rounded to it. A block's first token starts its scale anew; tokens behind the
    last are not kept. NaN and infinities are stored as NaN.

    A sequence whose ``start`` and ``count`` do not lie within the cache is left alone,
    and ``ExecutionError`` is raised by a later call or :func:`check_errors`.
    """
    if _direct(k_cache, v_cache, k_scale, v_scale, k, v, start, count):
        return _cache_append_now(k_cache, v_cache, k_scale, v_scale, k, v, start, count)
    return torch.ops.mlc.cache_append(k_cache, v_cache, k_scale, v_scale, k, v, start, count)


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count=None, *,
                    scale: float | None = None, cap: float = 0.0, slopes=None):
    """Attention of ``q [batch, tokens, heads, dim]`` (fp16 or bf16) over the cache that
    :func:`cache_append` filled: token ``t`` of sequence ``b`` stands at ``start[b] + t``
    and sees the keys up to there, its own included, so the new tokens are appended
    first. Tokens from ``count[b]`` on get zeros, as do sequences whose ``start`` and
    ``count`` do not lie within the cache (an ``ExecutionError`` later). ``scale``, ``cap``
    and ``slopes`` are those of :func:`attention`.
    """
    if _direct(q, k_cache, v_cache, k_scale, v_scale, start, count, slopes):
        return _cache_attention_now(q, k_cache, v_cache, k_scale, v_scale, start, count, scale,
                                    cap, slopes)
    return torch.ops.mlc.cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count,
                                         scale, cap, slopes)


class KeyValueCache(torch.nn.Module):
    """Keys and values of ``batch`` sequences of up to ``capacity`` tokens in 8 bits, as
    buffers of a module (:func:`cache_append`, :func:`cache_attention`)."""

    def __init__(self, batch: int, kv_heads: int, capacity: int, dim: int, *, block: int = 64,
                 device=None) -> None:
        super().__init__()
        _require(block in (32, 64, 128) and capacity % block == 0,
                 f"a capacity of {capacity} in blocks of {block}: a multiple of 32, 64 or 128 "
                 "tokens expected")
        shape = (batch, kv_heads, capacity, dim)
        for name in ("keys", "values"):
            self.register_buffer(name, torch.zeros(shape, dtype=torch.uint8, device=device)
                                 .view(_E4M3), persistent=False)
            self.register_buffer(f"{name[:-1]}_scales",
                                 torch.ones(*shape[:2], capacity // block, device=device),
                                 persistent=False)

    def append(self, k, v, start, count=None) -> None:
        cache_append(self.keys, self.values, self.key_scales, self.value_scales, k, v, start, count)

    def attend(self, q, start, count=None, **options):
        return cache_attention(q, self.keys, self.values, self.key_scales, self.value_scales,
                               start, count, **options)
