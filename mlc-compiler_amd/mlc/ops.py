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
inference: a tensor that asks for a gradient, backward or forward, is refused. Softmax
statistics and sums are held in fp32, the angles of ``rotary`` in 64 bits.
"""

from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from .codegen import hip_operators as plans
from .codegen.hip_operators import Operand, OperatorError
from .runtime import native, operators

__all__ = ["rotary", "rotary_frequencies", "attention", "cache_append", "cache_attention",
           "KeyValueCache", "check_errors", "OperatorError"]

_HALF = (torch.float16, torch.bfloat16)
_FLOATS = (*_HALF, torch.float32)
_INTS = (torch.int32, torch.int64)
_E4M3 = torch.float8_e4m3fn
_MAX = 2 ** 31 - 256
#: and of keys: kernels look some tiles past the last one
_MOST_KEYS = 2 ** 30


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
    _require(2.0 ** -100 <= value <= 2.0 ** 100, f"scale: a positive number between 2^-100 and 2^100 "
             f"expected, got {scale}")
    return value


def _cap(cap) -> float:
    value = float(cap)
    # a capped score is off by 2^-21 of the cap: at 1024 by what rounding its weight to fp16 is
    _require(value == 0.0 or 2.0 ** -20 <= value <= 2.0 ** 10, "cap: a positive number between 2^-20 and "
             f"1024, or 0 for none, expected, got {cap}")
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
    _require(abs(magnitude) <= torch.finfo(torch.float32).max,
             f"magnitude: a finite fp32 number expected, got {magnitude}")
    _require(q.shape[0] * q.shape[1] <= _MAX, "rotary: too many tokens for one call")
    _require(q.shape[2] + k.shape[2] <= 1 << 20, "rotary: too many heads for one call")
    _same(q, {"k": k, "positions": positions, "frequencies": frequencies})


def _check_attention(q, k, v, slopes, documents, prefix, scale, causal, cap) -> None:
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
    _require(keys <= _MOST_KEYS and queries * (heads // kv_heads) <= _MAX,
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
    _require(capacity <= _MOST_KEYS, "the cache's capacity is too large")
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


def _check_cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count, slopes, scale,
                           cap) -> None:
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

_plans = operators.Calls()
_is_compiling = torch.compiler.is_compiling
_stream_of = torch._C._cuda_getCurrentRawStream


def _operand(x) -> Operand | None:
    return None if x is None else Operand(tuple(x.shape), x.stride(), x.dtype,
                                          aligned=x.data_ptr() % 16 == 0)


def _add(signature: bytes, op: str, operands: tuple, options: tuple, results: int) -> None:
    """The launches of a call of a new signature, checked."""
    check, plan, names = _OPERATORS[op]
    check(*operands, *options)
    seen = tuple(map(_operand, operands))
    plans.require_aligned(dict(zip(names, seen)))
    made = plan(*seen, *options)
    changed = len(_CACHE) if op == "cache_append" else 0
    _plans.add(signature, made, names, changed, results, operands[0].get_device())


def check_errors() -> None:
    """Wait for the device and raise ``ExecutionError`` if an operator called so far
    met an invalid ``start`` or ``count``. Without it the next call of an operator
    that can meet one raises, once the call that met it is done."""
    operators.check_errors()


def _plan_attention(q, k, v, slopes, documents, prefix, scale, causal, cap):
    return plans.plan_attention(q, k, v, slopes, documents, prefix,
                                plans.score_scale(scale, q.shape[3]), causal, float(cap))


def _plan_cache_attention(q, kc, vc, ks, vs, start, count, slopes, scale, cap):
    return plans.plan_cache_attention(q, kc, vc, ks, vs, start, count, slopes,
                                      plans.score_scale(scale, q.shape[3]), float(cap))


_CACHE = ("k_cache", "v_cache", "k_scale", "v_scale")
#: operator -> its check, its plan (operands, then options) and its operands' names
_OPERATORS = {
    "rotary": (_check_rotary, plans.plan_rotary, ("q", "k", "positions", "frequencies")),
    "attention": (_check_attention, _plan_attention,
                  ("q", "k", "v", "slopes", "documents", "prefix")),
    "cache_append": (_check_cache_append, plans.plan_cache_append,
                     (*_CACHE, "k", "v", "start", "count")),
    "cache_attention": (_check_cache_attention, _plan_cache_attention,
                        ("q", *_CACHE, "start", "count", "slopes")),
}


_NUMBERS = {op: i for i, op in enumerate(_OPERATORS)}


_POLL, _DISPATCHED = 1, 2
_GRADIENT = ("an operand asks for a gradient, and the operators of mlc.ops are for inference: call "
             "them under torch.no_grad(), or, in forward mode, on the primal "
             "(torch.autograd.forward_ad.unpack_dual)")


def _now(op: str, operands: tuple, options: tuple, results: int, flags: int = _POLL) -> tuple | None:
    """The call, with so many results like the first operands, or None where they are not
    plain GPU tensors outside of any tracing. An operand that asks for a gradient is refused."""
    if _is_compiling():
        return None
    run = native.load_calls().call
    while True:
        out = run(_NUMBERS[op], operands, options, results, _stream_of, flags)
        if out is None or type(out) is tuple:
            return out
        if out is False:
            raise OperatorError(_GRADIENT)
        if out is True:
            if not torch.cuda.is_current_stream_capturing():
                operators.raise_pending(operators.device_modules(operands[0].get_device()))
            flags &= ~_POLL
        elif out is NotImplemented:
            with torch.cuda.device(operands[0].get_device()):
                return _now(op, operands, options, results, flags)
        elif out is Ellipsis:
            raise OperatorError(f"{op}: keys and values share a cache or its scales, or another "
                                "operand shares memory with them")
        elif type(out) is bytes:
            _add(out, op, operands, options, results)
        else:
            native.check(out, f"a launch of {op}")


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


def _asks_gradient(x) -> bool:
    return isinstance(x, torch.Tensor) and (
        (torch.is_grad_enabled() and x.requires_grad)
        or (torch._C._is_fwd_grad_enabled() and unpack_dual(x).tangent is not None))


@contextlib.contextmanager
def _untraced():
    """While torch.jit traces, sizes are tensors and what is done with them goes into its
    graph: not below an operator, which is in it as a whole."""
    state = torch._C._get_tracing_state()
    if state is not None:
        torch._C._set_tracing_state(None)
    try:
        yield
    finally:
        if state is not None:
            torch._C._set_tracing_state(state)


def _implement(op: str, split, results: int) -> None:
    """``mlc::op``: ``split`` puts the schema's arguments into operands and options,
    results are like the first operands."""
    check = _OPERATORS[op][0]

    def autograd(keys, *args):
        # a program that is exported is a graph, and refuses when it is run
        if not torch.compiler.is_exporting() and any(map(_asks_gradient, args)):
            raise OperatorError(_GRADIENT)
        with torch._C._AutoDispatchBelowAutograd():
            return overload.redispatch(keys & torch._C._after_autograd_keyset, *args)

    @_untraced()
    def gpu(*args):
        operands, options = split(*args)
        # what the dispatcher hands over may be a subclass
        plain = tuple(x if x is None or type(x) is torch.Tensor
                      else x.detach().as_subclass(torch.Tensor) for x in operands)
        with torch.no_grad():
            out = _now(op, plain, options, results, _POLL | _DISPATCHED)
        if out is None:
            check(*operands, *options)
        _require(out is not None, f"{op}: not plain tensors of one GPU")
        return tuple(out) if results > 1 else out[0] if results else None

    def fake(*args):
        operands, options = split(*args)
        check(*operands, *options)
        out = tuple(map(_like, operands[:results]))
        return out if results > 1 else out[0] if results else None

    @_untraced()
    def host(*args):
        from .runtime.executor import ExecutionError

        operands, options = split(*args)
        check(*operands, *options)
        raise ExecutionError("the operators of mlc.ops run on a ROCm GPU (torch device 'cuda'), "
                             "not on the CPU")

    overload = getattr(torch.ops.mlc, op).default
    _lib.impl(op, autograd, "Autograd", with_keyset=True)
    _lib.impl(op, gpu, "CUDA")
    _lib.impl(op, host, "CPU")
    torch.library.register_fake(f"mlc::{op}", fake, lib=_lib)


_implement("rotary", lambda q, k, p, f, i, m: ((q, k, p, f), (i, m)), 2)
_implement("attention", lambda q, k, v, scale, causal, cap, slopes, documents, prefix:
           ((q, k, v, slopes, documents, prefix), (scale, causal, cap)), 1)
_implement("cache_append", lambda *args: (args, ()), 0)
_implement("cache_attention", lambda q, kc, vc, ks, vs, start, count, scale, cap, slopes:
           ((q, kc, vc, ks, vs, start, count, slopes), (scale, cap)), 1)


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
    interleaved, magnitude = bool(interleaved), float(magnitude)
    out = _now("rotary", (q, k, positions, frequencies), (interleaved, magnitude), 2)
    if out is not None:
        return out[0], out[1]
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

    A score is ``q . k * scale`` (``1 / sqrt(dim)``); with ``cap`` (up to 1024) it becomes
    ``cap * tanh(score / cap)``; with ``slopes`` (float32[heads]) ``slope * |i - j|`` is
    taken off for query position ``i`` and key position ``j``. Queries stand at the last
    positions of the keys: query ``t`` at ``t + keys - queries``. What it sees:

    * ``causal``: keys up to its own position, and with ``prefix`` (int32[batch]) also
      keys below ``prefix``;
    * ``documents`` (int32[batch, keys]): of those the keys of its own document; a token
      of a negative document sees nothing and is seen by none.

    A query that sees nothing gets zeros. What is not seen has no influence, NaN and
    infinities included. Softmax weights are rounded to the type of ``q`` before they meet
    the values; a capped score is off by up to 2^-21 of the cap, whatever its size.
    """
    scale, causal, cap = None if scale is None else float(scale), bool(causal), float(cap)
    out = _now("attention", (q, k, v, slopes, documents, prefix), (scale, causal, cap), 1)
    if out is not None:
        return out[0]
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

    Operands that overlap the cache or its scales in memory are refused. A sequence whose
    ``start`` and ``count`` do not lie within the cache is left alone, and
    ``ExecutionError`` is raised by a later call or :func:`check_errors`.
    """
    if _now("cache_append", (k_cache, v_cache, k_scale, v_scale, k, v, start, count), (), 0) is not None:
        return None
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
    scale, cap = None if scale is None else float(scale), float(cap)
    out = _now("cache_attention", (q, k_cache, v_cache, k_scale, v_scale, start, count, slopes),
               (scale, cap), 1)
    if out is not None:
        return out[0]
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

    def _apply(self, fn, recurse=True):
        """Moves the buffers with the module but keeps their types: ``model.half()`` is for
        weights."""
        for name, x in self._buffers.items():
            y = fn(x)
            self._buffers[name] = y if y.dtype == x.dtype else x.to(y.device)
        return self

    def append(self, k, v, start, count=None) -> None:
        cache_append(self.keys, self.values, self.key_scales, self.value_scales, k, v, start, count)

    def attend(self, q, start, count=None, **options):
        return cache_attention(q, self.keys, self.values, self.key_scales, self.value_scales,
                               start, count, **options)
