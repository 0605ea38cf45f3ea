"""Operators of decoders, as functions on GPU tensors: positions turned into
queries and keys, attention whose masks are made from indices, a cache of keys and
values in 8 bits and the attention over it; norms, linear layers in 8 bits, and the
choice of a token.

    q, k = mlc.ops.rotary(q, k, positions, frequencies)
    out = mlc.ops.attention(q, k, v, causal=True)            # a prompt
    cache = mlc.ops.KeyValueCache(batch, kv_heads, capacity, dim, device="cuda")
    cache.append(k, v, start)                                # then, token by token
    out = cache.attend(q, start)

    codes, scales, x = mlc.ops.rms_norm(x, weight, residual, quantized=True)
    y = mlc.ops.scaled_product(codes, scales, *mlc.ops.quantize_weight(w))
    tokens = mlc.ops.sample(logits, uniform, temperature=t, top_p=p)

In attention and the cache tensors are token-major, ``[batch, tokens, heads, dim]``, as a
linear layer's output is viewed, rows elsewhere ``[rows, dim]`` or ``[batch, tokens, dim]``,
with any strides whose last is 1; results are contiguous. ``heads`` of the queries is a
multiple of ``kv_heads`` of keys and values: query head ``h`` reads
key head ``h // (heads // kv_heads)``.

Called with GPU tensors, each launches this build's kernels on the current stream.
Used in a module given to ``mlc.compile`` they become launches of the compiled
schedule; ``cache_append`` then changes the module's own buffers. They are for
inference: a tensor that asks for a gradient, backward or forward, is refused. Softmax
statistics and sums are held in fp32, the angles of ``rotary`` and the sums of ``sample`` in 64 bits.
"""

from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from .codegen import hip_decoder as decoder
from .codegen import hip_operators as plans
from .codegen.hip_operators import Operand, OperatorError
from .runtime import native, operators

__all__ = ["rotary", "rotary_frequencies", "attention", "cache_append", "cache_attention",
           "KeyValueCache", "rms_norm", "quantize", "quantize_weight", "scaled_product", "ScaledLinear",
           "sample", "check_errors", "OperatorError"]

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


def _lines(name: str, x, dtypes, most: int) -> None:
    _require(x.dim() in (2, 3), f"{name}: [rows, dim] or [batch, tokens, dim] expected, got {tuple(x.shape)}")
    _require(x.dtype in dtypes, f"{name}: one of {[str(d) for d in dtypes]} expected, got {x.dtype}")
    _require(1 <= x.shape[-1] <= most, f"{name}: a dim of 1 to {most} expected, got {x.shape[-1]}")
    _require(x.shape[-1] == 1 or x.stride(-1) == 1, f"{name}: the last dimension's stride is "
             f"{x.stride(-1)}, and 1 is expected")
    _require(math.prod(x.shape[:-1]) <= _MAX, f"{name}: too many rows for one call")


def _like_lines(name: str, x, first, of: str) -> None:
    _require(x.shape == first.shape and x.dtype == first.dtype,
             f"{name} {x.dtype}{list(x.shape)} and {of} {first.dtype}{list(first.shape)} differ")
    _require(x.shape[-1] == 1 or x.stride(-1) == 1, f"{name}: the last dimension's stride is "
             f"{x.stride(-1)}, and 1 is expected")


def _pieces(name: str, x) -> None:
    _require(x.shape[-1] % 16 == 0, f"{name}: a dim that is a multiple of 16 expected, got {x.shape[-1]}")


def _check_norm(x, weight, residual, eps, quantized) -> None:
    _lines("x", x, _FLOATS, decoder.MOST_DIM)
    if quantized:
        _pieces("x", x)
    _require(tuple(weight.shape) == (x.shape[-1],) and weight.dtype in (x.dtype, torch.float32)
             and weight.is_contiguous(), f"weight: contiguous {x.dtype}[{x.shape[-1]}] or float32 expected, "
             f"got {weight.dtype}{list(weight.shape)} with strides {weight.stride()}")
    _require(0.0 < eps <= torch.finfo(torch.float32).max, f"eps: a positive number expected, got {eps}")
    others = {"weight": weight}
    if residual is not None:
        _like_lines("residual", residual, x, "x")
        others["residual"] = residual
    _same(x, others)


def _check_quantize(x, gate) -> None:
    _lines("x", x, _FLOATS, 1 << 24)
    _pieces("x", x)
    if gate is not None:
        _like_lines("gate", gate, x, "x")
        _same(x, {"gate": gate})


def _result_number(dtype) -> int:
    _require(dtype in decoder.RESULTS, f"dtype: one of {[str(d) for d in decoder.RESULTS]} expected, "
             f"got {dtype}")
    return decoder.RESULTS.index(dtype)


def _check_product(a, a_scales, b, b_scales, bias, number) -> None:
    dtype = decoder.RESULTS[int(number)]
    _lines("a", a, (_E4M3,), 1 << 24)
    _lines("b", b, (_E4M3,), 1 << 24)
    _require(b.dim() == 2 and b.shape[1] == a.shape[-1],
             f"b {tuple(b.shape)}: [outputs, {a.shape[-1]}] expected")
    _pieces("a", a)
    blocks, outputs = decoder.blocks_of(a.shape[-1]), decoder.blocks_of(b.shape[0])
    for name, x, shape in (("a_scales", a_scales, (*a.shape[:-1], blocks)), ("b_scales", b_scales, (outputs, blocks))):
        _require(tuple(x.shape) == tuple(shape) and x.dtype == torch.float32,
                 f"{name}: float32{list(shape)} expected, got {x.dtype}{list(x.shape)}")
    for name, x in (("a", a), ("b", b)):
        _require(all(s % 16 == 0 for s, n in zip(x.stride()[:-1], x.shape) if n > 1),
                 f"{name}: rows of codes that lie on 16 bytes expected, got strides {x.stride()}")
    others = {"a_scales": a_scales, "b": b, "b_scales": b_scales}
    if bias is not None:
        _require(tuple(bias.shape) == (b.shape[0],) and bias.dtype in (dtype, torch.float32)
                 and bias.is_contiguous(), f"bias: contiguous {dtype}[{b.shape[0]}] or float32 expected, "
                 f"got {bias.dtype}{list(bias.shape)} with strides {bias.stride()}")
        others["bias"] = bias
    _same(a, others)


def _check_sample(logits, uniform, temperature, top_k, top_p, min_p) -> None:
    _require(logits.dim() == 2, f"logits: [batch, tokens] expected, got {tuple(logits.shape)}")
    _lines("logits", logits, _FLOATS, decoder.MOST_TOKENS)
    others = {"uniform": uniform, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    others = {name: x for name, x in others.items() if x is not None}
    for name, x in others.items():
        _vector(name, x, torch.int32 if name == "top_k" else torch.float32, logits.shape[0])
    _same(logits, others)


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


def _norm_of(residual: bool, quantized: bool) -> tuple:
    """The check, plan and operands' names of one of the four norms."""
    def with_options(f):
        if residual:
            return lambda x, weight, other, eps: f(x, weight, other, eps, quantized)
        return lambda x, weight, eps: f(x, weight, None, eps, quantized)

    return (with_options(_check_norm), with_options(decoder.plan_norm),
            ("x", "weight", "residual")[:3 if residual else 2])


def _plan_product(a, a_scales, b, b_scales, bias, number):
    return decoder.plan_product(a, a_scales, b, b_scales, bias, decoder.RESULTS[int(number)])


#: (with a residual, in 8 bits) -> the norm's name
_NORMS = {(False, False): "rms_norm", (True, False): "add_rms_norm",
          (False, True): "rms_norm_quantized", (True, True): "add_rms_norm_quantized"}
# in the order of the names that _calls.call knows
_OPERATORS |= {name: _norm_of(*kind) for kind, name in _NORMS.items()}
_OPERATORS |= {
    "quantize": (_check_quantize, decoder.plan_quantize, ("x", "gate")),
    "scaled_product": (_check_product, _plan_product, ("a", "a_scales", "b", "b_scales", "bias")),
    "sample": (_check_sample, decoder.plan_sample,
               ("logits", "uniform", "temperature", "top_k", "top_p", "min_p")),
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
_lib.define("rms_norm(Tensor x, Tensor weight, float eps) -> Tensor")
_lib.define("add_rms_norm(Tensor x, Tensor weight, Tensor residual, float eps) -> (Tensor, Tensor)")
_lib.define("rms_norm_quantized(Tensor x, Tensor weight, float eps) -> (Tensor, Tensor)")
_lib.define("add_rms_norm_quantized(Tensor x, Tensor weight, Tensor residual, float eps) -> "
            "(Tensor, Tensor, Tensor)")
_lib.define("quantize(Tensor x, Tensor? gate) -> (Tensor, Tensor)")
_lib.define("scaled_product(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor? bias, "
            "ScalarType dtype) -> Tensor")
_lib.define("sample(Tensor logits, Tensor uniform, Tensor? temperature, Tensor? top_k, Tensor? top_p, "
            "Tensor? min_p) -> Tensor")


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


def _implement(op: str, split, results: int, made=None) -> None:
    """``mlc::op``: ``split`` puts the schema's arguments into operands and options,
    results are like the first operands, or of the shapes and types that ``made`` gives."""
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
        if made is None:
            out = tuple(map(_like, operands[:results]))
        else:
            out = tuple(torch.empty(shape, dtype=dtype, device=operands[0].device)
                        for shape, dtype in made(*operands, *options))
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
_implement("rms_norm", lambda x, w, eps: ((x, w), (eps,)), 1)
_implement("add_rms_norm", lambda x, w, r, eps: ((x, w, r), (eps,)), 2,
           lambda x, w, r, eps: decoder.norm_results(x, r, False))
_implement("rms_norm_quantized", lambda x, w, eps: ((x, w), (eps,)), 2,
           lambda x, w, eps: decoder.norm_results(x, None, True))
_implement("add_rms_norm_quantized", lambda x, w, r, eps: ((x, w, r), (eps,)), 3,
           lambda x, w, r, eps: decoder.norm_results(x, r, True))
_implement("quantize", lambda *args: (args, ()), 2, lambda x, gate: decoder.eight_bits(x))
_implement("scaled_product", lambda a, a_scales, b, b_scales, bias, dtype:
           ((a, a_scales, b, b_scales, bias), (_result_number(dtype),)), 1,
           lambda a, a_scales, b, b_scales, bias, number:
           decoder.product_results(a, b, decoder.RESULTS[number]))
_implement("sample", lambda *args: (args, ()), 1, lambda logits, *_: decoder.sample_results(logits))


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


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6, quantized: bool = False):
    """``h / sqrt(mean(h^2) + eps) * weight`` for rows ``h`` of ``x [rows, dim]`` or
    ``[batch, tokens, dim]`` (fp16, bf16 or fp32, ``dim`` up to 32768), with ``weight``
    ``[dim]`` in the type of ``x`` or float32. With ``residual``, of the shape and type of
    ``x``, ``h = x + residual`` in fp32, and the sum, rounded to that type, comes back behind the
    norm; the norm itself is taken of the sum as it is before that.

    Returns the norm in the type of ``x``, or with ``quantized`` (``dim`` a multiple of 16)
    its codes and scales as :func:`quantize` gives them: ``y``, ``(y, sum)``, ``(codes,
    scales)`` or ``(codes, scales, sum)``. Sums of squares are held in 64 bits, the squares of
    eight neighbouring 16-bit values in fp32.
    """
    op = _NORMS[residual is not None, bool(quantized)]
    operands, eps = (x, weight) if residual is None else (x, weight, residual), float(eps)
    results = 1 + bool(quantized) + (residual is not None)
    out = _now(op, operands, (eps,), results)
    if out is None:
        return getattr(torch.ops.mlc, op)(*operands, eps)
    return out if results > 1 else out[0]


def quantize(x, gate=None):
    """``(codes, scales)`` of rows ``x [rows, dim]`` or ``[batch, tokens, dim]`` (fp16, bf16 or
    fp32, ``dim`` a multiple of 16), or of ``x * gate / (1 + e^-gate)`` with ``gate`` of the
    same shape and type.

    A scale, ``float32 [..., ceil(dim / 128)]``, is that of 128 neighbouring values of a
    row: their largest finite magnitude divided by 448, and 2^-126 or more. A code,
    ``float8_e4m3fn``, is a value divided by its scale; infinities and NaN become NaN.
    """
    out = _now("quantize", (x, gate), (), 2)
    return out if out is not None else torch.ops.mlc.quantize(x, gate)


def quantize_weight(weight):
    """``(codes, scales)`` of a weight ``[outputs, inputs]``, for :func:`scaled_product`: a scale
    for each 128 x 128 values, as :func:`quantize` has them for 128. Once, in torch, on the weight's
    device."""
    _require(weight.dim() == 2 and weight.is_floating_point(),
             f"weight: floating [outputs, inputs] expected, got {weight.dtype}{list(weight.shape)}")
    n, k = weight.shape
    _require(k % 16 == 0 and k > 0, f"weight: a multiple of 16 inputs expected, got {k}")
    rows, blocks = decoder.blocks_of(n), decoder.blocks_of(k)
    with torch.no_grad():
        whole = torch.zeros(rows * decoder.BLOCK, blocks * decoder.BLOCK, dtype=torch.float32,
                            device=weight.device)
        whole[:n, :k] = weight
        tiles = whole.view(rows, decoder.BLOCK, blocks, decoder.BLOCK)
        top = torch.where(tiles.isfinite(), tiles.abs(), 0.0).amax(dim=(1, 3))
        scales = (top / 448.0).clamp(min=2.0 ** -126)
        tiles /= scales[:, None, :, None]
        whole = torch.where(whole.isfinite(), whole, float("nan"))[:n, :k]
        return whole.contiguous().to(_E4M3), scales


def scaled_product(a, a_scales, b, b_scales, bias=None, *, dtype=torch.bfloat16):
    """Rows of codes ``a [rows, k]`` or ``[batch, tokens, k]`` times a weight of codes ``b
    [outputs, k]``, both ``float8_e4m3fn`` with ``k`` a multiple of 16 and rows on 16 bytes:

        out[m, n] = sum_j a[m, j] * a_scales[m, j / 128] * b[n, j] * b_scales[n / 128, j / 128] + bias[n]

    Scales are float32, ``[..., ceil(k / 128)]`` (:func:`quantize`) and ``[ceil(outputs / 128),
    ceil(k / 128)]`` (:func:`quantize_weight`), of any value; a block's two are multiplied in fp32. ``bias
    [outputs]`` is in ``dtype`` or float32. The result is ``dtype``: float16, bfloat16 or float32.

    Sums are held in fp32. In float32, and for few rows in any type, every product counts whole.
    In float16 and bfloat16 of more rows the matrix units take eight neighbouring products at once and
    cut each at 2^-13 of the largest one's power of two: a random sum is 1.3e-5 to 3e-5 of itself off, but one of
    large terms that cancel by as much of those, and a row's result depends in its last places on how many rows
    come with it.
    """
    number = _result_number(dtype)
    out = _now("scaled_product", (a, a_scales, b, b_scales, bias), (number,), 1)
    if out is not None:
        return out[0]
    return torch.ops.mlc.scaled_product(a, a_scales, b, b_scales, bias, dtype)


def sample(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token, ``int64 [batch]``, of each row of ``logits [batch, tokens]`` (fp16, bf16 or
    fp32) from the random numbers ``uniform`` (float32[batch], 0 or more and below 1).

    A token's weight is ``e^((logit - largest) / temperature)`` (float32[batch]; 0, or less than
    2^-100, takes the likeliest token, the first of several; without it 1). In the order of
    falling logits, and of indexes where they are equal, kept are

    * ``top_k`` (int32[batch]): the first so many; all where it is not positive;
    * ``top_p`` (float32[batch]): of those the ones in front of which less than ``top_p`` of
      their weight lies, the first always;
    * ``min_p`` (float32[batch]): of those the ones of ``min_p`` times the largest weight or more.

    The token is the first, by index, up to which more than ``uniform`` of the kept weight lies.
    Weights count in steps of 2^-40 of the largest, and of 2^-24 of the weight of the eight neighbouring
    tokens that they may be added with in fp32: one of 2^-25 beside one of 1 may never be drawn. A token whose
    border lies within 2^-20 of the random number, or of ``top_p`` or ``min_p``, may go to either side. Logits of
    -infinity are never taken; a row of nothing else gets -1. So does a row with NaN or +infinity among its
    logits, a random number outside its range, or an option that is NaN, negative or, for ``top_p`` and ``min_p``,
    above 1, for the temperature above 2^100: ``ExecutionError`` is raised by a later call or :func:`check_errors`.
    """
    out = _now("sample", (logits, uniform, temperature, top_k, top_p, min_p), (), 1)
    if out is not None:
        return out[0]
    return torch.ops.mlc.sample(logits, uniform, temperature, top_k, top_p, min_p)


class _KeepsTypes(torch.nn.Module):
    def _apply(self, fn, recurse=True):
        """Moves the buffers with the module but keeps their types: ``model.half()`` is for
        weights."""
        for name, x in self._buffers.items():
            if x is not None:
                y = fn(x)
                self._buffers[name] = y if y.dtype == x.dtype else x.to(y.device)
        return self


class ScaledLinear(_KeepsTypes):
    """A linear layer whose weight is held in 8 bits (:func:`scaled_product`), as buffers of a
    module. Called with rows it brings them into 8 bits itself; called with codes and scales
    (of :func:`rms_norm` or :func:`quantize`) it takes those."""

    def __init__(self, inputs: int, outputs: int, *, bias: bool = False, dtype=torch.bfloat16,
                 device=None) -> None:
        super().__init__()
        _require(inputs > 0 and inputs % 16 == 0, f"a multiple of 16 inputs expected, got {inputs}")
        _result_number(dtype)
        self.inputs, self.outputs, self.dtype = inputs, outputs, dtype
        self.register_buffer("codes", torch.zeros(outputs, inputs, dtype=torch.uint8, device=device)
                             .view(_E4M3))
        self.register_buffer("scales", torch.ones(decoder.blocks_of(outputs), decoder.blocks_of(inputs),
                                                  dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros(outputs, dtype=torch.float32, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, dtype=None) -> "ScaledLinear":
        """``linear`` in 8 bits, with results in ``dtype`` (that of its weight)."""
        w = linear.weight
        made = cls(w.shape[1], w.shape[0], bias=linear.bias is not None, dtype=dtype or w.dtype,
                   device=w.device)
        codes, scales = quantize_weight(w.detach())
        made.codes.copy_(codes)
        made.scales.copy_(scales)
        if linear.bias is not None:
            made.bias.copy_(linear.bias.detach())
        return made

    def forward(self, x, scales=None):
        if scales is None:
            x, scales = quantize(x)
        return scaled_product(x, scales, self.codes, self.scales, self.bias, dtype=self.dtype)


class KeyValueCache(_KeepsTypes):
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
                                 torch.ones(*shape[:2], capacity // block, dtype=torch.float32, device=device),
                                 persistent=False)

    def append(self, k, v, start, count=None) -> None:
        cache_append(self.keys, self.values, self.key_scales, self.value_scales, k, v, start, count)

    def attend(self, q, start, count=None, **options):
        return cache_attention(q, self.keys, self.values, self.key_scales, self.value_scales,
                               start, count, **options)
