"""Launches of the operators of ``mlc.ops``: rotary positions, attention with
masks made from indices, the 8-bit cache and the attention over it.

Their kernels are hand-written (``codegen/operators/*.hip``) and take every size
and stride as an argument; what is fixed when they are compiled is the element
type, the head size rounded up to a tile's, and which of the options the call
uses. ``plan_*`` picks the kernel from sizes, types and alignment alone and lays
its arguments out: pointers first, then what follows from the operands' shapes.
The same plan serves a direct call and a compiled model.
"""

from __future__ import annotations

import functools
import math
import pathlib
import struct
from dataclasses import dataclass

import torch

SOURCES = pathlib.Path(__file__).resolve().parent / "operators"
NAMES = {torch.float16: "mlc::f16", torch.bfloat16: "__bf16", torch.float32: "float"}
SHORT = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
LOG2E = math.log2(math.e)
#: HIP takes fewer than 2^32 threads a launch
MAX_THREADS = 2 ** 32 - 1
#: compute units of an MI355X
UNITS = 256


class OperatorError(ValueError):
    """Arguments that an operator of ``mlc.ops`` does not take."""


@dataclass(frozen=True)
class Operand:
    """A tensor as a plan sees it; ``offset`` in bytes from the pointer that a
    launch is given."""

    shape: tuple
    strides: tuple
    dtype: torch.dtype
    offset: int = 0
    #: whether pointer and offset together are a multiple of 16
    aligned: bool = True


def require_aligned(operands: dict) -> None:
    """Caches and their scales lie on 16 bytes: kernels take their rows in such pieces."""
    for name, x in operands.items():
        if name.endswith(("_cache", "_scale")) and not x.aligned:
            raise OperatorError(f"{name}: not on 16 bytes")


@dataclass(frozen=True)
class Launch:
    """One kernel launch: ``pointers`` names what its leading arguments point
    to (None: a null pointer), ``tail`` are the bytes behind them."""

    kernel: str  # the macro call that instantiates the kernel
    file: str
    symbol: str
    grid: int
    block: int
    pointers: tuple
    tail: bytes

    def arguments(self, pointers: dict) -> bytes:
        return struct.pack(f"<{len(self.pointers)}Q",
                           *[0 if p is None else pointers[p] for p in self.pointers]) + self.tail


@dataclass(frozen=True)
class Plan:
    launches: tuple
    #: bytes of memory that the launches share and nobody reads afterwards
    workspace: int = 0


@functools.lru_cache(maxsize=None)
def _text(file: str) -> str:
    return (SOURCES / "common.hip").read_text() + (SOURCES / f"{file}.hip").read_text()


def source(file: str, kernel: str) -> str:
    """The module that holds one kernel."""
    return f"{_text(file)}\n{kernel}\n"


def _grid(blocks: int, threads: int, what: str) -> int:
    if blocks * threads > MAX_THREADS:
        raise OperatorError(f"{what}: {blocks} workgroups of {threads} threads are more than one "
                            "launch takes; split the batch")
    return blocks


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _numel(x: Operand) -> int:
    return math.prod(x.shape)


# --------------------------------------------------------------------------
# rotary positions
# --------------------------------------------------------------------------

ROTARY_BLOCK, ROTARY_PAIRS, ROTARY_TOKENS = 256, 1024, 64


def rotary_kernel(dtype, v: int, interleaved: bool) -> tuple[str, str]:
    name = f"rotary_{SHORT[dtype]}_v{v}_{'pairs' if interleaved else 'halves'}"
    return f"ROTARY({name}, {NAMES[dtype]}, {v}, {str(bool(interleaved)).lower()})", name


def plan_rotary(q: Operand, k: Operand, positions: Operand, frequencies: Operand,
                interleaved: bool, magnitude: float) -> Plan:
    batch, seq, heads, dim = q.shape
    kv_heads = k.shape[2]
    turned = 2 * frequencies.shape[0]
    tokens = batch * seq
    if tokens * (heads + kv_heads) * dim == 0:
        return Plan(())
    run = turned if interleaved else turned // 2
    v = 16 // q.dtype.itemsize if q.aligned and k.aligned else 1
    while v > 1 and any(n % v for n in (dim, turned, run, *q.strides[:3], *k.strides[:3])):
        v //= 2
    # many workgroups first, so that some stream while others evaluate angles (4 x 4096 tokens,
    # 40 heads of 128: 16 tokens a workgroup 81 us, 1 69), then as many tokens of one as fit;
    # fewer than 2^20 rows of heads
    group = max(1, min(ROTARY_PAIRS // max(1, turned // 2), ROTARY_TOKENS, tokens // (64 * UNITS),
                       (1 << 20) // (heads + kv_heads)))
    blocks = min(_ceil(tokens, group), 1 << 22)
    pb, pt = (0, positions.strides[0]) if len(positions.shape) == 1 else positions.strides
    tail = struct.pack("<4q9q8ifi", q.offset, k.offset, positions.offset, frequencies.offset,
                       *q.strides[:3], *k.strides[:3], pb, pt, frequencies.strides[0],
                       tokens, seq, heads, kv_heads, dim, turned, group,
                       positions.dtype == torch.int64, magnitude, 0)
    kernel, name = rotary_kernel(q.dtype, v, interleaved)
    return Plan((Launch(kernel, "rotary", name, blocks, ROTARY_BLOCK,
                        ("q", "k", "positions", "frequencies", "out0", "out1"), tail),))


# --------------------------------------------------------------------------
# attention over keys and values in 16 bits
# --------------------------------------------------------------------------

ATTENTION_DIMS = (64, 96, 128, 256)


def _padded(dim: int, dims) -> int:
    return next(d for d in dims if d >= dim)


def score_scale(scale: float | None, dim: int) -> float:
    return 1.0 / math.sqrt(max(dim, 1)) if scale is None else float(scale)


def _factors(scale: float, cap: float) -> tuple[float, float]:
    """What a score is multiplied by, and the cap in log2 units: the kernels'
    exponentials are powers of two."""
    return (scale / cap, cap * LOG2E) if cap else (scale * LOG2E, 0.0)


def attention_kernel(dtype, dp: int, waves: int, source: str, scores: str, apart: bool
                     ) -> tuple[str, str]:
    name = (f"attention_{SHORT[dtype]}_{dp}_w{waves}_{source.lower()}"
            f"_{scores.lower()}{'_apart' if apart else ''}")
    return (f"ATTENTION({name}, {NAMES[dtype]}, {dp}, {waves}, {source}, {scores}, "
            f"{str(apart).lower()})"), name


def join_kernel(op: str, dtype, waves: int) -> tuple[str, str]:
    name = f"{op}_join_{SHORT[dtype]}_w{waves}"
    return f"{op.upper()}_JOIN({name}, {NAMES[dtype]}, {waves})", name


def _join(op: str, dtype, parts: int, rows: int, pointers: tuple, tail: bytes) -> Launch:
    """The launch that makes one of up to ``parts`` parts of each of ``rows`` rows: four
    waves a row take the latency of many parts side by side where rows are few."""
    waves = 4 if parts > 8 and rows <= 1 << 16 else 1
    kernel, name = join_kernel(op, dtype, waves)
    return Launch(kernel, op, name, _grid(rows, 64 * waves, op), 64 * waves, pointers, tail)


def attention_split(rows: int, pairs: int, keys: int, dim: int, teams: tuple, apart: tuple | None
                    ) -> tuple[bool, int, int]:
    """Whether the waves of a workgroup take keys apart, how many waves it has, and splits
    of the keys, by what the ways cost in us. ``teams`` and ``apart``: keys of a tile and the
    time of one, and for the second the waves.

    Waves that share tiles have 32 rows each, and two such workgroups fit a unit; waves
    apart have the same 32 rows, a quarter of the tiles one behind the other, four times the
    workgroups, and one fits a unit. Causal, bf16: 1000 tokens, 12 heads of 64 shared 18.6, apart
    11.2; 3 x 1024, 4 heads of 128 28.5, 17.4; 4096, 8 heads of 128 69, 83; 4 x 300, 32 heads over
    8 of 128 15, 31.

    All keys are priced for every row. A causal mask leaves out half of both ways' tiles, and
    without one the same ways are faster (18.5, 16.5; 29.9, 26.6; 93, 142; 19, 39). How much
    documents and prefixes leave out is known on the device alone; with documents: 4096 tokens, 8
    heads of 128, 8 documents 38, 64 and one 78, 137; 3 x 2021, 16 heads over 4 of 96, 8 documents
    41, 129; 4 x 1000, 16 heads of 64, 8 documents 18, 74; 6 x 999, 8 heads of 256, 5 documents 64,
    118; 300, 4 heads of 128, 2 documents 13.1, 11.9; 1000, 12 heads of 64, 4 documents 20.4, 20.5:
    what the rule takes is within 5 % of the better one in all of them.

    Splits fill the device where there are few workgroups. What they cost is a second
    launch and parts of O in fp32, written and read: 4 us and 8 bytes a value at 3 TB/s."""
    values = rows * pairs * (dim + 4)
    best = None

    def consider(is_apart: bool, waves: int, blocks: int, room: int, first: float, tiles: int, us: float):
        nonlocal best
        for n in range(1, max(1, min(room // blocks, tiles)) + 1):
            cost = max(1.0, blocks * n / room) * (first + _ceil(tiles, n) * us)
            cost += 4 + n * values * 8 / 3e6 if n > 1 else 0
            if best is None or cost < best[0]:
                best = cost, (is_apart, waves, n)

    waves = 4 if rows > 64 else 2 if rows > 32 else 1
    consider(False, waves, _ceil(rows, 32 * waves) * pairs, 2 * UNITS, 5, _ceil(keys, teams[0]), teams[1])
    if apart:
        n, us, waves = apart
        consider(True, waves, _ceil(rows, 32) * pairs, UNITS, 5.5, _ceil(keys, n * waves), us)
    return best[1]


def _strides(x: Operand | None, n: int) -> tuple:
    return x.strides[:n] if x is not None else (0,) * n


def _offset(x: Operand | None) -> int:
    return x.offset if x is not None else 0


def _attention(source: str, q: Operand, k: Operand, v: Operand, pairs: tuple, key_strides: tuple,
               masks: tuple, cache: tuple, causal: bool, factors: tuple) -> Plan:
    """Launches of ``attention.hip``. ``pairs``: kv_heads, keys; ``masks``: slopes, documents,
    prefix; ``cache``: key and value scales, start, count and the tokens of a
    scale, in logarithm."""
    batch, queries, heads, dim = q.shape
    kv_heads, keys = pairs
    slopes, documents, prefix = masks
    *scales, start, count, shift = cache
    codes = source == "CODES"
    dp, group = _padded(dim, CACHED_DIMS if codes else ATTENTION_DIMS), heads // kv_heads
    rows = queries * group
    # measured: 1 us for 64 keys of 64 values, 1.8 of 128; twice that through registers.
    # Waves apart take 32 keys of more than 64 values at a time, in 0.6 of it.
    us = (0.2 + dp / 80) * (1 if source == "DIRECT" else 2)
    teams = (32, us / 2) if codes or dp == 256 else (64, us)
    alone = (64, us, 4) if dp == 64 else (32, us * 0.6, 4) if dp < 256 else (32, us / 2, 2)
    apart, waves, splits = attention_split(rows, batch * kv_heads, keys, dim, teams, None if codes else alone)
    tiles = _ceil(rows, 32 if apart else 32 * waves)
    scores = ("DOCUMENTS" if documents is not None else
              "BIASED" if factors[1] or slopes is not None else "PLAIN")
    operands = {"q": q, "k": k, "v": v, "slopes": slopes, "documents": documents, "prefix": prefix,
                "k_scale": scales[0], "v_scale": scales[1], "start": start, "count": count}
    names = {"k": "k_cache", "v": "v_cache"} if codes else {}
    where = {n: names.get(n, n) if x is not None else None for n, x in operands.items()}
    pointers = (*list(where.values())[:6], "out0", "workspace" if splits > 1 else None,
                *list(where.values())[6:], "error" if codes else None)
    tail = struct.pack("<10q15q10i2f", *map(_offset, operands.values()), *q.strides[:3],
                       *key_strides, *_strides(slopes, 1), *_strides(documents, 2),
                       *_strides(prefix, 1), *_strides(start, 1), *_strides(count, 1),
                       batch, queries, keys, kv_heads, group, dim, causal, tiles, splits, shift,
                       *factors)
    kernel, name = attention_kernel(q.dtype, dp, waves, source, scores, apart)
    grid = _grid(tiles * batch * kv_heads * splits, 64 * waves, "attention")
    launch = Launch(kernel, "attention", name, grid, 64 * waves, pointers, tail)
    if splits == 1:
        return Plan((launch,))
    return Plan((launch, _join("attention", q.dtype, splits, batch * queries * heads, pointers, tail)),
                splits * batch * kv_heads * rows * (dim + 4) * 4)


def plan_attention(q: Operand, k: Operand, v: Operand, slopes: Operand | None,
                   documents: Operand | None, prefix: Operand | None, scale: float, causal: bool,
                   cap: float) -> Plan:
    if _numel(q) == 0:
        return Plan(())
    keys, kv_heads = k.shape[1:3]
    # a tile's rows are addressed by 32 bits from its first one
    direct = (q.shape[3] in ATTENTION_DIMS and keys > 0 and k.aligned and v.aligned
              and all(n % 8 == 0 for n in (*k.strides[:3], *v.strides[:3]))
              and max(k.strides[1], v.strides[1]) < 1 << 24)
    return _attention("DIRECT" if direct else "COPIED", q, k, v, (kv_heads, keys),
                      (*k.strides[:3], *v.strides[:3]), (slopes, documents, prefix),
                      (None, None, None, None, 0), causal, _factors(scale, cap))


# --------------------------------------------------------------------------
# the 8-bit cache
# --------------------------------------------------------------------------

def append_kernel(dtype, align: int, n: int, waves: int) -> tuple[str, str]:
    name = f"cache_append_{SHORT[dtype]}_a{align}_n{n}_w{waves}"
    return f"CACHE_APPEND({name}, {NAMES[dtype]}, {align}, {n}, {waves})", name


def plan_cache_append(k_cache: Operand, v_cache: Operand, k_scale: Operand, v_scale: Operand,
                      k: Operand, v: Operand, start: Operand, count: Operand | None) -> Plan:
    batch, heads, capacity, dim = k_cache.shape
    tokens = k.shape[1]
    block = capacity // k_scale.shape[2] if k_scale.shape[2] else 1
    if batch * heads * capacity * dim * tokens == 0:
        return Plan(())
    touched = min(capacity // block, (tokens + block - 2) // block + 1)
    pack = 8
    whole = all(n % pack == 0 for n in (*k.strides[:3], *v.strides[:3]))
    align = 16 if whole and k.aligned and v.aligned else k.dtype.itemsize
    # a workgroup's registers hold the new rows of a block: one wave where one
    # item of 8 values for each lane is enough
    items = min(tokens, block) * dim // 8
    waves = 1 if items <= 64 else 4
    n = 1 << (_ceil(items, 64 * waves) - 1).bit_length()
    off = lambda x: x.offset if x is not None else 0  # noqa: E731
    pair = lambda i: (k.strides[i], v.strides[i])  # noqa: E731
    tail = struct.pack("<8q8q6i", k_cache.offset, v_cache.offset, k_scale.offset, v_scale.offset,
                       k.offset, v.offset, start.offset, off(count), *pair(0), *pair(1), *pair(2),
                       start.strides[0], count.strides[0] if count is not None else 0,
                       tokens, heads, dim, capacity, block, touched)
    kernel, name = append_kernel(k.dtype, align, n, waves)
    grid = _grid(batch * touched * 2 * heads, 64 * waves, "cache_append")
    pointers = ("k_cache", "v_cache", "k_scale", "v_scale", "k", "v", "start",
                "count" if count is not None else None, "error")
    return Plan((Launch(kernel, "cache_append", name, grid, 64 * waves, pointers, tail),))


CACHED_DIMS = (64, 128, 256)
#: products of scores and values from which on rows go through tiles of 128
#: (``attention.hip``) and not of 16: keys are widened once for all of them, in more
#: launches of work that is fixed. Tiles of 128 / 16, 8 key heads of 128: 4 x 128 rows over
#: 2048 keys (1.1e9) 25 / 22 us, 4 x 512 (4.3e9) 39 / 53, 512 over 16384 (8.6e9) 61 / 97;
#: 2 x 488 rows of 2 heads over 8192 (2.0e9) 34 / 35, over 16384 (4.1e9) 41 / 55.
MANY_ROWS, MANY_PRODUCTS = 128, 3e9


def cached_kernel(dtype, dp: int, step: int, waves: int, general: bool) -> tuple[str, str]:
    name = f"cache_attention_{SHORT[dtype]}_{dp}_{step}_{waves}{'_general' if general else ''}"
    return (f"CACHE_ATTENTION({name}, {NAMES[dtype]}, {dp}, {step}, {waves}, "
            f"{str(general).lower()})"), name


def plan_cache_attention(q: Operand, k_cache: Operand, v_cache: Operand, k_scale: Operand,
                         v_scale: Operand, start: Operand, count: Operand | None,
                         slopes: Operand | None, scale: float, cap: float) -> Plan:
    batch, tokens, heads, dim = q.shape
    kv_heads, capacity = k_cache.shape[1:3]
    if _numel(q) == 0:
        return Plan(())
    group, block = heads // kv_heads, capacity // k_scale.shape[2] if k_scale.shape[2] else 32
    rows = tokens * group
    if rows >= MANY_ROWS and batch * heads * tokens * capacity * dim > MANY_PRODUCTS:
        strides = (kv_heads * capacity * dim, dim, capacity * dim)
        return _attention("CODES", q, k_cache, v_cache, (kv_heads, capacity), strides * 2,
                          (slopes, None, None), (k_scale, v_scale, start, count, block.bit_length() - 1),
                          True, _factors(scale, cap))
    dp = _padded(dim, CACHED_DIMS)
    row_tiles = _ceil(rows, 16)
    step = 64 if block % 64 == 0 else 32
    # A workgroup's waves go through a short cache at once; a longer one is cut into items,
    # as many as the device holds, none shorter than two steps of every wave.
    short = capacity <= (4096 if batch * kv_heads * row_tiles >= 2 * UNITS else 1024)
    waves = 8 if short and batch * kv_heads * row_tiles < UNITS and dp < 256 else 4
    shortest = 2 * 64 * waves
    most = 1 if short else _ceil(capacity, shortest)
    items = 0 if short else max(1, min(2 * UNITS // (kv_heads * row_tiles), batch * most))
    slots = min(items + batch, batch * most)
    general = bool(cap) or slopes is not None
    off = lambda x: x.offset if x is not None else 0  # noqa: E731
    tail = struct.pack("<8q6q8i2i2f", q.offset, k_cache.offset, v_cache.offset, k_scale.offset,
                       v_scale.offset, off(slopes), start.offset, off(count), *q.strides[:3],
                       slopes.strides[0] if slopes is not None else 0, start.strides[0],
                       count.strides[0] if count is not None else 0, batch, tokens, kv_heads,
                       group, dim, capacity, block.bit_length() - 1, row_tiles, items, shortest,
                       *_factors(scale, cap))
    kernel, name = cached_kernel(q.dtype, dp, step, waves, general)
    pointers = ("q", "k_cache", "v_cache", "k_scale", "v_scale",
                "slopes" if slopes is not None else None, "start",
                "count" if count is not None else None, "out0",
                "workspace" if most > 1 else None, "error")
    grid = _grid(slots * row_tiles * kv_heads, 64 * waves, "cache_attention")
    launches = [Launch(kernel, "cache_attention", name, grid, 64 * waves, pointers, tail)]
    workspace = 0
    if most > 1:  # a sequence may be cut
        workspace = _ceil(batch, 2) * 16 + slots * kv_heads * rows * (dim + 4) * 4
        launches.append(_join("cache_attention", q.dtype, min(most, slots), batch * tokens * heads,
                              pointers, tail))
    return Plan(tuple(launches), workspace)


#: operators of a captured graph -> the plan of their operands, by their names in
#: the operator's schema
PLANS = {
    "mlc.rotary.default": plan_rotary,
    "mlc.attention.default": lambda q, k, v, scale, causal, cap, slopes, documents, prefix:
        plan_attention(q, k, v, slopes, documents, prefix, score_scale(scale, q.shape[3]), causal, cap),
    "mlc.cache_append.default": plan_cache_append,
    "mlc.cache_attention.default":
        lambda q, k_cache, v_cache, k_scale, v_scale, start, count, scale, cap, slopes:
        plan_cache_attention(q, k_cache, v_cache, k_scale, v_scale, start, count, slopes,
                             score_scale(scale, q.shape[3]), cap),
}
#: those that can meet an invalid input
FLAGGING = ("mlc.cache_append.default", "mlc.cache_attention.default")


def all_kernels() -> list[tuple[str, str]]:
    """``(file, kernel)`` of everything that a plan can ask for."""
    out = []
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        out += [("rotary", rotary_kernel(dtype, v, i)[0]) for v in (8, 4, 2, 1)
                for i in (False, True) if v * dtype.itemsize <= 16]
        out += [("cache_append", append_kernel(dtype, a, n, w)[0]) for a in (16, dtype.itemsize)
                for n, w in ((1, 1), (1, 4), (2, 4), (4, 4), (8, 4), (16, 4))]
    for dtype in (torch.float16, torch.bfloat16):
        for source in ("COPIED", "DIRECT", "CODES"):
            for scores in ("PLAIN", "BIASED", "DOCUMENTS")[:2 if source == "CODES" else 3]:
                ways = [(dp, 4, False) for dp in CACHED_DIMS] if source == "CODES" else \
                    [(dp, w, False) for dp in ATTENTION_DIMS for w in (1, 2, 4)] + \
                    [(dp, 4 if dp < 256 else 2, True) for dp in ATTENTION_DIMS]
                out += [("attention", attention_kernel(dtype, dp, w, source, scores, apart)[0])
                        for dp, w, apart in ways]
        out += [("cache_attention", cached_kernel(dtype, dp, step, w, g)[0])
                for dp in CACHED_DIMS for w in (4, 8) if w < 8 or dp < 256 for step in (32, 64)
                for g in (False, True)]
        out += [(op, join_kernel(op, dtype, w)[0]) for op in ("attention", "cache_attention")
                for w in (1, 4)]
    return out
