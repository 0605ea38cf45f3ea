"""Launches of the operators of ``mlc.ops`` that stand around a decoder's attention: norms
and rows in 8 bits, products of scaled 8-bit values, the choice of a token.

Like those of ``hip_operators`` their plans follow from sizes, types and alignment alone and
serve direct calls and compiled models. Results have shapes and types of their own, which a
plan carries.
"""

from __future__ import annotations

import struct

import torch

from .hip_operators import (NAMES, SHORT, UNITS, Launch, Operand, OperatorError, Plan, _ceil, _grid,
                            _numel, _offset)

E4M3 = torch.float8_e4m3fn
#: values that share a scale
BLOCK = 128
#: types of a product's result, by the number that stands for one among a call's options
RESULTS = (torch.float16, torch.bfloat16, torch.float32)


def blocks_of(dim: int) -> int:
    return _ceil(dim, BLOCK)


def _rows(x: Operand | None) -> tuple[int, int, tuple]:
    """Rows of the last dimension, how many of them follow each other with the second stride, and
    the strides of both. What a dimension of one says of its stride means nothing."""
    if x is None:
        return 0, 1, (0, 0)
    if len(x.shape) == 3 and x.shape[1] != 1:
        return x.shape[0] * x.shape[1], max(1, x.shape[1]), (x.strides[0] if x.shape[0] > 1 else 0, x.strides[1])
    return x.shape[0], max(1, x.shape[0]), (0, x.strides[0] if x.shape[0] > 1 else 0)


def _in_packs(x: Operand | None, n: int) -> bool:
    """Whether rows begin on 16 bytes, as packs of ``n`` values do."""
    return x is None or (x.aligned and all(s % n == 0 for s in _rows(x)[2]))


# --------------------------------------------------------------------------
# rows
# --------------------------------------------------------------------------

#: values of a row in registers at most
MOST_DIM = 1 << 15
#: (waves of a row, packs of 8 values of a lane), shortest rows first. 2^25 values in bf16 with a residual, in us: rows
#: of 1024 by 1 wave of 2 packs 50.5 and by 4 of 1 52.5 (to codes 46.8 and 61), of 1168 by 1 of 4 65.6 and by 4 of 1
#: 53 (65.4 and 60), of 2048 53 and 45.5 (52.7 and 48.7); of 4096 by 1 of 8 68 and by 4 of 2 51.8 (70 and 46.4).
NORM_SHAPES = ((1, 1), (1, 2), (4, 1), (4, 2), (4, 4), (16, 2), (16, 4))
QUANTIZE_THREADS, QUANTIZE_PACKS = 256, 2


def norm_kernel(dtype, align: int, waves: int, n: int, eight: bool) -> tuple[str, str]:
    name = f"rms_norm_{SHORT[dtype]}_a{align}_w{waves}_n{n}{'_e4m3' if eight else ''}"
    return f"RMS_NORM({name}, {NAMES[dtype]}, {align}, {waves}, {n}, {str(eight).lower()})", name


def quantize_kernel(dtype, align: int, gated: bool) -> tuple[str, str]:
    name = f"quantize_{SHORT[dtype]}_a{align}{'_gated' if gated else ''}"
    return f"QUANTIZE({name}, {NAMES[dtype]}, {align}, {str(gated).lower()})", name


def eight_bits(x) -> tuple:
    """Shapes and types of the codes and scales of rows like ``x``."""
    return ((tuple(x.shape), E4M3), ((*x.shape[:-1], blocks_of(x.shape[-1])), torch.float32))


def norm_results(x, residual, quantized: bool) -> tuple:
    made = eight_bits(x) if quantized else ((tuple(x.shape), x.dtype),)
    return (*made, (tuple(x.shape), x.dtype)) if residual is not None else made


def _row_args(x: Operand, other: Operand | None, weight: Operand | None, eps: float) -> bytes:
    rows, seq, strides = _rows(x)
    return struct.pack("<3q4q4i2d", x.offset, _offset(other), _offset(weight), *strides,
                       *_rows(other)[2], rows, seq, x.shape[-1], weight is not None
                       and weight.dtype == torch.float32, eps, 1.0 / x.shape[-1])


def plan_norm(x: Operand, weight: Operand, residual: Operand | None, eps: float, quantized: bool) -> Plan:
    results = norm_results(x, residual, quantized)
    rows, _, _ = _rows(x)
    dim = x.shape[-1]
    if rows * dim == 0:
        return Plan((), results=results)
    align = 16 if dim % 8 == 0 and _in_packs(x, 8) and _in_packs(residual, 8) else x.dtype.itemsize
    waves, n = next((w, n) for w, n in NORM_SHAPES if 512 * w * n >= dim)
    kernel, name = norm_kernel(x.dtype, align, waves, n, quantized)
    grid = _grid(_ceil(rows, 4) if waves == 1 else rows, max(256, 64 * waves), "rms_norm")
    pointers = ("x", "residual" if residual is not None else None, "weight", "out0",
                "out1" if quantized else None,
                f"out{len(results) - 1}" if residual is not None else None)
    return Plan((Launch(kernel, "rows", name, grid, max(256, 64 * waves), pointers,
                        _row_args(x, residual, weight, eps)),), results=results)


def plan_quantize(x: Operand, gate: Operand | None) -> Plan:
    results = eight_bits(x)
    rows, _, _ = _rows(x)
    if _numel(x) == 0:
        return Plan((), results=results)
    align = 16 if _in_packs(x, 8) and _in_packs(gate, 8) else x.dtype.itemsize
    kernel, name = quantize_kernel(x.dtype, align, gate is not None)
    packs = rows * blocks_of(x.shape[-1]) * (BLOCK // 8)
    grid = _grid(_ceil(packs, QUANTIZE_THREADS * QUANTIZE_PACKS), QUANTIZE_THREADS, "quantize")
    return Plan((Launch(kernel, "rows", name, grid, QUANTIZE_THREADS,
                        ("x", "gate" if gate is not None else None, None, "out0", "out1", None),
                        _row_args(x, gate, None, 0.0)),), results=results)


# --------------------------------------------------------------------------
# products
# --------------------------------------------------------------------------

#: Few rows, up to 16: a workgroup reads all of them beside 16 rows of the weight, in 8 waves with 4 blocks each. Reading
#: them again and again ends that: 1 row, 4096 -> 8192 8.9 us and in tiles 11.2, 16 rows, 4096 -> 4096 7.5 and 10.8,
#: 8 rows, 4096 -> 8192 10.4 and 11.0; but 16 rows 12.0 and 11.4, 12288 -> 4096 15.8 and 14.9, 1 row, 4096 -> 16384 15.5
#: and 13.7, and 12288 -> 5120, one and a quarter rounds of long sums, 17.4 and 15.0.
FEW_ROWS, FEW_COLUMNS, FEW_SUM, FEW_VALUES, FEW_PRODUCTS = 16, 8192, 8192, 1 << 16, 1 << 29
#: In 16 waves where a unit has one workgroup and the sum more blocks than 8 waves ask for at once: 1 row, 12288 -> 4096
#: 10.9 us and with 8 waves 11.9, 16384 -> 4096 16.6 and 18.8; but 4096 -> 6144 9.6 and 8.6, 4096 -> 1024 6.0 and 5.7.
FEW_BLOCKS, FEW_WAVES = 4, (8, 16)
#: Tiles of many rows by the product's instructions, exact or not (rows of both operands, waves along both):
#: workgroups that a unit holds, and in us what one takes beside its steps, a step of one alone and of each of
#: many. Measured over 768 to 12288 inputs, 128 to 8192 rows and 2304 to 24576 outputs.
TILES = {False: {(256, 256, 4, 2): (1, 8.5, 1.7, 1.7), (128, 128, 2, 2): (2, 3.5, 0.75, 0.59),
                 (64, 64, 2, 2): (4, 2.5, 0.31, 0.21), (32, 64, 2, 2): (4, 2.5, 0.28, 0.155)},
         True: {(128, 128, 2, 2): (2, 3.5, 1.25, 1.05), (64, 64, 2, 2): (4, 2.5, 0.46, 0.36),
                (32, 64, 2, 2): (4, 2.5, 0.38, 0.22)}}
JOIN_THREADS = 256


def takes_rows(rows: int, n: int, k: int) -> bool:
    """Whether a workgroup reads all rows of a."""
    return (rows <= FEW_ROWS and n <= FEW_COLUMNS and rows * n <= FEW_VALUES and rows * n * k < FEW_PRODUCTS
            and (n <= 16 * UNITS or k <= FEW_SUM))


def is_exact(rows: int, n: int, k: int, dtype: torch.dtype) -> bool:
    """Whether products are taken of widened codes: where that costs nothing, or fp32 results show it."""
    return dtype == torch.float32 or takes_rows(rows, n, k)


def choose_tile(rows: int, n: int, blocks: int, dtype: torch.dtype) -> tuple[tuple, int]:
    """The tile, and splits of the sum, that cost least. A unit's workgroups share it, so a step takes
    as many times its work as there are, but not less than alone. Splits cost a second launch
    and parts in fp32, written and read: 4 us and 8 bytes a value at 3 TB/s."""
    best = None
    for tile, (room, first, alone, each) in TILES[dtype == torch.float32].items():
        tiles = _ceil(rows, tile[0]) * _ceil(n, tile[1])
        for splits in range(1, max(1, min(blocks // 2, 2 * UNITS // tiles)) + 1):
            steps = _ceil(blocks, splits)
            full, rest = divmod(tiles * splits, UNITS * room)
            cost = full * (first + steps * max(alone, room * each))
            if rest:
                cost += first + steps * max(alone, _ceil(rest, UNITS) * each)
            if splits > 1:
                cost += 4 + splits * rows * n * 8 / 3e6
            if best is None or cost < best[0]:
                best = cost, (tile, splits)
    return best[1]


def few_kernel(dtype, waves: int) -> tuple[str, str]:
    name = f"scaled_product_rows_{SHORT[dtype]}_w{waves}"
    return f"SCALED_PRODUCT_ROWS({name}, {NAMES[dtype]}, {FEW_BLOCKS}, {waves})", name


def tiles_kernel(dtype, tile: tuple) -> tuple[str, str]:
    name = f"scaled_product_tiles_{SHORT[dtype]}_{'_'.join(map(str, tile))}"
    return f"SCALED_PRODUCT_TILES({name}, {NAMES[dtype]}, {', '.join(map(str, tile))})", name


def product_join_kernel(dtype) -> tuple[str, str]:
    name = f"scaled_product_join_{SHORT[dtype]}"
    return f"SCALED_PRODUCT_JOIN({name}, {NAMES[dtype]})", name


def product_results(a, b, dtype) -> tuple:
    return (((*a.shape[:-1], b.shape[0]), dtype),)


def require_pieces(**operands) -> None:
    """Rows of codes are taken in pieces of 16 bytes."""
    for name, x in operands.items():
        if _numel(x) and not _in_packs(x, 16):
            raise OperatorError(f"{name}: rows of codes that lie on 16 bytes expected")


def _reach(x: Operand, strides: tuple) -> int:
    """Bytes from the first of the rows to the last."""
    shape = x.shape[:-1] if len(x.shape) == 3 else (1, x.shape[0])
    return sum((n - 1) * s for n, s in zip(shape, strides)) * x.dtype.itemsize


def plan_product(a: Operand, a_scales: Operand, b: Operand, b_scales: Operand, bias: Operand | None,
                 dtype: torch.dtype) -> Plan:
    results = product_results(a, b, dtype)
    require_pieces(a=a, b=b)
    rows, seq, strides = _rows(a)
    n, k = b.shape
    if rows * n == 0:
        return Plan((), results=results)
    blocks = blocks_of(k)
    splits, row_tiles = 1, 1
    scale_strides = _rows(a_scales)[2]
    regular = all(s[0] == s[1] * seq for s in (strides, scale_strides)) or rows == seq
    if regular:
        seq = rows
    pointers = ["a", "a_scales", "b", "b_scales", "bias" if bias is not None else None, "out0", None]
    if takes_rows(rows, n, k):
        waves = FEW_WAVES[n <= 16 * UNITS and blocks > FEW_WAVES[0] * FEW_BLOCKS]
        kernel, name = few_kernel(dtype, waves)
        grid, threads = _ceil(n, 16), 64 * waves
    else:
        tile, splits = choose_tile(rows, n, blocks, dtype)
        # bytes from where the kernel counts to the end of a row, or to a row's last scale
        most = max(tile[:2])
        far, scales_far = ((most * strides[1], most * 4 * scale_strides[1]) if regular
                           else (_reach(a, strides), _reach(a_scales, scale_strides)))
        reach = max(max(far, most * b.strides[0]) + k, scales_far + 4 * a_scales.strides[-1] * blocks)
        if reach >= 1 << 31:
            raise OperatorError("scaled_product: rows that lie too far apart: make them contiguous")
        row_tiles = _ceil(rows, tile[0])
        kernel, name = tiles_kernel(dtype, tile)
        grid, threads = row_tiles * _ceil(n, tile[1]) * splits, 64 * tile[2] * tile[3]
        if splits > 1:
            pointers[-1] = "workspace"
    tail = struct.pack("<5q8q8i", a.offset, a_scales.offset, b.offset, b_scales.offset, _offset(bias),
                       *strides, *scale_strides, a_scales.strides[-1], b.strides[0],
                       *b_scales.strides, rows, seq, n, k, splits, row_tiles,
                       bias is not None and bias.dtype == torch.float32, regular)
    launches = [Launch(kernel, "scaled_product", name, _grid(grid, threads, "scaled_product"), threads,
                       tuple(pointers), tail)]
    if splits > 1:
        kernel, name = product_join_kernel(dtype)
        launches.append(Launch(kernel, "scaled_product", name,
                               _grid(_ceil(rows * n, JOIN_THREADS), JOIN_THREADS, "scaled_product"),
                               JOIN_THREADS, tuple(pointers), tail))
    return Plan(tuple(launches), splits * rows * n * 4 if splits > 1 else 0, results=results)


# --------------------------------------------------------------------------
# the choice of a token
# --------------------------------------------------------------------------

#: sums of weights, whole numbers up to 2^40 each, stay below 2^63
MOST_TOKENS = 1 << 22
SAMPLE_THREADS = 1024


def sample_kernel(dtype) -> tuple[str, str]:
    name = f"sample_{SHORT[dtype]}"
    return f"SAMPLE({name}, {NAMES[dtype]})", name


def sample_results(logits) -> tuple:
    return (((logits.shape[0],), torch.int64),)


def plan_sample(logits: Operand, uniform: Operand, temperature: Operand | None, top_k: Operand | None,
                top_p: Operand | None, min_p: Operand | None) -> Plan:
    results = sample_results(logits)
    batch, size = logits.shape
    if batch == 0:
        return Plan((), results=results)
    options = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    rows = (uniform, *options.values())
    tail = struct.pack("<6q6q2i", logits.offset, *map(_offset, rows), logits.strides[0],
                       *(x.strides[0] if x is not None else 0 for x in rows), batch, size)
    kernel, name = sample_kernel(logits.dtype)
    pointers = ("logits", "uniform", *(n if x is not None else None for n, x in options.items()),
                "out0", "error")
    return Plan((Launch(kernel, "sample", name, _grid(batch, SAMPLE_THREADS, "sample"), SAMPLE_THREADS,
                        pointers, tail),), results=results)


#: operators of a captured graph -> the plan of their operands, by their names in the schema
PLANS = {
    "mlc.rms_norm.default": lambda x, weight, eps: plan_norm(x, weight, None, eps, False),
    "mlc.add_rms_norm.default": lambda x, weight, residual, eps: plan_norm(x, weight, residual, eps, False),
    "mlc.rms_norm_quantized.default": lambda x, weight, eps: plan_norm(x, weight, None, eps, True),
    "mlc.add_rms_norm_quantized.default": lambda x, weight, residual, eps:
        plan_norm(x, weight, residual, eps, True),
    "mlc.quantize.default": plan_quantize,
    "mlc.scaled_product.default": plan_product,
    "mlc.sample.default": plan_sample,
}
#: those that can meet an invalid input
FLAGGING = ("mlc.sample.default",)


def all_kernels() -> list[tuple[str, str]]:
    """``(file, kernel)`` of everything that a plan can ask for."""
    out = []
    for dtype in RESULTS:
        aligns = sorted({16, dtype.itemsize})
        for w, n in NORM_SHAPES:
            out += [("rows", norm_kernel(dtype, a, w, n, e)[0]) for a in aligns for e in (False, True)]
        out += [("rows", quantize_kernel(dtype, a, g)[0]) for a in aligns for g in (False, True)]
        out += [("scaled_product", few_kernel(dtype, waves)[0]) for waves in FEW_WAVES]
        out += [("scaled_product", product_join_kernel(dtype)[0]),
                ("sample", sample_kernel(dtype)[0])]
        out += [("scaled_product", tiles_kernel(dtype, t)[0]) for t in TILES[dtype == torch.float32]]
    return out
