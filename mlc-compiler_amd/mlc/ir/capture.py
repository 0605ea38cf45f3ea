"""Front end: ``nn.Module`` -> graph IR, through ``torch.export``.

Capture happens in two stages:

1. **Export.** The model is exported in eval mode at the example shapes, and
   the exported program is decomposed with torch's core-ATen table widened by
   :data:`FORCE_DECOMPOSE` (softmax, layer norm, gelu, ... arrive as the
   reductions and pointwise chains they are made of, which fusion needs to
   see).
2. **Translation.** One walk over the exported FX graph emits graph-IR nodes.
   Each ``call_function`` is routed by what it is: a split (rewritten as one
   slice view per piece), an ``addmm`` with unit scalings (rewritten as
   ``mm`` + a fusable bias ``add``, so half-precision GEMMs keep their dtype:
   torch's own ``addmm`` decomposition computes in fp32), a view (a restride
   of its source's buffer, or a copy plus a restride when no restride can
   express it), an op with no rule (kept whole and typed from the exporter's
   metadata), or an op with a rule (typed by :mod:`mlc.ir.shapes`).

Reference behaviour followed: ``mlc/ir/capture.py:38-387``. Kept identical
because later stages depend on them: the two op tables below (they fix the
export graph), value and buffer names (the FX name; ``<fx>_mm`` for the GEMM
of a split ``addmm``; ``<fx>_<i>`` for the pieces of a split or the results
of a multi-result op; ``copy<n>`` for an inserted copy -- the planner breaks
ties by buffer name), slices as the view form of split pieces, and the node
order.
"""

from __future__ import annotations

import contextlib
import operator
import warnings
from typing import Any, Callable, Sequence

import torch
from torch.export import export

from . import shapes
from .graph import Graph, Node, Value
from .ops import NonViewable, OpClass, op_class
from .types import Buffer, Layout

#: core-ATen ops that are decomposed all the same, because each of them wraps a
#: row reduction or an elementwise chain the fusion passes must be able to
#: see (``addmm`` is not among them: see the module docstring)
FORCE_DECOMPOSE = [
    "_softmax",
    "_log_softmax",
    "native_layer_norm",
    "gelu",
    "silu",
    "var_mean.correction",
    "std_mean.correction",
    "split_with_sizes",
    "native_batch_norm",
    "_native_batch_norm_legit_no_training",
]

#: checks export records as nodes; a static-shape program has nothing to do
#: for them at run time
DROP_OPS = {
    "aten._assert_tensor_metadata.default",
    "aten._assert_async.msg",
    "aten._assert_async.default",
    "aten._assert_scalar.default",
    "aten.sym_constrain_range.default",
    "aten.sym_constrain_range_for_size.default",
    "aten._functional_assert_scalar.default",
}

_ADDMM = "aten.addmm.default"
_UNBIND = "aten.unbind.int"
_SPLIT_BY_CHUNK = "aten.split.Tensor"
_SPLIT_BY_SIZES = "aten.split_with_sizes.default"
#: how the exporter writes an op that changes its operands
_IN_PLACE = "auto_functionalized_v2"


class CaptureError(Exception):
    """The model cannot be captured as a static-shape inference graph."""


# --------------------------------------------------------------------------
# stage 1: export
# --------------------------------------------------------------------------

def _aten_overload(spec: str):
    """``"name"`` or ``"name.overload"`` -> the ATen overload, or ``None``
    when this torch has no such op."""
    base, _, overload = spec.partition(".")
    packet = getattr(torch.ops.aten, base, None)
    return None if packet is None else getattr(packet, overload or "default", None)


def _decomposition_table(extra: Sequence[str]) -> dict:
    from torch._decomp import core_aten_decompositions, get_decompositions

    table = dict(core_aten_decompositions())
    table.update(get_decompositions([o for o in map(_aten_overload, extra) if o is not None]))
    return table


@contextlib.contextmanager
def _in_eval_mode(model: torch.nn.Module):
    restore = model.training
    model.eval()
    try:
        yield model
    finally:
        model.train(restore)


def _shared_buffers(model: torch.nn.Module) -> tuple[str, str] | None:
    """Two names of buffers that share memory."""
    seen: dict[int, str] = {}
    for name, x in model.named_buffers(remove_duplicate=False):
        if x is None or not x.numel() or x.is_meta:
            continue
        other = seen.setdefault(x.untyped_storage().data_ptr(), name)
        if other != name:
            return other, name
    return None


def _export(model: torch.nn.Module, example: tuple, extra: Sequence[str]):
    with _in_eval_mode(model), torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        try:
            return export(model, example).run_decompositions(_decomposition_table(extra))
        except AssertionError as e:  # what the exporter makes of a change seen under two names
            shared = _shared_buffers(model)
            if shared is None:
                raise
            raise CaptureError(f"{shared[0]} and {shared[1]} share memory, and a buffer that changes "
                               "may have one name only: keep a cache that several modules use in one "
                               "of them and hand it to the others' calls") from e


def capture(model: torch.nn.Module, example_inputs: tuple, *, name: str | None = None,
            extra_decompositions: Sequence[str] = FORCE_DECOMPOSE) -> Graph:
    """The graph of ``model`` at the shapes (and dtypes) of ``example_inputs``."""
    program = _export(model, tuple(example_inputs), extra_decompositions)
    graph = Graph(name or type(model).__name__)
    call_spec = getattr(program, "call_spec", None)
    graph.meta["in_spec"] = None if call_spec is None else call_spec.in_spec
    graph.meta["out_spec"] = getattr(program, "_out_spec", None)
    _Translation(graph, program).run()
    graph.topo_check()
    return graph


# --------------------------------------------------------------------------
# stage 2: translation
# --------------------------------------------------------------------------

def _static_type(fx: torch.fx.Node) -> tuple[tuple[int, ...], torch.dtype]:
    fake = fx.meta.get("val")
    if fake is None or not hasattr(fake, "shape"):
        raise CaptureError(f"the exporter recorded no tensor type for {fx.name}")
    return _type_of(fake, fx.name)


def _type_of(fake, where: str) -> tuple[tuple[int, ...], torch.dtype]:
    if any(isinstance(d, torch.SymInt) for d in fake.shape):
        raise CaptureError(f"{where} has a symbolic shape {tuple(fake.shape)}; "
                           "only static shapes compile")
    return tuple(int(d) for d in fake.shape), fake.dtype


def _result_names(base: str, count: int) -> list[str]:
    return [base] if count == 1 else [f"{base}_{i}" for i in range(count)]


def _unit_scalings(args: list, kwargs: dict) -> bool:
    """``addmm`` with ``beta == alpha == 1`` (every ``nn.Linear``)."""
    beta = kwargs["beta"] if "beta" in kwargs else (args[3] if len(args) > 3 else 1)
    alpha = kwargs["alpha"] if "alpha" in kwargs else (args[4] if len(args) > 4 else 1)
    return beta == 1 and alpha == 1


def _split_pieces(op: str, args: list, kwargs: dict, shape: tuple[int, ...]):
    """``(dim, piece sizes, squeeze)`` of a split-like op over ``shape``."""
    rank = len(shape)
    dim_at = 1 if op == _UNBIND else 2
    dim = kwargs.get("dim", args[dim_at] if len(args) > dim_at else 0) % rank
    extent = shape[dim]
    if op == _UNBIND:
        return dim, [1] * extent, True
    if op == _SPLIT_BY_CHUNK:
        chunk = args[1] if len(args) > 1 else kwargs["split_size"]
        return dim, [min(chunk, extent - lo) for lo in range(0, extent, chunk)], False
    sizes = args[1] if len(args) > 1 else kwargs["split_sizes"]
    return dim, list(sizes), False


class _Translation:
    """One pass over an exported program's FX graph, appending to ``graph``."""

    def __init__(self, graph: Graph, program) -> None:
        self.graph = graph
        self.program = program
        #: FX node -> the value (or list of values) it became
        self.bound: dict[torch.fx.Node, Value | list[Value]] = {}
        #: lifted tensors by state-dict key; parameters and buffers win over
        #: constants of the same key
        self.lifted = {**dict(getattr(program, "constants", None) or {}),
                       **dict(program.state_dict)}
        self.routes: dict[str, Callable] = {
            "split": self._split,
            "addmm": self._addmm,
            "view": self._view,
            "opaque": self._opaque,
            "typed": self._typed,
        }

    # -- the walk ---------------------------------------------------------------
    def run(self) -> None:
        fx_graph = self.program.graph_module.graph
        signature = self.program.graph_signature
        placeholders = [n for n in fx_graph.nodes if n.op == "placeholder"]
        if len(placeholders) != len(signature.input_specs):
            raise CaptureError(f"{len(placeholders)} placeholders but "
                               f"{len(signature.input_specs)} input specs in the export")
        spec_of = dict(zip(placeholders, signature.input_specs))
        for fx in fx_graph.nodes:
            if fx.op == "placeholder":
                self._placeholder(fx, spec_of[fx])
            elif fx.op == "call_function":
                self._call(fx)
            elif fx.op == "output":
                self._outputs(fx, list(signature.output_specs))
            elif fx.op == "get_attr":
                raise CaptureError(f"the export kept a module attribute ({fx.target}) "
                                   "instead of lifting it to an input")
            else:
                raise CaptureError(f"FX node {fx.name} of kind {fx.op!r} cannot be captured")

    # -- operands ---------------------------------------------------------------
    def _operand(self, a: Any):
        """An FX argument with every node replaced by its value."""
        if isinstance(a, torch.fx.Node):
            bound = self.bound[a]
            if isinstance(bound, list):
                raise CaptureError(f"{a.name} has several results and is read without "
                                   "selecting one")
            return bound
        if isinstance(a, (list, tuple)):
            return type(a)(self._operand(x) for x in a)
        if isinstance(a, torch.SymInt):
            raise CaptureError(f"symbolic integer argument {a}; only static shapes compile")
        return a

    # -- emission helpers ---------------------------------------------------------
    def _fresh(self, name: str, shape, dtype) -> Value:
        """A value over a new contiguous intermediate buffer."""
        shape = tuple(shape)
        return Value(name, Buffer(name, shape, dtype, "intermediate"), Layout.contiguous(shape))

    def _emit(self, op: str, args, kwargs: dict, outputs: list[Value], **meta) -> Node:
        node = Node(op, tuple(args), kwargs, outputs=outputs)
        node.meta.update(meta)
        self.graph.add_node(node)
        return node

    @staticmethod
    def _single_or_list(outputs: list[Value]):
        return outputs[0] if len(outputs) == 1 else outputs

    # -- placeholders -------------------------------------------------------------
    def _placeholder(self, fx: torch.fx.Node, spec) -> None:
        from torch.export.graph_signature import InputKind

        shape, dtype = _static_type(fx)
        from_caller = spec.kind == InputKind.USER_INPUT
        buffer = Buffer(fx.name, shape, dtype, "input" if from_caller else "param")
        value = Value(fx.name, buffer, Layout.contiguous(shape))
        if from_caller:
            self.graph.inputs.append(value)
        else:
            tensor = self.lifted.get(spec.target)
            if tensor is None:
                raise CaptureError(f"the export lifted {spec.target!r} into an input but "
                                   "holds no tensor for it")
            self.graph.params.append(value)
            self.graph.param_tensors[value.name] = tensor.detach()
            self.graph.param_origin[value.name] = spec.target
        self.bound[fx] = value

    # -- call_function --------------------------------------------------------------
    def _call(self, fx: torch.fx.Node) -> None:
        if fx.target is operator.getitem:
            source, which = fx.args
            self.bound[fx] = self.bound[source][which]
            return
        op = str(fx.target)
        if op in DROP_OPS:
            return
        if op == _IN_PLACE:
            self.bound[fx] = self._in_place(fx)
            return
        args = [self._operand(a) for a in fx.args]
        kwargs = {key: self._operand(v) for key, v in fx.kwargs.items()}
        self.bound[fx] = self.routes[self._route(op, args, kwargs)](fx, op, args, kwargs)

    @staticmethod
    def _route(op: str, args: list, kwargs: dict) -> str:
        if op in (_UNBIND, _SPLIT_BY_CHUNK, _SPLIT_BY_SIZES):
            return "split"
        if op == _ADDMM and _unit_scalings(args, kwargs):
            return "addmm"
        kind = op_class(op)
        if kind is OpClass.VIEW:
            return "view"
        if kind is OpClass.OPAQUE:
            return "opaque"
        return "typed"

    def _typed(self, fx, op, args, kwargs):
        """An op with a rule: result types from the shape rules (the
        exporter's are kept in ``export_val`` to check them against)."""
        types = shapes.infer(op, args, kwargs)
        outputs = [self._fresh(nm, shape, dtype)
                   for nm, (shape, dtype) in zip(_result_names(fx.name, len(types)), types)]
        self._emit(op, args, kwargs, outputs, export_val=fx.meta.get("val"), target=fx.target)
        return self._single_or_list(outputs)

    def _opaque(self, fx, op, args, kwargs):
        """An op with no rule: it runs as one torch call, a fusion barrier,
        with result types taken from the exporter."""
        if op.startswith("mlc."):
            args = self._rows_together(fx.target, args)
        recorded = fx.meta.get("val")
        results = list(recorded) if isinstance(recorded, (list, tuple)) else [recorded]
        outputs = []
        for nm, fake in zip(_result_names(fx.name, len(results)), results):
            if fake is None or not hasattr(fake, "shape"):
                raise CaptureError(f"{op} (no lowering rule) returns something other than a "
                                   "tensor, which a compiled graph cannot hold")
            outputs.append(self._fresh(nm, *_type_of(fake, fx.name)))
        self._emit(op, args, kwargs, outputs, export_val=recorded, target=fx.target,
                   types_from_export=True, opaque=True)
        return self._single_or_list(outputs)

    def _rows_together(self, target, args: list) -> list:
        """Operands of an operator of ``mlc.ops`` with the rows of heads in one piece and a
        cache whole, as its checks found the exporter's tensors: a value here may lie
        otherwise in its buffer (results are contiguous, whatever torch makes them)."""
        out = []
        for a, v in zip(target._schema.arguments, args):
            if isinstance(v, Value) and v.numel:
                cache = a.name.endswith(("_cache", "_scale"))
                if cache and v.layout.strides != Layout.contiguous(v.shape).strides:
                    raise CaptureError(f"{target}: {a.name} is a view of a buffer that lies otherwise: "
                                       "give the buffer itself")
                if not cache and v.rank == 4 and v.shape[3] > 1 and v.layout.strides[3] != 1:
                    v = self._contiguous_copy(v)
            out.append(v)
        return out

    def _in_place(self, fx) -> list:
        """An operator of ``mlc.ops`` that changes its operands: they have to be
        buffers of the module, whole, and the compiled schedule changes those.
        Its results are values over the same buffers, which later readers of
        them read, so that they run after it."""
        target = fx.args[0]
        if target.namespace != "mlc":
            raise CaptureError(f"{target} changes its operands: only side-effect-free inference "
                               "graphs and the operators of mlc.ops compile")
        bases = [self._operand(x) for x in fx.kwargs["_all_bases"]]
        args, changed = [], []
        for a in target._schema.arguments:
            if a.alias_info is None or not a.alias_info.is_write:
                args.append(self._operand(fx.kwargs[a.name]))
                continue
            base: Value = bases[fx.kwargs[f"_{a.name}_base_index"]]
            window = [n for n in fx.kwargs if n.startswith(f"_{a.name}_")
                      and n != f"_{a.name}_base_index"]
            if window or base.buffer.kind != "param" or base.layout != Layout.contiguous(base.buffer.shape):
                raise CaptureError(f"{target}: {a.name} is changed in place, so it has to be a "
                                   "whole buffer of the module (register_buffer)")
            if any(base is v for v in changed):
                raise CaptureError(f"{target}: one buffer is given for two operands that change")
            args.append(base)
            changed.append(base)
        args = self._rows_together(target, args)
        outputs = {id(v): Value(f"{fx.name}_{i}", v.buffer, v.layout) for i, v in enumerate(changed)}
        self._emit(str(target), args, {}, list(outputs.values()), target=target,
                   types_from_export=True, opaque=True, pin=True)
        return [None] * max(1, len(target._schema.returns)) + [outputs.get(id(v), v) for v in bases]

    def _check_changes(self) -> None:
        """A buffer's old contents cannot be read beside the new ones: nothing
        orders such a reader before the change. So what a pass reads of a buffer
        it reads after its last change."""
        readers: dict[int, list[Node]] = self.graph.use_map()
        windows: dict[int, list[Value]] = {}
        for node in self.graph.nodes:
            if node.meta.get("is_view"):
                windows.setdefault(id(node.args[0]), []).append(node.out)
        for node in self.graph.nodes:
            if not node.meta.get("pin"):
                continue
            changed = {id(v.buffer) for v in node.outputs}
            for v in node.unique_tensor_args():
                if id(v.buffer) not in changed:
                    continue
                seen = [v]
                while seen:
                    at = seen.pop()
                    seen += windows.get(id(at), [])
                    others = [n for n in readers.get(id(at), []) if n is not node]
                    returned = any(at is o for o in self.graph.outputs)
                    if not others and not returned:
                        continue
                    by = others[0].op if others else "the module's result"
                    if v.producer is not None and v.producer.meta.get("pin"):
                        raise CaptureError(f"{v.name} is changed once more after {by} read it: {node.op} "
                                           "may change a buffer again only where nothing has read it "
                                           "in between. Compile one step and call it twice")
                    raise CaptureError(f"{v.name} is read by another operator beside {node.op}, which "
                                       f"changes it ({by}): read it after the change")

    def _view(self, fx, op, args, kwargs) -> Value:
        """A restride of the source's buffer. When the requested view needs
        data movement (a reshape across a permuted layout), the source is
        first copied into a contiguous buffer and the view restrides that."""
        try:
            layout = shapes.infer_view(op, args, kwargs)
        except NonViewable:
            args = [self._contiguous_copy(args[0]), *args[1:]]
            layout = shapes.infer_view(op, args, kwargs)
        source: Value = args[0]
        if layout.max_offset() > source.buffer.numel:
            raise CaptureError(f"{op} would address {layout} past the end of {source.buffer}")
        out = Value(fx.name, source.buffer, layout)
        self._emit(op, args, kwargs, [out], export_val=fx.meta.get("val"),
                   target=fx.target, is_view=True)
        return out

    def _contiguous_copy(self, source: Value) -> Value:
        out = self._fresh(self.graph.fresh_name("copy"), source.shape, source.dtype)
        self._emit("mlc.copy", (source,), {}, [out], target=None)
        return out

    def _addmm(self, fx, op, args, kwargs) -> Value:
        """``addmm(bias, a, b)`` as ``mm(a, b)`` (an extern GEMM in the
        operands' own dtype) followed by a pointwise ``add`` of the bias,
        which fuses into whatever consumes it."""
        bias, lhs, rhs = args[:3]
        mm_shape, mm_dtype = shapes.infer_matmul("aten.mm.default", [lhs, rhs], {})
        product = self._fresh(f"{fx.name}_mm", mm_shape, mm_dtype)
        self._emit("aten.mm.default", (lhs, rhs), {}, [product], target=torch.ops.aten.mm.default)
        sum_shape, sum_dtype = shapes.infer_pointwise("aten.add.Tensor", [product, bias], {})
        out = self._fresh(fx.name, sum_shape, sum_dtype)
        self._emit("aten.add.Tensor", (product, bias), {}, [out], export_val=fx.meta.get("val"),
                   target=torch.ops.aten.add.Tensor)
        return out

    def _split(self, fx, op, args, kwargs) -> list[Value]:
        """Each piece of a split (or unbind) is a slice view of the source's
        buffer; an unbind piece also drops the split dimension."""
        source: Value = args[0]
        dim, sizes, squeeze = _split_pieces(op, args, kwargs, source.shape)
        pieces: list[Value] = []
        lo = 0
        for i, size in enumerate(sizes):
            hi = lo + size
            layout = source.layout.slice(dim, lo, hi)
            piece = Value(f"{fx.name}_{i}", source.buffer,
                          layout.squeeze([dim]) if squeeze else layout)
            self._emit("aten.slice.Tensor", (source, dim, lo, hi, 1), {}, [piece],
                       is_view=True, from_split=True)
            pieces.append(piece)
            lo = hi
        return pieces

    # -- output -------------------------------------------------------------------
    def _outputs(self, fx: torch.fx.Node, specs: list) -> None:
        from torch.export.graph_signature import OutputKind

        results = fx.args[0]
        results = list(results) if isinstance(results, (list, tuple)) else [results]
        for position, result in enumerate(results):
            kind = specs[position].kind if position < len(specs) else OutputKind.USER_OUTPUT
            if kind == OutputKind.BUFFER_MUTATION and self._operand(result).buffer.kind == "param" \
                    and self._operand(result).producer.meta.get("pin"):
                continue  # changed where it is
            if kind != OutputKind.USER_OUTPUT:
                raise CaptureError(f"result {position} of the export is a {kind}, not a user "
                                   "output: only side-effect-free inference graphs compile")
            if result is None:
                raise CaptureError(f"result {position} is None; every result must be a tensor")
            value = self._operand(result)
            self.graph.outputs.append(value)
            if value.buffer.kind == "intermediate":
                value.buffer.kind = "output"
        self._check_changes()
