"""Direct calls of the operators of ``mlc.ops``: their code objects, loaded once a
device, and the table of their launches.

A call's plan follows from shapes, strides, types and options alone, so it is kept
under them; ``_calls.call`` (``csrc/mlc_calls.cpp``) puts addresses in at every call and
launches on torch's current stream. Memory that a call's launches share is allocated
for that call through torch, on its stream: calls on several streams and calls captured
into several graphs have memory of their own.
"""

from __future__ import annotations

import ctypes

import torch

from ..codegen import hip_operators
from ..codegen.hip_operators import Launch, Plan
from . import native

#: what a kernel leaves in the invalid-input word, and the message for it
INVALID = {1: ("an embedding id was outside its table (torch raises IndexError for such an "
               "id); the rows it addressed were written as zeros"),
           2: ("start and count of a sequence lay outside its cache, or count above the new "
               "tokens: nothing was written for it, and its attention is zeros"),
           3: ("a row of sample had NaN or +infinity among its logits, or a random number or an option "
               "outside its range: its token is -1")}


class OperatorModules:
    """The operators' kernels on one device, in a context of the runtime library."""

    def __init__(self, index: int, ctx=None) -> None:
        self.lib = native.load_library()
        self.index = index
        self._ctx = ctx
        if ctx is None:
            self._ctx = ctypes.c_void_p()
            native.check(self.lib.mlc_ctx_create(index, ctypes.byref(self._ctx)), "mlc_ctx_create")
        self._modules: list[ctypes.c_void_p] = []
        self._functions: dict[str, int] = {}
        self._error_word: int | None = None

    def function(self, launch: Launch) -> int:
        fn = self._functions.get(launch.symbol)
        return fn if fn is not None else self._load(launch)

    def _load(self, launch: Launch) -> int:
        text = hip_operators.source(launch.file, launch.kernel)
        _, path = native.compile_code_object(text)
        if torch.cuda.is_current_stream_capturing():
            raise native.NativeError(f"{launch.symbol} is not loaded yet, and loading it while a "
                                     "graph is captured is not possible: call it once before")
        image = path.read_bytes()
        buf = ctypes.create_string_buffer(image, len(image))
        mod, fn = ctypes.c_void_p(), ctypes.c_void_p()
        native.check(self.lib.mlc_module_load(self._ctx, buf, len(image), ctypes.byref(mod)),
                     "mlc_module_load")
        self._modules.append(mod)
        native.check(self.lib.mlc_function(mod, launch.symbol.encode(), ctypes.byref(fn)),
                     f"mlc_function({launch.symbol})")
        self._functions[launch.symbol] = fn.value
        return fn.value

    @property
    def context(self) -> int:
        return self._ctx.value

    def error_word(self) -> int:
        if self._error_word is None:
            word = ctypes.c_void_p()
            native.check(self.lib.mlc_error_word(self._ctx, ctypes.byref(word)), "mlc_error_word")
            self._error_word = word.value
        return self._error_word

    def pending(self) -> int:
        """The invalid-input word as completed kernels left it."""
        if self._error_word is None:
            return 0
        value = ctypes.c_int32()
        native.check(self.lib.mlc_error_poll(self._ctx, ctypes.byref(value)), "mlc_error_poll")
        return value.value

    def clear(self) -> None:
        native.check(self.lib.mlc_error_clear(self._ctx), "mlc_error_clear")

    def close(self) -> None:
        for mod in self._modules:
            self.lib.mlc_module_unload(mod)
        self._modules, self._functions = [], {}


_devices: dict[int, OperatorModules] = {}


def device_modules(index: int) -> OperatorModules:
    found = _devices.get(index)
    if found is None:
        with torch.cuda.device(index):
            found = _devices.setdefault(index, OperatorModules(index))
    return found


#: calls kept: with ever new sizes it starts again
MOST_CALLS = 4096


class Calls(dict):
    """Signature (bytes) -> the ``Plan`` of its calls, which ``_calls.call`` launches."""

    def add(self, signature: bytes, plan: Plan, operands: tuple, changed: int, results: int,
            device: int) -> None:
        """``operands``: their names, of which the first ``changed`` change. Functions are
        loaded, arguments laid out but for the addresses: of the operands, the results, the
        shared memory, nothing and the invalid-input word."""
        modules = device_modules(device)
        flags = any("error" in x.pointers for x in plan.launches)
        names = (*operands, *(f"out{i}" for i in range(results)), "workspace", None, "error")
        place = {n: i for i, n in enumerate(names)}
        with torch.cuda.device(device):
            launches = tuple((modules.function(x), x.grid, x.block, bytes(place[p] for p in x.pointers),
                              x.tail) for x in plan.launches)
        address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
        if len(self) >= MOST_CALLS:
            self.clear()
        native.load_calls().add(signature, len(names), changed, address(modules.lib.mlc_launch), launches,
                                plan.workspace, address(modules.lib.mlc_error_poll) if flags else 0,
                                modules.context if flags else 0, modules.error_word() if flags else 0,
                                tuple((dtype, shape) for shape, dtype in plan.results))
        self[signature] = plan

    def clear(self) -> None:
        native.load_calls().clear()
        super().clear()


def raise_pending(modules: OperatorModules) -> None:
    from .executor import ExecutionError

    code = modules.pending()
    modules.clear()
    raise ExecutionError(INVALID.get(code, f"an operator flagged an invalid input ({code})"))


def check_errors() -> None:
    """Wait for every device that operators ran on and raise for an invalid input."""
    from . import hip_runtime

    hip_runtime.close_late()
    for index, modules in list(_devices.items()):
        torch.cuda.synchronize(index)
        if modules.pending():
            raise_pending(modules)
