"""Direct calls of the operators of ``mlc.ops``: their code objects, loaded once a
device, and their launches on torch's current stream of the operands' device.

A call's plan follows from shapes, strides, types and options alone, so it is kept
under them; addresses are put in at every call. Memory that a call's launches share
is allocated for that call through torch, on its stream: calls on several streams
and calls captured into several graphs have memory of their own.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from ..codegen import hip_operators
from ..codegen.hip_operators import Launch, Plan
from . import native

#: what a kernel leaves in the invalid-input word, and the message for it
INVALID = {1: ("an embedding id was outside its table (torch raises IndexError for such an "
               "id); the rows it addressed were written as zeros"),
           2: ("start and count of a sequence lay outside its cache, or count above the new "
               "tokens: nothing was written for it, and its attention is zeros")}


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


class Call:
    """The launches of one signature on one device: functions loaded, arguments laid
    out but for the addresses, which ``run`` gets in the order of the operands and
    results."""

    def __init__(self, plan: Plan, operands: tuple, device: int) -> None:
        self.plan = plan
        self.modules = device_modules(device)
        self.device, self.workspace = device, plan.workspace
        self.flags = any("error" in x.pointers for x in plan.launches)
        error = self.modules.error_word() if self.flags else 0
        # where a launch's pointers are in ``at`` with the workspace and constants behind it
        names = [*operands, *sorted({p for x in plan.launches for p in x.pointers
                                     if p is not None and p.startswith("out")})]
        self.tail = (0, error)
        place = {n: i for i, n in enumerate((*names, "workspace", None, "error"))}
        self.launches = []
        with torch.cuda.device(device):
            for x in plan.launches:
                layout = struct.Struct(f"<{len(x.pointers)}Q{len(x.tail)}s")
                self.launches.append((self.modules.function(x), x.grid, x.block, layout.pack,
                                      tuple(place[p] for p in x.pointers), x.tail, layout.size))
        self._launch = self.modules.lib.mlc_launch

    def run(self, at: list, like) -> None:
        """Launch on torch's current stream of the device. ``like``: a tensor on it."""
        if _current_device() != self.device:
            with torch.cuda.device(self.device):
                return self.run(at, like)
        if self.flags and self.modules.pending() and not torch.cuda.is_current_stream_capturing():
            raise_pending(self.modules)
        space = None
        if self.workspace:
            space = like.new_empty(self.workspace, dtype=torch.uint8)
            at.append(space.data_ptr())
        else:
            at.append(0)
        at += self.tail
        stream = _current_stream(self.device)
        for fn, grid, block, pack, place, tail, size in self.launches:
            rc = self._launch(fn, grid, block, 0, pack(*[at[i] for i in place], tail), size, stream)
            if rc:
                native.check(rc, "mlc_launch")


def raise_pending(modules: OperatorModules) -> None:
    from .executor import ExecutionError

    code = modules.pending()
    modules.clear()
    raise ExecutionError(INVALID.get(code, f"an operator flagged an invalid input ({code})"))


def check_errors() -> None:
    """Wait for every device that operators ran on and raise for an invalid input."""
    for index, modules in list(_devices.items()):
        torch.cuda.synchronize(index)
        if modules.pending():
            raise_pending(modules)


def _current_device() -> int:
    return torch._C._cuda_getDevice()


def _current_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)
