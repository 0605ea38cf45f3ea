"""Calls of ``mlc.ops`` that something else looks on or that hand it memory in unusual
ways: tracing, modes, gradients of both directions, overlapping and lazily copied
operands, many sequences of uneven lengths."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mlc
import operators_reference as ref
from mlc import ops
from test_operators import BF, E4M3, FULL, HALF, _heads, _refused, filled, gpu, host, ints, normal, parts


# --------------------------------------------------------------------------
# what looks on
# --------------------------------------------------------------------------

@gpu
def test_a_traced_call_is_the_operator():
    """torch.jit's tracer sees the operator and not the allocation of its result."""
    q, k, v = _heads(1, 5, 70, 2, 1, 64, HALF)
    cache, start = filled(1, 1, 128, 64), ints([70])

    def f(q, k, v):
        cache.append(k[:, :5], v[:, :5], start)
        return ops.attention(q, k, v, causal=True), cache.attend(q, start)

    traced = torch.jit.trace(f, (q, k, v), check_trace=False)
    kinds = [n.kind() for n in traced.graph.nodes()]
    for name in ("cache_append", "attention", "cache_attention"):
        assert f"mlc::{name}" in kinds, kinds
    q, k, v = _heads(1, 5, 70, 2, 1, 64, HALF, seed=20)
    got = traced(q, k, v)
    ref.close(got[0], *ref.attention(q, k, v, causal=True))
    ref.close(got[1], *ref.cache_attention(q, *parts(cache), start))


@gpu
def test_function_modes_see_the_operator():
    from torch.overrides import TorchFunctionMode

    class Log(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    seen = []
    q, k, v = _heads(1, 5, 70, 2, 1, 64, HALF)
    want = ops.attention(q, k, v)
    with Log():
        assert torch.equal(ops.attention(q, k, v), want)
    assert any("mlc.attention" in x for x in seen), seen
    with torch.device("cuda"):  # a mode too, for factories only
        assert torch.equal(ops.attention(q, k, v), want)
    traced = torch.jit.trace(lambda q: ops.attention(q, k, v), (q,), check_trace=False)
    with Log():  # the traced operator, called below Python's modes
        assert torch.equal(traced(q), want)


@gpu
def test_functions_that_torch_compiles_or_records_call_the_operators():
    from torch.fx.experimental.proxy_tensor import make_fx

    a, b = filled(1, 2, 128, 64), filled(1, 2, 128, 64)
    f, _ = ops.rotary_frequencies(64, device="cuda")
    q, k, start = normal(1, 1, 4, 64), normal(1, 1, 2, 64, seed=1), ints([5])

    def step(cache, q, k, start):
        q, k = ops.rotary(q, k, start, f)
        cache.append(k, k, start)
        return cache.attend(q, start) * 2.0, ops.attention(q, k, k)

    with torch.no_grad():
        compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
        for i in range(2):
            for x, y in zip(compiled(a, q, k, start + i), step(b, q, k, start + i)):
                assert torch.equal(x, y)
            for x, y in zip(parts(a), parts(b)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for pre in (False, True):
        recorded = make_fx(lambda q, k: ops.attention(q, k, k), pre_dispatch=pre)(q, k)
        assert "mlc.attention.default" in [str(n.target) for n in recorded.graph.nodes]
        assert torch.equal(recorded(q, k), ops.attention(q, k, k))


@gpu
def test_the_profiler_records_each_call_once():
    from torch.profiler import ProfilerActivity, profile

    q, k, v = _heads(1, 5, 70, 2, 1, 64, HALF)
    ops.attention(q, k, v)
    with profile(activities=[ProfilerActivity.CPU], record_shapes=True) as p:
        ops.attention(q, k, v)
        torch.ops.mlc.attention(q, k, v, None, False, 0.0, None, None, None)
    found = [e for e in p.events() if e.name == "mlc::attention"]
    assert len(found) == 2, [e.name for e in p.events()]
    assert found[0].input_shapes[:3] == [list(q.shape), list(k.shape), list(v.shape)]

# --------------------------------------------------------------------------
# gradients
# --------------------------------------------------------------------------

def test_operands_with_a_forward_gradient_are_refused():
    import torch.autograd.forward_ad as forward

    q = host(1, 1, 2, 64)
    with forward.dual_level():
        dual = forward.make_dual(q, torch.ones_like(q))
        with torch.no_grad():  # forward mode goes on there
            _refused(lambda: ops.attention(dual, q, q), "gradient")
        _refused(lambda: ops.attention(q, q, dual), "gradient")
        with torch.inference_mode():  # and not there
            _refused(lambda: ops.attention(dual, q, q), "ROCm GPU")
    _refused(lambda: ops.attention(q, q, q), "ROCm GPU")


def _dispatched(q, start, parts):
    """A call of each operator through torch's dispatcher, by its name."""
    f = torch.ones(32, dtype=torch.float64, device=q.device)
    o = torch.ops.mlc
    return {"rotary": lambda: o.rotary(q, q, start, f, False, 1.0),
            "attention": lambda: o.attention(q, q, q, None, False, 0.0, None, None, None),
            "cache_append": lambda: o.cache_append(*parts, q, q, start, None),
            "cache_attention": lambda: o.cache_attention(q, *parts, start, None, None, 0.0, None)}


@pytest.mark.parametrize("op", ("rotary", "attention", "cache_append", "cache_attention"))
def test_the_dispatcher_refuses_operands_that_ask_for_gradients(op):
    import torch.autograd.forward_ad as forward
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        cache = ops.KeyValueCache(1, 2, 64, 64, device="cuda")
        q = torch.zeros(1, 1, 2, 64, dtype=HALF, device="cuda", requires_grad=True)
        start = torch.zeros(1, dtype=torch.int32, device="cuda")
        _refused(_dispatched(q, start, parts(cache))[op], "gradient")
        with torch.no_grad():
            _dispatched(q, start, parts(cache))[op]()
        _dispatched(q.detach(), start, parts(cache))[op]()
    q, start, cache = host(1, 1, 2, 64), torch.zeros(1, dtype=torch.int32), ops.KeyValueCache(1, 2, 64, 64)
    with forward.dual_level():
        dual = forward.make_dual(q, torch.ones_like(q))
        with torch.no_grad():
            _refused(_dispatched(dual, start, parts(cache))[op], "gradient")
    _refused(_dispatched(q, start, parts(cache))[op], "ROCm GPU")


def test_a_compiled_function_refuses_operands_that_ask_for_gradients():
    w = torch.zeros(64, 64, dtype=HALF, requires_grad=True)
    x = host(1, 3, 2, 64)
    seen = []

    def f(x):
        return ops.attention(x @ w, x, x)

    def backend(gm, example):
        seen.append([str(n.target) for n in gm.graph.nodes])
        return gm.forward

    with pytest.raises(Exception, match="gradient"):
        torch.compile(f, backend=backend, fullgraph=True)(x)
    with torch.no_grad(), pytest.raises(Exception, match="ROCm GPU"):
        torch.compile(f, backend=backend, fullgraph=True)(x)
    assert any("mlc.attention" in n for n in seen[-1])


def test_transforms_that_differentiate_are_refused():
    q, t = host(1, 3, 2, 64), torch.ones(1, 3, 2, 64, dtype=HALF)
    _refused(lambda: torch.func.grad(lambda x: ops.attention(x, q, q).sum())(q), "gradient")
    _refused(lambda: torch.func.jvp(lambda x: ops.attention(x, q, q), (q,), (t,)), "gradient")


def test_a_module_whose_weights_ask_for_gradients_is_exported():
    """The program is a graph; who asks it for a gradient is refused then."""

    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.proj = torch.nn.Linear(64, 64).half()

        def forward(self, x):
            y = self.proj(x)
            return ops.attention(y, y, y)

    program = torch.export.export(M().eval(), (host(1, 3, 2, 64),))
    assert any("mlc.attention" in str(n.target) for n in program.graph.nodes)

# --------------------------------------------------------------------------
# memory
# --------------------------------------------------------------------------

def _pool():
    codes = torch.zeros(3, 2, 64, 64, dtype=torch.uint8, device="cuda").view(E4M3)
    return codes, torch.ones(3, 2, 4, device="cuda")


@gpu
def test_operands_that_lie_in_a_cache_that_changes_are_refused():
    """In part, too: two caches or scales cut out of one pool, scales inside of keys."""
    codes, scales = _pool()
    apart, ones = torch.zeros_like(codes), torch.ones_like(scales)
    scales, ones = scales[..., :2].contiguous(), ones[..., :2].contiguous()
    k, start = normal(2, 1, 2, 64), ints([0, 0])
    one = (codes[:2], apart[:2], scales[:2], ones[:2])
    inside = codes[1:].view(torch.uint8).flatten()[:2 * 2 * 2 * 4].view(FULL).view(2, 2, 2)
    inside.fill_(1.0)
    for bad in ((codes[:2], codes[1:], scales[:2], ones[:2]), (*one[:2], scales[:2], scales[1:]),
                (codes[:2], apart[:2], inside, ones[:2])):
        _refused(lambda: ops.cache_append(*bad, k, k, start), "share")
    rows = codes[:2].view(torch.uint8).flatten()[:2 * 2 * 64 * 2].view(HALF).view(2, 1, 2, 64)
    _refused(lambda: ops.cache_append(*one, rows, k, start), "share")
    _refused(lambda: ops.cache_append(*one, k, k, scales.flatten()[:2].view(torch.int32)), "share")
    ops.cache_append(codes[:1], codes[1:2], scales[:1], scales[1:2], k[:1], k[:1], start[:1])  # side by side
    ops.check_errors()


@gpu
def test_autograd_sees_that_a_cache_changed():
    cache = filled(1, 1, 64, 64)
    k, start = normal(1, 1, 1, 64), ints([3])
    before = [x._version for x in parts(cache)]
    cache.append(k, k, start)
    assert all(x._version > b for x, b in zip(parts(cache), before))
    w = torch.ones_like(cache.key_scales, requires_grad=True)
    y = (w * cache.key_scales).sum()  # keeps the scales for its backward
    cache.append(k, k, start)
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    before = [x._version for x in parts(cache)]
    cache.attend(normal(1, 1, 2, 64), start)
    assert [x._version for x in parts(cache)] == before
    with torch.inference_mode():  # which counts no versions
        other = filled(1, 1, 64, 64)
        other.append(k, k, start)
    other.append(k, k, start)


class _Step(torch.nn.Module):
    def __init__(self, cache):
        super().__init__()
        self.cache = cache

    def forward(self, k, start):
        self.cache.append(k, k, start)
        return self.cache.attend(k, start)


@gpu
@pytest.mark.parametrize("config", [{}, {"memory_planning": False}, {"cuda_graphs": False}],
                         ids=("graph", "unplanned", "planned"))
def test_autograd_sees_that_a_compiled_model_changed_its_cache(config):
    m = _Step(filled(1, 2, 64, 64))
    args = normal(1, 1, 2, 64), ints([3])
    compiled = mlc.compile(m, args, mlc.Config(**config))
    for _ in range(2):
        before = [x._version for x in parts(m.cache)]
        compiled(*args)
        assert all(x._version > b for x, b in zip(parts(m.cache), before))


@gpu
@pytest.mark.parametrize("name", ("keys", "value_scales"))
def test_a_compiled_model_refuses_a_cache_off_16_bytes(name):
    cache = filled(1, 2, 128, 64)
    x = cache._buffers[name]
    raw = torch.zeros(x.numel() * x.element_size() + 16, dtype=torch.uint8, device="cuda")
    at = raw[4:4 + x.numel() * x.element_size()].view(x.dtype if x.dtype == E4M3 else FULL).view(x.shape)
    at.copy_(x)
    cache._buffers[name] = at
    args = normal(1, 1, 2, 64), ints([0])
    _refused(lambda: cache.append(args[0], args[0], args[1]), "16 bytes")
    with pytest.raises(ops.OperatorError, match="16 bytes"):
        mlc.compile(_Step(cache), args)(*args)


@gpu
def test_a_lazy_copy_of_a_cache_is_changed_and_its_source_is_not():
    cache = filled(1, 2, 128, 64)
    copy = [torch._lazy_clone(x) for x in parts(cache)]
    kept = [x.clone().view(torch.uint8) for x in parts(cache)]
    k, start = normal(1, 3, 2, 64, spread=50.0), ints([62])
    wants = [ref.cache_append(c, s, k, start) for c, s in ((cache.keys, cache.key_scales),
                                                           (cache.values, cache.value_scales))]
    ops.cache_append(*copy, k, k, start)
    for (codes, scales), c, s in zip(wants, copy[:2], copy[2:]):
        assert torch.equal(c.view(torch.uint8).cpu(), torch.from_numpy(codes))
        assert torch.equal(s.double().cpu(), torch.from_numpy(scales))
    for x, y in zip(parts(cache), kept):
        assert torch.equal(x.view(torch.uint8), y)


@gpu
def test_an_input_that_lies_in_a_cache_that_changes_is_read_as_it_was():
    """By a compiled model whose inputs are read in place."""

    class M(_Step):
        def forward(self, k, start, x):
            y = super().forward(k, start)
            return y, x * 2.0 + y[..., :2].reshape(1, 2, 2).float() * 0.0  # behind the change

    m = M(filled(1, 2, 128, 64))
    k, start = normal(1, 1, 2, 64), ints([0])
    for config in ({}, {"memory_planning": False, "cuda_graphs": False}, {"cuda_graphs": False}):
        compiled = mlc.compile(m, (k, start, m.cache.key_scales.clone()), mlc.Config(**config))
        for i in range(2):
            m.cache.key_scales.fill_(2.0 ** (20 + i))  # the append starts it anew
            want = m.cache.key_scales * 2.0
            assert torch.equal(compiled(k, start, m.cache.key_scales)[1], want)

# --------------------------------------------------------------------------
# over the cache
# --------------------------------------------------------------------------

def _items(lengths, kv_heads, capacity, dim=64, block=64):
    """How the kernel cuts sequences of these lengths, ``[first item, items]`` of each, from the
    memory that its launches share."""
    from mlc.codegen import hip_operators as plans
    from mlc.runtime import native, operators

    batch = len(lengths)
    cache = ops.KeyValueCache(batch, kv_heads, capacity, dim, block=block, device="cuda")
    q, start = normal(batch, 1, kv_heads, dim), ints([n - 1 for n in lengths])
    operands = {"q": q, **dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), parts(cache))), "start": start}
    plan = plans.plan_cache_attention(*map(ops._operand, operands.values()), None, None, 0.125, 0.0)
    modules, launch, out = operators.device_modules(0), plan.launches[0], torch.empty_like(q)
    space = torch.zeros(plan.workspace, dtype=torch.uint8, device="cuda")
    at = {n: x.data_ptr() for n, x in operands.items()}
    at.update(out0=out.data_ptr(), workspace=space.data_ptr(), error=modules.error_word())
    args = launch.arguments(at)
    native.check(modules.lib.mlc_launch(modules.function(launch), launch.grid, launch.block, 0, args, len(args),
                                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    return space.view(torch.int32)[:2 * batch].view(batch, 2).tolist(), launch.grid // kv_heads


@gpu
@pytest.mark.parametrize("lengths", [
    [819 + 117 * i for i in range(64)],          # as many sequences as items are wanted
    [65536] + [200] * 255,                       # one that is long among many
    [1] * 69 + [32768],
    [8192] * 3 + [64] * 5,
], ids=("even", "one", "tokens", "few"))
def test_the_cache_is_cut_into_even_items_however_many_sequences(lengths):
    """None is longer than two even shares, rounded up to whole steps of 64 keys."""
    found, slots = _items(lengths, 8, max(lengths) + 63 & ~63)
    at = 0
    for first, n in found:  # one behind the other, and within the launch
        assert first == at and n >= 1
        at += n
    assert at <= slots
    even = max(sum(lengths) / 64, 512)
    assert max(-(-n // of) for n, (_, of) in zip(lengths, found)) <= 2 * (even + 64)


@gpu
def test_cache_attention_of_many_sequences_of_uneven_lengths():
    lengths = [1 + 37 * i for i in range(65)] + [1, 64, 65, 8192, 8191]
    cache = filled(len(lengths), 8, 8192, 64)
    q, start = normal(len(lengths), 1, 8, 64, dtype=BF), ints([n - 1 for n in lengths])
    got = cache.attend(q, start)
    some = [0, 30, 63, 64, 65, 66, 67, 68, 69]
    held = [x[some] for x in (x.view(torch.uint8) for x in parts(cache))]
    held = [x.view(y.dtype) for x, y in zip(held, parts(cache))]
    ref.close(got[some], *ref.cache_attention(q[some], *held, start[some]))


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
@pytest.mark.parametrize("options", ({}, {"scale": 2.0 ** -60}, {"cap": 5.0}), ids=("", "scale", "cap"))
def test_blocks_of_zero_scale_behind_a_row_and_under_it(way, options):
    """A mask's -infinity is not multiplied by a factor of zero: a scale of zero, or one of
    2^-126 (of a block of zeros) times a small ``scale``."""
    cache = filled(2, 1, 256, 64)
    cache.key_scales[0, 0, 1:3] = torch.tensor([0.0, 2.0 ** -126])
    cache.key_scales[1, 0] = 2.0 ** -126
    q, start = normal(2, 70, 2, 64, dtype=BF), ints([90, 186])
    got = cache.attend(q, start, **options)
    assert got.isfinite().all()
    ref.close(got, *ref.cache_attention(q, *parts(cache), start, **options))

# --------------------------------------------------------------------------
# in compiled models
# --------------------------------------------------------------------------

@gpu
def test_many_layers_over_caches_of_their_own_are_the_direct_calls_to_the_bit():
    """Every attention over a cache is used, so all of them are in the graph, replayed
    between other work."""

    class Layers(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.caches = torch.nn.ModuleList(filled(2, 2, 2048, 64, seed=i) for i in range(12))
            f, _ = ops.rotary_frequencies(64, device="cuda")
            self.register_buffer("f", f)

        def forward(self, q, k, start):
            for cache in self.caches:
                q, b = ops.rotary(q, k, start.unsqueeze(1), self.f)
                cache.append(b, k, start)
                q = cache.attend(q, start)
            return q

    m, other = Layers(), Layers()
    q, k = normal(2, 1, 4, 64, dtype=BF), normal(2, 1, 2, 64, dtype=BF, seed=1)
    compiled = mlc.compile(m, (q, k, ints([0, 0])))
    assert sum("mlc.cache_attention" in x.summary() for x in compiled.schedule) == 12
    for i, at in enumerate(([5, 1999], [6, 2000], [2047, 0])):
        got = compiled(q * (1 + i), k, ints(at)).clone()
        assert torch.equal(got, other(q * (1 + i), k, ints(at)))
        for a, b in zip(m.caches, other.caches):
            for x, y in zip(parts(a), parts(b)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    compiled.check_errors()


@gpu
def test_many_appends_of_one_pass_round_as_direct_calls():
    """Token by token into one block, each larger than those before, so that the scale grows and
    codes are rounded again and again: a first call that makes a graph runs once for its caller."""

    class Appends(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = filled(2, 2, 64, 64)

        def forward(self, k, start):
            for i in range(k.shape[1]):
                self.cache.append(k[:, i:i + 1], k[:, i:i + 1], start + i)
            return self.cache.attend(k[:, :1], start)

    m, other = Appends(), Appends()
    k = normal(2, 20, 2, 64, spread=2.0 ** -5) * torch.arange(20, device="cuda").exp2()[:, None, None].sqrt()
    k = (k * normal(2, 20, 2, 64, dtype=FULL, seed=3, spread=5.0).exp2()).half()
    compiled = mlc.compile(m, (k, ints([1, 7])))
    for start in ([1, 7], [21, 30]):
        compiled(k, ints(start))
        other(k, ints(start))
        for x, y in zip(parts(m.cache), parts(other.cache)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_a_cache_changed_again_after_it_was_read_is_refused_by_its_reason():
    from mlc.ir.capture import CaptureError, capture

    class Twice(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.cache = ops.KeyValueCache(2, 2, 128, 64)

        def forward(self, k, start):
            self.cache.append(k, k, start)
            a = self.cache.attend(k, start)
            self.cache.append(a, a, start + 1)
            return self.cache.attend(a, start + 1)

    with pytest.raises(CaptureError, match="changed once more after mlc.cache_attention.default read it"):
        capture(Twice(), (host(2, 1, 2, 64), torch.zeros(2, dtype=torch.int32)))


def test_a_cache_under_several_names_is_refused_by_its_reason():
    from mlc.ir.capture import CaptureError, capture

    class Layer(torch.nn.Module):
        def __init__(self, cache, fills):
            super().__init__()
            self.cache, self.fills = cache, fills

        def forward(self, k, start):
            if self.fills:
                self.cache.append(k, k, start)
            return self.cache.attend(k, start)

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            cache = ops.KeyValueCache(2, 2, 128, 64)
            self.one, self.two = Layer(cache, True), Layer(cache, False)

        def forward(self, k, start):
            return self.two(self.one(k, start), start)

    with pytest.raises(CaptureError, match="one.cache.keys and two.cache.keys share memory"):
        capture(Model(), (host(2, 1, 2, 64), torch.zeros(2, dtype=torch.int32)))
