"""The measured operators of 8-bit decoders: what stands around and between their
products, the products themselves, and the choice of the next token.

* ``norm``: root-mean-square norm, with the residual's addition in front of it, in
  the input's type or in 8 bits with a scale for each 128 values of a row
  (``mlc.ops.rms_norm``);
* ``quantize``: a row in that form, as it is or gated (``mlc.ops.quantize``);
* ``product``: rows in that form times a weight in 8 bits with a scale for each
  128 x 128 values (``mlc.ops.scaled_product``);
* ``sample``: one token of each row of logits from a given random number, with
  temperature, top-k, top-p and min-p of its own (``mlc.ops.sample``).

Rows are the last dimension: ``[batch, tokens, width]`` with scales
``[batch, tokens, ceil(width / 128)]``; a weight is ``[outputs, inputs]``.
"""

from __future__ import annotations

import functools
import math
import pathlib
import sys

import torch

#: False: the plain forms; True: the framework's operators
own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
BLOCK = 128
LEAST_SCALE = 2.0 ** -126
EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _ops():
    package = str(pathlib.Path.cwd() / "mlc-compiler_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import mlc

    return mlc.ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _norm(name, batch, tokens, width, dtype, residual=True, quantized=False):
    return {"name": name, "op": "norm", "batch": batch, "tokens": tokens, "width": width,
            "dtype": dtype, "residual": residual, "quantized": quantized}


def _quantize(name, batch, tokens, width, dtype, gated=False):
    return {"name": name, "op": "quantize", "batch": batch, "tokens": tokens, "width": width,
            "dtype": dtype, "gated": gated}


def _product(name, batch, tokens, inputs, outputs, dtype, bias=False):
    return {"name": name, "op": "product", "batch": batch, "tokens": tokens, "inputs": inputs,
            "outputs": outputs, "dtype": dtype, "bias": bias}


def _sample(name, batch, vocabulary, dtype, temperature=True, top_k=0, top_p=0.0, min_p=0.0,
            spread=2.5, padded=False):
    return {"name": name, "op": "sample", "batch": batch, "vocabulary": vocabulary, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "spread": spread, "padded": padded}


def listed():
    return [
        # one new token of one request, width 768: launch latency
        _norm("norm-step-b1", 1, 1, 768, "fp16", residual=False),
        # prompts on their way into the next 8-bit product
        _norm("norm-b4-s2048-8bit", 4, 2048, 4096, "bf16", quantized=True),
        # what attention gives for one new token of each of 32 requests
        _quantize("quantize-step-b32", 32, 1, 4096, "fp16"),
        # between a decoder's two halves of its gated layer, at an odd number of tokens
        _quantize("quantize-b3-s2021-gated", 3, 2021, 12288, "bf16", gated=True),
        # one new token of one request through a merged projection: the weight is all there is
        _product("product-step-b1", 1, 1, 4096, 6144, "bf16"),
        # one new token of each of 32 requests through a gated layer's two halves
        _product("product-step-b32", 32, 1, 4096, 24576, "bf16"),
        # a short prompt at an odd length through a projection of width 768, with a bias, in fp32
        _product("product-b3-s333-bias", 3, 333, 768, 2304, "fp32", bias=True),
        # long prompts back to the model's width: the largest work
        _product("product-b4-s2048", 4, 2048, 12288, 4096, "bf16"),
        # one request, the 50257 tokens of a small decoder, a padded row of them
        _sample("sample-b1-v50257", 1, 50257, "fp32", top_k=50, top_p=0.9, padded=True),
        # requests that go by the distribution's body, rows of an odd number of tokens
        _sample("sample-b32-v50257-min-p", 32, 50257, "fp16", min_p=0.05),
        # a large serving batch over a large vocabulary: all of it counts towards top-p
        _sample("sample-b256-v131072-top-p", 256, 131072, "bf16", top_p=0.9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c) -> float:
    """Seconds, roughly, at rates every path reaches: only to bound a draw."""
    w = work(c)
    extra = 0.0
    if c["op"] == "sample":  # a sorted copy and sums in 64 bits
        extra = 100.0 * c["batch"] * c["vocabulary"]
    elif c["op"] == "product":
        extra = 8.0 * (c["inputs"] * (c["outputs"] + c["batch"] * c["tokens"]))
    return w["flops"] / 1e14 + (4 * w["bytes"] + extra) / 3e12


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("norm", "quantize", "product", "product", "sample", "sample"))
        dtype = rng.choice(("fp16", "bf16", "fp32"))
        batch, tokens = _log_int(rng, 1, 32), rng.choice((1, _log_int(rng, 1, 4096)))
        if op == "norm":
            quantized = rng.random() < 0.5
            width = _log_int(rng, 4, 1024) * 16 if quantized or rng.random() < 0.7 \
                else _log_int(rng, 3, 16384)
            c = _norm("", batch, tokens, width, dtype, rng.random() < 0.7, quantized)
        elif op == "quantize":
            c = _quantize("", batch, tokens, _log_int(rng, 4, 1792) * 16, dtype, rng.random() < 0.5)
        elif op == "product":
            inputs = _log_int(rng, 1, 128) * 128 if rng.random() < 0.7 else _log_int(rng, 4, 768) * 16
            outputs = _log_int(rng, 1, 256) * 64 if rng.random() < 0.7 else _log_int(rng, 16, 50257)
            c = _product("", batch, tokens, inputs, outputs, dtype, rng.random() < 0.3)
        else:
            c = _sample("", _log_int(rng, 1, 256), _log_int(rng, 1000, 200000), dtype,
                        rng.random() < 0.8, rng.choice((0, 0, 1, _log_int(rng, 2, 1000))),
                        rng.choice((0.0, 0.5, 0.9, 0.99)), rng.choice((0.0, 0.0, 0.01, 0.1)),
                        rng.choice((1.0, 2.5, 4.0)), rng.random() < 0.5)
        del c["name"]
        if _cost(c) <= limit and work(c)["bytes"] <= 1 << 30:
            return c


def _blocks(n):
    return -(-n // BLOCK)


def work(c):
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "sample":
        values = c["batch"] * c["vocabulary"]
        each = 12 + 4 * sum(1 for o in ("temperature", "top_k", "top_p", "min_p") if c[o])
        return {"bytes": values * size + c["batch"] * each, "flops": 4 * values}
    rows = c["batch"] * c["tokens"]
    if c["op"] == "product":
        k, n = c["inputs"], c["outputs"]
        held = rows * k + n * k + 4 * _blocks(k) * (rows + _blocks(n))
        return {"bytes": held + rows * n * size + (n * size if c["bias"] else 0),
                "flops": 2 * rows * n * k}
    values = rows * c["width"]
    eight = values + 4 * rows * _blocks(c["width"])
    if c["op"] == "quantize":
        return {"bytes": values * size * (2 if c["gated"] else 1) + eight, "flops": 4 * values}
    return {"bytes": values * size * (3 if c["residual"] else 1) + c["width"] * size
            + (eight if c["quantized"] else values * size), "flops": 5 * values}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, spread=1.0):
        x = torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32)
        return x.mul_(spread).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda", dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def activations(self, batch, tokens, width, dtype, spread=1.0):
        """Channels of very different sizes, a few far above the others."""
        size = self.normal(width, spread=0.4).exp()
        size[self.order(width)[:max(1, width // 500)]] *= 12.0
        return (self.normal(batch, tokens, width, spread=spread) * size).to(dtype)


def _in_blocks(x, rows):
    """Codes and scales of ``x`` [n, k], a scale for each ``rows`` x 128 values."""
    n, k = x.shape
    whole = x.new_zeros(-(-n // rows) * rows, _blocks(k) * BLOCK)
    whole[:n, :k] = x
    tiles = whole.view(-1, rows, _blocks(k), BLOCK)
    scale = (tiles.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp(min=LEAST_SCALE)
    codes = (tiles / scale[:, None, :, None]).view(whole.shape)[:n, :k]
    return codes.contiguous().to(E4M3), scale


def prepare(c, seed):
    r = _Random(seed)
    dtype, s = DTYPES[c["dtype"]], {"case": c}
    if c["op"] == "sample":
        b, v = c["batch"], c["vocabulary"]
        # a body of tokens, and a few that the model is sure of, more in some rows than in others
        x = r.normal(b, v, spread=c["spread"])
        x.scatter_add_(1, (r.uniform(b, 12) * v).long(), 10.0 * r.uniform(b, 12) * r.uniform(b, 1))
        wide = -(-v // 64) * 64 if c["padded"] else v
        held = torch.full((b, wide), 1e4, dtype=dtype, device="cuda")  # behind the last: not read
        held[:, :v] = x
        s["logits"] = held[:, :v]
        s["uniform"] = r.uniform(b).clamp(max=1.0 - 2.0 ** -24)
        turn = r.order(b)
        if c["temperature"]:  # one request in eight takes its likeliest token
            s["temperature"] = torch.where(turn % 8 == 7, 0.0, 0.6 + 0.1 * (turn % 7)).float()
        if c["top_k"]:
            s["top_k"] = (c["top_k"] + turn % 5).to(torch.int32)
        if c["top_p"]:
            s["top_p"] = (c["top_p"] - 0.02 * (turn % 4)).float()
        if c["min_p"]:
            s["min_p"] = (c["min_p"] * (1 + turn % 3)).float()
        return s
    b, t = c["batch"], c["tokens"]
    if c["op"] == "product":
        k, n = c["inputs"], c["outputs"]
        a, a_scale = _in_blocks(r.activations(1, b * t, k, torch.float32)[0], 1)
        s["a"], s["a_scale"] = a.view(b, t, k), a_scale.view(b, t, -1)
        s["b"], s["b_scale"] = _in_blocks(r.normal(n, k, spread=k ** -0.5), BLOCK)
        if c["bias"]:
            s["bias"] = r.normal(n, dtype=dtype)
        return s
    s["x"] = r.activations(b, t, c["width"], dtype)
    if c["op"] == "norm":
        s["weight"] = (1.0 + r.normal(c["width"], spread=0.2)).to(dtype)
        if c["residual"]:
            s["residual"] = r.activations(b, t, c["width"], dtype, spread=3.0)
    elif c["gated"]:
        s["gate"] = r.activations(b, t, c["width"], dtype)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _own(c, s)
    return {"norm": _plain_norm, "quantize": _plain_quantize, "product": _plain_product,
            "sample": _plain_sample}[c["op"]](c, s)


def _own(c, s):
    ops = _ops()
    if c["op"] == "norm":
        return ops.rms_norm(s["x"], s["weight"], s.get("residual"), eps=EPS, quantized=c["quantized"])
    if c["op"] == "quantize":
        return ops.quantize(s["x"], s.get("gate"))
    if c["op"] == "product":
        return ops.scaled_product(s["a"], s["a_scale"], s["b"], s["b_scale"], s.get("bias"),
                                  dtype=DTYPES[c["dtype"]])
    return ops.sample(s["logits"], s["uniform"], temperature=s.get("temperature"),
                      top_k=s.get("top_k"), top_p=s.get("top_p"), min_p=s.get("min_p"))


def _plain_eight(x):
    """``x`` in 32 bits as codes and the scale of each 128 values of a row."""
    k = x.shape[-1]
    whole = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k))
    tiles = whole.unflatten(-1, (-1, BLOCK))
    scale = (tiles.abs().amax(-1) / E4M3_MAX).clamp(min=LEAST_SCALE)
    codes = (tiles / scale.unsqueeze(-1)).flatten(-2)[..., :k]
    return codes.to(E4M3), scale


def _plain_norm(c, s):
    x = s["x"].float()
    if c["residual"]:
        x = x + s["residual"].float()
    y = x * ((x * x).mean(-1, keepdim=True) + EPS).rsqrt() * s["weight"].float()
    out = _plain_eight(y) if c["quantized"] else (y.to(s["x"].dtype),)
    if c["residual"]:
        out = (*out, x.to(s["x"].dtype))
    return out if len(out) > 1 else out[0]


def _plain_quantize(c, s):
    x = s["x"].float()
    if c["gated"]:
        g = s["gate"].float()
        x = x * (g / (1.0 + (-g).exp()))
    return _plain_eight(x)


def _plain_product(c, s):
    k, n = c["inputs"], c["outputs"]
    a = s["a"].float() * s["a_scale"].repeat_interleave(BLOCK, -1)[..., :k]
    scale = s["b_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    out = a.view(-1, k) @ (s["b"].float() * scale).t()
    if c["bias"]:
        out = out + s["bias"].float()
    return out.view(c["batch"], c["tokens"], n).to(DTYPES[c["dtype"]])


def _plain_sample(c, s):
    # in 64 bits: a token is next to the border of what its row keeps, or of what is drawn
    x, wanted = s["logits"].double(), s["uniform"].double().unsqueeze(-1)
    b, v = x.shape
    t = s["temperature"].double().unsqueeze(-1) if c["temperature"] else x.new_ones(b, 1)
    w = ((x - x.amax(-1, keepdim=True)) / torch.where(t == 0, 1.0, t)).exp()
    order = x.sort(dim=-1, descending=True, stable=True).indices
    ranked, place = w.gather(-1, order), torch.arange(v, device=x.device)
    kept = (t != 0) | (place == 0)
    if c["top_k"]:
        kept = kept & (place < s["top_k"].unsqueeze(-1))
    if c["top_p"]:
        held = ranked * kept
        before = held.cumsum(-1) - held
        kept = kept & ((before < s["top_p"].double().unsqueeze(-1) * held.sum(-1, keepdim=True))
                       | (place == 0))
    if c["min_p"]:
        kept = kept & (ranked >= s["min_p"].double().unsqueeze(-1))
    mass = (w * torch.zeros_like(kept).expand(b, v).scatter(-1, order, kept.expand(b, v))).cumsum(-1)
    return (mass <= wanted * mass[:, -1:]).sum(-1)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    return {"norm": _exact_norm, "quantize": _exact_quantize, "product": _exact_product,
            "sample": _exact_sample}[c["op"]](c, s)


def _exact_eight(y):
    """Each block by itself; a quotient goes to the nearest value of e4m3's ladder, a tie
    to the one with the even code."""
    ladder = torch.arange(127, dtype=torch.uint8, device=y.device).view(E4M3).double()
    codes, scales = torch.empty_like(y), []
    for lo in range(0, y.shape[-1], BLOCK):
        part = y[..., lo:lo + BLOCK]
        scale = torch.maximum(part.abs().amax(-1) / E4M3_MAX, y.new_tensor(LEAST_SCALE))
        scales.append(scale)
        q = (part / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
        above = torch.bucketize(q.abs(), ladder).clamp(1, 126)
        up, down = ladder[above] - q.abs(), q.abs() - ladder[above - 1]
        rises = (up < down) | ((up == down) & (above % 2 == 0))
        codes[..., lo:lo + BLOCK] = torch.where(rises, ladder[above], ladder[above - 1]) * q.sign()
    return codes, torch.stack(scales, -1)


def _exact_norm(c, s):
    h = s["x"].double()
    if c["residual"]:
        h = s["residual"].double().add(h)
    length = torch.linalg.vector_norm(h, dim=-1, keepdim=True)
    y = s["weight"].double() * h / (length ** 2 / c["width"] + EPS).sqrt()
    out = [*_exact_eight(y)] if c["quantized"] else [y]
    if c["residual"]:
        out.append(h)
    return tuple(out) if len(out) > 1 else out[0]


def _exact_quantize(c, s):
    y = s["x"].double()
    if c["gated"]:
        y = y * s["gate"].double() * torch.special.expit(s["gate"].double())
    return _exact_eight(y)


def _exact_product(c, s):
    k, n = c["inputs"], c["outputs"]
    a, a_scale = s["a"].view(-1, k), s["a_scale"].view(-1, _blocks(k)).double()
    out = torch.zeros(len(a), n, dtype=torch.float64, device="cuda")
    for i in range(_blocks(k)):
        at = slice(i * BLOCK, (i + 1) * BLOCK)
        by = s["b_scale"][:, i].double().repeat_interleave(BLOCK)[:n]
        out += (a[:, at].double() @ s["b"][:, at].double().t()) * a_scale[:, i, None] * by
    if c["bias"]:
        out += s["bias"].double()
    return out.view(c["batch"], c["tokens"], n)


def _exact_sample(c, s):
    """Row by row, on the host in numpy's 64 bits."""
    import numpy as np

    logits = s["logits"].double().cpu().numpy()
    option = {n: s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p")
              if n in s}
    uniform, tokens = s["uniform"].double().cpu().numpy(), []
    for b, x in enumerate(logits):
        t = option["temperature"][b] if "temperature" in option else 1.0
        if t == 0:
            tokens.append(int(np.argmax(x)))
            continue
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / t)
        n = len(w)
        if "top_k" in option:
            n = min(n, int(option["top_k"][b]))
        if "top_p" in option:
            sums = np.cumsum(w[:n])
            n = min(n, int(np.searchsorted(sums, option["top_p"][b] * sums[-1])) + 1)
        if "min_p" in option:
            n = min(n, int(np.count_nonzero(w >= option["min_p"][b])))
        back = np.argsort(order[:n])
        sums = np.cumsum(w[:n][back])
        at = int(np.searchsorted(sums, uniform[b] * sums[-1], side="right"))
        tokens.append(int(order[:n][back][min(at, n - 1)]))
    return torch.tensor(tokens)
