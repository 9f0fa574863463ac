"""Operators on matrices held in blocks of small floating-point numbers, as cases that can be timed and compared.

A block is a run of 16 or 32 neighbours along one axis of a matrix that share a scale. Three formats:

    mxfp4   4-bit numbers (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), blocks of 32, each with a
            power of two: the smallest that brings the block's largest magnitude to 6 or below
    nvfp4   the same numbers, blocks of 16, each with an 8-bit scale (E4M3) times one power of two for the
            whole matrix: the block's largest magnitude / 6 / that power of two, rounded to E4M3, from 2^-9 to 448
    mxfp8   8-bit numbers (E4M3, up to 448), blocks of 32, each with a power of two as above, where
            a number that is not zero never becomes zero: its sign is kept

Numbers are rounded to nearest, ties to even. Kinds of cases:

    quant       a matrix into 4-bit blocks and back to the values that they stand for
    product     C = relu?(W * X) + beta * C with weights kept in 4-bit blocks and inputs quantised on the way
    checkpoint  an activation into 8-bit blocks and back
    grad        what a fully-connected layer's backward pass does with its input's 8-bit record: the weight
                gradient E * X^T, and the deltas of the layer below masked where its ReLU's output X was not positive

`listed()` gives the standing cases, `draw(rng)` another one of the same ranges, `prepare(case, seed)` what a
program has in hand before the call, `run(state)` one pass, `exact(case, seed)` the same in 64 bits and
`work(case)` the bytes and operations that a pass cannot do without.
"""
import math

import torch

own = False     # true: the library's operators; false: their plain form

_TORCH = {"f16": torch.float16, "f32": torch.float32}
_BYTES = {"f16": 2, "f32": 4}
# format -> (block, largest number, its exponent, its mantissa, smallest exponent of a normal number, mantissa bits)
_FORMATS = {"mxfp4": (32, 6.0, 2, 1.5, 0, 1), "nvfp4": (16, 6.0, 2, 1.5, 0, 1), "mxfp8": (32, 448.0, 8, 1.75, -6, 3)}


# ---- the cases -------------------------------------------------------------------------------------
def listed():
    return [
        # the weights of AlexNet's first fully-connected layer, laid out along the inputs for its forward product
        dict(name="quant_weights_nvfp4", kind="quant", fmt="nvfp4", dtype="f16", rows=4096, cols=9216, axis=1, what="weights"),
        # a minibatch of that layer's inputs: the product sums over the features, so blocks run down the columns
        dict(name="quant_inputs_mxfp4", kind="quant", fmt="mxfp4", dtype="f16", rows=9216, cols=128, axis=0, what="relu"),
        # odd sizes everywhere, from 32 bits: 1001 classes, 4096 features and a bias
        dict(name="quant_odd_f32", kind="quant", fmt="nvfp4", dtype="f32", rows=1001, cols=4097, axis=1, what="weights"),
        # one image through a hidden layer: the weights are read once for one column, latency counts
        dict(name="product_one_column", kind="product", fmt="nvfp4", m=4096, n=1, k=4096, relu=True, beta=0.0),
        # AlexNet's first fully-connected layer, a minibatch of 128
        dict(name="product_fc", kind="product", fmt="nvfp4", m=4096, n=128, k=9216, relu=True, beta=0.0),
        # odd sizes everywhere: 1001 classes, a last minibatch of 125, 4096 features and a bias, added to what is there
        dict(name="product_ragged", kind="product", fmt="mxfp4", m=1001, n=125, k=4097, relu=False, beta=1.0),
        # a large square product: bound by the tensor cores
        dict(name="product_square", kind="product", fmt="nvfp4", m=8192, n=8192, k=8192, relu=True, beta=0.0),
        # the record of a fully-connected layer's input, short: latency counts
        dict(name="checkpoint_fc", kind="checkpoint", dtype="f16", rows=9216, cols=128),
        # the record of a convolution's output: 192 feature maps of 27x27 for 128 images
        dict(name="checkpoint_maps", kind="checkpoint", dtype="f16", rows=139968, cols=128),
        # backward pass of AlexNet's first fully-connected layer: few images, a large gradient to write
        dict(name="grad_fc", kind="grad", m=4096, k=9216, n=128),
        # odd sizes everywhere: the last minibatch of an epoch, 1001 classes, 4096 features and a bias
        dict(name="grad_ragged", kind="grad", m=1001, k=4097, n=125),
        # a hidden layer over many examples: bound by the tensor cores
        dict(name="grad_long", kind="grad", m=4096, k=4096, n=8192),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm; now and then a multiple of 8."""
    v = max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    return max(8, v // 8 * 8) if v > 16 and rng.random() < 0.4 else v


def draw(rng):
    kind = rng.choice(["quant", "product", "product", "checkpoint", "grad"])
    if kind == "quant":
        return dict(kind=kind, fmt=rng.choice(["mxfp4", "nvfp4"]), dtype=rng.choice(["f16", "f16", "f32"]),
                    rows=_log(rng, 16, 6000), cols=_log(rng, 16, 6000), axis=rng.choice([0, 1]),
                    what=rng.choice(["weights", "relu"]))
    if kind == "product":
        while True:
            c = dict(kind=kind, fmt=rng.choice(["mxfp4", "nvfp4"]), m=_log(rng, 16, 8192), n=_log(rng, 1, 8192),
                     k=_log(rng, 16, 16384), relu=rng.random() < 0.5, beta=rng.choice([0.0, 0.0, 1.0]))
            if work(c)["flops"] <= 1.0e12:
                return c
    if kind == "checkpoint":
        while True:
            c = dict(kind=kind, dtype=rng.choice(["f16", "f16", "f32"]), rows=_log(rng, 64, 200000), cols=_log(rng, 1, 1024))
            if c["rows"] * c["cols"] <= 17000000:
                return c
    while True:
        c = dict(kind=kind, m=_log(rng, 16, 8192), k=_log(rng, 16, 9216), n=_log(rng, 1, 8192))
        if work(c)["flops"] <= 5.0e11 and c["m"] * c["k"] <= 40000000:
            return c


# ---- what a pass needs -----------------------------------------------------------------------------
def _stored(size, fmt):
    """Bytes of a matrix in blocks."""
    block = _FORMATS[fmt][0]
    return size * (1.0 if fmt == "mxfp8" else 0.5) + size / block


def work(case):
    c = case
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        out = 2.0 * m * n * (2 if c["beta"] else 1)
        return {"bytes": _stored(m * k, c["fmt"]) + 2.0 * k * n + out, "flops": 2.0 * m * n * k}
    if c["kind"] == "grad":
        # the record is read once and serves both, the deltas below are read and written
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": 2.0 * m * n + _stored(k * n, "mxfp8") + 2.0 * m * k + 4.0 * k * n, "flops": 2.0 * m * n * k}
    size = c["rows"] * c["cols"]
    fmt = "mxfp8" if c["kind"] == "checkpoint" else c["fmt"]
    return {"bytes": 2.0 * _BYTES[c["dtype"]] * size + _stored(size, fmt), "flops": 4.0 * size}


# ---- inputs ----------------------------------------------------------------------------------------
def _values(gen, shape, what, dtype):
    x = torch.randn(shape, generator=gen, device="cuda")
    if what == "weights":       # rows of different sizes, a few large entries
        x *= 0.02 * torch.exp(0.5 * torch.randn((shape[0], 1), generator=gen, device="cuda"))
    elif what == "relu":        # half of them zero, features of different sizes
        x = torch.relu(x) * torch.exp(torch.randn((shape[0], 1), generator=gen, device="cuda"))
    else:                       # deltas
        x *= 0.01
    return x.to(_TORCH[dtype])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c = case
    if c["kind"] == "quant":
        return {"A": _values(gen, (c["rows"], c["cols"]), c["what"], c["dtype"])}
    if c["kind"] == "checkpoint":
        return {"A": _values(gen, (c["rows"], c["cols"]), "relu", c["dtype"])}
    if c["kind"] == "product":
        return {"W": _values(gen, (c["m"], c["k"]), "weights", "f16"), "X": _values(gen, (c["k"], c["n"]), "relu", "f16"),
                "start": _values(gen, (c["m"], c["n"]), "relu", "f16") if c["beta"] else None}
    return {"E": _values(gen, (c["m"], c["n"]), "deltas", "f16"), "X": _values(gen, (c["k"], c["n"]), "relu", "f16"),
            "D": _values(gen, (c["k"], c["n"]), "deltas", "f16")}


def _scale(what):
    """One power of two for a whole nvfp4 matrix that brings its blocks' scales into the range of E4M3."""
    return 2.0 ** -10 if what == "weights" else 2.0 ** -4


# ---- plain form ------------------------------------------------------------------------------------
def _pow2(e):
    """2^e for whole e, exactly: the bits of a 64-bit number."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_plain(y, fmt):
    """Magnitudes, divided by their scale, to the numbers of a format."""
    _, top, _, _, low, bits = _FORMATS[fmt]
    _, ex = torch.frexp(y)
    step = _pow2((ex - 1).clamp(min=low) - bits)
    q = (torch.round(y / step) * step).clamp(max=top)
    return torch.where((q == 0) & (y > 0), torch.full_like(q, 2.0 ** (low - bits)), q) if fmt == "mxfp8" else q


def _blocks_plain(A, fmt, axis, scale=1.0):
    """The values that A's blocks along `axis` stand for, in 32 bits. Scales and quotients in 64: a number next to
    the border between two has to fall on its own side."""
    block, top, emax, mant, _, _ = _FORMATS[fmt]
    x = (A if axis == 1 else A.t()).float()
    rows, cols = x.shape
    pad = -cols % block
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], dim=1)
    x = x.reshape(rows, -1, block)
    amax = x.abs().amax(dim=2, keepdim=True).double()
    if fmt == "nvfp4":
        s = amax / (top * scale)
        _, ex = torch.frexp(s)
        step = _pow2((ex - 1).clamp(min=-6) - 3)
        s = (torch.round(s / step) * step).clamp(2.0 ** -9, 448.0) * scale
    else:
        f, ex = torch.frexp(amax)
        e = torch.where(amax > 0, ex - 1 - emax + (2.0 * f > mant).int(), torch.zeros_like(ex))
        s = _pow2(e)
    q = _round_plain(x.abs().double() / s, fmt) * s
    q = torch.copysign(q, x.double()).float().reshape(rows, -1)[:, :cols]
    return q if axis == 1 else q.t()


# ---- preparation and passes ------------------------------------------------------------------------
def _tensor(ng, t):
    """A library tensor over a device array."""
    import numpy as np
    from nervanagpu_b200.nervanagpu import GPUTensor
    dtype = np.float16 if t.dtype == torch.float16 else np.float32
    return GPUTensor(ng, tuple(t.shape), dtype, gpudata=t.data_ptr())


def prepare(case, seed):
    c = case
    s = {"case": c, "in": _inputs(c, seed)}
    t = s["in"]
    if not own:
        if c["kind"] == "product":
            s["W"] = _blocks_plain(t["W"], c["fmt"], 1, _scale("weights"))
        elif c["kind"] == "grad":
            s["X"] = _blocks_plain(t["X"], "mxfp8", 1).half()
        return s
    from nervanagpu_b200 import NervanaGPU
    ng = s["ng"] = NervanaGPU()
    if c["kind"] in ("quant", "checkpoint"):
        s["out"] = torch.empty_like(t["A"])
        s["A"], s["O"] = _tensor(ng, t["A"]), _tensor(ng, s["out"])
        if c["kind"] == "quant":
            s["Q"] = ng.block_empty((c["rows"], c["cols"]), c["fmt"], axis=c["axis"], scale=_scale(c["what"]) if c["fmt"] == "nvfp4" else 1.0)
        else:
            s["Q"] = ng.block_empty((c["rows"], c["cols"]), "mxfp8")
    elif c["kind"] == "product":
        nv = c["fmt"] == "nvfp4"
        s["out"] = torch.empty((c["m"], c["n"]), device="cuda", dtype=torch.float16)
        s["W"] = ng.block_empty((c["m"], c["k"]), c["fmt"], axis=1, scale=_scale("weights") if nv else 1.0)
        s["Q"] = ng.block_empty((c["k"], c["n"]), c["fmt"], axis=0, scale=_scale("relu") if nv else 1.0)
        ng.quantize(_tensor(ng, t["W"]), s["W"])
        s["X"], s["C"] = _tensor(ng, t["X"]), _tensor(ng, s["out"])
    else:
        s["out"] = torch.empty((c["m"], c["k"]), device="cuda", dtype=torch.float16)
        s["Q"] = ng.block_empty((c["k"], c["n"]), "mxfp8")
        ng.quantize(_tensor(ng, t["X"]), s["Q"])
        s["E"], s["C"], s["D"] = _tensor(ng, t["E"]), _tensor(ng, s["out"]), _tensor(ng, t["D"])
    ng.synchronize()
    return s


def run(state):
    s = state
    c, t = s["case"], s["in"]
    if own:
        return _run_own(s, c, t)
    if c["kind"] == "quant":
        return _blocks_plain(t["A"], c["fmt"], c["axis"], _scale(c["what"])).to(t["A"].dtype).contiguous()
    if c["kind"] == "checkpoint":
        return _blocks_plain(t["A"], "mxfp8", 1).to(t["A"].dtype)
    if c["kind"] == "product":
        y = torch.matmul(s["W"], _blocks_plain(t["X"], c["fmt"], 0, _scale("relu")))
        if c["relu"]:
            y = y.clamp(min=0.0)
        if c["beta"]:
            y = y + c["beta"] * t["start"].float()
        return y.half()
    dw = torch.matmul(t["E"].float(), s["X"].float().t())
    return dw.half(), torch.where(s["X"] > 0, t["D"], torch.zeros_like(t["D"]))


def _run_own(s, c, t):
    ng = s["ng"]
    if c["kind"] in ("quant", "checkpoint"):
        ng.quantize(s["A"], s["Q"])
        ng.dequantize(s["Q"], s["O"])
        return s["out"]
    if c["kind"] == "product":
        if c["beta"]:
            s["out"].copy_(t["start"])      # the sum that the product is added to
        ng.quantize(s["X"], s["Q"])
        ng.block_dot(s["W"], s["Q"], s["C"], beta=c["beta"], relu=c["relu"])
        return s["out"]
    ng.block_dot(s["E"], s["Q"].T, s["C"])
    ng.relu_mask(s["Q"], s["D"])
    return s["out"], t["D"]


# ---- the definition in 64 bits ---------------------------------------------------------------------
def _numbers(fmt):
    """The numbers of a format from zero up, and the borders between neighbours. The number with an even last
    bit has an even place in the list and takes the border."""
    if fmt == "mxfp8":
        q = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    else:
        q = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    q = torch.tensor(q, dtype=torch.float64, device="cuda")
    return q, (q[1:] + q[:-1]) / 2


def _nearest(y, fmt):
    q, border = _numbers(fmt)
    lo = torch.searchsorted(border, y, right=False)     # on a border: the lower neighbour
    hi = torch.searchsorted(border, y, right=True)      # on a border: the upper neighbour
    return q[torch.where(lo % 2 == 0, lo, hi)]


def _blocks_exact(A, fmt, axis, scale=1.0):
    block, top = _FORMATS[fmt][:2]
    if axis == 0:
        return _blocks_exact(A.t(), fmt, 1, scale).t()
    parts = []
    for x in torch.split(A, max(block, (1 << 24) // max(1, A.shape[0]) // block * block), dim=1):
        x = x.double()
        n = x.shape[1]
        full = torch.zeros(x.shape[0], -(-n // block) * block, dtype=torch.float64, device="cuda")
        full[:, :n] = x
        mag = full.abs().view(x.shape[0], -1, block)
        amax = mag.max(dim=2).values
        if fmt == "nvfp4":
            s = _nearest(amax / top / scale, "mxfp8")
            s = torch.where(s == 0, torch.full_like(s, 2.0 ** -9), s) * scale
        else:
            powers = torch.tensor([2.0 ** e for e in range(-180, 160)], dtype=torch.float64, device="cuda")
            s = powers[torch.searchsorted(powers * top, amax)]      # the smallest with which s * top >= amax
        y = mag / s[:, :, None]
        q = _nearest(y, fmt)
        if fmt == "mxfp8":
            q = torch.where((q == 0) & (y > 0), torch.full_like(q, 2.0 ** -9), q)
        q = (q * s[:, :, None]).reshape(x.shape[0], -1)[:, :n]
        parts.append(torch.where(x < 0, -q, q))
    return torch.cat(parts, dim=1)


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "quant":
        return _blocks_exact(t["A"], c["fmt"], c["axis"], _scale(c["what"]) if c["fmt"] == "nvfp4" else 1.0).contiguous()
    if c["kind"] == "checkpoint":
        return _blocks_exact(t["A"], "mxfp8", 1)
    if c["kind"] == "product":
        y = _blocks_exact(t["W"], c["fmt"], 1, _scale("weights")) @ _blocks_exact(t["X"], c["fmt"], 0, _scale("relu"))
        if c["relu"]:
            y = torch.relu(y)
        return y + c["beta"] * t["start"].double() if c["beta"] else y
    x = _blocks_exact(t["X"], "mxfp8", 1)
    return t["E"].double() @ x.t(), t["D"].double() * (t["X"] > 0)
