"""Dense projections in 8-bit floating point: what is timed and compared.

Four operators, in the order a feed-forward block of a decoder layer runs them:

  norm      H = X + R, RMSNorm(H; gamma) in 8 bits
  gate_up   silu(X Wg^T) * (X Wu^T) in 8 bits, from 8-bit activations and weights
  project   Y = R + X W^T in f32, or X W^T in bf16, from 8-bit activations and weights
  quantize  a matrix in 8 bits: activations with a scale for each row, weights
            with a scale for each 128 rows

A matrix in 8 bits [rows x cols] is its codes, e4m3 bytes [rows x pitch] with
pitch the next multiple of 128 columns and zeros past `cols`, and its scales,
powers of two held as their e8m0 byte, one for each 128 columns of `block`
rows (1 or 128): [ceil(rows / block) x spitch], spitch the column blocks
rounded up to a multiple of 4, 1 past the last block. A scale is the smallest
power of two with the block's largest finite magnitude at most 448 scales.

``listed()`` names the fixed cases, ``draw`` makes more of the same ranges,
``prepare`` builds a program's inputs (library buffers when the library is
called, plain tensors otherwise; the same values), ``run`` is one pass,
``work`` the bytes and operations it cannot do without, ``exact`` the same
results in 64 bits, before their rounding to an output's type.
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = 128
TOP = 448.0  # e4m3's largest value
TYPES = ["f32", "bf16"]


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # One token's attention output (24 heads of 256) before its projection: the smallest call.
        dict(name="quantize_token", kind="quantize", rows=1, cols=6144, block=1, type="f32"),
        # A layer's bf16 weights (hidden 2560 to 10240 channels) once at load.
        dict(name="quantize_weights", kind="quantize", rows=10240, cols=2560, block=128, type="bf16"),
        # A decode step of five sequences between two blocks.
        dict(name="norm_batch5", kind="norm", rows=5, cols=2560, residual=True, type="f32"),
        # A prompt between two blocks: a sublayer's bf16 output into the f32 residual stream.
        dict(name="norm_prompt", kind="norm", rows=4096, cols=2560, residual=True, type="bf16"),
        # One token's projection from the hidden state: latency and the weights' bytes.
        dict(name="project_token", kind="project", tokens=1, cols=2560, rows=10240, residual=False, type="f32"),
        # A decode step of 32 sequences: attention's output projection into the residual stream.
        dict(name="project_batch32", kind="project", tokens=32, cols=6144, rows=2560, residual=True, type="f32"),
        # A short prompt of ragged length, output rows that fill no tile.
        dict(name="project_ragged", kind="project", tokens=333, cols=2500, rows=5003, residual=False, type="bf16"),
        # A prompt's attention output into the residual stream, sums to f32.
        dict(name="project_prompt_f32", kind="project", tokens=2048, cols=6144, rows=2560, residual=True, type="f32"),
        # Several long prompts in one batch.
        dict(name="project_prompt", kind="project", tokens=8192, cols=2560, rows=10240, residual=False, type="bf16"),
        # One token's feed-forward input.
        dict(name="gate_up_token", kind="gate_up", tokens=1, cols=2560, ff=8192),
        # A step of many sequences, a hidden size that ends inside a block.
        dict(name="gate_up_batch96", kind="gate_up", tokens=96, cols=2560, ff=6000),
        # A long prompt through a wide feed-forward block: the largest call.
        dict(name="gate_up_prompt", kind="gate_up", tokens=4096, cols=4096, ff=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng):
    n = _log(rng, 64, 8192)
    return n if rng.random() < 0.5 else max(64, 64 * round(n / 64))


def draw(rng):
    kind = rng.choice(["quantize", "norm", "project", "project", "gate_up", "gate_up"])
    cols = _cols(rng)
    if kind == "quantize":
        return dict(kind=kind, rows=_log(rng, 1, min(16384, (1 << 26) // cols)), cols=cols, block=rng.choice([1, 128]),
                    type=rng.choice(TYPES))
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, min(16384, (1 << 25) // cols)), cols=cols, residual=rng.random() < 0.7,
                    type=rng.choice(TYPES))
    if kind == "project":
        rows = _log(rng, 16, 12288)
        kept = rng.choice(["f32", "f32 with R", "bf16"])
        return dict(kind=kind, tokens=_log(rng, 1, min(8192, 2 * 10 ** 11 // (cols * rows))), cols=cols, rows=rows,
                    residual=kept == "f32 with R", type=kept[:4].strip())
    ff = _log(rng, 64, 8192)
    return dict(kind=kind, tokens=_log(rng, 1, min(8192, 10 ** 11 // (cols * ff))), cols=cols, ff=ff)


# ------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, seed, sigma=1.0):
    return torch.randn(shape, generator=_gen(seed), device="cuda") * sigma


def _hidden(rows, cols, seed):
    """Activations as a decoder has them: normal, some columns many times larger, a few far out."""
    columns = torch.exp(_normal((cols,), seed + 1, 0.8))
    x = _normal((rows, cols), seed) * columns
    return torch.where(x.abs() > 3.5 * columns, 4 * x, x)


def _blocks(rows, block):
    return -(-rows // block)


def _quantize(x, block):
    """(codes, scales) of x in 32 bits: amax, its power of two, one rounding."""
    rows, cols = x.shape
    up, kb = _blocks(rows, block), _blocks(cols, BLOCK)
    p = torch.zeros((up * block, kb * BLOCK), device=x.device)
    p[:rows, :cols] = x
    b = p.view(up, block, kb, BLOCK)
    amax = torch.where(b.isfinite(), b, 0.0).abs().amax((1, 3))
    m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1; at most 448 2^s for s = e - 9, one more past 7/8
    s = torch.where(amax > 0, (e - 9 + (m > 0.875)).clamp(min=-127), 0)
    y = torch.ldexp(b, -s[:, None, :, None])
    codes = torch.where(y.isfinite(), y, math.nan).to(torch.float8_e4m3fn).view(up * block, kb * BLOCK)[:rows]
    scales = torch.full((up, 4 * _blocks(kb, 4)), 127, dtype=torch.uint8, device=x.device)
    scales[:, :kb] = (s + 127).to(torch.uint8)
    return codes, scales.view(torch.float8_e8m0fnu)


def _dequantize(codes, scales, block):
    rows, pitch = codes.shape
    s = scales.float()[:, : pitch // BLOCK].repeat_interleave(block, 0)[:rows].repeat_interleave(BLOCK, 1)
    return codes.float() * s


def _weights(rows, cols, seed):
    w = _normal((rows, cols), seed, cols ** -0.5)
    return w * torch.exp(_normal((rows, 1), seed + 1, 0.3))


def _dtype(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float32


def _inputs(case, seed):
    """The pass's inputs by name."""
    kind, seed = case["kind"], 100 * seed
    if kind == "quantize":
        x = _weights(case["rows"], case["cols"], seed) if case["block"] > 1 else _hidden(case["rows"], case["cols"], seed)
        return {"X": x.to(_dtype(case))}
    cols = case["cols"]
    if kind == "norm":
        t = {"X": _hidden(case["rows"], cols, seed).to(_dtype(case)), "gamma": 1 + _normal((cols,), seed + 5, 0.1)}
        if case["residual"]:
            t["R"] = _hidden(case["rows"], cols, seed + 10)
        return t
    t = {}
    t["X"], t["Xs"] = _quantize(_hidden(case["tokens"], cols, seed), 1)
    if kind == "gate_up":
        t["Wg"], t["Wgs"] = _quantize(_weights(case["ff"], cols, seed + 20), BLOCK)
        t["Wu"], t["Wus"] = _quantize(_weights(case["ff"], cols, seed + 30), BLOCK)
        return t
    t["W"], t["Ws"] = _quantize(_weights(case["rows"], cols, seed + 20), BLOCK)
    if case["residual"]:
        t["R"] = _hidden(case["tokens"], case["rows"], seed + 40)
    return t


# ------------------------------------------------------------------ prepare
_held = {}


def _backend():
    """The program's one context on the GPU."""
    if "backend" not in _held:
        import stratacuda_amd as sm

        _held["backend"] = sm.Backend(0)
    return _held["backend"]


class _Owned:
    """A library buffer freed with its last user, readable as a torch tensor of bytes."""

    def __init__(self, nbytes):
        self.buf = _backend().alloc_bytes(nbytes)
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (self.buf.handle, False),
                                         "version": 2, "strides": None}

    def __del__(self):
        try:
            _backend().free(self.buf)
        except Exception:
            pass


def _empty(shape, dtype):
    """(buffer, tensor over it); the tensor keeps the buffer."""
    nbytes = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    held = _Owned(nbytes)
    return held.buf, torch.as_tensor(held, device="cuda").view(dtype).view(shape)


def _put(t):
    buf, view = _empty(t.shape, t.dtype)
    view.view(torch.uint8).copy_(t.contiguous().view(torch.uint8))
    return buf, view


def _empty_f8(rows, cols):
    kb = _blocks(cols, BLOCK)
    return _empty((rows, kb * BLOCK), torch.float8_e4m3fn), _empty((rows, 4 * _blocks(kb, 4)), torch.float8_e8m0fnu)


def prepare(case, seed):
    t = _inputs(case, seed)
    if not own:
        return {"case": case, "in": t}
    # The library takes the buffers that it allocated: the same inputs there,
    # and the outputs and workspace that a program keeps.
    s = {"case": case, "in": {k: _put(v) for k, v in t.items()}}
    kind = case["kind"]
    if kind == "quantize":
        up, kb = _blocks(case["rows"], case["block"]), _blocks(case["cols"], BLOCK)
        s["codes"] = _empty((case["rows"], kb * BLOCK), torch.float8_e4m3fn)
        s["scales"] = _empty((up, 4 * _blocks(kb, 4)), torch.float8_e8m0fnu)
    elif kind == "norm":
        s["codes"], s["scales"] = _empty_f8(case["rows"], case["cols"])
        if case["residual"]:
            s["H"] = _empty((case["rows"], case["cols"]), torch.float32)
    elif kind == "project":
        s["Y"] = _empty((case["tokens"], case["rows"]), _dtype(case))
    else:
        s["codes"], s["scales"] = _empty_f8(case["tokens"], case["ff"])
        s["workspace"] = _empty((_backend().f8_gate_up_workspace_bytes(case["tokens"], case["ff"]),), torch.uint8)
    torch.cuda.synchronize()  # the library's stream starts from finished inputs
    return s


# ---------------------------------------------------------------------- run
def _run_own(s):
    be, c = _backend(), s["case"]
    t = {k: v[0] for k, v in s["in"].items()}
    if c["kind"] == "quantize":
        be.f8_quantize(t["X"], c["rows"], c["cols"], c["block"], s["codes"][0], s["scales"][0],
                       type=c["type"])
    elif c["kind"] == "norm":
        if c["residual"]:
            be.f8_norm(t["X"], t["gamma"], EPS, c["rows"], c["cols"], s["codes"][0], s["scales"][0], residual=t["R"],
                       H=s["H"][0], type=c["type"])
            return {"H": s["H"][1], "codes": s["codes"][1], "scales": s["scales"][1]}
        be.f8_norm(t["X"], t["gamma"], EPS, c["rows"], c["cols"], s["codes"][0], s["scales"][0], type=c["type"])
    elif c["kind"] == "project":
        be.f8_project(t["X"], t["Xs"], c["tokens"], c["cols"], t["W"], t["Ws"], c["rows"], s["Y"][0],
                      residual=t.get("R"), type=c["type"])
        return {"Y": s["Y"][1]}
    else:
        be.f8_gate_up(t["X"], t["Xs"], c["tokens"], c["cols"], t["Wg"], t["Wgs"], t["Wu"], t["Wus"], c["ff"],
                      s["codes"][0], s["scales"][0], s["workspace"][0])
    return {"codes": s["codes"][1], "scales": s["scales"][1]}


def run(state):
    if own:
        return _run_own(state)
    c, t = state["case"], state["in"]
    if c["kind"] == "quantize":
        codes, scales = _quantize(t["X"].float(), c["block"])
        return {"codes": codes, "scales": scales}
    if c["kind"] == "norm":
        h = t["X"].float() + t["R"] if c["residual"] else t["X"].float()
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * t["gamma"]
        codes, scales = _quantize(y, 1)
        return {"H": h, "codes": codes, "scales": scales} if c["residual"] else {"codes": codes, "scales": scales}
    x = _dequantize(t["X"], t["Xs"], 1)
    if c["kind"] == "project":
        y = x @ _dequantize(t["W"], t["Ws"], BLOCK).T
        return {"Y": y + t["R"] if c["residual"] else y.to(_dtype(c))}
    g, u = x @ _dequantize(t["Wg"], t["Wgs"], BLOCK).T, x @ _dequantize(t["Wu"], t["Wus"], BLOCK).T
    codes, scales = _quantize(g / (1 + torch.exp(-g)) * u, 1)
    return {"codes": codes, "scales": scales}


# ---------------------------------------------------------------- the bound
def work(case):
    kind, cols, size = case["kind"], case["cols"], 2 if case.get("type") == "bf16" else 4
    f8 = lambda rows, n, block: rows * n + _blocks(rows, block) * _blocks(n, BLOCK)  # noqa: E731
    if kind in ("quantize", "norm"):
        n = case["rows"] * cols
        if kind == "quantize":
            return {"bytes": n * size + f8(case["rows"], cols, case["block"]), "flops": 3 * n}
        return {"bytes": n * (size + (8 if case["residual"] else 0)) + 4 * cols + f8(case["rows"], cols, 1), "flops": 8 * n}
    n = case["tokens"]
    if kind == "project":
        rows = case["rows"]
        return {"bytes": f8(n, cols, 1) + f8(rows, cols, BLOCK) + n * rows * size * (2 if case["residual"] else 1),
                "flops": 2 * n * rows * cols}
    return {"bytes": f8(n, cols, 1) + 2 * f8(case["ff"], cols, BLOCK) + f8(n, case["ff"], 1), "flops": 4 * n * case["ff"] * cols}


# ------------------------------------------------------------------ 64 bits
def _exact_f8(y, block):
    """What codes and scales stand for: y over its block's scale, not rounded, and the scale."""
    rows, cols = y.shape
    kb = _blocks(cols, BLOCK)
    wide = torch.nn.functional.pad(y, (0, kb * BLOCK - cols))
    tall = torch.nn.functional.pad(wide, (0, 0, 0, _blocks(rows, block) * block - rows))
    amax = tall.abs().unfold(0, block, block).unfold(1, BLOCK, BLOCK).amax((-1, -2))
    e = torch.ceil(torch.log2(amax / TOP))
    e = e + (amax > TOP * torch.exp2(e)).double() - (amax <= TOP * torch.exp2(e - 1)).double()
    scale = torch.exp2(torch.where(amax > 0, e, torch.zeros_like(e)))
    each = scale.repeat_interleave(block, 0)[:rows].repeat_interleave(BLOCK, 1)
    return {"codes": wide / each, "scales": torch.nn.functional.pad(scale, (0, -kb % 4), value=1.0)}


def _value(codes, scales, block):
    v = codes.double()
    s = torch.exp2(scales.view(torch.uint8).double() - 127)
    row = torch.arange(v.shape[0], device="cuda") // block
    return v * s[row][:, torch.arange(v.shape[1], device="cuda") // BLOCK]


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_f8(t["X"].double(), case["block"])
    if kind == "norm":
        h = t["X"].double() + (t["R"].double() if case["residual"] else 0.0)
        out = _exact_f8(h / (h.square().sum(-1, keepdim=True) / case["cols"] + EPS).sqrt() * t["gamma"].double(), 1)
        return dict(out, H=h) if case["residual"] else out
    x = _value(t["X"], t["Xs"], 1)
    if kind == "project":
        y = x @ _value(t["W"], t["Ws"], BLOCK).T
        return {"Y": y + t["R"].double() if case["residual"] else y}
    g = x @ _value(t["Wg"], t["Wgs"], BLOCK).T
    return _exact_f8(torch.sigmoid(g) * g * (x @ _value(t["Wu"], t["Wus"], BLOCK).T), 1)
