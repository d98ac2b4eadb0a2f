"""Measured cases of the 8-bit block-scaled operators: quantisation with a power-of-two scale for each block of 128, the
matrix product of such operands, the 8-bit activation checkpoint (its restoration and its use in a backward pass), and the
linear layer that runs them together.

With ``own`` false, ``run`` computes the operators in elementary torch operations in 32 bits; with ``own`` true it calls
``qgemm_b200``. A quantised matrix is a float8_e4m3fn tensor of codes with one float8_e8m0fnu scale for each 128 elements of
the axis a product sums over: a row-form [R, C] matrix has scales [ceil(C/128), R] (or [ceil(C/128), ceil(R/128)] where a
scale covers a square of 128 x 128).
"""
import math

import torch

own = False

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one token's activations on their way into a layer while text is generated: latency
        {"name": "quant_token", "op": "quantize", "rows": 1, "cols": 7168, "type": "bf16", "square": False, "form": "row"},
        # the gradient of a training step's layer output, wanted along both axes by the two backward products
        {"name": "quant_grad_both", "op": "quantize", "rows": 4096, "cols": 7168, "type": "bf16", "square": False, "form": "both"},
        # a fp32 master weight after an optimiser step: squares, in both orders
        {"name": "quant_weight", "op": "quantize", "rows": 11008, "cols": 4096, "type": "fp32", "square": True, "form": "both"},
        # the saved 8-bit activation of a long batch turned into the operand of the weight gradient
        {"name": "ckpt_turn", "op": "requantize", "rows": 16384, "cols": 7168},
        # a ragged batch's saved activation restored for a recomputation
        {"name": "ckpt_restore", "op": "dequantize", "rows": 1537, "cols": 4104, "type": "bf16", "square": False},
        # one token against a layer's weight, and a small serving batch against a wide one
        {"name": "mm_token", "op": "mm", "M": 1, "N": 7168, "K": 2048, "out": "bf16", "a_square": False, "b_square": True, "accumulate": False},
        {"name": "mm_batch64", "op": "mm", "M": 64, "N": 28672, "K": 8192, "out": "fp16", "a_square": False, "b_square": True, "accumulate": False},
        # a layer's forward product over a prompt or a training batch
        {"name": "mm_forward", "op": "mm", "M": 4096, "N": 7168, "K": 7168, "out": "bf16", "a_square": False, "b_square": True, "accumulate": False},
        # a weight gradient added to the fp32 sum of earlier micro-batches, over an odd number of tokens
        {"name": "mm_wgrad_add", "op": "mm", "M": 7168, "N": 2048, "K": 4001, "out": "fp32", "a_square": False, "b_square": False, "accumulate": True},
        # the largest product of the repository's own benchmark
        {"name": "mm_8192", "op": "mm", "M": 8192, "N": 8192, "K": 8192, "out": "bf16", "a_square": False, "b_square": True, "accumulate": False},
        # a training step's layer, forward and backward: bf16 activations and fp32 weights; and a ragged small one
        {"name": "linear_step", "op": "linear", "tokens": 6144, "in": 2048, "out_f": 7168, "type": "bf16", "wtype": "fp32"},
        {"name": "linear_ragged", "op": "linear", "tokens": 333, "in": 1040, "out_f": 520, "type": "fp16", "wtype": "fp16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Any operator, any size from single rows to the listed ones' largest, odd ones as often as even ones."""
    op = rng.choice(["quantize", "requantize", "dequantize", "mm", "mm", "linear"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("quantize", "requantize", "dequantize"):
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 1, min(16384, max(1, (40 << 20) // rows)))
        case = {"op": op, "rows": rows, "cols": cols}
        if op != "requantize":
            case |= {"type": kind, "square": rng.random() < 0.4}
        if op == "quantize":
            case["form"] = rng.choice(["row", "column", "both"])
        return case
    if op == "mm":
        M, K = _log(rng, 1, 8192), _log(rng, 64, 16384)
        N = _log(rng, 16, 16384)
        while 2.0 * M * N * K > 1.0e12 or N * K > 240e6:
            K = max(64, K // 2 + 1)
        add = kind == "fp32" and rng.random() < 0.5
        return {"op": op, "M": M, "N": N, "K": K, "out": kind, "a_square": rng.random() < 0.2, "b_square": rng.random() < 0.6, "accumulate": add}
    tokens, fin, fout = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
    while 6.0 * tokens * fin * fout > 6.0e11:
        tokens = max(1, tokens // 2)
    return {"op": op, "tokens": tokens, "in": fin, "out_f": fout, "type": kind, "wtype": rng.choice(["bf16", "fp32"]) if kind == "bf16" else kind}


# ------------------------------------------------------------------------------------------------ inputs
def _activations(rows, cols, gen, dtype=torch.float32):
    """Values as a layer meets them: each token at its own level, a few channels far above the others."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    x *= torch.exp(torch.randn(rows, 1, device="cuda", generator=gen) * 0.7)
    x *= torch.where(torch.rand(1, cols, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
    return x.to(dtype)


def _weights(rows, cols, gen, dtype=torch.float32):
    return (torch.randn(rows, cols, device="cuda", generator=gen) / math.sqrt(cols)).to(dtype)


def _padded(codes):
    """The same codes with rows that start on 16-byte boundaries, as the product asks for."""
    rows, cols = codes.shape
    out = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=codes.device)
    out[:, :cols] = codes.view(torch.uint8)
    return out.view(E4M3)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "quantize":
        make = _weights if case["square"] else _activations
        s["x"] = make(case["rows"], case["cols"], gen, TYPES[case["type"]])
    elif op in ("requantize", "dequantize"):
        q, e = _quant(_activations(case["rows"], case["cols"], gen), case.get("square", False))
        s["q"], s["scale"] = _padded(q), e
    elif op == "mm":
        q, e = _quant(_activations(case["M"], case["K"], gen), case["a_square"])
        s["a"], s["a_scale"] = _padded(q), e
        q, e = _quant(_weights(case["N"], case["K"], gen), case["b_square"])
        s["b"], s["b_scale"] = _padded(q), e
        if case["accumulate"]:
            s["sum"] = torch.randn(case["M"], case["N"], device="cuda", generator=gen)
        else:
            s["c"] = torch.zeros(case["M"], case["N"], device="cuda", dtype=TYPES[case["out"]])
    else:
        s["x"] = _activations(case["tokens"], case["in"], gen, TYPES[case["type"]]).requires_grad_(True)
        s["w"] = _weights(case["out_f"], case["in"], gen, TYPES[case["wtype"]]).requires_grad_(True)
        s["dy"] = (_activations(case["tokens"], case["out_f"], gen) * 1e-2).to(TYPES[case["type"]])
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _pow2(e):
    """2^e in 32 bits for whole e in [-126, 127], and 2^-127."""
    return torch.where(e < -126, torch.full_like(e, 0x400000), (e + 127).clamp(min=0) << 23).to(torch.int32).view(torch.float32)


def _spread(s, rows, cols):
    """A value for each block, [blocks of columns, rows or blocks of rows], over all elements."""
    s = s.t()
    if s.shape[0] != rows:
        s = s.repeat_interleave(128, 0)[:rows]
    return s.repeat_interleave(128, 1)[:, :cols]


def _quant(x, square):
    """Codes and scales of x [R, C] along its rows."""
    rows, cols = x.shape
    x = x.float()
    pad_r, pad_c = (-rows % 128 if square else 0), -cols % 128
    p = torch.nn.functional.pad(x, (0, pad_c, 0, pad_r))
    if square:
        amax = p.abs().view(p.shape[0] // 128, 128, p.shape[1] // 128, 128).amax((1, 3))
    else:
        amax = p.abs().view(rows, p.shape[1] // 128, 128).amax(2)
    amax = amax.t().contiguous()
    m, e = torch.frexp(amax)
    e = (e.to(torch.int32) - 9 + (m > 0.875)).clamp(min=-127)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    bad = ~torch.isfinite(amax)
    codes = (x * _spread(_pow2(torch.where(bad, torch.zeros_like(e), -e)), rows, cols)).to(E4M3)
    codes = torch.where(_spread(bad, rows, cols), torch.full_like(codes.view(torch.uint8), 0x7F), codes.view(torch.uint8)).view(E4M3)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8).view(E8M0)
    return codes, scale


def _value(q, scale):
    rows, cols = q.shape
    return q.float() * _spread(scale.float(), rows, cols)


def _turned(x, square):
    """The column form of x: codes and scales of its transpose."""
    return _quant(x.float().t(), square)


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        out = ()
        if s["form"] in ("row", "both"):
            out += _quant(s["x"], s["square"])
        if s["form"] in ("column", "both"):
            out += _turned(s["x"], s["square"])
        return out
    if op == "requantize":
        return _turned(_value(s["q"], s["scale"]), False)
    if op == "dequantize":
        return _value(s["q"], s["scale"]).to(TYPES[s["type"]])
    if op == "mm":
        c = _value(s["a"], s["a_scale"]) @ _value(s["b"], s["b_scale"]).t()
        return s["sum"] + c if s["accumulate"] else c.to(TYPES[s["out"]])
    with torch.no_grad():
        x = _value(*_quant(s["x"], False))
        w = _value(*_quant(s["w"], True))
        dy_row = _value(*_quant(s["dy"], False))
        dy_col = _value(*_turned(s["dy"], False))
        x_col = _value(*_turned(x, False))
        return (x @ w.t()).to(s["x"].dtype), (dy_row @ w).to(s["x"].dtype), (dy_col @ x_col.t()).to(s["w"].dtype)


def _run_own(s):
    import qgemm_b200 as q
    op = s["op"]
    if op == "quantize":
        return q.quantize_block(s["x"], square=s["square"], form=s["form"])
    if op == "requantize":
        return q.requantize_block(s["q"], s["scale"])
    if op == "dequantize":
        return q.dequantize_block(s["q"], s["scale"], TYPES[s["type"]])
    if op == "mm":
        c = s["sum"].clone() if s["accumulate"] else s["c"]
        q.fp8_block_mm_e8m0(s["a"], s["b"], s["a_scale"], s["b_scale"], c, accumulate=s["accumulate"])
        return c
    from qgemm_b200.linear import fp8_linear
    y = fp8_linear(s["x"], s["w"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"]))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ work and definition
def work(case):
    op = case["op"]
    blocks = lambda n: -(-n // 128)  # noqa: E731
    if op in ("quantize", "requantize", "dequantize"):
        r, c = case["rows"], case["cols"]
        along = blocks(c) * (blocks(r) if case.get("square") else r)
        across = blocks(r) * (blocks(c) if case.get("square") else c)
        if op == "requantize":
            return {"bytes": 2 * r * c + along + across, "flops": 3 * r * c}
        if op == "dequantize":
            return {"bytes": (1 + BYTES[case["type"]]) * r * c + along, "flops": r * c}
        forms = 2 if case["form"] == "both" else 1
        scales = (along if case["form"] != "column" else 0) + (across if case["form"] != "row" else 0)
        return {"bytes": (BYTES[case["type"]] + forms) * r * c + scales, "flops": (1 + forms) * r * c}
    if op == "mm":
        M, N, K = case["M"], case["N"], case["K"]
        scales = blocks(K) * ((blocks(M) if case["a_square"] else M) + (blocks(N) if case["b_square"] else N))
        c_bytes = M * N * BYTES[case["out"]] * (2 if case["accumulate"] else 1)
        return {"bytes": M * K + N * K + scales + c_bytes, "flops": 2.0 * M * N * K}
    t, i, o = case["tokens"], case["in"], case["out_f"]
    a, w = BYTES[case["type"]], BYTES[case["wtype"]]
    return {"bytes": a * (2 * t * i + 2 * t * o) + 2 * w * i * o, "flops": 6.0 * t * i * o}


def _ideal(x, square):
    """The quantised matrix by its definition, in 64 bits: (codes as numbers, exponents of the scales [blocks, rows])."""
    rows, cols = x.shape
    x = x.double()
    step_r = 128 if square else 1
    nb_r, nb_c = -(-rows // step_r), -(-cols // 128)
    full = torch.zeros(nb_r * step_r, nb_c * 128, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    tiles = full.reshape(nb_r, step_r, nb_c, 128)
    ratio = torch.linalg.vector_norm(tiles, ord=math.inf, dim=(1, 3)) / 448.0
    mant, expo = torch.frexp(ratio)  # ratio = mant * 2^expo with 1/2 <= mant < 1: the least power of two not below it
    expo = torch.where(mant == 0.5, expo - 1, expo).double()
    expo = torch.where(ratio == 0, torch.zeros_like(expo), expo.clamp(min=-127.0))
    y = tiles * torch.exp2(-expo)[:, None, :, None]
    grid = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp(min=-6.0) - 3.0)
    codes = torch.round(y / grid) * grid  # half to even: the codes' last bit
    return codes.reshape(nb_r * step_r, nb_c * 128)[:rows, :cols], expo.t().contiguous()


def _ideal_value(codes, expo):
    rows, cols = codes.shape
    at_r = torch.arange(rows, device=codes.device)
    if expo.shape[1] != rows:
        at_r = at_r // 128
    at_c = torch.arange(cols, device=codes.device) // 128
    return codes * torch.exp2(expo)[at_c[None, :], at_r[:, None]]


def _held(q, scale):
    return _ideal_value(q.double(), scale.view(torch.uint8).double() - 127.0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        out = []
        for form, x in (("row", s["x"]), ("column", s["x"].t())):
            if case["form"] in (form, "both"):
                codes, expo = _ideal(x, case["square"])
                out += [codes, torch.exp2(expo)]
        return out
    if op == "requantize":
        codes, expo = _ideal(_held(s["q"], s["scale"]).t(), False)
        return [codes, torch.exp2(expo)]
    if op == "dequantize":
        return _held(s["q"], s["scale"])
    if op == "mm":
        c = torch.matmul(_held(s["a"], s["a_scale"]), _held(s["b"], s["b_scale"]).t())
        return c + s["sum"].double() if case["accumulate"] else c
    x, w, dy = (s[k].detach() for k in ("x", "w", "dy"))
    xv, wv = _ideal_value(*_ideal(x, False)), _ideal_value(*_ideal(w, True))
    along, across = _ideal_value(*_ideal(dy, False)), _ideal_value(*_ideal(dy.t(), False))
    x_across = _ideal_value(*_ideal(xv.t(), False))
    return [torch.matmul(xv, wv.t()), torch.matmul(along, wv), torch.matmul(across, x_across.t())]
