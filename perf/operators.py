"""Cases of the microscaled 4-bit (MXFP4) operators of `kubernetes_amd.ops.hip_kernels`.

  mxfp4_quantize(x)                  -> q, scale     values to e2m1 codes and an e8m0 scale for each 32 of them
  mxfp4_dequantize(q, scale, ...)    -> x            the values that codes and scales stand for
  gemm_mxfp4_nt(a, sa, b, sb, ...)   -> a @ b.T      the product of two such matrices

Kinds of cases:
  quantize    values to 4 bits; the result is returned as the values it stands for, in x's type
  dequantize  a stored matrix to a wider type
  product     both operands stored in 4 bits
  linear      activations that arrive wide, quantised and multiplied with a stored weight

Sizes are those of the burn-in and of the tests of the framework's other matrix products, and generic ones.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token's activations on their way into a product
        {"name": "quantize-token", "kind": "quantize", "m": 1, "k": 8192, "type": "bf16", "view": "rows"},
        # an operand of the burn-in's size, a large weight
        {"name": "quantize-8192", "kind": "quantize", "m": 8192, "k": 8192, "type": "bf16", "view": "rows"},
        # rows that end inside a block, out of a wider matrix, from a checkpoint in 32 bits
        {"name": "quantize-odd", "kind": "quantize", "m": 1000, "k": 2041, "type": "fp32", "view": "slice"},
        # blocks along the other axis, as the products of a backward pass need them
        {"name": "quantize-transposed", "kind": "quantize", "m": 4096, "k": 8192, "type": "bf16", "view": "transposed"},
        # a stored weight for a path that computes in bf16
        {"name": "dequantize-8192", "kind": "dequantize", "m": 8192, "k": 8192, "type": "bf16"},
        # a small odd one, looked at in 32 bits
        {"name": "dequantize-odd", "kind": "dequantize", "m": 1000, "k": 2041, "type": "fp32"},
        # a single token through a layer
        {"name": "product-token", "kind": "product", "m": 1, "n": 4096, "k": 4096, "type": "bf16"},
        # a batch of sequences, a token each, through a large layer
        {"name": "product-batch", "kind": "product", "m": 32, "n": 8192, "k": 8192, "type": "bf16"},
        # nothing divides anything
        {"name": "product-odd", "kind": "product", "m": 1000, "n": 521, "k": 265, "type": "fp32"},
        # a prompt through a layer that is not large enough to fill the card with the largest tiles
        {"name": "product-prompt", "kind": "product", "m": 2048, "n": 1024, "k": 4096, "type": "bf16"},
        # the burn-in's product
        {"name": "product-8192", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "type": "fp32"},
        # wide activations of a short prompt, quantised and multiplied
        {"name": "linear-prompt", "kind": "linear", "m": 512, "n": 4096, "k": 4096, "type": "bf16"},
    ]


def _size(rng, low, high, step):
    """Spread over the logarithm; half of them on a multiple of `step`, half as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        v = max(step, v // step * step)
    return max(low, min(high, v))


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "dequantize", "product", "product", "linear"])
    case = {"kind": kind, "m": _size(rng, 1, 8192, 16), "k": _size(rng, 32, 8192, 128)}
    if kind == "quantize":
        case["type"] = rng.choice(["bf16", "fp16", "fp32"])
        case["view"] = rng.choice(["rows", "slice", "transposed"])
    elif kind == "dequantize":
        case["type"] = rng.choice(["bf16", "fp16", "fp32"])
    elif kind == "product":
        case["n"] = _size(rng, 16, 8192, 64)
        case["type"] = rng.choice(["bf16", "fp32"])
    else:
        case["n"] = _size(rng, 16, 8192, 64)
        case["type"] = "bf16"
    return case


# ---------------------------------------------------------------------------
# inputs

def _values(m, k, gen, dtype, spread):
    """Normal values; a few channels are much larger, as activations have them."""
    x = torch.randn(m, k, device="cuda", generator=gen)
    big = torch.rand(k, device="cuda", generator=gen) < 0.01
    return (x * torch.where(big, 20.0, 1.0) * spread).to(dtype)


def _packed(x):
    """A stored matrix: codes [m, 16 * blocks] and scales [m, blocks], both bytes."""
    code, scale = _codes(x)
    lo, hi = code[:, 0::2], code[:, 1::2]
    return (lo | (hi << 4)).contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, kind = case["m"], case["k"], case["kind"]
    state = dict(case, dtype=_TYPES[case["type"]])
    if kind == "quantize":
        if case["view"] == "transposed":
            state["x"] = _values(k, m, gen, state["dtype"], 1.0).t()
        elif case["view"] == "slice":
            state["x"] = _values(m, k + 71, gen, state["dtype"], 1.0)[:, 64:64 + k]
        else:
            state["x"] = _values(m, k, gen, state["dtype"], 1.0)
    elif kind == "dequantize":
        state["q"], state["scale"] = _packed(_values(m, k, gen, torch.float32, 0.05))
    else:
        a = _values(m, k, gen, torch.bfloat16, 1.0)
        if kind == "product":
            state["a"], state["a_scale"] = _packed(a)
        else:
            state["x"] = a
        state["b"], state["b_scale"] = _packed(_values(case["n"], k, gen, torch.bfloat16, 0.02))
    return state


# ---------------------------------------------------------------------------
# plain forms, in 32 bits

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes(x):
    """e2m1 codes [m, 32 * blocks] and e8m0 scales [m, blocks] of x [m, k]."""
    m, k = x.shape
    nb = (k + 31) // 32
    v = torch.zeros(m, nb * 32, device=x.device)
    v[:, :k] = x
    v = v.view(m, nb, 32)
    amax = v.abs().amax(dim=2)
    _, e = torch.frexp(amax)                       # amax = f * 2^e, f in [0.5, 1)
    s = torch.where(amax > 0, (e - 1 - 2 + 127).clamp(min=0), 0)
    v = torch.ldexp(v, (127 - s)[:, :, None])
    u = v.abs()
    # half-way values go to the even code
    code = ((u > 0.25).to(torch.uint8) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) + (u > 5.0))
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    return code.view(m, nb * 32), s.to(torch.uint8)


def _stand_for(code, scale):
    grid = torch.tensor(_GRID + tuple(-g for g in _GRID), device=code.device)
    v = grid[code.int()].view(scale.shape[0], scale.shape[1], 32)
    return torch.ldexp(v, (scale.int() - 127)[:, :, None]).view(code.shape)


def _unpacked(q):
    return torch.stack((q & 15, q >> 4), dim=2).view(q.shape[0], -1)


def run(state):
    kind, k, dtype = state["kind"], state["k"], state["dtype"]
    if own:
        from kubernetes_amd.ops import hip_kernels as hk
        if kind == "quantize":
            q, scale = hk.mxfp4_quantize(state["x"])
            return hk.mxfp4_dequantize(q, scale, k=k, dtype=dtype)
        if kind == "dequantize":
            return hk.mxfp4_dequantize(state["q"], state["scale"], k=k, dtype=dtype)
        if kind == "product":
            a, a_scale = state["a"], state["a_scale"]
        else:
            a, a_scale = hk.mxfp4_quantize(state["x"])
        return hk.gemm_mxfp4_nt(a, a_scale, state["b"], state["b_scale"], out_fp32=dtype == torch.float32)
    if kind == "quantize":
        return _stand_for(*_codes(state["x"]))[:, :k].to(dtype)
    if kind == "dequantize":
        return _stand_for(_unpacked(state["q"]), state["scale"])[:, :k].to(dtype)
    if kind == "product":
        a = _stand_for(_unpacked(state["a"]), state["a_scale"])
    else:
        a = _stand_for(*_codes(state["x"]))
    b = _stand_for(_unpacked(state["b"]), state["b_scale"])
    return (a @ b.t()).to(dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    m, k = case["m"], case["k"]
    size = 4 if case["type"] == "fp32" else 2
    nb = (k + 31) // 32
    if case["kind"] == "quantize":
        return {"bytes": 2 * m * k * size, "flops": 3 * m * k}
    if case["kind"] == "dequantize":
        return {"bytes": m * nb * 17 + m * k * size, "flops": m * k}
    n = case["n"]
    a_bytes = m * nb * 17 if case["kind"] == "product" else m * k * 2
    return {"bytes": a_bytes + n * nb * 17 + m * n * size, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _bits_to_values(q, scale):
    """Sign, exponent and fraction of each code by arithmetic, times 2^(scale - 127)."""
    out = torch.empty(q.shape[0], q.shape[1], 2, device=q.device, dtype=torch.float64)
    for half in (0, 1):
        c = (q.int() >> (4 * half)) & 15
        e, f = (c >> 1) & 3, (c & 1).double()
        v = torch.where(e == 0, 0.5 * f, (1.0 + 0.5 * f) * torch.exp2((e - 1).double()))
        out[:, :, half] = torch.where(c >= 8, -v, v)
    out = out.view(q.shape[0], -1, 32)
    return (out * torch.exp2(scale.double() - 127.0)[:, :, None]).view(q.shape[0], -1)


def _rounded(x):
    """x [m, k] on its blocks' grids: steps of half the leading power of two, of 0.5 below 1, at most 6."""
    m, k = x.shape
    nb = -(-k // 32)
    v = torch.nn.functional.pad(x.double(), (0, nb * 32 - k)).reshape(m * nb, 32)
    top = v.abs().max(dim=1).values
    unit = torch.exp2(torch.floor(torch.log2(top)).clamp(min=-125.0) - 2.0)[:, None]
    w = v / unit
    step = torch.exp2(torch.floor(torch.log2(w.abs().clamp(min=1.0)))) / 2
    w = (torch.round(w / step) * step).clamp(-6.0, 6.0) * unit
    return w.view(m, nb * 32)


def exact(case, seed):
    state = prepare(case, seed)
    kind, k = case["kind"], case["k"]
    if kind == "quantize":
        return _rounded(state["x"])[:, :k]
    if kind == "dequantize":
        return _bits_to_values(state["q"], state["scale"])[:, :k]
    a = _bits_to_values(state["a"], state["a_scale"]) if kind == "product" else _rounded(state["x"])
    return a @ _bits_to_values(state["b"], state["b_scale"]).t()
