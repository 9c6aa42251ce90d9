"""The microscaled 4-bit (MXFP4) operators of the linear path, as measured cases.

MXFP4: blocks of 32 consecutive values along the last dimension share one
power-of-two scale 2^(floor(log2 amax) - 2), held as an E8M0 byte (exponent +
127); each value is an E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives), rounded to nearest, ties to even, saturating at 6.  A block that
holds an infinity or a NaN has the NaN scale.  Two codes per byte, the even
index in the low half.  Scales lie in 512-byte tiles of 128 rows x 4 blocks
(row r, block c at (r % 32) * 16 + (r // 32) * 4 + c), tiles of a row group
consecutive along K and padded to a multiple of 256 values.

Operators (``op`` of a case):
  quant    activations to MXFP4, and the values that it stands for
  silu     silu(gate) * up, to MXFP4, and its values
  rmsnorm  residual add, RMSNorm, to MXFP4, its values and the new residual
  gemm     MXFP4 activations x MXFP4 weight^T (+ bias), bf16 or fp16
  mlp      the gated MLP: quantise, gate_up with silu * up and requantisation,
           down, from 16-bit activations to 16-bit outputs
"""
import importlib
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6


def listed():
    return [
        # one token's hidden state in front of qkv: pure latency
        {"name": "quant 1x5120", "op": "quant", "m": 1, "k": 5120, "ld": 5120, "dtype": "bf16"},
        # a prefill batch's attention output, a slice of a wider buffer's rows
        {"name": "quant 4096x8192 of 10240", "op": "quant", "m": 4096, "k": 8192, "ld": 10240, "dtype": "bf16"},
        # decode batch in front of down_proj
        {"name": "silu 33x25600", "op": "silu", "m": 33, "k": 25600, "ld": 51200, "dtype": "bf16"},
        # prefill in front of down_proj, half precision
        {"name": "silu 4096x12288 fp16", "op": "silu", "m": 4096, "k": 12288, "ld": 24576, "dtype": "fp16"},
        # one token through the norm in front of gate_up
        {"name": "rmsnorm 1x5120", "op": "rmsnorm", "m": 1, "k": 5120, "ld": 5120, "dtype": "bf16"},
        # a ragged prefill batch through the norm
        {"name": "rmsnorm 4097x5120", "op": "rmsnorm", "m": 4097, "k": 5120, "ld": 5120, "dtype": "bf16"},
        # gate_up for one token: the weight stream
        {"name": "gemm 1x51200x5120", "op": "gemm", "m": 1, "n": 51200, "k": 5120, "bias": False, "dtype": "bf16"},
        # down for a small decode batch: few output tiles, a long K
        {"name": "gemm 32x5120x25600", "op": "gemm", "m": 32, "n": 5120, "k": 25600, "bias": False, "dtype": "bf16"},
        # qkv with bias for a ragged mixed batch
        {"name": "gemm 333x10240x5120 bias", "op": "gemm", "m": 333, "n": 10240, "k": 5120, "bias": True, "dtype": "fp16"},
        # gate_up of a prefill batch
        {"name": "gemm 4096x51200x5120", "op": "gemm", "m": 4096, "n": 51200, "k": 5120, "bias": False, "dtype": "bf16"},
        # a decode batch through a whole MLP
        {"name": "mlp 16x4096x12288", "op": "mlp", "m": 16, "k": 4096, "i": 12288, "dtype": "bf16"},
        # a prefill batch through a whole MLP
        {"name": "mlp 8192x4096x12288", "op": "mlp", "m": 8192, "k": 4096, "i": 12288, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "silu", "rmsnorm", "gemm", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    m = _log(rng, 1, 8192)
    if op in ("quant", "rmsnorm"):
        k = 32 * _log(rng, 2, 256)
        return {"op": op, "m": m, "k": k, "ld": k + 8 * rng.choice([0, 0, 1, 40]), "dtype": dtype}
    if op == "silu":
        i = 32 * _log(rng, 2, 800)
        m = min(m, max(1, (1 << 27) // i))
        return {"op": op, "m": m, "k": i, "ld": 2 * i + 8 * rng.choice([0, 0, 3]), "dtype": dtype}
    if op == "gemm":
        k = 32 * _log(rng, 2, 800)
        n = _log(rng, 16, 51200)
        m = max(1, min(m, (1 << 40) // (n * k)))
        n = n if rng.random() < 0.25 else -(-n // 16) * 16
        return {"op": op, "m": m, "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": dtype}
    k = 32 * _log(rng, 4, 160)
    i = 32 * _log(rng, 4, 800)
    i = i if rng.random() < 0.25 else -(-i // 128) * 128
    return {"op": op, "m": max(1, min(m, (1 << 40) // (3 * i * k))), "k": k, "i": i, "dtype": dtype}


# ------------------------------------------------------------------ the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(m, k, ld, dtype, g):
    """Unit-normal rows with a few large channels, a view of rows `ld` apart."""
    x = torch.randn(m, ld, device="cuda", generator=g)
    x *= 1 + 12 * (torch.rand(ld, device="cuda", generator=g) > 0.998)
    return x.to(_TYPES[dtype])[:, :k]


def _pack(values):
    """Packed codes and scale bytes [R, K / 32] of fp32 rows (to make weights and activations to multiply)."""
    r, k = values.shape
    b = values.reshape(r, k // 32, 32)
    e = (torch.frexp(b.abs().amax(-1))[1] - 3).clamp(-127, 127)
    a = torch.ldexp(b, -e[..., None]).reshape(r, k)
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=values.device)
    c = torch.bucketize(a.abs(), grid, out_int32=True).to(torch.uint8) | ((a < 0).to(torch.uint8) << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _tiles(s):
    """Scale bytes [R, C] in the tiled order of the operators."""
    r, c = s.shape
    rb, ch = -(-r // 128), 2 * -(-c // 8)
    p = torch.zeros(rb * 128, ch * 4, dtype=torch.uint8, device=s.device)
    p[:r, :c] = s
    return p.view(rb, 4, 32, ch, 4).permute(0, 3, 2, 1, 4).reshape(rb, ch, 512).contiguous()


def _packed_normal(r, k, sigma, g):
    data = torch.empty(r, k // 2, dtype=torch.uint8, device="cuda")
    scale = torch.empty(r, k // 32, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // k)
    for at in range(0, r, step):
        w = torch.randn(min(step, r - at), k, device="cuda", generator=g) * sigma
        data[at:at + step], scale[at:at + step] = _pack(w)
    return data, _tiles(scale)


def prepare(case, seed):
    g = _generator(seed)
    op, m, k, dtype = case["op"], case["m"], case["k"], case["dtype"]
    t = _TYPES[dtype]
    s = {"op": op, "dtype": t}
    if op == "quant":
        s["x"] = _activations(m, k, case["ld"], dtype, g)
    elif op == "silu":
        s["x"] = _activations(m, 2 * k, case["ld"], dtype, g)
    elif op == "rmsnorm":
        s["x"] = _activations(m, k, case["ld"], dtype, g)
        s["residual"] = _activations(m, k, case["ld"], dtype, g)
        s["weight"] = (1 + 0.1 * torch.randn(k, device="cuda", generator=g)).to(t)
    elif op == "gemm":
        s["a"] = _packed_normal(m, k, 1.0, g)
        s["w"] = _packed_normal(case["n"], k, 0.02, g)
        s["bias"] = (0.1 * torch.randn(case["n"], device="cuda", generator=g)).to(t) if case["bias"] else None
    else:
        i = case["i"]
        s["x"] = _activations(m, k, k, dtype, g)
        s["gate_up"] = _packed_normal(2 * i, k, 0.02, g)
        s["down"] = _packed_normal(k, i, 0.02, g)
    return s


# ------------------------------------------------------------------ plain forms
def _quantised(y):
    """The MXFP4 values of [M, K] rows (32 or 64 bits), in the type of y."""
    m, k = y.shape
    b = y.reshape(m, k // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = torch.ldexp(b, -e)
    r = a.abs().clamp(max=6)
    step = torch.where(r < 2, 0.5, torch.where(r < 4, 1.0, 2.0)).to(y.dtype)
    v = torch.ldexp(torch.round(r / step) * step * torch.sign(a), e)
    return torch.where(amax.float().isfinite(), v, torch.nan).reshape(m, k)


def _values(packed):
    """fp32 values of packed rows and their scale tiles."""
    data, tiles = packed
    r, k = data.shape[0], 2 * data.shape[1]
    rb, ch = tiles.shape[0], tiles.shape[1]
    s = tiles.view(rb, ch, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, ch * 4)[:r, :k // 32].int() - 127
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=data.device)
    table = torch.cat([table, -table])
    codes = torch.stack([data & 15, data >> 4], dim=-1)
    v = table[codes.int()].reshape(r, k // 32, 32)
    return torch.ldexp(v, s[..., None]).reshape(r, k)


def _plain(state):
    op = state["op"]
    if op == "quant":
        return _quantised(state["x"].float()).bfloat16()
    if op == "silu":
        g, u = state["x"].double().chunk(2, dim=1)  # 64 bits: values next to a rounding border
        return _quantised(g / (1 + torch.exp(-g)) * u).bfloat16()
    if op == "rmsnorm":
        v = state["x"].float() + state["residual"].float()
        state["residual"].copy_(v)
        v = v.double()
        y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + _EPS) * state["weight"].double()
        return _quantised(y).bfloat16(), state["residual"]
    if op == "gemm":
        y = _values(state["a"]) @ _values(state["w"]).T
        return (y if state["bias"] is None else y + state["bias"].float()).to(state["dtype"])
    gu = _quantised(state["x"].float()) @ _values(state["gate_up"]).T
    g, u = gu.double().chunk(2, dim=1)
    y = _quantised(g / (1 + torch.exp(-g)) * u).float()
    return (y @ _values(state["down"]).T).to(state["dtype"])


def run(state):
    if not own:
        return _plain(state)
    ops = importlib.import_module("mini-sglang-fork_b200").ops
    op = state["op"]
    if op == "quant":
        return ops.mxfp4_dequant(ops.mxfp4_quant(state["x"]))
    if op == "silu":
        return ops.mxfp4_dequant(ops.mxfp4_silu_and_mul_quant(state["x"]))
    if op == "rmsnorm":
        q, residual = ops.mxfp4_rmsnorm_quant(state["x"], state["weight"], _EPS, state["residual"])
        return ops.mxfp4_dequant(q), residual
    if op == "gemm":
        return ops.mxfp4_gemm(ops.MXFP4Tensor(*state["a"]), ops.MXFP4Tensor(*state["w"]), state["bias"],
                              out_dtype=state["dtype"])
    y = ops.mxfp4_gate_up_silu_quant(ops.mxfp4_quant(state["x"]), ops.MXFP4Tensor(*state["gate_up"]))
    return ops.mxfp4_gemm(y, ops.MXFP4Tensor(*state["down"]), out_dtype=state["dtype"])


def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    four = lambda r, c: r * c * 17 / 32  # noqa: E731  codes and scales
    if op == "quant":  # read, the 4-bit form, its values
        return {"bytes": 2 * m * k + four(m, k) + 2 * m * k, "flops": 4 * m * k}
    if op == "silu":
        return {"bytes": 4 * m * k + four(m, k) + 2 * m * k, "flops": 10 * m * k}
    if op == "rmsnorm":
        return {"bytes": 6 * m * k + 2 * k + four(m, k) + 2 * m * k, "flops": 10 * m * k}
    if op == "gemm":
        n = case["n"]
        return {"bytes": four(m, k) + four(n, k) + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    i = case["i"]
    return {"bytes": 2 * m * k + four(2 * i, k) + four(k, i) + 2 * m * k, "flops": 6 * m * i * k}


# ------------------------------------------------------------------ 64 bits
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(y):
    """MXFP4 values by the definition: the nearest E2M1 number of each scaled value, the even code on a tie."""
    m, k = y.shape
    b = y.view(m, k // 32, 32)
    amax = b.abs().amax(-1, keepdim=True)
    p = torch.where(amax > 0, torch.floor(torch.log2(amax)), torch.full_like(amax, -125.0))
    p = torch.where(torch.exp2(p) > amax, p - 1, p)  # log2 rounded up at a power of two
    p = torch.where((torch.exp2(p + 1) <= amax) & (amax > 0), p + 1, p)
    scale = torch.exp2((p - 2).clamp(-127, 127))
    t = b.abs() / scale
    best = torch.zeros_like(t)
    for code in range(1, 8):  # ties go up exactly where the upper code is even
        border = (_GRID[code - 1] + _GRID[code]) / 2
        best = torch.where(t >= border if code % 2 == 0 else t > border, torch.full_like(t, _GRID[code]), best)
    out = torch.where(b < 0, -best, best) * scale
    return torch.where(amax <= torch.finfo(torch.float32).max, out, torch.full_like(out, math.nan)).view(m, k)


def _decoded(packed):
    data, tiles = packed
    r, k = data.shape[0], 2 * data.shape[1]
    row = torch.arange(r, device=data.device)[:, None]
    blk = torch.arange(k // 32, device=data.device)[None, :]
    s = tiles[row // 128, blk // 4, row % 32 * 16 + row % 128 // 32 * 4 + blk % 4]
    out = torch.empty(r, k, dtype=torch.float64, device=data.device)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=data.device)
    for half in (0, 1):
        c = (data >> (4 * half)) & 15
        out[:, half::2] = grid[(c & 7).long()] * (1 - 2 * (c >> 3).double())
    return out * torch.exp2(s.double() - 127).repeat_interleave(32, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        return _nearest(state["x"].double().contiguous())
    if op in ("silu", "mlp"):
        if op == "silu":
            gu = state["x"].double()
        else:
            gu = _nearest(state["x"].double().contiguous()) @ _decoded(state["gate_up"]).T
        i = gu.shape[1] // 2
        y = _nearest((gu[:, i:] * gu[:, :i] * torch.sigmoid(gu[:, :i])).contiguous())
        return y if op == "silu" else y @ _decoded(state["down"]).T
    if op == "rmsnorm":
        v = state["x"].double() + state["residual"].double()
        y = v / torch.sqrt((v * v).sum(1, keepdim=True) / v.shape[1] + _EPS) * state["weight"].double()
        return _nearest(y), v
    y = _decoded(state["a"]) @ _decoded(state["w"]).T
    return y if state["bias"] is None else y + state["bias"].double()
