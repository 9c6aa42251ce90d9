"""CPU: the MXFP4 entry points' exports and refusals, the scale layout, the
oracle's own format -- no GPU calls."""
from __future__ import annotations

import os
import re

import pytest
import torch

from conftest import ROOT
from oracle import mxfp4_oracle as O


def test_library_exports_the_declared_entries(pkg):
    src = open(os.path.join(ROOT, "include", "mxfp4.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = sorted(set(re.findall(r"\b(mxfp4_[a-z0-9_]+)\s*\(", src)))
    assert sorted(pkg._lib.MXFP4_SIGNATURES) == names
    lib = pkg.load_library()
    for n in names:
        assert hasattr(lib, n), n


def test_host_validation(pkg):
    """Bad arguments come back as a status and a message before any CUDA call."""
    lib = pkg.load_library()
    L = pkg._lib
    msg = lib.w8a8_last_error
    # (x, ldx, dtype, data, scales, M, K)
    assert lib.mxfp4_quant(None, 64, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"null" in msg()
    assert lib.mxfp4_quant(16, 64, 2, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"bf16 or fp16" in msg()
    assert lib.mxfp4_quant(16, 48, 0, 16, 16, 4, 48, None) == L.ERR_INVALID_ARG and b"multiple of 32" in msg()
    assert lib.mxfp4_quant(16, 32, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"stride" in msg()
    assert lib.mxfp4_quant(16, 68, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"stride" in msg()
    assert lib.mxfp4_quant(18, 64, 0, 16, 16, 4, 64, None) == L.ERR_ALIGNMENT
    assert lib.mxfp4_quant(16, 64, 0, 16, 16, -1, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_quant(None, 64, 0, None, None, 0, 64, None) == L.OK
    assert lib.mxfp4_dequant(16, 16, 16, 3, 4, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_dequant(16, 16, 24, 0, 4, 64, None) == L.ERR_ALIGNMENT
    assert lib.mxfp4_dequant(None, None, None, 0, 0, 64, None) == L.OK
    assert lib.mxfp4_silu_mul_quant(16, 64, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"2I" in msg()
    assert lib.mxfp4_silu_mul_quant(16, 96, 0, 16, 16, 4, 48, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_rmsnorm_quant(16, 64, None, 64, None, 1e-6, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_rmsnorm_quant(16, 64, None, 64, 16, -1.0, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG and b"eps" in msg()
    assert lib.mxfp4_rmsnorm_quant(16, 64, None, 64, 16, float("nan"), 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_rmsnorm_quant(16, 1 << 16, None, 64, 16, 1e-6, 0, 16, 16, 4, 1 << 16, None) == L.ERR_UNSUPPORTED
    assert lib.mxfp4_rmsnorm_quant(16, 64, 16, 32, 16, 1e-6, 0, 16, 16, 4, 64, None) == L.ERR_INVALID_ARG
    # (a, as, b, bs, bias, C, dtype, M, N, K)
    assert lib.mxfp4_gemm(16, 16, 16, 16, None, None, 0, 4, 64, 64, None) == L.ERR_INVALID_ARG and b"null" in msg()
    assert lib.mxfp4_gemm(16, 16, 16, 16, None, 16, 0, 4, 64, 80, None) == L.ERR_INVALID_ARG and b"multiple of 32" in msg()
    assert lib.mxfp4_gemm(16, 16, 16, 16, None, 16, 2, 4, 64, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_gemm(24, 16, 16, 16, None, 16, 0, 4, 64, 64, None) == L.ERR_ALIGNMENT
    assert lib.mxfp4_gemm(16, 16, 16, 16, None, 16, 0, 1 << 28, 64, 64, None) == L.ERR_UNSUPPORTED
    assert lib.mxfp4_gemm(None, None, None, None, None, None, 0, 0, 64, 64, None) == L.OK
    assert lib.mxfp4_gemm_silu_quant(16, 16, 16, 16, None, 0, 16, 16, 4, 96, 64, None) == L.ERR_UNSUPPORTED
    assert lib.mxfp4_gemm_silu_quant(16, 16, 16, 16, None, 0, None, 16, 4, 128, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_gemm_silu_quant(None, None, None, None, None, 0, None, None, 0, 128, 64, None) == L.OK
    assert lib.mxfp4_gemm_silu_quant_halves(16, 16, 16, 16, None, 0, 16, 16, 4, 80, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_gemm_silu_quant_halves(16, 16, 16, None, None, 0, 16, 16, 4, 96, 64, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_gemm_silu_quant_halves(None, None, None, None, None, 0, None, None, 0, 96, 64, None) == L.OK
    # (scales, half scales, I, K)
    assert lib.mxfp4_half_scales(16, 16, 80, 64, None) == L.ERR_INVALID_ARG and b"multiples of 32" in msg()
    assert lib.mxfp4_half_scales(16, 16, 96, 40, None) == L.ERR_INVALID_ARG
    assert lib.mxfp4_half_scales(None, 16, 96, 64, None) == L.ERR_INVALID_ARG and b"null" in msg()
    assert lib.mxfp4_half_scales(16, 24, 96, 64, None) == L.ERR_ALIGNMENT
    assert lib.mxfp4_half_scales(16, 16, 1 << 28, 64, None) == L.ERR_UNSUPPORTED
    assert lib.mxfp4_half_scales(None, None, 0, 64, None) == L.OK
    assert lib.mxfp4_scale_bytes(129, 288) == 2 * 4 * 512 and lib.mxfp4_scale_bytes(4, 40) == 0


@pytest.mark.parametrize("r,c", [(1, 1), (5, 8), (128, 9), (129, 33), (300, 4)])
def test_scale_tiles_round_trip(pkg, r, c):
    plain = torch.randint(0, 256, (r, c), dtype=torch.uint8, generator=torch.Generator().manual_seed(r + c))
    tiles = pkg.ops.mxfp4_tile_scales(plain)
    assert tuple(tiles.shape) == pkg.ops.mxfp4_scale_shape(r, 32 * c)
    assert tiles.numel() == pkg.load_library().mxfp4_scale_bytes(r, 32 * c)
    assert torch.equal(tiles, O.tile(plain.long()))
    t = pkg.ops.MXFP4Tensor(torch.zeros(r, 16 * c, dtype=torch.uint8), tiles)
    assert torch.equal(pkg.ops.mxfp4_plain_scales(t), plain)


def test_tensor_refusals(pkg):
    E = pkg.W8A8Error
    T = pkg.ops.MXFP4Tensor
    data = torch.zeros(4, 32, dtype=torch.uint8)
    tiles = torch.zeros(pkg.ops.mxfp4_scale_shape(4, 64), dtype=torch.uint8)
    assert tuple(T(data, tiles).shape) == (4, 64)
    for d, s in ((data.int(), tiles), (data[:, :24], tiles), (data[:, :24].contiguous(), tiles), (data[None], tiles),
                 (data, tiles[:, :1]), (data, tiles.int()), (data.t(), tiles), (data, tiles.flatten())):
        with pytest.raises(E, match="MXFP4Tensor"):
            T(d, s)


def test_ops_refuse_cpu_tensors_and_bad_operands(pkg):
    E, ops = pkg.W8A8Error, pkg.ops
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = ops.MXFP4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(ops.mxfp4_scale_shape(4, 64), dtype=torch.uint8))
    w = ops.MXFP4Tensor(torch.zeros(256, 32, dtype=torch.uint8),
                        torch.zeros(ops.mxfp4_scale_shape(256, 64), dtype=torch.uint8))
    short = ops.MXFP4Tensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(ops.mxfp4_scale_shape(4, 32), dtype=torch.uint8))
    for call in (lambda: ops.mxfp4_quant(x), lambda: ops.mxfp4_silu_and_mul_quant(x),
                 lambda: ops.mxfp4_rmsnorm_quant(x, x[0], 1e-6), lambda: ops.mxfp4_dequant(q),
                 lambda: ops.mxfp4_gemm(q, w), lambda: ops.mxfp4_gate_up_silu_quant(q, w)):
        with pytest.raises(E, match="no CPU path"):
            call()
    with pytest.raises(E, match="shape mismatch"):
        ops.mxfp4_gemm(short, w)
    with pytest.raises(E, match="bias"):
        ops.mxfp4_gemm(q, w, torch.zeros(128, dtype=torch.bfloat16))
    with pytest.raises(E, match="bias"):
        ops.mxfp4_gemm(q, w, torch.zeros(256, dtype=torch.float16))
    with pytest.raises(E, match="bf16 or fp16"):
        ops.mxfp4_gemm(q, w, out_dtype=torch.float32)
    with pytest.raises(E, match="bf16, fp16 or fp32"):
        ops.mxfp4_dequant(q, torch.float64)


def test_oracle_codes_are_the_nearest_values():
    """The restatement itself: every code is a nearest grid value, and each of
    the 16 codes decodes to its own value."""
    g = torch.Generator().manual_seed(3)
    t = torch.randn(1000, generator=g, dtype=torch.float64) * 3
    c = O.codes(t)
    grid = torch.tensor(O.GRID, dtype=torch.float64)
    best = (t.abs()[:, None] - grid).abs().amin(1)
    assert torch.equal((t.abs() - grid[c & 7]).abs(), best)
    y = torch.randn(7, 96, generator=g, dtype=torch.float64)
    c, b = O.quant(y)
    assert torch.equal(O.unpack(O.pack(c)), c) and torch.equal(O.untile(O.tile(b), 7, 3), b)
    assert ((O.values(c, b) - y).abs() <= torch.exp2((b - 127).double()).repeat_interleave(32, 1) * 2).all()
