"""GPU: the gate_up product's epilogue, code by code (its result is the
quantisation of the exact silu(gate) * up of its fp32 sums, which these tests
make exact), and products whose K several CTAs or SM pairs share."""
from __future__ import annotations

import pytest
import torch

from oracle import mxfp4_oracle as O
from test_mxfp4_gpu import _gemm_bound, _gen, _no_timeouts, _operand, _same  # noqa: F401

pytestmark = pytest.mark.gpu

BITS = 24


def _sums(pkg, dev, values, m, k):
    """Operands whose product is exactly `values` (fp32 [N]) in each of `m` rows:
    a is 1 in the first column of every 32-value block, and a weight row has one
    bit of its value in each of 24 blocks, spread over K from the highest down,
    so that every partial sum is a 24-bit number."""
    n = values.numel()
    a = torch.zeros(m, k, dtype=torch.long)
    a[:, ::32] = 2  # the code of 1
    a = pkg.MXFP4Tensor(O.pack(a).to(dev), O.tile(torch.full((m, k // 32), 127)).to(dev))
    mant, exp = torch.frexp(values.double().abs())
    whole = (mant * 2 ** BITS).long()  # 24 bits, the highest set
    assert torch.equal(whole.double() * torch.exp2((exp - BITS).double()), values.double().abs())
    codes = torch.zeros(n, k, dtype=torch.long)
    scales = torch.zeros(n, k // 32, dtype=torch.long)
    for b in range(BITS):
        at = b * (k // 32) // BITS
        bit = (whole >> (BITS - 1 - b)) & 1
        codes[:, 32 * at] = bit * torch.where(values < 0, 10, 2)
        scales[:, at] = (exp - 1 - b + 127).clamp(min=0)
        assert ((exp - 1 - b + 127 >= 0) | (bit == 0)).all()
    return a, pkg.MXFP4Tensor(O.pack(codes).to(dev), O.tile(scales).to(dev))


def _check(pkg, dev, gate, up, m, k):
    i = gate.numel()
    a, w = _sums(pkg, dev, torch.cat([gate, up]), m, k)
    y = pkg.mxfp4_gate_up_silu_quant(a, w)
    want, byte = O.quant(O.silu_mul(gate, up)[None])
    _same(y, want.expand(m, i), byte.expand(m, -1))


# K 768: one share of K; 4096 and 8192: several CTAs, or two SM pairs, share a block's
SHAPES = [(1, 128, 768), (20, 160, 768), (64, 256, 1536), (100, 384, 768), (300, 416, 768),
          (1, 256, 8192), (17, 160, 8192), (50, 128, 12288), (130, 256, 4096), (300, 352, 8192)]


@pytest.mark.parametrize("m,i,k", SHAPES)
def test_values_next_to_borders(pkg, cuda_dev, m, i, k):
    """Products within fp32's rounding of a border between two codes, in a block
    whose scale is 1 (its first product is near 6), and largest products next to
    a power of two."""
    g = _gen(m + i)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for seed in range(3):
        target = borders[torch.randint(0, 7, (i,), generator=g)]
        target[::32] = 6.3
        target[32::64] = 4.0  # just below or above: the block's scale hangs on it
        target *= torch.randint(0, 2, (i,), generator=g) * 2 - 1
        gate = torch.where(torch.rand(i, generator=g) < 0.5, 1.0, -1.0) * torch.rand(i, generator=g) * 12 + 0.01
        up = (target.double() / O.silu_mul(gate, torch.ones(i))).float()
        _check(pkg, cuda_dev, gate, up, m, k)


@pytest.mark.parametrize("m,i,k", [(1, 128, 768), (20, 160, 768), (100, 384, 768), (17, 160, 8192), (300, 352, 8192)])
def test_far_gates(pkg, cuda_dev, m, i, k):
    """Gates between -40 and -190, where the sigmoid leaves fp32's range, under
    ups that lift the product back into it (up to 2^127): the values, some next to
    a border; blocks that mix them with ordinary gates, and blocks of one gate."""
    g = _gen(m + i)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.3, 1.0, 0.1])
    for seed in range(6):
        gate = -torch.rand(i, generator=g) * (45, 85, 150, 150, 150, 8)[seed] - (40.0 if seed < 5 else 84.0)
        if seed == 3:
            gate[::3] = torch.randn(gate[::3].numel(), generator=g) * 4 + 0.01
        if seed >= 4:
            gate = gate[::32].repeat_interleave(32)
        shape = O.silu_mul(gate, torch.ones(i))
        target = borders[torch.randint(0, 10, (i,), generator=g)].double()
        target[::32] = 6.3
        # each block's scale: within fp32's range, and such that every up is below 2^127
        most = torch.floor(torch.log2(shape.abs().reshape(-1, 32).amin(1)) + 127 - 3).clamp(max=20)
        target *= torch.exp2(torch.maximum(most - (0, 3, 6, 9, 12, 20)[seed], torch.full_like(most, -95.0))).repeat_interleave(32)
        up = (target / shape).float().clamp(-1.7e38, 1.7e38)
        up *= (torch.randint(0, 2, (i,), generator=g) * 2 - 1)
        want = O.silu_mul(gate, up)
        assert (want.abs() > 0).any() and (gate < -40).any()
        _check(pkg, cuda_dev, gate, up, m, k)


@pytest.mark.parametrize("m,k", [(1, 768), (40, 768), (100, 768), (64, 8192), (300, 8192)])
def test_gates_and_ups_that_are_not_finite(pkg, cuda_dev, m, k):
    """Infinite and NaN sums make their blocks NaN, next to values of any size; a
    product beyond fp32 does, one whose factors' product alone overflows does not;
    blocks without them are not touched."""
    i, big = 384, 2.0 ** 127
    g = _gen(m)
    gate, up = (torch.randn(i, generator=g) + 0.01 for _ in range(2))
    gate[1] = gate[6 * 32] = -1000.0
    gate[2 * 32], up[2 * 32] = 300.0, 1e37       # 3e39
    gate[3 * 32], up[3 * 32] = -20.0, 1.5 * big  # -20 e^-20 1.5 2^127: finite
    gate[4 * 32], up[4 * 32] = -95.0, -big
    a, w = _sums(pkg, cuda_dev, torch.cat([gate, up]), m, k)
    # a column that no other value uses: 4 times 2^127, or the NaN scale
    plain = pkg.ops.mxfp4_plain_scales(w).cpu()
    codes = O.unpack(w.data)
    want_g, want_u = gate.clone(), up.clone()
    free = next(c for c in range(k // 32) if c not in {b * (k // 32) // BITS for b in range(BITS)}) if k > 768 else None
    for row, code, byte in ((6 * 32, 6, 254), (7 * 32 + 5, 14, 254), (8 * 32 + 31, 0, 255), (i + 9 * 32 + 1, 6, 254),
                            (i + 10 * 32 + 2, 0, 255)):
        at = 0 if free is None else free
        codes[row] = 0  # its own value goes
        codes[row, 32 * at] = code
        plain[row, at] = byte
        (want_g if row < i else want_u)[row % i] = float("nan") if byte == 255 else float("inf") * (-1 if code == 14 else 1)
    w = pkg.MXFP4Tensor(O.pack(codes).to(cuda_dev), pkg.ops.mxfp4_tile_scales(plain).to(cuda_dev))
    y = pkg.mxfp4_gate_up_silu_quant(a, w)
    want, byte = O.quant(O.silu_mul(want_g, want_u)[None])
    assert (byte[0] == 255).nonzero().flatten().tolist() == [2, 6, 7, 8, 9, 10]
    _same(y, want.expand(m, i), byte.expand(m, -1))


def _exact_sums(a, w, av, wv):
    """The products' sums, which fp32 holds exactly in any order: each product is
    a multiple of the unit below, and no partial sum reaches 2^24 of them."""
    def least(t):
        r, k = t.shape
        return O.untile(t.scales, r, k // 32).min().item() - 127

    unit = 2.0 ** (least(a) + least(w) - 2)
    assert (av.abs() @ wv.abs().T).max() < 2 ** 23 * unit
    return av @ wv.T


# K 4096 and more with few blocks: two SM pairs, or up to eight CTAs, share a block's K
@pytest.mark.parametrize("m,i,k", [(1, 128, 4096), (16, 256, 8192), (40, 160, 12288), (64, 128, 16384), (64, 416, 8192),
                                   (65, 128, 4096), (129, 256, 8192), (200, 416, 8192), (256, 128, 25600), (333, 96, 8192),
                                   (500, 608, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shares_of_k(pkg, cuda_dev, m, i, k, dtype):
    """With and without biases, the intermediate size a multiple of 128 or not."""
    a, av = _operand(pkg, m, k, 1.0, m + k, cuda_dev)
    w, wv = _operand(pkg, 2 * i, k, 0.05, i + k, cuda_dev)
    full = _exact_sums(a, w, av.to(cuda_dev), wv.to(cuda_dev)).cpu()
    bias = torch.randint(-8, 9, (2 * i,), generator=_gen(i)).to(dtype) / 16
    for b in (None, bias):
        gu = (full if b is None else full + b.double()).float()
        y = pkg.mxfp4_gate_up_silu_quant(a, w, None if b is None else b.to(cuda_dev), dtype)
        _same(y, *O.quant(O.silu_mul(gu[:, :i], gu[:, i:])))


@pytest.mark.parametrize("m,n,k", [(129, 500, 4096), (129, 256, 25600), (200, 1000, 8192), (256, 1280, 8192), (333, 643, 4096),
                                   (333, 640, 25600), (500, 250, 8192), (500, 2056, 4096), (1000, 130, 4128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_product_shares_of_k(pkg, cuda_dev, m, n, k, dtype):
    """The plain product where two SM pairs share a block's K: ragged M, N and K,
    with and without a bias."""
    a, av = _operand(pkg, m, k, 1.0, m + k, cuda_dev, spread=1)
    w, wv = _operand(pkg, n, k, 0.05, n + k, cuda_dev, spread=2)
    av, wv = av.to(cuda_dev), wv.to(cuda_dev)
    ref, mag = (av @ wv.T).cpu(), (av.abs() @ wv.abs().T).cpu()
    bias = (0.1 * torch.randn(n, generator=_gen(n))).to(dtype)
    for b in (None, bias):
        want = ref if b is None else ref + b.double()
        out = pkg.mxfp4_gemm(a, w, None if b is None else b.to(cuda_dev), out_dtype=dtype)
        err = (out.cpu().double() - want).abs()
        assert (err <= _gemm_bound(k, mag, want, dtype)).all()
