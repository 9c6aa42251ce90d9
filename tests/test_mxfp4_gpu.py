"""GPU: the MXFP4 operators against 64-bit restatements (oracle/mxfp4_oracle.py).

The quantisers are compared code by code and scale by scale: their result is
defined by the exact value, so there is no tolerance.  The product is compared
within the bound of its arithmetic (``_gemm_bound``).
"""
from __future__ import annotations

import pytest
import torch

from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _no_timeouts(pkg, cuda_dev):
    yield
    torch.cuda.synchronize()
    assert pkg.ops.device_error() == 0, "a bounded wait gave up"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(q, want_codes, want_bytes):
    """An MXFP4Tensor holds these codes and scale bytes (a zero's sign apart),
    and zero scale bytes in the padding along K."""
    r, k = want_codes.shape
    assert tuple(q.shape) == (r, k)
    got_b = O.untile(q.scales, r, k // 32)
    assert torch.equal(got_b, want_bytes), (got_b != want_bytes).nonzero()[:4]
    got = O.unpack(q.data)
    zero = ((got & 7) == 0) & ((want_codes & 7) == 0)
    bad = (got != want_codes) & ~zero
    assert not bad.any(), (bad.nonzero()[:4], got[bad][:4], want_codes[bad][:4])
    cols = 4 * q.scales.shape[1]
    assert (O.untile(q.scales, r, cols)[:, k // 32:] == 0).all()


def _operand(pkg, r, k, sigma, seed, dev, spread=0):
    """A random MXFP4 operand and its fp64 values; `spread` widens the range of
    the block scales by that many powers of two."""
    g = _gen(seed)
    y = torch.randn(r, k, generator=g, dtype=torch.float64) * sigma
    if spread:
        y *= torch.exp2(torch.randint(-spread, spread + 1, (r, k // 32), generator=g).double()).repeat_interleave(32, 1)
    c, b = O.quant(y)
    t = pkg.ops.MXFP4Tensor(O.pack(c).to(dev), O.tile(b).to(dev))
    return t, O.values(c, b)


def _gemm_bound(k, mag, ref, dtype):
    """Half a step of the output type, plus fp32 accumulation: each of the K/32
    block sums is exact (64 products of 4-bit numbers), and each addition of
    one to the running sum may lose one fp32 step (2^-23, truncation allowed
    for) of the sum of magnitudes `mag`."""
    return torch.finfo(dtype).eps / 2 * ref.abs() + (k // 32 + 2) * 2.0 ** -23 * mag + 1e-30


# ------------------------------------------------------------------ quantisers
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (1, 5120, 0), (3, 64, 8), (33, 288, 0), (129, 1056, 40),
                                     (1000, 512, 0), (257, 8192, 8)])
def test_quant(pkg, cuda_dev, m, k, pad, dtype):
    x = (torch.randn(m, k + pad, generator=_gen(m + k)) * torch.exp2(
        torch.randint(-12, 10, (m, 1), generator=_gen(k)).float())).to(dtype).to(cuda_dev)[:, :k]
    q = pkg.ops.mxfp4_quant(x)
    _same(q, *O.quant(x.cpu().double()))
    for t in (torch.bfloat16, torch.float32):
        assert torch.equal(pkg.ops.mxfp4_dequant(q, t).cpu().double(), O.decode(q.data, q.scales))
    assert torch.equal(pkg.ops.mxfp4_dequant(q, torch.float16).cpu(), O.decode(q.data, q.scales).half())


def test_quant_every_bf16(pkg, cuda_dev):
    """Every bf16 pattern in blocks whose largest magnitude spans the type."""
    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16)
    v = bits.view(torch.bfloat16)
    x = torch.cat([v.reshape(-1, 32), v[torch.randperm(65536, generator=_gen(0))].reshape(-1, 32)])
    x = torch.cat([x.reshape(-1, 256)[:, torch.randperm(256, generator=_gen(i))] for i in range(2)]).to(cuda_dev)
    _same(pkg.ops.mxfp4_quant(x), *O.quant(x.cpu().double()))


@pytest.mark.parametrize("dtype", TYPES)
def test_quant_borders_and_extremes(pkg, cuda_dev, dtype):
    """Ties, saturation, zeros, subnormals, the type's ends, infinities and NaN."""
    fi = torch.finfo(dtype)
    rows = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5]
    for amax in (4.0, 6.0, 7.5):
        rows.append([amax] + [s * t for t in ties for s in (1, -1)] + [0.0] * 15)
    rows.append([0.0] * 32)
    rows.append([-0.0] * 32)
    rows.append([fi.max, fi.min] + [1.0] * 30)
    rows.append([fi.tiny] * 16 + [-fi.tiny] * 16)
    rows.append([fi.smallest_normal / 8 if dtype == torch.float16 else 2.0 ** -133] * 32)
    rows.append([float("inf")] + [1.0] * 31)
    rows.append([1.0] * 31 + [float("-inf")])
    rows.append([1.0] * 16 + [float("nan")] + [1.0] * 15)
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).to(cuda_dev)
    q = pkg.ops.mxfp4_quant(x)
    _same(q, *O.quant(x.cpu().double()))
    v = pkg.ops.mxfp4_dequant(q)
    assert v[-3:].isnan().all() and v[:-3].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,i,pad,sigma", [(1, 32, 0, 1.0), (33, 25600, 0, 1.0), (7, 96, 8, 4.0), (300, 1184, 0, 12.0),
                                           (2050, 768, 24, 1.0), (64, 512, 0, 60.0)])
def test_silu_quant(pkg, cuda_dev, m, i, pad, sigma, dtype):
    x = (torch.randn(m, 2 * i + pad, generator=_gen(m + i)) * sigma).to(dtype).to(cuda_dev)[:, :2 * i]
    q = pkg.ops.mxfp4_silu_and_mul_quant(x)
    g, u = x.cpu().chunk(2, dim=1)
    _same(q, *O.quant(O.silu_mul(g, u)))


def test_silu_quant_extremes(pkg, cuda_dev):
    """Far gates of both signs, the type's lowest value as a masked gate,
    subnormal gates under large ups, infinities and NaN, zero rows."""
    lo, hi = torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max
    inf, nan = float("inf"), float("nan")
    gates = [-30.0, -39.9, -41.0, -60.0, -87.0, -88.5, -90.0, -100.0, -120.0, -199.0, -201.0, -1e4, lo, 50.0, 1e4, hi,
             1e-38, 1e-39, -3e-40, 2.0 ** -101, 0.0, -0.0]
    ups = [1.0, -3.0, 1e30, hi, 1e-30, 0.0]
    rows = []
    for g in gates:
        for u in ups:
            rows.append(([g] * 32, [u * (1 + j / 64) if abs(u) < 1e38 else u for j in range(32)]))
    for g, u in ((inf, 1.0), (-inf, 1.0), (nan, 1.0), (1.0, inf), (1.0, nan), (0.0, inf)):
        rows.append(([g] + [1.0] * 31, [u] + [1.0] * 31))
    rows.append(([0.0] * 32, [0.0] * 32))
    x = torch.cat([torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])], 1).bfloat16().to(cuda_dev)
    q = pkg.ops.mxfp4_silu_and_mul_quant(x)
    g, u = x.cpu().chunk(2, dim=1)
    _same(q, *O.quant(O.silu_mul(g, u)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (1, 5120, 0), (37, 1056, 8), (300, 5120, 0), (5, 8192, 40),
                                     (3, 12288, 0), (2, 32768, 0), (700, 256, 0)])
def test_rmsnorm_quant(pkg, cuda_dev, m, k, pad, with_res, dtype):
    g = _gen(m + k)
    x = torch.randn(m, k + pad, generator=g).to(dtype).to(cuda_dev)[:, :k]
    res = torch.randn(m, k + pad, generator=g).to(dtype).to(cuda_dev) if with_res else None
    w = (1 + 0.1 * torch.randn(k, generator=g)).to(dtype).to(cuda_dev)
    before = res.clone() if with_res else None
    y, r = O.rmsnorm(x.cpu(), w.cpu(), 1e-6, before[:, :k].cpu() if with_res else None)
    q, out = pkg.ops.mxfp4_rmsnorm_quant(x, w, 1e-6, res[:, :k] if with_res else None)
    _same(q, *O.quant(y))
    if with_res:
        assert torch.equal(out.cpu(), r) and out.data_ptr() == res.data_ptr()
        assert torch.equal(res[:, k:], before[:, k:])  # what lies between the rows stays
    else:
        assert out is x


def test_rmsnorm_quant_extremes(pkg, cuda_dev):
    """Rows of zeros, tiny and huge values (a mean square outside fp32), eps 0,
    infinities and NaN."""
    k = 64
    g = _gen(5)
    base = torch.randn(k, generator=g)
    rows = [torch.zeros(k), base * 1e-36, base * 1e-39, base * 1e37, base, base.clone(), base.clone()]
    rows[5][7] = float("inf")
    rows[6][9] = float("nan")
    x = torch.stack(rows).bfloat16().to(cuda_dev)
    w = torch.ones(k, dtype=torch.bfloat16, device=cuda_dev)
    for eps in (1e-6, 0.0):
        y, _ = O.rmsnorm(x.cpu(), w.cpu(), eps)
        q, _ = pkg.ops.mxfp4_rmsnorm_quant(x, w, eps)
        _same(q, *O.quant(y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(8, 1056), (600, 5120)])
def test_rmsnorm_quant_rows_that_are_not_finite(pkg, cuda_dev, m, k, dtype):
    """Infinities and NaN in some rows' input, residual and weight: zeros and NaN
    blocks in those rows, and no other row is touched."""
    g = _gen(m + k)
    x, r = (torch.randn(m, k, generator=g).to(dtype) for _ in range(2))
    x[1, 40] = float("inf")
    x[2, 700] = float("-inf")
    r[2, 3] = float("inf")
    x[3, 5] = float("nan")
    x[4, 100], r[4, 100] = float("inf"), float("-inf")
    x[5, 64:96] = float("inf")
    for special in (None, float("inf"), float("nan"), 0.0):
        w = (1 + 0.1 * torch.randn(k, generator=_gen(k))).to(dtype)
        if special is not None:
            w[300] = special
        y, want = O.rmsnorm(x, w, 1e-6, r)
        q, out = pkg.ops.mxfp4_rmsnorm_quant(x.to(cuda_dev), w.to(cuda_dev), 1e-6, r.to(cuda_dev))
        _same(q, *O.quant(y))
        assert torch.equal(out.cpu().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))


@pytest.mark.parametrize("seed,row", [(463, 57), (688, 14), (1247, 29), (3629, 59)])
@pytest.mark.parametrize("whole", [False, True])
def test_rmsnorm_quant_next_to_a_border(pkg, cuda_dev, seed, row, whole):
    """Rows in which a value is so close to a rounding border that a sum of
    squares with fp32 additions in it gives the neighbouring code; alone and
    among others."""
    g = _gen(seed)
    x = torch.randn(64, 2048, generator=g).bfloat16()
    r = torch.randn(64, 2048, generator=g).bfloat16()
    w = (1 + 0.3 * torch.randn(2048, generator=g)).bfloat16()
    if whole:
        x, r = x.repeat(8, 1), r.repeat(8, 1)
    else:
        x, r = x[row:row + 1].contiguous(), r[row:row + 1].contiguous()
    y, _ = O.rmsnorm(x, w, 1e-6, r)
    q, _ = pkg.ops.mxfp4_rmsnorm_quant(x.to(cuda_dev), w.to(cuda_dev), 1e-6, r.to(cuda_dev))
    _same(q, *O.quant(y))


def test_rmsnorm_quant_tiny_values_under_large_weights(pkg, cuda_dev):
    """v / rms or weight / rms below fp32's range, lifted back into it by the other
    factor: 1e-38 / 1e10 times 1e30 is 1e-18, in blocks of their own and next to
    zeros, and 1e10 / 1e10 times 1e-36 stays what it is."""
    k = 256
    g = _gen(11)
    x = torch.randn(8, k, generator=g)
    x[:, :64] *= 1e10
    x[0, 64:] *= 1e-38
    x[1, 64:] *= 1e-30
    x[2, 64:] *= 1e-36
    x[3, 64:] = 0.0
    x[4, 64:] *= 1e-38
    x[4, 70:90] = 0.0
    x[5, 64:] *= 1e-28
    x[6, :32] = 0.0
    x[7, 32:64] *= 1e-5
    x = x.bfloat16().to(cuda_dev)
    w = (torch.randn(k, generator=g) * 1e30).bfloat16()
    w[:32] = 1.0
    w[32:48] = 1e-30
    w[48:64] = 1e-36
    w[64:96] = 0.0
    w[128:160] = 2.0
    w[224:] = 1e-30
    w = w.to(cuda_dev)
    for res in (None, torch.zeros_like(x)):
        y, _ = O.rmsnorm(x.cpu(), w.cpu(), 1e-6, None if res is None else res.cpu())
        q, _ = pkg.ops.mxfp4_rmsnorm_quant(x, w, 1e-6, res)
        _same(q, *O.quant(y))


# --------------------------------------------------------------------- product
@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 16, 32), (16, 128, 256), (1, 1, 32), (5, 130, 96), (16, 384, 1056), (17, 200, 512),
                                   (32, 256, 2080), (33, 512, 768), (64, 1000, 4096), (65, 384, 320), (128, 256, 1024),
                                   (129, 257, 288), (300, 1024, 512), (1, 2048, 8192), (513, 640, 1280),
                                   # 256 x 256 blocks: whole, ragged in M, N and K, several per SM pair
                                   (4096, 1024, 256), (2000, 2040, 544), (129, 9600, 96), (1025, 4099, 320),
                                   (3000, 8192, 1056)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gemm(pkg, cuda_dev, m, n, k, dtype):
    a, av = _operand(pkg, m, k, 1.0, m + k, cuda_dev)
    w, wv = _operand(pkg, n, k, 0.05, n + k, cuda_dev, spread=2)
    bias = (0.1 * torch.randn(n, generator=_gen(n))).to(dtype).to(cuda_dev)
    ref = (av.to(cuda_dev) @ wv.to(cuda_dev).T).cpu()
    mag = (av.abs().to(cuda_dev) @ wv.abs().to(cuda_dev).T).cpu()
    for b in (None, bias):
        want = ref if b is None else ref + b.cpu().double()
        out = pkg.ops.mxfp4_gemm(a, w, b, out_dtype=dtype)
        assert out.dtype == dtype and tuple(out.shape) == (m, n)
        err = (out.cpu().double() - want).abs()
        bound = _gemm_bound(k, mag, want, dtype)
        assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (40, 128, 1024), (200, 384, 256), (512, 512, 2048), (1024, 2560, 256)])
def test_gemm_nan_scales_and_wide_scales(pkg, cuda_dev, m, n, k):
    """A NaN-scaled block makes its output row (or column) NaN and no other;
    scales at both ends of E8M0 multiply as numbers."""
    a, av = _operand(pkg, m, k, 1.0, 1, cuda_dev, spread=8)
    w, wv = _operand(pkg, n, k, 1.0, 2, cuda_dev, spread=8)
    plain = pkg.ops.mxfp4_plain_scales(a).clone()
    plain[m // 2, k // 64] = 255
    a = pkg.ops.MXFP4Tensor(a.data, pkg.ops.mxfp4_tile_scales(plain))
    wplain = pkg.ops.mxfp4_plain_scales(w).clone()
    wplain[n // 3] = 0  # 2^-127
    wplain[n - 1, 0] = 255
    w = pkg.ops.MXFP4Tensor(w.data, pkg.ops.mxfp4_tile_scales(wplain))
    out = pkg.ops.mxfp4_gemm(a, w).cpu()
    av, wv = O.decode(a.data, a.scales), O.decode(w.data, w.scales)
    want = av @ wv.T
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[m // 2] = True
    nan[:, n - 1] = True
    assert torch.equal(out.isnan(), nan)
    err = (out.double() - want).abs()
    bound = _gemm_bound(k, av.nan_to_num(0).abs() @ wv.nan_to_num(0).abs().T, want, torch.bfloat16)
    assert (err[~nan] <= bound[~nan]).all()


def _silu_gemm_check(y, gv, uv, slack):
    """`y` quantises, block by block, some value within a relative `slack` of
    silu(g) * u (g, u fp64, exact): codes between those of the two ends under
    the scale of one of the two ends."""
    want = O.silu_mul(gv, uv)
    r, k = want.shape
    byte = O.untile(y.scales, r, k // 32)
    _, lo_b = O.quant(want * (1 - slack))
    _, hi_b = O.quant(want * (1 + slack))
    assert ((byte == lo_b) | (byte == hi_b)).all()
    got = O.values(O.unpack(y.data), byte).abs()
    lo = O.values(*O.quant(want * (1 - slack), byte)).abs()
    hi = O.values(*O.quant(want * (1 + slack), byte)).abs()
    assert ((got >= lo) & (got <= hi)).all()
    sign = O.values(O.unpack(y.data), byte) * want
    assert (sign >= 0).all()
    cols = 4 * y.scales.shape[1]
    assert (O.untile(y.scales, r, cols)[:, k // 32:] == 0).all()


@pytest.mark.parametrize("m,i,k", [(1, 128, 64), (16, 256, 512), (9, 384, 1056), (32, 128, 288), (50, 512, 256), (64, 128, 2048),
                                   (100, 256, 96), (128, 384, 1024), (130, 128, 512), (333, 768, 640),
                                   (2000, 640, 544), (129, 4992, 96), (3000, 2048, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gate_up_silu_quant(pkg, cuda_dev, m, i, k, dtype):
    _gate_up_check(pkg, cuda_dev, m, i, k, dtype)


def _gate_up_check(pkg, cuda_dev, m, i, k, dtype):
    """The fused epilogue on operands whose sums are exact in fp32 (block
    scales within a few powers of two, K small: every product is a multiple of
    2^-2 of the smallest scale product and the sums stay below 2^22 of those),
    so that only silu's own evaluation (2^-18 relative) lies between its result
    and the definition."""
    a, av = _operand(pkg, m, k, 1.0, m + k, cuda_dev)
    w, wv = _operand(pkg, 2 * i, k, 0.05, i + k, cuda_dev)
    bias = torch.randint(-8, 9, (2 * i,), generator=_gen(i)).to(dtype) / 16
    full = (av.to(cuda_dev) @ wv.to(cuda_dev).T).cpu()
    assert torch.equal(full.float().double(), full)
    for b in (None, bias):
        gu = full if b is None else full + b.double()
        y = pkg.ops.mxfp4_gate_up_silu_quant(a, w, None if b is None else b.to(cuda_dev), dtype)
        assert tuple(y.shape) == (m, i)
        _silu_gemm_check(y, gu[:, :i], gu[:, i:], 2.0 ** -17)


@pytest.mark.parametrize("m,i,k", [(3, 32, 64), (40, 160, 512), (300, 96, 256)])
def test_gate_up_silu_quant_ragged(pkg, cuda_dev, m, i, k):
    """I % 128 != 0: the up rows start inside a scale tile and the last tile is
    not full; held to the definition as the full tiles are."""
    _gate_up_check(pkg, cuda_dev, m, i, k, torch.bfloat16)


@pytest.mark.parametrize("m,i,k", [(1, 32, 32), (1, 4896, 512), (16, 224, 1056), (33, 288, 4096), (64, 5216, 288),
                                   (65, 32, 64), (130, 416, 768), (257, 1312, 320), (1000, 10912, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gate_up_silu_quant_ragged_sizes(pkg, cuda_dev, m, i, k, dtype):
    _gate_up_check(pkg, cuda_dev, m, i, k, dtype)
