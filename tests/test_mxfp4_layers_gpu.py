"""GPU: the MXFP4 layer classes against the 64-bit restatement, the operators
together as a decoder layer runs them (eager, captured, on several streams),
and the calls at the edges: no rows, rows inside larger buffers, more than 2^32
values, refused alignments."""
from __future__ import annotations

import subprocess
import sys
import threading

import pytest
import torch

from conftest import ROOT
from oracle import mxfp4_oracle as O
from test_mxfp4_gpu import _gemm_bound, _gen, _operand, _same

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _tp1(pkg, cuda_dev):
    pkg.reset_tp_info()
    pkg.set_tp_info(0, 1)
    yield
    pkg.reset_tp_info()
    torch.cuda.synchronize()
    assert pkg.ops.device_error() == 0, "a bounded wait gave up"


def _load(pkg, layer, dev, seed, dtype=torch.bfloat16, prefix="x"):
    """Loads random weights into a layer through the checkpoint loader."""
    g = _gen(seed)
    items = []
    for key, t in layer.state_dict(prefix=prefix).items():
        if key.endswith("weight_scale"):
            continue
        if key.endswith("weight") and t.dim() == 2:  # a packed linear weight
            n, k = t.shape[0], 2 * t.shape[1]
            w = (torch.randn(n, k, generator=g) * 0.05).to(dtype)
            items.append((key, w))
        else:
            items.append((key, (1 + 0.1 * torch.randn(t.shape, generator=g)).to(dtype)))
    sd = {}
    for key, w in items:
        if w.dim() == 2:
            q = pkg.ops.mxfp4_quant(w.to(dev))
            sd[key], sd[key + "_scale"] = q.data, q.scales
        else:
            sd[key] = w.to(dev)
    layer.load_state_dict(sd, prefix=prefix)
    return layer


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 7, 64, 300])
def test_each_layer_class(pkg, cuda_dev, m, dtype):
    L, h, hd, nq, nkv, inter = pkg.mxfp4, 512, 64, 8, 2, 768
    layers = [L.LinearQKVMerged(h, hd, nq, nkv, True, dtype), L.LinearOProj(nq * hd, h, False, dtype),
              L.LinearColParallelMerged(h, [inter, inter], False, dtype), L.LinearRowParallel(inter, h, False, dtype),
              L.LinearReplicated(h, 250, True, dtype)]
    for i, layer in enumerate(layers):
        _load(pkg, layer, cuda_dev, i + 10 * m, dtype)
        k = layer.local_input_size
        x = torch.randn(m, k, generator=_gen(m + i)).to(dtype)
        y = layer.forward(x.to(cuda_dev))
        assert y.dtype == dtype and tuple(y.shape) == (m, layer.local_output_size)
        av = O.values(*O.quant(x.double()))
        wv = O.decode(layer.weight, layer.weight_scale)
        want = av @ wv.T + (0 if layer.bias is None else layer.bias.cpu().double())
        assert ((y.cpu().double() - want).abs() <= _gemm_bound(k, av.abs() @ wv.abs().T, want, dtype)).all()


def test_loader_on_the_device(pkg, cuda_dev):
    """Quantise-at-load with the CUDA quantiser: the layer's weight is the
    restatement's quantisation of the checkpoint's."""
    w = (torch.randn(96, 128, generator=_gen(0)) * 0.02).bfloat16()
    sd = pkg.load_mxfp4_state_dict([("m.o_proj.weight", w)], 0, 1, 1, device=cuda_dev)
    assert sd["m.o_proj.weight"].is_cuda
    c, b = O.quant(w.double())
    assert torch.equal(O.unpack(sd["m.o_proj.weight"]), c)
    assert torch.equal(O.untile(sd["m.o_proj.weight_scale"], 96, 4), b)


class _Decoder:
    """The linear path of a decoder layer, the attention replaced by the q
    slice of the qkv output (a strided view)."""

    def __init__(self, pkg, dev, h=512, nq=8, nkv=2, hd=64, inter=1024, seed=0):
        L = pkg.mxfp4
        self.pkg, self.nq = pkg, nq * hd
        self.n1 = _load(pkg, L.RMSNormFusedQuant(h, 1e-6), dev, seed)
        self.qkv = _load(pkg, L.LinearQKVMerged(h, hd, nq, nkv, True), dev, seed + 1)
        self.o = _load(pkg, L.LinearOProj(nq * hd, h, False), dev, seed + 2)
        self.n2 = _load(pkg, L.RMSNormFusedQuant(h, 1e-6), dev, seed + 3)
        self.mlp = _load(pkg, L.GatedMLP(h, inter), dev, seed + 4)

    def __call__(self, x, residual):
        q, residual = self.n1.forward(x, residual)
        attn = self.qkv.forward(q)[:, :self.nq]
        q, residual = self.n2.forward(self.o.forward(attn), residual)
        return self.mlp.forward(q), residual


def _inputs(m, dev, seed, h=512):
    g = _gen(seed)
    return (torch.randn(m, h, generator=g).bfloat16().to(dev), torch.randn(m, h, generator=g).bfloat16().to(dev))


@pytest.mark.parametrize("m", [1, 5, 40, 130, 700])
def test_decoder_layer(pkg, cuda_dev, m):
    """Step by step against the restatement, each step from the kernel's own
    input, so that every tolerance is one step's."""
    d = _Decoder(pkg, cuda_dev)
    x, r = _inputs(m, cuda_dev, m)
    y_ref, r_ref = O.rmsnorm(x.cpu(), d.n1.weight.cpu(), 1e-6, r.cpu())
    q, r1 = d.n1.forward(x, r)
    _same(q, *O.quant(y_ref))
    assert torch.equal(r1.cpu(), r_ref)

    def linear(a, layer, out):
        av, wv = O.decode(a.data, a.scales), O.decode(layer.weight, layer.weight_scale)
        want = av @ wv.T + (0 if layer.bias is None else layer.bias.cpu().double())
        bound = _gemm_bound(av.shape[1], av.abs() @ wv.abs().T, want, out.dtype)
        assert ((out.cpu().double() - want).abs() <= bound).all()

    qkv = d.qkv.forward(q)
    linear(q, d.qkv, qkv)
    a = pkg.mxfp4_quant(qkv[:, :d.nq])
    _same(a, *O.quant(qkv[:, :d.nq].cpu().double()))
    o = d.o.forward(a)
    linear(a, d.o, o)
    y_ref, r_ref = O.rmsnorm(o.cpu(), d.n2.weight.cpu(), 1e-6, r1.cpu())
    q2, r2 = d.n2.forward(o, r1)
    _same(q2, *O.quant(y_ref))
    y = d.mlp.gate_up_proj.forward_silu_quant(q2)
    out = d.mlp.down_proj.forward(y)
    linear(y, d.mlp.down_proj, out)
    # and the same as one call
    x, r = _inputs(m, cuda_dev, m)
    out2, r3 = d(x, r)
    assert torch.equal(out2, out) and torch.equal(r3, r2)


def test_decoder_layer_captured(pkg, cuda_dev):
    """Two captured graphs of the same layers (no workspace is shared), their
    replays interleaved on two streams with new inputs each time, give what
    eager calls give, bit for bit."""
    d = _Decoder(pkg, cuda_dev)
    sizes = (3, 300)
    want = {(m, s): d(*_inputs(m, cuda_dev, s)) for m in sizes for s in range(3)}
    graphs = []
    for m in sizes:
        stream = torch.cuda.Stream()
        x, r = _inputs(m, cuda_dev, 0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            rr = r.clone()
            out = d(x, rr)
        graphs.append((m, g, stream, x, r, out))
    for s in range(3):
        got = []
        for m, g, stream, x, r, out in graphs:
            with torch.cuda.stream(stream):
                a, b = _inputs(m, cuda_dev, s)
                x.copy_(a)
                r.copy_(b)
                g.replay()
                got.append((m, [t.clone() for t in out]))
        torch.cuda.synchronize()
        for m, out in got:
            for u, v in zip(out, want[m, s]):
                assert torch.equal(u, v)


@pytest.mark.parametrize("m", [5, 40, 300])
def test_ragged_gated_mlp_captured(pkg, cuda_dev, m):
    """An intermediate size that is no multiple of 128: two captured graphs of
    one layer follow weights that are changed in place between replays, and give
    what eager calls give, bit for bit."""
    layer = _load(pkg, pkg.mxfp4.GatedMLP(512, 416), cuda_dev, 1)
    other = _load(pkg, pkg.mxfp4.GatedMLP(512, 416), cuda_dev, 2)
    xs = [torch.randn(m, 512, generator=_gen(s)).bfloat16().to(cuda_dev) for s in range(3)]
    want = [[n.forward(x).clone() for x in xs] for n in (layer, other)]
    assert not torch.equal(want[0][0], want[1][0])
    graphs = []
    for _ in range(2):
        x, stream = xs[0].clone(), torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = layer.forward(x)
        graphs.append((g, stream, x, out))
    for n, expected in enumerate(want):
        if n == 1:
            torch.cuda.synchronize()
            for mine, theirs in ((layer.gate_up_proj, other.gate_up_proj), (layer.down_proj, other.down_proj)):
                mine.weight.copy_(theirs.weight)
                mine.weight_scale.copy_(theirs.weight_scale)
            torch.cuda.synchronize()
        for s in range(3):
            for j, (g, stream, x, out) in enumerate(graphs):
                with torch.cuda.stream(stream):
                    x.copy_(xs[(s + j) % 3])
                    g.replay()
            torch.cuda.synchronize()
            for j, (g, stream, x, out) in enumerate(graphs):
                assert torch.equal(out, expected[(s + j) % 3])



def test_streams_at_once(pkg, cuda_dev):
    """The same weights used from four streams at once, operands made on the
    stream that uses them."""
    d = _Decoder(pkg, cuda_dev)
    want = [d(*_inputs(m, cuda_dev, m))[0] for m in (1, 33, 129, 520)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in want]
    for _ in range(5):
        got = []
        for m, s in zip((1, 33, 129, 520), streams):
            with torch.cuda.stream(s):
                got.append(d(*_inputs(m, cuda_dev, m))[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


_FIRST = """
import importlib, sys, torch
sys.path.insert(0, {root!r})
p = importlib.import_module("mini-sglang-fork_b200")
x = torch.randn(20, 4096, device="cuda").bfloat16()
w = torch.randn(512, 4096, device="cuda").bfloat16()
n = torch.ones(4096, device="cuda").bfloat16()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q, _ = p.mxfp4_rmsnorm_quant(x, n, 1e-6)
    b = p.mxfp4_quant(w)
    y = p.mxfp4_gemm(q, b)
    z = p.mxfp4_dequant(p.mxfp4_gate_up_silu_quant(q, b))
g.replay()
torch.cuda.synchronize()
q, _ = p.mxfp4_rmsnorm_quant(x, n, 1e-6)
assert torch.equal(y, p.mxfp4_gemm(q, p.mxfp4_quant(w)))
assert torch.equal(z, p.mxfp4_dequant(p.mxfp4_gate_up_silu_quant(q, p.mxfp4_quant(w))))
print("captured first")
"""


def test_first_calls_may_be_captured(cuda_dev):
    """A process whose first MXFP4 calls are inside a capture: whatever is set
    up once per device does not disturb it."""
    r = subprocess.run([sys.executable, "-c", _FIRST.format(root=ROOT)], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


def test_calls_from_two_threads(pkg, cuda_dev):
    d = _Decoder(pkg, cuda_dev)
    want = {m: d(*_inputs(m, cuda_dev, m))[0] for m in (4, 200)}
    torch.cuda.synchronize()
    bad = []

    def work(m):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not torch.equal(d(*_inputs(m, cuda_dev, m))[0], want[m]):
                    bad.append(m)

    threads = [threading.Thread(target=work, args=(m,)) for m in want]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_residual_is_the_input(pkg, cuda_dev):
    """The same tensor as x and residual: v = 2x, written back in place."""
    x, _ = _inputs(9, cuda_dev, 0)
    w = torch.ones(512, dtype=torch.bfloat16, device=cuda_dev)
    y, r = O.rmsnorm(x.cpu(), w.cpu(), 1e-6, x.cpu())
    q, out = pkg.mxfp4_rmsnorm_quant(x, w, 1e-6, x)
    _same(q, *O.quant(y))
    assert torch.equal(out.cpu(), r) and torch.equal(x.cpu(), r)


def _far(pkg, dev, negative):
    """Operands with gates around 2^22 and ups around 2^112; `negative`: every
    gate below zero."""
    k, i = 64, 128
    a, _ = _operand(pkg, 3, k, 1.0, 0, dev)
    w, _ = _operand(pkg, 2 * i, k, 1.0, 1, dev)
    data, wdata = a.data.clone(), w.data.clone()
    if negative:
        data &= 0x77  # magnitudes
        wdata[:i] |= 0x88
    scale = torch.full((3, 2), 127 + 20, dtype=torch.uint8, device=dev)
    wscale = torch.full((2 * i, 2), 127, dtype=torch.uint8, device=dev)
    wscale[i:] = 127 + 90
    a = pkg.MXFP4Tensor(data, pkg.ops.mxfp4_tile_scales(scale))
    w = pkg.MXFP4Tensor(wdata, pkg.ops.mxfp4_tile_scales(wscale))
    gu = O.decode(a.data, a.scales) @ O.decode(w.data, w.scales).T
    return pkg.mxfp4_dequant(pkg.mxfp4_gate_up_silu_quant(a, w)).cpu(), gu[:, :i], gu[:, i:]


def test_gated_product_far_gates(pkg, cuda_dev):
    """Gates whose exp overflows give zeros, not NaN, next to ups that overflow
    with them."""
    y, g, u = _far(pkg, cuda_dev, negative=True)
    assert (g < -200).all() and ((g * u).abs() > O.FP32_MAX).any()
    assert (y == 0).all()


def test_gated_product_overflow(pkg, cuda_dev):
    """A product beyond fp32 makes its block NaN, and no block without one."""
    y, g, u = _far(pkg, cuda_dev, negative=False)
    over = (O.silu_mul(g, u).abs() > O.FP32_MAX).reshape(3, 4, 32).any(-1)
    assert over.any()
    assert torch.equal(y.isnan().reshape(3, 4, 32), over[..., None].expand(3, 4, 32))


@pytest.mark.parametrize("m,n,k", [(1, 640, 5120), (40, 512, 8192), (100, 1024, 2048), (200, 512, 8192), (1000, 768, 256)])
def test_results_do_not_depend_on_timing(pkg, cuda_dev, m, n, k):
    """Shares of K are added in a fixed order: repeated calls give the same bits,
    other work on the device or not."""
    a, _ = _operand(pkg, m, k, 1.0, 0, cuda_dev, spread=6)
    w, _ = _operand(pkg, n, k, 1.0, 1, cuda_dev, spread=6)
    first = pkg.mxfp4_gemm(a, w)
    gated = pkg.mxfp4_gate_up_silu_quant(a, w)
    side = torch.cuda.Stream()
    noise = torch.randn(1 << 24, device=cuda_dev)
    for _ in range(10):
        with torch.cuda.stream(side):
            noise.mul_(1.0001)
        assert torch.equal(pkg.mxfp4_gemm(a, w), first)
        again = pkg.mxfp4_gate_up_silu_quant(a, w)
        assert torch.equal(again.data, gated.data)
        assert torch.equal(pkg.ops.mxfp4_plain_scales(again), pkg.ops.mxfp4_plain_scales(gated))


def test_weight_quantised_right_before_use(pkg, cuda_dev):
    """A weight that the kernel just before writes is read as written (launches
    overlap their predecessor's end)."""
    g = _gen(0)
    x = torch.randn(2, 4096, generator=g).bfloat16().to(cuda_dev)
    ws = [torch.randn(1024, 4096, generator=g).bfloat16().to(cuda_dev) for _ in range(4)]
    a = pkg.mxfp4_quant(x)
    want = [pkg.mxfp4_gemm(a, pkg.mxfp4_quant(w)) for w in ws]
    torch.cuda.synchronize()
    for _ in range(20):
        for w, r in zip(ws, want):
            q = pkg.mxfp4_quant(w)
            assert torch.equal(pkg.mxfp4_gemm(a, q), r)
            del q


def test_no_rows(pkg, cuda_dev):
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=cuda_dev)
    w, _ = _operand(pkg, 256, 64, 1.0, 0, cuda_dev)
    q = pkg.mxfp4_quant(x)
    assert tuple(q.shape) == (0, 64) and pkg.mxfp4_dequant(q).shape == (0, 64)
    assert pkg.mxfp4_gemm(q, w).shape == (0, 256)
    assert pkg.mxfp4_gate_up_silu_quant(q, w).shape == (0, 128)
    assert pkg.mxfp4_silu_and_mul_quant(x).shape == (0, 32)
    q, r = pkg.mxfp4_rmsnorm_quant(x, torch.ones(64, dtype=torch.bfloat16, device=cuda_dev), 1e-6, x.clone())
    assert tuple(q.shape) == (0, 64) and r.shape == (0, 64)


@pytest.mark.parametrize("m,n", [(5, 264), (5, 33), (100, 130), (300, 520), (300, 130)])
def test_out_inside_a_larger_buffer(pkg, cuda_dev, m, n):
    """Only the result's rows are written."""
    a, _ = _operand(pkg, m, 64, 1.0, 0, cuda_dev)
    w, _ = _operand(pkg, n, 64, 1.0, 1, cuda_dev)
    want = pkg.mxfp4_gemm(a, w)
    big = torch.full((m + 16, n), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    start = 8 if n % 8 else 3  # a 16-byte aligned row
    out = pkg.mxfp4_gemm(a, w, out=big[start:start + m])
    assert out.data_ptr() == big[start:].data_ptr() and torch.equal(out, want)
    assert (big[:start] == 7).all() and (big[start + m:] == 7).all()


def test_refusals_on_the_device(pkg, cuda_dev):
    E = pkg.W8A8Error
    buf = torch.zeros(4 * 64 + 8, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(E, match="aligned"):
        pkg.mxfp4_quant(buf[1:1 + 256].view(4, 64))
    with pytest.raises(E, match="stride"):
        pkg.mxfp4_quant(torch.zeros(4, 70, dtype=torch.bfloat16, device=cuda_dev)[:, :64])
    with pytest.raises(E, match="stride"):
        pkg.mxfp4_quant(torch.zeros(1, 64, dtype=torch.bfloat16, device=cuda_dev).expand(4, 64))
    with pytest.raises(E, match="unit column stride"):
        pkg.mxfp4_quant(torch.zeros(64, 64, dtype=torch.bfloat16, device=cuda_dev).t()[:, :32])
    with pytest.raises(E, match="2-D bf16 or fp16"):
        pkg.mxfp4_quant(torch.zeros(4, 64, device=cuda_dev))
    with pytest.raises(E, match="multiple of 32"):
        pkg.mxfp4_quant(torch.zeros(4, 48, dtype=torch.bfloat16, device=cuda_dev))
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(E, match="weight"):
        pkg.mxfp4_rmsnorm_quant(x, torch.ones(64, dtype=torch.float16, device=cuda_dev), 1e-6)
    with pytest.raises(E, match="residual"):
        pkg.mxfp4_rmsnorm_quant(x, x[0], 1e-6, torch.zeros(4, 64, dtype=torch.float16, device=cuda_dev))
    with pytest.raises(E, match="stride"):
        pkg.mxfp4_rmsnorm_quant(x, x[0], 1e-6, torch.zeros(1, 64, dtype=torch.bfloat16, device=cuda_dev).expand(4, 64))
    a, _ = _operand(pkg, 4, 64, 1.0, 0, cuda_dev)
    w, _ = _operand(pkg, 100, 64, 1.0, 1, cuda_dev)
    with pytest.raises(E, match="gate; up"):
        pkg.mxfp4_gate_up_silu_quant(a, w)
    with pytest.raises(E, match="contiguous"):
        pkg.mxfp4_gemm(a, w, out=torch.empty(100, 4, dtype=torch.bfloat16, device=cuda_dev).t())
    with pytest.raises(E, match="several devices|no CPU path"):
        pkg.mxfp4_gemm(a, pkg.MXFP4Tensor(w.data.cpu(), w.scales.cpu()))


def test_more_than_2_to_32_values(pkg, cuda_dev):
    """Offsets beyond 32 bits, in values and in bytes."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    m, k = 840_000, 5120
    x = torch.empty(m, k, dtype=torch.bfloat16, device=cuda_dev)
    x.view(-1, 64 * k)[:] = torch.randn(64 * k, generator=_gen(0)).bfloat16().to(cuda_dev)
    x[-100:] = torch.randn(100, k, generator=_gen(1)).bfloat16().to(cuda_dev)
    q = pkg.mxfp4_quant(x)
    c, b = O.quant(x[-130:].cpu().double())
    assert torch.equal(O.unpack(q.data[-130:]), c)
    last = pkg.mxfp4_dequant(q)[-130:]
    assert torch.equal(last.cpu().double(), O.values(c, b))
    del x, q, last
    m, n = 50_000, 51_200
    a, av = _operand(pkg, m, 32, 1.0, 2, cuda_dev)
    w, wv = _operand(pkg, n, 32, 1.0, 3, cuda_dev)
    out = pkg.mxfp4_gemm(a, w)
    rows = torch.tensor([0, m // 2, m - 1])
    want = av[rows] @ wv.T
    assert ((out[rows.to(cuda_dev)].cpu().double() - want).abs()
            <= _gemm_bound(32, av[rows].abs() @ wv.abs().T, want, torch.bfloat16)).all()
