"""CPU: the MXFP4 layers' sizes and state-dict contract, the MXFP4 checkpoint
loader, and the row-parallel composition over gloo (world_size 2), with the
64-bit restatement in the place of the CUDA operators."""
from __future__ import annotations

import multiprocessing as mp
import os
import sys
import traceback

import pytest
import torch

from conftest import ROOT
from oracle import mxfp4_oracle as O

HIDDEN, NQ, NKV, HD, INTER = 128, 4, 2, 32, 256


def _quantise(w):
    c, b = O.quant(w.double())
    return O.pack(c), b.to(torch.uint8)


def _checkpoint(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s, scale=0.05: (torch.randn(*s, generator=g) * scale).to(dtype)  # noqa: E731
    p = "model.layers.0."
    return [("model.embed_tokens.weight", rnd(100, HIDDEN)),
            (p + "input_layernorm.weight", rnd(HIDDEN, scale=1.0)),
            (p + "self_attn.q_proj.weight", rnd(NQ * HD, HIDDEN)), (p + "self_attn.q_proj.bias", rnd(NQ * HD)),
            (p + "self_attn.k_proj.weight", rnd(NKV * HD, HIDDEN)), (p + "self_attn.k_proj.bias", rnd(NKV * HD)),
            (p + "self_attn.v_proj.weight", rnd(NKV * HD, HIDDEN)), (p + "self_attn.v_proj.bias", rnd(NKV * HD)),
            (p + "self_attn.o_proj.weight", rnd(HIDDEN, NQ * HD)),
            (p + "mlp.gate_proj.weight", rnd(INTER, HIDDEN)), (p + "mlp.up_proj.weight", rnd(INTER, HIDDEN)),
            (p + "mlp.down_proj.weight", rnd(HIDDEN, INTER))]


def _packed_checkpoint():
    """The same checkpoint already in MXFP4 (codes and plain scales)."""
    items = []
    for k, v in _checkpoint():
        if "proj.weight" in k:
            d, s = _quantise(v)
            items += [(k, d), (k + "_scale", s)]
        else:
            items.append((k, v))
    return items


@pytest.mark.parametrize("world", [1, 2])
def test_loader_shards_of_the_unsharded_quantisation(pkg, world):
    """Every rank's dequantised weight is its slice of the whole weight's
    dequantised values; scales come in tiles; a packed checkpoint gives the
    same state dict."""
    full = dict(_checkpoint())
    p = "model.layers.0."
    val = lambda k: O.values(*O.quant(full[p + k].double()))  # noqa: E731
    for r in range(world):
        sd = pkg.load_mxfp4_state_dict(_checkpoint(), r, world, NKV, quantise=_quantise)
        got = lambda k: O.decode(sd[p + k + ".weight"], sd[p + k + ".weight_scale"])  # noqa: E731
        part = lambda t, d: t.chunk(world, dim=d)[r]  # noqa: E731
        assert torch.equal(got("self_attn.o_proj"), part(val("self_attn.o_proj.weight"), 1))
        assert torch.equal(got("mlp.down_proj"), part(val("mlp.down_proj.weight"), 1))
        assert torch.equal(got("mlp.gate_up_proj"), torch.cat([part(val("mlp.gate_proj.weight"), 0),
                                                               part(val("mlp.up_proj.weight"), 0)]))
        assert torch.equal(got("self_attn.qkv_proj"),
                           torch.cat([part(val(f"self_attn.{x}_proj.weight"), 0) for x in "qkv"]))
        assert sd[p + "self_attn.qkv_proj.bias"].dtype == torch.bfloat16
        again = pkg.load_mxfp4_state_dict(_packed_checkpoint(), r, world, NKV)
        assert sorted(again) == sorted(sd)
        for k in sd:
            assert torch.equal(again[k], sd[k]), k


def test_loaded_state_fits_the_layers(pkg):
    pkg.reset_tp_info()
    try:
        for r in range(2):
            pkg.set_tp_info(r, 2)
            sd = pkg.load_mxfp4_state_dict(_checkpoint(torch.float16), r, 2, NKV, quantise=_quantise, dtype=torch.float16)
            L, t = pkg.mxfp4, torch.float16
            p = "model.layers.0."
            for key, layer in ((p + "self_attn.qkv_proj", L.LinearQKVMerged(HIDDEN, HD, NQ, NKV, True, t)),
                               (p + "self_attn.o_proj", L.LinearOProj(NQ * HD, HIDDEN, False, t)),
                               (p + "mlp", L.GatedMLP(HIDDEN, INTER, t)),
                               (p + "input_layernorm", L.RMSNormFusedQuant(HIDDEN, 1e-6, t))):
                layer.load_state_dict({k: v for k, v in sd.items() if k.startswith(key + ".")}, prefix=key)
            pkg.reset_tp_info()
    finally:
        pkg.reset_tp_info()


def test_loader_refusals(pkg):
    E = pkg.W8A8Error
    w = torch.zeros(64, 96)
    with pytest.raises(E, match="do not divide"):  # three blocks of 32 over two ranks
        pkg.load_mxfp4_state_dict([("a.o_proj.weight", w)], 0, 2, 1, quantise=_quantise)
    with pytest.raises(E, match="no MXFP4 layer"):
        pkg.load_mxfp4_state_dict([("m.mlp.experts.0.gate_proj.weight", w)], 0, 1, 1, quantise=_quantise)
    with pytest.raises(E, match="uint8"):
        pkg.load_mxfp4_state_dict([("a.o_proj.weight_scale", torch.zeros(64))], 0, 1, 1, quantise=_quantise)
    with pytest.raises(E, match="incomplete"):
        pkg.load_mxfp4_state_dict([("a.q_proj.weight", w)], 0, 1, 1, quantise=_quantise)
    with pytest.raises(E, match="multiple of 32"):
        pkg.mxfp4.LinearReplicated(80, 64, False)


def test_state_dict_contract(pkg):
    layer = pkg.mxfp4.LinearReplicated(64, 48, has_bias=True)
    assert sorted(layer.state_dict()) == ["bias", "weight", "weight_scale"]
    good = {"weight": torch.zeros(48, 32, dtype=torch.uint8), "bias": torch.zeros(48, dtype=torch.bfloat16),
            "weight_scale": torch.zeros(pkg.ops.mxfp4_scale_shape(48, 64), dtype=torch.uint8)}
    layer.load_state_dict(dict(good))
    assert layer._weight().data is layer.weight and layer._weight() is layer._weight()
    first = layer._weight()
    layer.load_state_dict({k: v.clone() for k, v in good.items()})
    assert layer._weight() is not first  # another weight, another operand
    with pytest.raises(ValueError):
        layer.load_state_dict({**good, "weight_scale": torch.zeros(48, 2, dtype=torch.uint8)})


def _fp32_weights():
    """fp32 values between the bf16 ones: next to every border, next to powers of
    two (a block's scale), at both ends of the type, infinities and NaN."""
    g = torch.Generator().manual_seed(7)
    rows = [torch.randn(64, generator=g) * 0.02 for _ in range(60)]
    ulp = torch.tensor([1 - 2.0 ** -20, 1 + 2.0 ** -20, 1.0, 1 - 2.0 ** -24, 1 + 2.0 ** -23])
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.5, 4.0, 6.0])
    near = (borders[:, None] * ulp).flatten()  # 50 values
    for e in (-100, -10, 0, 3, 100):
        for top in (4.0, 4.0 * (1 - 2.0 ** -24), 7.9999, 8.0 * (1 - 2.0 ** -24)):
            row = torch.cat([near[:31], torch.tensor([top]), near[-31:].clamp(max=top), torch.tensor([top])])
            rows.append(row * 2.0 ** e * (torch.randint(0, 2, (64,), generator=g) * 2 - 1))
    bits = torch.randint(0, 2 ** 31 - 1, (200, 64), generator=g, dtype=torch.int64).to(torch.int32)
    rows += list((bits & 0x007fffff).view(torch.float32))  # subnormals
    rows += list(bits.view(torch.float32))  # anything, infinities' exponents among them
    last = torch.randn(4, 64, generator=g)
    last[0, 5], last[1, 40], last[2, 3] = float("inf"), float("nan"), torch.finfo(torch.float32).max
    last[3, 0] = torch.tensor(0x7f800001, dtype=torch.int32).view(torch.float32)  # a NaN in its last bit alone
    return torch.stack(rows + list(last))


def test_fp32_checkpoint_is_quantised_as_it_is(pkg, monkeypatch):
    """The codes and scales of an fp32 weight are the nearest to its own values, not
    to those of its bf16 rounding."""
    def quant(x):
        assert x.dtype in (torch.bfloat16, torch.float16)
        c, b = O.quant(x.double())
        return pkg.MXFP4Tensor(O.pack(c), O.tile(b))

    monkeypatch.setattr(pkg.ops, "mxfp4_quant", quant)
    w = _fp32_weights()
    c, b = O.quant(w.double())
    assert not torch.equal(O.quant(w.bfloat16().double())[0], c)
    for t in (w, w.t().contiguous().t()):
        data, scales = pkg.weights.mxfp4_quantiser(torch.device("cpu"))(t)
        assert torch.equal(O.unpack(data), c) and torch.equal(scales.long(), b)


def test_fp16_row_parallel_is_refused_with_the_peer_memory_plugin(pkg):
    """The peer-memory all-reduce sums bf16: a layer whose every forward would fail
    there is not made; other types, plugins and a single rank are."""
    from importlib import import_module

    D = import_module(pkg.__name__ + ".distributed")
    plugins, L, E = D.DistributedCommunicator.plugins, pkg.mxfp4, pkg.W8A8Error
    pkg.reset_tp_info()
    try:
        pkg.set_tp_info(0, 2)
        L.LinearOProj(128, 64, False, torch.float16)
        D.DistributedCommunicator.plugins = plugins + [D.PeerMemDistributedImpl(object())]
        for make in (lambda t: L.LinearOProj(128, 64, False, t), lambda t: L.LinearRowParallel(128, 64, False, t),
                     lambda t: L.GatedMLP(64, 128, t)):
            make(torch.bfloat16)
            with pytest.raises(E, match="peer-memory"):
                make(torch.float16)
        L.LinearReplicated(128, 64, False, torch.float16)
        D.DistributedCommunicator.plugins = D.DistributedCommunicator.plugins + [D.TorchDistributedImpl()]
        L.LinearOProj(128, 64, False, torch.float16)  # the last plugin is the one in use
        D.DistributedCommunicator.plugins = plugins + [D.PeerMemDistributedImpl(object())]
        pkg.reset_tp_info()
        pkg.set_tp_info(0, 1)
        L.LinearOProj(128, 64, False, torch.float16)
    finally:
        D.DistributedCommunicator.plugins = plugins
        pkg.reset_tp_info()


def _patch(pkg):
    """The operators' restatements in the place of the CUDA ones."""
    ops = pkg.ops

    def tensor(y):
        c, b = O.quant(y)
        return ops.MXFP4Tensor(O.pack(c), O.tile(b))

    def gemm(a, w, bias=None, out=None, out_dtype=torch.bfloat16):
        y = O.decode(a.data, a.scales) @ O.decode(w.data, w.scales).T
        return (y if bias is None else y + bias.double()).to(out_dtype)

    def gated(a, w, bias=None, dtype=torch.bfloat16):
        g, u = (O.decode(a.data, a.scales) @ O.decode(w.data, w.scales).T).chunk(2, dim=1)
        return tensor(O.silu_mul(g, u))

    ops.mxfp4_quant = lambda x: tensor(x.double())
    ops.mxfp4_gemm, ops.mxfp4_gate_up_silu_quant = gemm, gated


def _rank(rank, world, port, q):
    try:
        sys.path.insert(0, ROOT)
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        import importlib
        from datetime import timedelta

        import torch.distributed as dist

        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=60))
        pkg = importlib.import_module("mini-sglang-fork_b200")
        _patch(pkg)
        x = torch.randn(5, HIDDEN, generator=torch.Generator().manual_seed(1)).bfloat16()
        key = "model.layers.0.mlp"

        def mlp(r, n):
            pkg.reset_tp_info()
            pkg.set_tp_info(r, n)
            m = pkg.mxfp4.GatedMLP(HIDDEN, INTER)
            sd = pkg.load_mxfp4_state_dict(_checkpoint(), r, n, NKV, quantise=_quantise)
            m.load_state_dict({k: v for k, v in sd.items() if k.startswith(key + ".")}, prefix=key)
            return m

        got = mlp(rank, world).forward(x)
        whole = mlp(0, 1)
        want = whole.forward(x).double()
        y = whole.gate_up_proj.forward_silu_quant(x)
        down = whole.down_proj
        dist.destroy_process_group()
        # every rank's partial, their sum and the unsharded result are rounded to
        # bf16: half a step (2^-8) of each, the partials' magnitudes being at
        # most that of the products' sum
        mags = O.decode(y.data, y.scales).abs() @ O.decode(down.weight, down.weight_scale).abs().T
        err = ((got.double() - want).abs() - 2.0 ** -8 * (mags + 2 * want.abs())).max()
        q.put((rank, "ok" if err <= 0 else f"off by {err} more than the bound"))
    except BaseException:  # noqa: BLE001
        q.put((rank, traceback.format_exc()))


def test_row_parallel_over_gloo():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29700 + os.getpid() % 200
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        out = dict(q.get(timeout=120) for _ in procs)
    finally:
        for p in procs:
            p.join(timeout=20)
            if p.is_alive():
                p.kill()
    assert out == {0: "ok", 1: "ok"}, out
