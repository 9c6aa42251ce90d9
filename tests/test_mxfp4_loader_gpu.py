"""GPU: quantise-at-load of fp32 checkpoints for the MXFP4 layers."""
from __future__ import annotations

import pytest
import torch

from oracle import mxfp4_oracle as O
from test_mxfp4_layers_cpu import _fp32_weights

pytestmark = pytest.mark.gpu


def test_fp32_checkpoint(pkg, cuda_dev):
    """The state dict holds the codes and scales nearest to the checkpoint's own
    fp32 values."""
    w = _fp32_weights()
    sd = pkg.load_mxfp4_state_dict([("m.o_proj.weight", w)], 0, 1, 1, device=cuda_dev)
    c, b = O.quant(w.double())
    got = O.unpack(sd["m.o_proj.weight"])
    zero = ((got & 7) == 0) & ((c & 7) == 0)  # (a zero's sign apart)
    assert ((got == c) | zero).all()
    assert torch.equal(O.untile(sd["m.o_proj.weight_scale"], w.shape[0], 2), b)
