"""MXFP4 (microscaled 4-bit) linear layers with mini-sglang's operator surface.

The same class names and constructor signatures as the W8A8 layers of
``layers.py`` (and so as mini-sglang's bf16 ones, M/layers/linear.py:13-127),
plus a trailing ``dtype``: the model's 16-bit type, which outputs, biases and
norm weights have.  ``weight`` is uint8 ``[N_local, K_local / 2]`` (two E2M1
codes per byte) and ``weight_scale`` the E8M0 scales in the tiles that the
tensor core reads (``ops.mxfp4_scale_shape``); ``weights.load_mxfp4_state_dict``
makes both from a checkpoint.  Activations are quantised per 32 values on the
way in, or arrive as an :class:`~.ops.MXFP4Tensor` from the layer before.

Row-parallel layers hold a K-shard and sum over ranks with the plugin stack's
``all_reduce`` after the product (the fused reduce exists for W8A8 only).  The
peer-memory plugin sums bf16 only: with it, fp16 row-parallel layers are refused.
Every local input size must be a multiple of 32.
"""
from __future__ import annotations

from typing import List, Optional, Tuple, Union

import torch

from . import _lib, ops
from .distributed import PeerMemDistributedImpl, communicator, div_even, get_tp_info
from .layers import BaseOP
from .ops import MXFP4Tensor

__all__ = [
    "LinearReplicated",
    "LinearColParallelMerged",
    "LinearQKVMerged",
    "LinearOProj",
    "LinearRowParallel",
    "RMSNormFusedQuant",
    "GatedMLP",
    "silu_and_mul_quant",
]

silu_and_mul_quant = ops.mxfp4_silu_and_mul_quant

Activation = Union[torch.Tensor, MXFP4Tensor]


class _LinearTPImpl(BaseOP):
    """MXFP4 counterpart of ``_LinearTPImpl`` (M/layers/linear.py:13-32)."""

    def __init__(self, full_isize: int, full_osize: int, local_isize: int, local_osize: int, has_bias: bool,
                 dtype: torch.dtype):
        if local_isize % 32:
            raise _lib.W8A8Error(_lib.ERR_INVALID_ARG,
                                 f"MXFP4 linear: the local input size {local_isize} must be a multiple of 32")
        self.full_input_size = full_isize
        self.full_output_size = full_osize
        self.local_input_size = local_isize
        self.local_output_size = local_osize
        self._dtype = dtype
        self._packed: Optional[MXFP4Tensor] = None
        self.weight = torch.empty(local_osize, local_isize // 2, dtype=torch.uint8)
        self.weight_scale = torch.empty(ops.mxfp4_scale_shape(local_osize, local_isize), dtype=torch.uint8)
        self.bias = torch.empty(local_osize, dtype=dtype) if has_bias else None

    def _weight(self) -> MXFP4Tensor:
        """``weight`` and ``weight_scale`` as one operand (remade when either
        attribute has been replaced)."""
        w = self._packed
        if w is None or w.data is not self.weight or w.scales is not self.weight_scale:
            w = self._packed = MXFP4Tensor(self.weight, self.weight_scale)
        return w

    def _quantize_input(self, x: Activation) -> MXFP4Tensor:
        return x if isinstance(x, MXFP4Tensor) else ops.mxfp4_quant(x)

    def forward(self, x: Activation) -> torch.Tensor:
        return ops.mxfp4_gemm(self._quantize_input(x), self._weight(), self.bias, out_dtype=self._dtype)


class LinearReplicated(_LinearTPImpl):
    """Unsharded MXFP4 linear (M/layers/linear.py:35-53)."""

    def __init__(self, input_size: int, output_size: int, has_bias: bool, dtype: torch.dtype = torch.bfloat16):
        super().__init__(input_size, output_size, input_size, output_size, has_bias, dtype)


class LinearColParallelMerged(_LinearTPImpl):
    """Column-parallel merged linear, e.g. gate_up (M/layers/linear.py:56-68)."""

    def __init__(self, input_size: int, output_sizes: List[int], has_bias: bool,
                 dtype: torch.dtype = torch.bfloat16):
        tp_info = get_tp_info()
        tp_output_sizes = [div_even(size, tp_info.size) for size in output_sizes]
        super().__init__(input_size, sum(output_sizes), input_size, sum(tp_output_sizes), has_bias, dtype)

    def forward_silu_quant(self, x: Activation) -> MXFP4Tensor:
        """For a [gate; up] merge: MXFP4 ``silu(gate) * up``
        (:func:`ops.mxfp4_gate_up_silu_quant`)."""
        return ops.mxfp4_gate_up_silu_quant(self._quantize_input(x), self._weight(), self.bias, self._dtype)


class LinearQKVMerged(_LinearTPImpl):
    """Column-parallel q|k|v over heads, kv replicated when kv_heads < tp
    (M/layers/linear.py:71-88)."""

    def __init__(self, hidden_size: int, head_dim: int, num_qo_heads: int, num_kv_heads: int, has_bias: bool,
                 dtype: torch.dtype = torch.bfloat16):
        tp_info = get_tp_info()
        local_num_qo = div_even(num_qo_heads, tp_info.size)
        local_num_kv = div_even(num_kv_heads, tp_info.size, allow_replicate=True)
        full_osize = (num_qo_heads + 2 * num_kv_heads) * head_dim
        local_osize = (local_num_qo + 2 * local_num_kv) * head_dim
        super().__init__(hidden_size, full_osize, hidden_size, local_osize, has_bias, dtype)


class _RowParallel(_LinearTPImpl):
    """Row-parallel forward: local product of the K-shard, then the sum over
    ranks (M/layers/linear.py:102-106,123-127)."""

    def __init__(self, input_size: int, output_size: int, has_bias: bool, dtype: torch.dtype = torch.bfloat16):
        tp_info = get_tp_info()
        self._comm = communicator()
        self._tp_size = tp_info.size
        if tp_info.size > 1 and dtype is not torch.bfloat16 and self._comm.plugins \
                and isinstance(self._comm.plugins[-1], PeerMemDistributedImpl):
            raise _lib.W8A8Error(_lib.ERR_UNSUPPORTED, "MXFP4 row-parallel linear: the peer-memory all-reduce sums bf16, "
                                 f"not {dtype}; use bf16, or another all-reduce plugin")
        super().__init__(input_size, output_size, div_even(input_size, tp_info.size), output_size, has_bias, dtype)

    def forward(self, x: Activation) -> torch.Tensor:
        y = super().forward(x)
        return self._comm.all_reduce(y) if self._tp_size > 1 else y


class LinearOProj(_RowParallel):
    """o_proj (M/layers/linear.py:91-106)."""


class LinearRowParallel(_RowParallel):
    """down_proj (M/layers/linear.py:109-127)."""


class RMSNormFusedQuant(BaseOP):
    """``RMSNormFused`` (M/layers/norm.py:23-38) with the following MXFP4
    layer's input quantisation fused in: ``forward(x, residual)`` returns
    ``(MXFP4Tensor, residual)``, the residual updated in place to ``x +
    residual`` (or ``x`` itself without one)."""

    def __init__(self, size: int, eps: float, dtype: torch.dtype = torch.bfloat16) -> None:
        self.eps = eps
        self.weight = torch.empty(size, dtype=dtype)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> Tuple[MXFP4Tensor, torch.Tensor]:
        return ops.mxfp4_rmsnorm_quant(x, self.weight, self.eps, residual)


class GatedMLP(BaseOP):
    """MXFP4 ``GatedMLP`` (M/models/utils.py:25-50): gate_up with SiLU*mul and
    requantisation in its epilogue, then down.  Between the two nothing but the
    4-bit product reaches memory."""

    def __init__(self, hidden_size: int, intermediate_size: int, dtype: torch.dtype = torch.bfloat16):
        self.gate_up_proj = LinearColParallelMerged(hidden_size, [intermediate_size, intermediate_size],
                                                    has_bias=False, dtype=dtype)
        self.down_proj = LinearRowParallel(intermediate_size, hidden_size, has_bias=False, dtype=dtype)

    def forward(self, x: Activation) -> torch.Tensor:
        y = self.gate_up_proj.forward_silu_quant(x)
        del x
        return self.down_proj.forward(y)
