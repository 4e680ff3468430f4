"""Linear layers with packed 4-bit weights and 16-bit activations for decoding batches.

A weight-only layer (``INT4_AWQ_CFG``, ``INT4_BLOCKWISE_WEIGHT_ONLY_CFG``, ``NVFP4_MLP_WEIGHT_ONLY_CFG`` after
``compress``) dequantises its whole weight to memory in every forward pass.  For a few rows the products of
``ops.int4_linear`` / ``ops.nvfp4_linear`` read the packed weight once instead.  They keep the sums in fp32 and do not
round the dequantised weight to 16 bits, so results differ from the dequantising path in the last bits; layers use them
after ``enable_real_quant_gemm(model, weight_only=True)`` (or ``compress(model, {"weight_only_gemm": True})``)."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd import Function

from .. import ops
from ..qtensor import INT4QTensor, NVFP4QTensor, QTensorWrapper
from .gemm_registry import gemm_registry

__all__ = ["WeightOnlyLinear", "weight_only_gemm", "WEIGHT_ONLY_MAX_ROWS"]

# Rows up to which any layer uses the packed weight (one launch); more go through the dequantised weight and a library
# GEMM.  Measured on the device (us, packed against dequantised): at 32 rows INT4 6.6 / 8.3 on 1024 x 1024, 7.5 / 17 on
# 2048 x 2048, 12.7 / 48 on 4096 x 4096, NVFP4 5.9 / 5.3, 6.9 / 7.3 and 11.6 / 13.5; smaller layers lose up to 3 us from 17
# rows on, and gain 14 us of host time where calls are not captured.
WEIGHT_ONLY_MAX_ROWS = {INT4QTensor: 32, NVFP4QTensor: 32}

# INT4 dequantises more slowly, so that large layers gain from several launches too.  A launch costs about 6 us and 0.4 us a
# million weights, the other path 5 us and 2.7 us a million; and a further launch 10 us of host time, which the last
# two sizes need to hide: 64 rows 14.6 / 17 us on 2048 x 2048 (12.8 / 8.1 on 1024 x 1024), 128 rows 61 / 72 us on 5120 x 5120
# (50 / 48 on 4096 x 4096), 272 / 783 on 8192 x 28672; 256 rows 92 / 53 on 4096 x 4096.
_INT4_MAX_ROWS = 128
_INT4_WEIGHTS_PER_LAUNCH_PAIR = 1 << 21


def _takes_packed(kind, rows: int, n: int, k: int) -> bool:
    """Whether ``rows`` rows go to the packed [n, k] weight: in one launch, or in several where the weight is large."""
    if rows <= WEIGHT_ONLY_MAX_ROWS[kind]:
        return True
    launches = -(-rows // ops._w4_max_rows(k))
    return (kind is INT4QTensor and rows <= _INT4_MAX_ROWS
            and launches * (launches - 1) * _INT4_WEIGHTS_PER_LAUNCH_PAIR <= n * k)


def weight_only_gemm(quant_module, input_tensor, bias=None):
    """``input [..., k]`` times the module's packed 4-bit weight ``[n, k]``."""
    wq, weight = quant_module.weight_quantizer, quant_module.weight
    n, k = weight.metadata["shape"]
    packed = weight.data.reshape(n, k // 2)
    block = wq.block_sizes[-1]
    if weight.metadata["qtensor_class"] is INT4QTensor:
        return ops.int4_linear(input_tensor, packed, wq._scale, block, bias)
    return ops.nvfp4_linear(input_tensor, packed, wq._scale, wq._double_scale, bias, block)


def _layout_covered(module) -> bool:
    """Whether the module's weight is packed in a layout that the products read: what lasts from call to call."""
    wq, weight = module.weight_quantizer, module.weight
    if not isinstance(weight, QTensorWrapper) or not hasattr(wq, "_scale"):
        return False
    kind, shape, dtype = (weight.metadata[key] for key in ("qtensor_class", "shape", "dtype"))
    if kind not in (INT4QTensor, NVFP4QTensor) or len(shape) != 2 or dtype not in (torch.float16, torch.bfloat16):
        return False
    block = (getattr(wq, "block_sizes", None) or {}).get(-1)
    if not isinstance(block, int) or weight.data.numel() * 2 != shape[0] * shape[1]:      # padded rows
        return False
    if kind is INT4QTensor:
        return wq._scale.dtype == dtype and ops._int4_sizes(shape[1], block)
    return hasattr(wq, "_double_scale") and ops._nvfp4_sizes(shape[1], block)


def _covered(module, input) -> bool:
    """Whether the products take this call: the weight's layout, and inputs and autocast as they are now."""
    if not _layout_covered(module):
        return False
    weight = module.weight
    shape, dtype = weight.metadata["shape"], weight.metadata["dtype"]
    if not (weight.data.is_cuda and input.is_cuda) or dtype != input.dtype or input.shape[-1] != shape[1]:
        return False
    # F.linear would cast both
    return not (torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != dtype)


def _weight_only_availability_check(module, input, args, kwargs) -> bool:
    """The answer is remembered by the layer, so nothing that changes from call to call may go into it: the products
    look at the input themselves."""
    from ..nn import RealQuantLinear, TensorQuantizer

    if not (isinstance(module, RealQuantLinear) and isinstance(getattr(module, "input_quantizer", None), TensorQuantizer)
            and isinstance(getattr(module, "weight_quantizer", None), TensorQuantizer)):
        return False
    return (getattr(module, "_weight_only_gemm", False) and not module.input_quantizer.is_enabled
            and module.weight_quantizer.is_enabled and _layout_covered(module))


class WeightOnlyLinear(Function):
    """Autograd wrapper: forward on the packed weight, the input's gradient through the dequantised weight (the
    packed weight itself is not trained)."""

    @staticmethod
    def forward(ctx, quant_module, input_tensor, weight, bias=None):
        ctx.quant_module = quant_module
        ctx.save_for_backward(weight)
        ctx.bias_grad = bias is not None and bias.requires_grad
        return weight_only_gemm(quant_module, input_tensor, bias)

    @staticmethod
    def backward(ctx, grad_outputs):
        weight, = ctx.saved_tensors
        grad_input = grad_bias = None
        if ctx.needs_input_grad[1]:
            grad_input = grad_outputs @ ctx.quant_module.weight_quantizer.dequantize(weight)
        if ctx.bias_grad:
            grad_bias = grad_outputs.sum(dim=list(range(grad_outputs.dim() - 1)))
        return None, grad_input, None, grad_bias


def _weight_only_linear(quant_module, input, weight, bias=None):
    x = quant_module.input_quantizer(input)               # a disabled quantiser still applies its AWQ pre-quant scale
    if not _covered(quant_module, x) or not _takes_packed(weight.metadata["qtensor_class"], x.numel() // x.shape[-1],
                                                          *weight.metadata["shape"]):
        return F.linear(x, quant_module._quantized_weight(), bias)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return WeightOnlyLinear.apply(quant_module, x, weight, bias)
    return weight_only_gemm(quant_module, x, bias)


gemm_registry.register(gemm_func=_weight_only_linear, availability_check=_weight_only_availability_check)
