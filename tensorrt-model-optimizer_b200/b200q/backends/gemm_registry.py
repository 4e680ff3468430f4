"""Registry of low-precision GEMM implementations (reference:
modelopt/torch/quantization/backends/gemm_registry.py:31-156).

An entry is a GEMM callable ``f(module, input, weight, bias, *args, **kwargs)`` plus a predicate
``check(module, input, args, kwargs)``; a ``RealQuantLinear`` asks the registry once for the first
entry whose predicate accepts it and keeps the answer.

The tensor-core kernels never synchronise: error bits of their bounded device-side waits collect in
a per-device status word, which ``backends.check_gemm_status(device)`` reads (and raises on)."""
from __future__ import annotations

from typing import Callable

from torch import nn

__all__ = ["GEMMRegistry", "gemm_registry", "enable_real_quant_gemm", "disable_real_quant_gemm",
           "is_real_quant_gemm_enabled"]


class GEMMRegistry:
    def __init__(self):
        self._registry: list[dict] = []

    def register(self, gemm_func: Callable, availability_check: Callable | None = None) -> None:
        self._registry.append({"gemm_func": gemm_func,
                               "availability_check": availability_check or (lambda module, input, args, kwargs: True)})

    def unregister(self, gemm_func: Callable) -> None:
        self._registry = [e for e in self._registry if e["gemm_func"] != gemm_func]

    def find_match(self, module: nn.Module, input, *args, **kwargs) -> Callable | None:
        for e in self._registry:
            if e["availability_check"](module, input, args, kwargs):
                return e["gemm_func"]
        return None

    def __contains__(self, gemm_func: Callable) -> bool:
        return any(e["gemm_func"] == gemm_func for e in self._registry)


gemm_registry = GEMMRegistry()


def _both_quantizers_enabled(module) -> bool:
    iq, wq = getattr(module, "input_quantizer", None), getattr(module, "weight_quantizer", None)
    return bool(iq is not None and wq is not None and iq.is_enabled and wq.is_enabled)


def _only_weight_quantizer_enabled(module) -> bool:
    iq, wq = getattr(module, "input_quantizer", None), getattr(module, "weight_quantizer", None)
    return bool(iq is not None and wq is not None and not iq.is_enabled and wq.is_enabled)


def enable_real_quant_gemm(model: nn.Module, weight_only: bool = False) -> None:
    """Mark every module whose input and weight quantisers are both enabled to use a registered
    real-quant GEMM.  ``weight_only`` marks those too whose weight quantiser alone is enabled: with a packed
    4-bit weight and few rows they then read the packed weight instead of dequantising it first.  Without it, layers that
    an earlier call marked in that way lose the mark: the last call says which layers are marked."""
    for module in model.modules():
        if _both_quantizers_enabled(module):
            _set_weight_only(module, False)
            module._use_real_quant_gemm = True
        elif weight_only and _only_weight_quantizer_enabled(module):
            _set_weight_only(module, True)
            module._use_real_quant_gemm = True
        elif getattr(module, "_weight_only_gemm", False):
            _set_weight_only(module, False)
            module._use_real_quant_gemm = False


def _set_weight_only(module: nn.Module, value: bool) -> None:
    """A layer whose mark changes asks the registry again: what it remembers was matched for the other mark."""
    if getattr(module, "_weight_only_gemm", False) != value:
        module._weight_only_gemm = value
        module.__dict__.pop("_real_quant_gemm_impl", None)


def disable_real_quant_gemm(model: nn.Module) -> None:
    for module in model.modules():
        if hasattr(module, "_use_real_quant_gemm"):
            _set_weight_only(module, False)
            module._use_real_quant_gemm = False


def is_real_quant_gemm_enabled(model: nn.Module) -> bool:
    return any(getattr(module, "_use_real_quant_gemm", False) for module in model.modules())
