"""Refusals of the 4-bit products that need no GPU, and the switch of the weight-only layers."""
import ctypes

import pytest
import torch
from torch import nn


def test_cpu_tensors_are_refused():
    from b200q import ops

    x, packed, scales = torch.zeros(1, 128, dtype=torch.float16), torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.int4_linear(x, packed, scales, 128)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.nvfp4_linear(x, packed, torch.zeros(4, 8, dtype=torch.uint8), torch.ones(()))


def test_status_codes():
    from b200q import _cabi

    lib = _cabi.lib
    buf = ctypes.create_string_buffer(512)
    p = (ctypes.addressof(buf) + 31) & ~31
    NULL, DTYPE, ALIGN, SHAPE, UNSUPPORTED = -1, -2, -3, -4, -7

    def int4(**kw):
        a = dict(x=p, xs=128, dtype=2, codes=p, scales=p, block=128, bias=None, out=p, os=16, rows=1, n=16, k=128, ws=None, wsb=0, status=p)
        a.update(kw)
        return lib.b200q_int4_linear(*a.values(), None)

    def nvfp4(**kw):
        a = dict(x=p, xs=128, dtype=2, codes=p, scales=p, block=16, scale2=p, bias=None, out=p, os=16, rows=1, n=16, k=128, ws=None, wsb=0, status=p)
        a.update(kw)
        return lib.b200q_nvfp4_linear(*a.values(), None)

    for f in (int4, nvfp4):
        for name in ("x", "codes", "scales", "out", "status"):
            assert f(**{name: None}) == NULL, name
        assert f(dtype=0) == DTYPE
        for kw in (dict(rows=0), dict(n=0), dict(k=0), dict(k=48), dict(xs=-8), dict(os=15)):
            assert f(**kw) == SHAPE, kw
        for kw in (dict(rows=33), dict(k=1 << 25, block=32)):
            assert f(**kw) == UNSUPPORTED, kw
        for kw in (dict(x=p + 8), dict(xs=132), dict(codes=p + 4), dict(scales=p + 1)):
            assert f(**kw) == ALIGN, kw
    assert nvfp4(scale2=None) == NULL and nvfp4(block=64) == UNSUPPORTED
    assert int4(block=96) == SHAPE and int4(block=16) == UNSUPPORTED and int4(block=0) == SHAPE
    assert lib.b200q_w4_linear_max_rows(4096) == 32 and lib.b200q_w4_linear_max_rows(4095) == 0
    assert lib.b200q_w4_linear_workspace(33, 16, 128, 128) == SHAPE


def test_switch_marks_weight_only_layers_when_asked():
    import b200q as mtq

    model = nn.Sequential(nn.Linear(128, 16))
    mtq.replace_quant_module(model)
    mtq.set_quantizer_by_cfg(model, mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG["quant_cfg"])
    mtq.backends.enable_real_quant_gemm(model)
    assert not mtq.backends.is_real_quant_gemm_enabled(model)
    mtq.backends.enable_real_quant_gemm(model, weight_only=True)
    assert mtq.backends.is_real_quant_gemm_enabled(model)
    mtq.backends.disable_real_quant_gemm(model)
    assert not mtq.backends.is_real_quant_gemm_enabled(model)


def test_the_last_call_says_which_layers_are_marked():
    import b200q as mtq

    model = nn.Sequential(nn.Linear(128, 16))
    mtq.replace_quant_module(model)
    mtq.set_quantizer_by_cfg(model, mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG["quant_cfg"])
    mtq.backends.enable_real_quant_gemm(model, weight_only=True)
    assert mtq.backends.is_real_quant_gemm_enabled(model)
    mtq.backends.enable_real_quant_gemm(model)               # weight-only layers are not asked for any more
    assert not mtq.backends.is_real_quant_gemm_enabled(model)
    mtq.backends.enable_real_quant_gemm(model, weight_only=True)
    assert mtq.backends.is_real_quant_gemm_enabled(model)


def test_status_word_needs_a_place_for_its_address():
    from b200q import _cabi

    assert _cabi.lib.b200q_gemm_status_word(None) == -1
