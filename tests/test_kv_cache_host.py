"""Refusals of the KV-cache operators that need no GPU: CPU tensors, and the C ABI's status codes for bad
arguments (nothing is launched)."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    from b200q import ops

    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    cache = (torch.zeros(1, 1, 16, 32, dtype=torch.uint8), torch.zeros(1, 1, 16, 4, dtype=torch.uint8))
    s = torch.ones(())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.kv_step(i, i, i, i, i.view(1, 1), 16, 1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.nvfp4_kv_append(x, x, torch.zeros(1, dtype=torch.int64), cache, cache, s, s)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.nvfp4_kv_attention(x, cache, cache, s, s, i.view(1, 1), i)


def test_status_codes():
    from b200q import _cabi

    lib = _cabi.lib
    buf = ctypes.create_string_buffer(512)
    p = (ctypes.addressof(buf) + 31) & ~31
    NULL, DTYPE, ALIGN, SHAPE, UNSUPPORTED, CAPACITY = -1, -2, -3, -4, -7, -9

    def step(**kw):
        a = dict(lens=p, new=p, free=p, nfree=1, taken=p, table=p, stride=1, width=1, requests=1, page=16, tokens=1, slots=p,
                 positions=p, cu=p, lens_out=p, taken_out=p, status=p)
        a.update(kw)
        return lib.b200q_kv_step(*a.values(), None)

    for name in ("lens", "new", "free", "taken", "table", "slots", "positions", "cu", "lens_out", "taken_out", "status"):
        assert step(**{name: None}) == NULL, name
    for kw in (dict(requests=0), dict(page=0), dict(tokens=-1), dict(nfree=-1), dict(width=-1), dict(stride=0)):
        assert step(**kw) == SHAPE, kw
    assert step(requests=8193) == UNSUPPORTED

    def append(**kw):
        a = dict(k=p, ks=64, kh=64, v=p, vs=64, vh=64, dtype=2, slots=p, tokens=1, heads=1, dim=64, k2=p, v2=p, kc=p, ksc=p, vc=p,
                 vsc=p, pages=1, page=16, kv=None, vv=None)
        a.update(kw)
        return lib.b200q_nvfp4_kv_append(*a.values(), None)

    for name in ("k", "v", "slots", "k2", "v2", "kc", "ksc", "vc", "vsc"):
        assert append(**{name: None}) == NULL, name
    assert append(dtype=5) == DTYPE
    for kw in (dict(tokens=0), dict(heads=0), dict(dim=24), dict(pages=0), dict(page=0)):
        assert append(**kw) == SHAPE, kw
    for kw in (dict(k=p + 16), dict(ks=65), dict(vh=8), dict(kc=p + 4), dict(vv=p + 2)):
        assert append(**kw) == ALIGN, kw
    assert append(pages=1 << 30, page=64) == UNSUPPORTED

    def attention(**kw):
        a = dict(q=p, qs=64, qh=64, dtype=2, kc=p, ks=p, vc=p, vs=p, k2=p, v2=p, table=p, stride=1, width=1, lens=p, cu=None,
                 requests=1, tokens=1, heads=1, group=1, dim=64, pages=1, page=16, scale=1.0, out=p, lse=None, tail=1, ws=p,
                 ws_bytes=1 << 40)
        a.update(kw)
        return lib.b200q_nvfp4_kv_attention(*a.values(), None)

    for name in ("q", "kc", "ks", "vc", "vs", "k2", "v2", "table", "lens", "out", "ws"):
        assert attention(**{name: None}) == NULL, name
    assert attention(dtype=0) == DTYPE
    for kw in (dict(requests=0), dict(tokens=2), dict(heads=0), dict(group=0), dict(pages=0), dict(page=24), dict(stride=-1), dict(width=-1)):
        assert attention(**kw) == SHAPE, kw
    for kw in (dict(dim=96), dict(width=1 << 20, stride=1 << 20, page=1 << 12), dict(heads=1 << 20, page=1 << 12)):
        assert attention(**kw) == UNSUPPORTED, kw
    for kw in (dict(q=p + 8), dict(qs=65), dict(qh=4), dict(kc=p + 8), dict(out=p + 4), dict(ws=p + 8)):
        assert attention(**kw) == ALIGN, kw
    assert lib.b200q_nvfp4_kv_attention_workspace(1, 1, 1, 1, 96) == SHAPE


def test_status_codes_of_the_step_that_says_what_is_seen():
    from b200q import _cabi

    buf = ctypes.create_string_buffer(512)
    p = (ctypes.addressof(buf) + 31) & ~31

    def step(**kw):
        a = dict(lens=p, new=p, free=p, nfree=1, taken=p, table=p, stride=1, width=1, requests=1, page=16, tokens=1, slots=p,
                 positions=p, cu=p, lens_out=p, taken_out=p, status=p, seen=p)
        a.update(kw)
        return _cabi.lib.b200q_kv_step_seen(*a.values(), None)

    for name in ("lens", "new", "free", "taken", "table", "slots", "positions", "cu", "lens_out", "taken_out", "status"):
        assert step(**{name: None}) == -1, name
    assert step(requests=0) == -4 and step(stride=0) == -4 and step(requests=8193) == -7
    assert step(requests=8193, seen=None) == -7
