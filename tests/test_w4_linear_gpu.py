"""Products of a few rows with 4-bit weights (INT4 with group scales, NVFP4) against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
E2M1 = [0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6]


def _int4(n, k, block, dtype, seed):
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(n, k, generator=g, device=DEV) * torch.logspace(-3, 0, n, device=DEV).unsqueeze(1)).to(dtype)
    packed, scales = ops.int4_quantize(w.reshape(-1), block)
    packed = packed.reshape(n, k // 2)
    c = torch.stack((packed >> 4, packed & 15), -1).reshape(n, k // block, block).double()
    return packed, scales, ((c - 8) / scales.reshape(n, -1, 1).double()).reshape(n, k)


def _nvfp4(n, k, dtype, seed, block=16):
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(n, k, generator=g, device=DEV) * torch.logspace(-3, 0, n, device=DEV).unsqueeze(1)).to(dtype)
    packed, scales, s2 = ops.nvfp4_quantize(w, block=block)
    lut = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    v = lut[torch.stack((packed & 15, packed >> 4), -1).reshape(n, k).long()]
    return packed, scales, s2, (v.reshape(n, -1, block) * scales.float().double().unsqueeze(-1)).reshape(n, k) * s2.double()


def _close(out, x, w, bias=None):
    """Half a step of the output's type, the fp32 sums (k + 8 operations, each off by at most 2^-23 of the sum of
    magnitudes; the tensor core may truncate where it adds), the group's reciprocal and its product (2^-22), and x's
    smallest elements in fp16 (2^-38 of the row's largest).  Results beyond the type's largest number are infinite: both
    sides are compared cut off there."""
    ref = x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    if bias is not None:
        ref = ref + bias.double()
        size = size + bias.double().abs()
    info = torch.finfo(out.dtype)
    tol = (info.eps / 2 * ref.abs().clamp(min=info.tiny) + size * ((x.shape[-1] + 8) * 2.0 ** -23 + 2.0 ** -21)
           + 2.0 ** -38 * x.double().abs().amax(-1, keepdim=True) * w.abs().sum(1)) * 1.01
    assert out.shape == ref.shape
    out, ref = (t.clamp(-info.max, info.max) for t in (out.double(), ref))
    assert float(((out - ref).abs() - tol).max()) <= 0


def _x(m, k, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(100 + seed)
    x = torch.randn(m, k, generator=g, device=DEV)
    x[:, ::53] *= 30
    return x.to(dtype)


SIZES = [(1, 32), (16, 128), (17, 160), (33, 2080), (100, 4096), (4097, 256), (48, 14336), (64, 8320)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 3, 8, 9, 16, 27, 32])
@pytest.mark.parametrize("n,k", SIZES)
def test_nvfp4_linear(dtype, m, n, k):
    from b200q import ops

    packed, scales, s2, w = _nvfp4(n, k, dtype, seed=n + m)
    x = _x(m, k, dtype, m)
    _close(ops.nvfp4_linear(x, packed, scales, s2), x, w)


@pytest.mark.parametrize("m", [1, 5, 12, 32])
@pytest.mark.parametrize("n,k", [(1, 32), (20, 96), (17, 288), (100, 4096), (16, 8224)])
def test_nvfp4_linear_with_scale_blocks_of_32(m, n, k):
    from b200q import ops

    packed, scales, s2, w = _nvfp4(n, k, torch.bfloat16, seed=n + m, block=32)
    x = _x(m, k, torch.bfloat16, m)
    _close(ops.nvfp4_linear(x, packed, scales, s2, block=32), x, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 2, 7, 13, 30])
@pytest.mark.parametrize("n,k,block", [(1, 32, 32), (20, 96, 32), (15, 64, 64), (77, 2112, 64), (16, 128, 128), (130, 2688, 128),
                                       (4099, 384, 128), (40, 14336, 128), (33, 1024, 256), (7, 8192, 1024), (24, 28672, 32)])
def test_int4_linear(dtype, m, n, k, block):
    from b200q import ops

    packed, scales, w = _int4(n, k, block, dtype, seed=n + m)
    x = _x(m, k, dtype, m)
    _close(ops.int4_linear(x, packed, scales, block), x, w)


@pytest.mark.parametrize("m,k", [(33, 512), (70, 128), (40, 28672)])
def test_more_rows_than_one_launch_takes(m, k):
    from b200q import ops

    packed, scales, s2, w = _nvfp4(50, k, torch.bfloat16, seed=1)
    x = _x(m, k, torch.bfloat16)
    _close(ops.nvfp4_linear(x, packed, scales, s2), x, w)


def test_bias_shapes_and_strides():
    from b200q import ops

    n, k = 70, 512
    packed, scales, s2, w = _nvfp4(n, k, torch.float16, seed=1)
    bias = torch.randn(n, device=DEV)                     # cast to x's dtype
    x = _x(6, k, torch.float16)
    want = ops.nvfp4_linear(x, packed, scales, s2, bias)
    _close(want, x, w, bias.half())
    assert torch.equal(ops.nvfp4_linear(x.view(2, 3, k), packed, scales, s2, bias), want.view(2, 3, n))
    assert torch.equal(ops.nvfp4_linear(x[0], packed, scales, s2, bias), want[0])
    wide = torch.zeros(6, 2 * k, dtype=x.dtype, device=DEV)
    wide[:, k:] = x
    assert torch.equal(ops.nvfp4_linear(wide[:, k:], packed, scales, s2, bias), want)      # strided rows
    odd = torch.zeros(6, k + 1, dtype=x.dtype, device=DEV)
    odd[:, 1:] = x
    assert torch.equal(ops.nvfp4_linear(odd[:, 1:], packed, scales, s2, bias), want)       # unaligned: copied
    assert torch.equal(ops.nvfp4_linear(x[:1].expand(6, k), packed, scales, s2, bias), want[:1].expand(6, n))
    assert ops.nvfp4_linear(x[:0], packed, scales, s2).shape == (0, n)
    shifted = torch.empty(n * k // 2 + 1, dtype=torch.uint8, device=DEV)[1:].view(n, k // 2)
    shifted.copy_(packed)
    assert torch.equal(ops.nvfp4_linear(x, shifted, scales, s2, bias), want)


@pytest.mark.parametrize("block", [16, 32])
def test_scales_at_odd_addresses(block):
    from b200q import ops

    packed, scales, s2, _ = _nvfp4(20, 96, torch.bfloat16, seed=3, block=block)
    x = _x(3, 96, torch.bfloat16)
    odd = torch.empty(scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:]
    odd.copy_(scales.view(torch.uint8).flatten())
    want = ops.nvfp4_linear(x, packed, scales, s2, block=block)
    assert torch.equal(ops.nvfp4_linear(x, packed, odd.view(torch.float8_e4m3fn).view(20, -1), s2, block=block), want)


@pytest.mark.parametrize("scale", [1e-36, 1e-5, 1e5, 1e36])
def test_bf16_rows_of_any_magnitude(scale):
    from b200q import ops

    packed, scales, s2, w = _nvfp4(40, 1024, torch.bfloat16, seed=1)
    x = (_x(5, 1024, torch.bfloat16).float() * scale).bfloat16()
    x[1] *= 2.0 ** -60 if scale > 1 else 1                 # rows are scaled one by one
    assert torch.isfinite(x).all()
    _close(ops.nvfp4_linear(x, packed, scales, s2), x, w)
    packed, scales, w = _int4(40, 1024, 128, torch.bfloat16, seed=2)
    _close(ops.int4_linear(x, packed, scales, 128), x, w)


@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 9, 20])
def test_fp16_rows_of_any_magnitude(m, block):
    """Rows from the smallest numbers of the type (2^-24 and few bits) to its largest, each as exact as the others.  The
    weights are large enough for the smallest rows' results to be normal numbers."""
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(m)
    w = (torch.randn(40, 1024, generator=g, device=DEV) * 100).half()
    packed, scales = ops.int4_quantize(w.reshape(-1), block)
    packed = packed.reshape(40, 512)
    c = torch.stack((packed >> 4, packed & 15), -1).reshape(40, 1024 // block, block).double()
    w = ((c - 8) / scales.reshape(40, -1, 1).double()).reshape(40, 1024)
    size = torch.logspace(-24, 0, m, base=2, device=DEV).unsqueeze(1)
    x = (torch.randn(m, 1024, generator=g, device=DEV).clamp(-2, 2) * size * 4).half()
    assert torch.isfinite(x).all()
    _close(ops.int4_linear(x, packed, scales, block), x, w)
    big = (torch.randn(m, 1024, generator=g, device=DEV).clamp(-2, 2) * 32752).half()      # up to 65504
    small = w / 4096                                                                       # the same codes, smaller weights
    _close(ops.int4_linear(big, packed, (scales.float() * 4096).half(), block), big, small)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_not_finite_rows_stay_alone(dtype):
    from b200q import ops

    packed, scales, w = _int4(64, 512, 128, dtype, seed=4)
    x = _x(9, 512, dtype)
    want = ops.int4_linear(x, packed, scales, 128)
    y = x.clone()
    y[2, 77], y[8, 500] = math.inf, math.nan
    got = ops.int4_linear(y, packed, scales, 128)
    keep = [0, 1, 3, 4, 5, 6, 7]
    assert torch.equal(got[keep], want[keep])
    assert torch.isnan(got[8]).all()
    zero = w[:, 77] == 0
    assert torch.isnan(got[2][zero]).all()                # inf * 0
    assert torch.equal(got[2][~zero], torch.copysign(torch.full_like(got[2], math.inf), w[:, 77].to(dtype))[~zero])


def test_zero_blocks_and_zero_rows():
    from b200q import ops

    w = torch.randn(20, 256, device=DEV).bfloat16()
    w[3], w[5, :128] = 0, 0
    packed, scales = ops.int4_quantize(w.reshape(-1), 128)                 # 7 / 0 = inf: the block's weights are 0
    x = _x(4, 256, torch.bfloat16)
    x[2] = 0
    out = ops.int4_linear(x, packed.view(20, 128), scales, 128)
    assert torch.isfinite(out).all() and (out[:, 3] == 0).all() and (out[2] == 0).all()


def test_deterministic_and_on_two_streams():
    from b200q import ops

    packed, scales, s2, _ = _nvfp4(512, 8192, torch.bfloat16, seed=1)
    xs = [_x(16, 8192, torch.bfloat16, s) for s in range(2)]
    want = [ops.nvfp4_linear(x, packed, scales, s2) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.nvfp4_linear(xs[i], packed, scales, s2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_captured_and_replayed():
    from b200q import ops

    packed, scales, w = _int4(300, 1024, 64, torch.float16, seed=2)
    x = _x(3, 1024, torch.float16, 1)
    ops.int4_linear(x, packed, scales, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.int4_linear(x, packed, scales, 64)
    for seed in (5, 6):
        x.copy_(_x(3, 1024, torch.float16, seed))
        graph.replay()
        assert torch.equal(out, ops.int4_linear(x, packed, scales, 64))


def test_refusals():
    from b200q import ops

    packed, scales, w = _int4(16, 256, 128, torch.float16, seed=2)
    x = _x(2, 256, torch.float16)
    with pytest.raises(TypeError):
        ops.int4_linear(x.float(), packed, scales.float(), 128)
    with pytest.raises(TypeError):
        ops.int4_linear(x, packed, scales.bfloat16(), 128)
    for args in ((x[:, :128], packed, scales, 128), (x, packed, scales[:5], 128), (x, packed, scales, 64), (x, packed, scales, 16),
                 (x, packed, scales, 96), (x, packed.view(-1), scales, 128), (x, packed, scales, 128, torch.zeros(3, device=DEV))):
        with pytest.raises(ValueError):
            ops.int4_linear(*args)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.int4_linear(x.cpu(), packed, scales, 128)
    with pytest.raises(TypeError):
        ops.nvfp4_linear(x, packed, scales, torch.ones((), device=DEV))
    with pytest.raises(ValueError):
        ops.nvfp4_linear(x, packed, scales.view(-1).view(torch.uint8)[: 16 * 4], torch.ones((), device=DEV), block=64)
    assert not ops.nvfp4_linear_supported(x[:, :16], 16, 16) and not ops.int4_linear_supported(x, 256, 16)
    assert ops.nvfp4_linear_supported(x, 256, 32) and ops.int4_linear_supported(x, 256, 256)


# ------------------------------------------------------- several tiles a CTA, sums that leave no room ----

# (rows, n, k) whose CTAs walk over several tiles on 148 SMs: with K whole, over the warps of a tile, over CTAs, and over both
WALKS = [(1, 40003, 256), (1, 40003, 640), (1, 40003, 2304), (8, 8203, 6400), (9, 4099, 2688), (9, 40003, 1024),
         (9, 4099, 12672), (16, 4099, 5632), (17, 4099, 3584), (32, 40003, 256), (32, 4099, 2304), (32, 4099, 5632)]


FORMATS = [("int4", 32), ("int4", 64), ("int4", 128), ("int4", 256), ("nvfp4", 16), ("nvfp4", 32)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,fmt,block", [w + f for w in WALKS for f in FORMATS if w[2] % f[1] == 0])
def test_ctas_that_walk_over_several_tiles(m, n, k, fmt, block, dtype):
    """x holds small integers, so that every sum of 128 elements (INT4: of a group where that is less) is exact in fp32:
    INT4 adds integers, NVFP4 multiples of 2^-5 below 2^7.  What is left is counted from those sums S: each is off by
    3 * 2^-24 (reciprocal or scale2, product), and the additions that follow (INT4: one for each S; in either format the
    joins of at most 16 warps and 16 CTAs) by 2^-24 each of at most the sum of |S|.  NVFP4's chain over a warp's elements
    stays exact: partial sums below 2^17, multiples of 2^-5.  Weights rounded to 16 bits would be off by far more.  The
    reference's own 64 bits count too, where a sum cancels: k products and additions of 2^-53 of the sum of magnitudes."""
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(m + n + k)
    x = torch.randint(-4, 5, (m, k), generator=g, device=DEV).to(dtype)
    packed = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV).to(torch.uint8)
    if fmt == "int4":
        scales = (torch.rand(n * (k // block), 1, generator=g, device=DEV) * 180 + 20).to(dtype)
        out = ops.int4_linear(x, packed, scales, block)
    else:
        s2 = torch.tensor(0.00123, device=DEV)
        scales = torch.randint(0x30, 0x49, (n, k // block), generator=g, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn)
        out = ops.nvfp4_linear(x, packed, scales, s2, block=block)
    unit = min(block, 128) if fmt == "int4" else 128
    adds = (k // unit if fmt == "int4" else 0) + 40
    lut = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    xg = x.double().unflatten(1, (-1, unit)).transpose(0, 1)               # [groups, m, unit]
    for at in range(0, n, 4096):
        c = packed[at:at + 4096]
        if fmt == "int4":
            w = (torch.stack((c >> 4, c & 15), -1).reshape(c.shape[0], -1, block).double() - 8) / scales.view(n, -1, 1)[at:at + 4096].double()
        else:
            w = lut[torch.stack((c & 15, c >> 4), -1).reshape(c.shape[0], -1, block).long()]
            w = w * scales[at:at + 4096].float().double().unsqueeze(-1) * s2.double()
        w = w.reshape(c.shape[0], -1, unit).permute(1, 2, 0)               # [groups, unit, n]
        parts = xg @ w
        ref, size = parts.sum(0), parts.abs().sum(0)
        own = (k + 2) * 2.0 ** -53 * (xg.abs() @ w.abs()).sum(0)
        got = out[:, at:at + 4096].double()
        info = torch.finfo(dtype)
        top = torch.maximum(ref.abs(), got.abs()).clamp(min=info.tiny)
        half = torch.exp2(torch.floor(torch.log2(top))) * info.eps / 2
        assert float(((got - ref).abs() - half - size * adds * 2.0 ** -24 - own).max()) <= 0


def test_replays_keep_the_error_word():
    """A first product under capture: replays must not clear the error bits that were collected before them.  In a process
    of its own, since the word is made by a process's first product."""
    import subprocess
    import sys

    code = """
import sys
sys.path[:0] = %r
import torch
from b200q import ops
packed, scales = ops.int4_quantize(torch.randn(64 * 512, device="cuda").bfloat16(), 128)
packed = packed.view(64, 256)
x = torch.randn(3, 512, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.int4_linear(x, packed, scales, 128)
ops.check_qgemm_status("cuda")                          # clean before the first replay
graph.replay()
ops.check_qgemm_status("cuda")
assert torch.equal(out, ops.int4_linear(x, packed, scales, 128))
ops.qgemm_status("cuda").fill_(4)                       # as a wait that ran out would leave it
graph.replay()
try:
    ops.check_qgemm_status("cuda")
except RuntimeError:
    ops.check_qgemm_status("cuda")                      # told once
else:
    raise AssertionError("the error bits are lost")
""" % sys.path
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
