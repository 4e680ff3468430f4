"""Weight-only layers on their packed 4-bit weights, the NVFP4 KV cache class, and a decoding step of both."""
import copy

import pytest
import torch
import torch.nn.functional as F
from torch import nn

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Mlp(nn.Module):
    def __init__(self, hidden=256, inner=384, bias=True):
        super().__init__()
        self.mlp = nn.Sequential(nn.Linear(hidden, inner, bias=bias), nn.SiLU(), nn.Linear(inner, hidden, bias=bias))

    def forward(self, x):
        return self.mlp(x)


def _compressed(cfg, dtype=torch.bfloat16, config=None, seed=0):
    import b200q as mtq

    torch.manual_seed(seed)
    model = Mlp().to(dtype).cuda()
    data = torch.randn(64, 256, device=DEV, dtype=dtype) * torch.linspace(0.1, 3, 256, device=DEV, dtype=dtype)
    mtq.quantize(model, copy.deepcopy(cfg), lambda m: m(data))
    mtq.compress(model, config)
    return model


def _weights64(model):
    return [m.weight_quantizer.dequantize(m.weight).double() for m in model.mlp if hasattr(m, "weight_quantizer")]


CFGS = ["INT4_AWQ_CFG", "INT4_BLOCKWISE_WEIGHT_ONLY_CFG", "NVFP4_MLP_WEIGHT_ONLY_CFG"]


@pytest.mark.parametrize("name", CFGS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layers_read_the_packed_weight(name, dtype):
    import b200q as mtq

    cfg = getattr(mtq, name)
    plain, fast = (_compressed(cfg, dtype, config) for config in (None, {"weight_only_gemm": True}))
    calls = []
    from b200q import ops
    real = ops._w4_linear
    try:
        ops._w4_linear = lambda *a, **k: (calls.append(a[0]), real(*a, **k))[1]
        for rows in ((1,), (5,), (2, 3), (32,)):
            x = torch.randn(*rows, 256, device=DEV, dtype=dtype)
            calls.clear()
            with torch.no_grad():
                want = plain(x)
            assert not calls                                 # nothing changes without the switch
            with torch.no_grad():
                got = fast(x)
            assert len(calls) == 2 and got.shape == want.shape
            # the fast path in 64 bits, layer by layer, from the same packed weights
            y = x.double().detach()
            size = 0
            for m in fast.mlp:
                if hasattr(m, "weight_quantizer"):
                    s = m.input_quantizer.pre_quant_scale
                    h = y if s is None else (y.to(dtype) * s).double()
                    w = m.weight_quantizer.dequantize(m.weight).double()
                    y, size = F.linear(h, w, m.bias.double()).detach(), (h.abs() @ w.abs().t() + m.bias.double().abs()).detach()
                else:
                    y = m(y)
            # dequantised weights rounded to 16 bits here, outputs and activations of two layers rounded there: four
            # roundings of half a step each, on sums whose magnitudes add up to `size`
            assert float(((got.double() - y).abs() - 4 * torch.finfo(dtype).eps / 2 * size).max()) <= 0
            assert float(((got.double() - want.double()).abs() - 8 * torch.finfo(dtype).eps / 2 * size).max()) <= 0
    finally:
        ops._w4_linear = real


@pytest.mark.parametrize("name", CFGS)
def test_many_rows_take_the_dequantising_path(name):
    import b200q as mtq
    from b200q.backends.weight_only_gemm import WEIGHT_ONLY_MAX_ROWS

    plain, fast = (_compressed(getattr(mtq, name), config=c) for c in (None, {"weight_only_gemm": True}))
    limit = WEIGHT_ONLY_MAX_ROWS[fast.mlp[0].weight.metadata["qtensor_class"]]
    x = torch.randn(limit + 1, 256, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(fast(x), plain(x)) and not torch.equal(fast(x[:-1]), plain(x[:-1]))


def test_switching_on_and_off():
    import b200q as mtq

    model = _compressed(mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG)
    x = torch.randn(3, 256, device=DEV, dtype=torch.bfloat16)
    plain = model(x)
    mtq.backends.enable_real_quant_gemm(model)               # without weight_only: as before
    assert torch.equal(model(x), plain)
    mtq.backends.enable_real_quant_gemm(model, weight_only=True)
    fast = model(x)
    mtq.backends.disable_real_quant_gemm(model)
    assert torch.equal(model(x), plain) and not torch.equal(fast, plain)


def test_layers_that_are_not_marked_keep_their_gemm():
    """An NVFP4 layer whose input quantiser is switched off after compress runs what it ran before."""
    import b200q as mtq
    from b200q import ops

    torch.manual_seed(0)
    layer = nn.Sequential(nn.Linear(256, 64)).bfloat16().cuda()
    x = torch.randn(4, 256, device=DEV, dtype=torch.bfloat16)
    mtq.quantize(layer, copy.deepcopy(mtq.NVFP4_DEFAULT_CFG), lambda m: m(x))
    mtq.compress(layer)
    want = layer(x)
    del layer[0]._real_quant_gemm_impl
    mtq.disable_quantizer(layer, "*input_quantizer")
    assert torch.equal(layer(x), want)
    mtq.backends.enable_real_quant_gemm(layer, weight_only=True)
    got = layer(x)
    m = layer[0]
    assert torch.equal(got, ops.nvfp4_linear(x, m.weight.data, m.weight_quantizer._scale, m.weight_quantizer._double_scale, m.bias))
    mtq.enable_quantizer(layer, "*input_quantizer")
    mtq.backends.enable_real_quant_gemm(layer)                     # both enabled again: the layer's own GEMM again
    assert torch.equal(layer(x), want)


def test_autocast_to_another_type():
    import b200q as mtq

    torch.manual_seed(0)
    layer = nn.Sequential(nn.Linear(256, 64)).half().cuda()
    mtq.quantize(layer, copy.deepcopy(mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG), lambda m: None)
    mtq.compress(layer, {"weight_only_gemm": True})
    x = torch.randn(4, 256, device=DEV, dtype=torch.float16)
    assert layer(x).dtype == torch.float16
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert layer(x).dtype == torch.bfloat16


def test_other_types_and_empty_inputs_fall_back():
    import b200q as mtq

    model = _compressed(mtq.INT4_AWQ_CFG, torch.float32, {"weight_only_gemm": True})
    plain = _compressed(mtq.INT4_AWQ_CFG, torch.float32)
    x = torch.randn(3, 256, device=DEV)
    with pytest.warns(UserWarning, match="no real-quant GEMM"):
        assert torch.equal(model(x), plain(x))               # fp32: not covered
    fast = _compressed(mtq.INT4_AWQ_CFG, config={"weight_only_gemm": True})
    assert fast(torch.empty(0, 256, device=DEV, dtype=torch.bfloat16)).shape == (0, 256)


@pytest.mark.parametrize("name", CFGS)
def test_gradients(name):
    """The input's and the biases' gradients: against the formula on the dequantised weights, and against
    differences of the layer itself."""
    import b200q as mtq

    model = _compressed(getattr(mtq, name), torch.float16, {"weight_only_gemm": True})
    layer = model.mlp[0]
    x = torch.randn(4, 256, device=DEV, dtype=torch.float16).requires_grad_()
    g = torch.randn(4, 384, device=DEV, dtype=torch.float16)
    layer.bias.grad = None
    layer(x).backward(g)
    w = layer.weight_quantizer.dequantize(layer.weight).double()
    s = layer.input_quantizer.pre_quant_scale
    s = 1.0 if s is None else s.double()
    want = (g.double() @ w) * s
    size = (g.double().abs() @ w.abs()) * s
    assert float(((x.grad.double() - want).abs() - (4 * 2.0 ** -11 * size + 2.0 ** -24)).max()) <= 0
    assert float(((layer.bias.grad.double() - g.double().sum(0)).abs() - 4 * 2.0 ** -11 * g.double().abs().sum(0)).max()) <= 0
    # the layer is linear: the difference along a direction is its derivative, whatever the step
    d = torch.randn(4, 256, device=DEV, dtype=torch.float16)
    with torch.no_grad():
        diff = (layer(x + d).double() - layer(x - d).double()) * g.double()
    moved = ((x + d).double() - (x - d).double()) * x.grad.double()
    slack = 2.0 ** -11 * 8 * ((x.abs().double() + d.abs().double()) * size).sum()     # outputs rounded, twice
    assert abs(float(diff.sum() - moved.sum())) <= float(slack)


def test_restored_model_keeps_the_switch():
    import b200q as mtq

    model = _compressed(mtq.INT4_AWQ_CFG, config={"weight_only_gemm": True})
    x = torch.randn(2, 256, device=DEV, dtype=torch.bfloat16)
    again = Mlp().bfloat16().cuda()
    mtq.restore_from_modelopt_state(again, mtq.modelopt_state(model))
    again.load_state_dict(model.state_dict())
    assert mtq.backends.is_real_quant_gemm_enabled(again)
    assert torch.equal(again(x), model(x))


# ------------------------------------------------------------------------------------ KV cache ----

def _quantizer(amax, **kw):
    import b200q as mtq

    q = mtq.nn.TensorQuantizer(mtq.config.QuantizerAttributeConfig(
        num_bits=(2, 1), block_sizes={-1: 16, "type": "dynamic", "scale_bits": (4, 3)}, **kw)).cuda()
    q.amax = torch.tensor(float(amax), device=DEV)
    return q


def _cache(amax=4.3, **kw):
    import b200q as mtq

    sizes = dict(num_pages=24, kv_heads=2, head_dim=64, max_requests=3, page_size=16)
    sizes.update(kw)
    quantizers = [(_quantizer(amax), _quantizer(amax + 1)) for _ in range(2)]
    return mtq.NVFP4KVCache.from_quantizers(quantizers, **sizes), quantizers


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_cache_attends_like_fake_quantised_keys_and_values():
    cache, quantizers = _cache()
    g = torch.Generator(device=DEV).manual_seed(1)
    held = [[[], []] for _ in range(3)]
    for new in ([20, 3, 0], [1, 1, 7], [2, 0, 1]):
        t = sum(new)
        step = cache.step(_int32(new), t)
        for layer, (kq, vq) in enumerate(quantizers):
            q = torch.randn(t, 8, 64, generator=g, device=DEV).bfloat16()
            k, v = (torch.randn(t, 2, 64, generator=g, device=DEV).bfloat16() for _ in range(2))
            cache.append(layer, k, v, step)
            out = cache.attend(layer, q, step)
            if layer:
                continue
            at = 0
            for r, m in enumerate(new):
                held[r][0].append(kq(k[at:at + m]).double())
                held[r][1].append(vq(v[at:at + m]).double())
                K, V = torch.cat(held[r][0]), torch.cat(held[r][1])
                for i in range(m):
                    see = K.shape[0] - m + i + 1
                    z = torch.einsum("hgd,nhd->hgn", q[at + i].double().view(2, 4, 64), K[:see]) / 8
                    want = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), V[:see]).reshape(8, 64)
                    # fake-quantised values are rounded to bf16, the cache's are not: 2^-8 of each in the scores
                    # (the sum of magnitudes below 40 / 8 at |k| < 4.3) and in the result
                    assert float((out[at + i].double() - want).abs().max()) <= 2.0 ** -8 * (2 * 5 + 2) * float(V[:see].abs().max())
                at += m
    cache.check()


def test_cache_release_and_refusal():
    cache, _ = _cache(num_pages=4)
    step = cache.step(_int32([30, 16, 1]), 47)               # 2 + 1 + 1 pages
    cache.check()
    assert cache.lens.tolist() == [30, 16, 1] and int(cache.taken) == 4 and (step.slots >= 0).all()
    cache.step(_int32([2, 1, 1]), 4)                         # request 1 needs a page
    assert cache.lens.tolist() == [32, 16, 2]
    with pytest.raises(RuntimeError, match="no free page"):
        cache.check()
    cache.check()
    pages = set(cache.block_table[0, :2].tolist())
    cache.release(0)
    assert cache.lens.tolist() == [0, 16, 2] and int(cache.taken) == 2 and (cache.block_table[0] == -1).all()
    cache.step(_int32([1, 1, 0]), 2)
    cache.check()
    assert {int(cache.block_table[0, 0]), int(cache.block_table[1, 1])} == pages
    with pytest.raises(IndexError):
        cache.release(3)


def test_cache_step_captured_and_replayed():
    from b200q import ops

    cache, _ = _cache(num_pages=30)
    dense = {r: [] for r in range(3)}
    q, k, v = (torch.zeros(3, h, 64, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    new = _int32([1, 1, 1])

    def one():
        st = cache.step(new, 3)
        kv, vv = cache.append(0, k, v, st, return_values=True)
        return cache.attend(0, q, st), kv, vv

    one()
    cache.lens.zero_(), cache.taken.zero_(), cache.block_table.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, kv, vv = one()
    cache.lens.zero_(), cache.taken.zero_(), cache.block_table.fill_(-1)
    g = torch.Generator(device=DEV).manual_seed(3)
    for n in range(40):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for r in range(3):
            dense[r].append((kv[r].double(), vv[r].double()))
    assert cache.lens.tolist() == [40] * 3
    cache.check()
    for r in range(3):
        K, V = (torch.stack([p[i] for p in dense[r]]) for i in range(2))
        z = torch.einsum("hgd,nhd->hgn", q[r].double().view(2, 2, 64), K) / 8
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), V).reshape(4, 64)
        assert float((out[r].double() - want).abs().max()) <= 2.0 ** -8 * (2 * 5 + 2) * float(V.abs().max())


def test_cache_refuses_other_formats():
    import b200q as mtq

    fp8 = mtq.nn.TensorQuantizer(mtq.config.QuantizerAttributeConfig(num_bits=(4, 3))).cuda()
    fp8.amax = torch.tensor(3.0, device=DEV)
    good, sizes = _quantizer(4.0), dict(num_pages=4, kv_heads=1, head_dim=64, max_requests=1)
    off, rotated = _quantizer(4.0), _quantizer(4.0)
    off.disable()
    rotated._rotate = True
    for bad in (fp8, off):
        with pytest.raises(ValueError):
            mtq.NVFP4KVCache.from_quantizers([(good, bad)], **sizes)
    with pytest.raises(NotImplementedError):
        mtq.NVFP4KVCache.from_quantizers([(rotated, good)], **sizes)
    for wrong in (dict(head_dim=96), dict(page_size=24), dict(num_pages=0)):
        with pytest.raises(ValueError):
            mtq.NVFP4KVCache([], **{**sizes, **wrong})
    with pytest.raises(RuntimeError):
        mtq.NVFP4KVCache([], **sizes, device="cpu")


# ------------------------------------------------------------------------------------ together ----

def test_decoding_step_of_a_4_bit_model():
    """Attention and MLP layers with INT4 weights over an NVFP4 cache: a prompt, then tokens one by one, against the
    same layers with dequantised weights and fake-quantised keys and values over the whole sequence."""
    import b200q as mtq

    heads, kv, dim, hidden = 4, 2, 64, 256

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.qkv = nn.Linear(hidden, (heads + 2 * kv) * dim, bias=False)
            self.o = nn.Linear(heads * dim, hidden, bias=False)
            self.mlp = Mlp(hidden, 512)

    torch.manual_seed(0)
    block = Block().bfloat16().cuda()
    mtq.quantize(block, copy.deepcopy(mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG))
    mtq.compress(block, {"weight_only_gemm": True})
    cache, ((kq, vq), _) = _cache(2.2, kv_heads=kv, head_dim=dim, max_requests=2)

    def forward(x, attend):
        q, k, v = block.qkv(x).unflatten(-1, (heads + 2 * kv, dim)).split([heads, kv, kv], -2)
        x = x + block.o(attend(q, k, v).flatten(-2))
        return x + block.mlp(x)

    xs = [torch.randn(n, hidden, device=DEV).bfloat16() for n in (37, 12)]
    outs = [[], []]
    for new in ([30, 6], *[[1, 1]] * 6, [1, 0]):
        at = [sum(len(o) for o in outs[r]) for r in range(2)]
        x = torch.cat([xs[r][at[r]:at[r] + new[r]] for r in range(2)])
        st = cache.step(_int32(new), x.shape[0])

        def attend(q, k, v):
            cache.append(0, k, v, st)
            return cache.attend(0, q, st)

        y = forward(x, attend)
        outs[0].append(y[:new[0]])
        outs[1].append(y[new[0]:])
    cache.check()
    mtq.backends.disable_real_quant_gemm(block)
    for r in range(2):
        n = xs[r].shape[0]

        def dense(q, k, v):
            k, v = kq(k.contiguous()), vq(v.contiguous())
            z = torch.einsum("ihgd,nhd->hgin", q.float().view(n, kv, heads // kv, dim), k.float()) / 8
            z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
            return torch.einsum("hgin,nhd->ihgd", torch.softmax(z, -1), v.float()).reshape(n, heads, dim).bfloat16()

        want = forward(xs[r], dense).float()
        got = torch.cat(outs[r]).float()
        # the two differ by roundings to bf16 in between (a dozen of 2^-8 on values of the output's size)
        assert float((got - want).norm() / want.norm()) <= 12 * 2.0 ** -8


@pytest.mark.parametrize("refused", ["no page", "row full", "too few rows"])
def test_rows_of_a_refused_request_see_nothing(refused):
    """A refused request's rows have no keys of their own in the cache: they are zero with log-sum -inf, and the other
    requests' rows are what they are without it."""
    from b200q import ops

    cache, _ = _cache(num_pages=4 if refused == "no page" else 24, max_pages_per_request=2 if refused == "row full" else 4)
    g = torch.Generator(device=DEV).manual_seed(2)

    def step(new, rows):
        t = sum(new)
        st = cache.step(_int32(new), rows)
        q = torch.randn(t, 8, 64, generator=g, device=DEV).bfloat16()
        k, v = (torch.randn(t, 2, 64, generator=g, device=DEV).bfloat16() for _ in range(2))
        cache.append(0, k[:rows], v[:rows], st)
        return q, st, cache.attend(0, q[:rows], st, return_lse=True)

    first = [20, 30, 16] if refused != "no page" else [20, 16, 1]
    step(first, sum(first))
    cache.check()
    held = cache.lens.tolist()
    new = [1, 5, 2] if refused != "too few rows" else [1, 2, 5]
    rows = sum(new) if refused != "too few rows" else sum(new) - 1
    bad = 1 if refused != "too few rows" else 2
    q, st, (out, lse) = step(new, rows)
    with pytest.raises(RuntimeError):
        cache.check()
    assert cache.lens.tolist() == [n + (m if r != bad else 0) for r, (n, m) in enumerate(zip(held, new))]
    rows_of = [slice(a, b) for a, b in zip(st.cu_new.tolist(), st.cu_new.tolist()[1:])]
    assert (st.slots[rows_of[bad]] == -1).all()
    assert (out[rows_of[bad]] == 0).all() and (lse[rows_of[bad]] == -float("inf")).all()
    see = cache.lens.clone()
    see[bad] = 0
    kc, vc, k2, v2 = cache.layers[0]
    want, wlse = ops.nvfp4_kv_attention(q[:rows], kc, vc, k2, v2, cache.block_table, see, cu_q=st.cu_new, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    assert all((lse[rows_of[r]] > -float("inf")).all() for r in range(3) if r != bad)


@pytest.mark.parametrize("name", CFGS)
def test_a_first_call_that_is_not_covered_is_not_remembered(name):
    """A marked layer whose first call runs under autocast to another type, or with another input type, still reads the
    packed weight in the calls that are covered."""
    import b200q as mtq
    from b200q import ops

    x = torch.randn(4, 256, device=DEV, dtype=torch.float16)
    want = _compressed(getattr(mtq, name), torch.float16, {"weight_only_gemm": True})(x)
    calls, real = [], ops._w4_linear
    try:
        ops._w4_linear = lambda *a, **k: (calls.append(a[0]), real(*a, **k))[1]
        model = _compressed(getattr(mtq, name), torch.float16, {"weight_only_gemm": True})
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert model(x).dtype == torch.bfloat16
        assert not calls
        assert torch.equal(model(x), want) and len(calls) == 2
        calls.clear()
        model = _compressed(getattr(mtq, name), torch.float16, {"weight_only_gemm": True})
        with pytest.raises(RuntimeError):
            model(x.float())                                 # as F.linear says it of two types
        assert not calls
        assert torch.equal(model(x), want) and len(calls) == 2
    finally:
        ops._w4_linear = real


def test_cache_refuses_quantisers_with_a_pre_quant_scale():
    """A scale that the quantiser puts on its input first would be missing from the cache's keys."""
    import b200q as mtq

    good, scaled = _quantizer(4.0), _quantizer(4.0)
    scaled.pre_quant_scale = torch.full((64,), 0.5, device=DEV)
    for pair in ((scaled, good), (good, scaled)):
        with pytest.raises(NotImplementedError, match="pre-quant"):
            mtq.NVFP4KVCache.from_quantizers([pair], num_pages=4, kv_heads=1, head_dim=64, max_requests=1)


def test_cache_of_a_model_calibrated_by_quantize():
    """``quantize`` with NVFP4_KV_CFG on registered attention modules, a cache from their calibrated quantisers, and each
    layer's attention against the module's fake-quantised keys and values in 64 bits; a later prompt exceeds the calibrated
    range.  Counted: the result's half step, P in fp16 (2^-11 of each weight, 2^-25 below its normal range), the scores in
    fp32 (dim + 8 operations of 2^-23 on the sum of magnitudes, twice in a weight's ratio to the sum) and the fake-quantised
    values' own fp32 (2^-24, in the scores twice and in the result)."""
    import b200q as mtq

    heads, group, dim = 2, 3, 64

    class Attention(nn.Module):
        def forward(self, q, k, v):
            n = k.shape[0]
            z = torch.einsum("ihgd,nhd->hgin", q.view(-1, heads, group, dim), k) * dim ** -0.5
            z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
            return torch.einsum("hgin,nhd->ihgd", torch.softmax(z, -1), v).reshape(n, heads * group, dim)

    class QuantAttention(Attention):
        def _setup(self):
            self.q_bmm_quantizer, self.k_bmm_quantizer, self.v_bmm_quantizer = (mtq.nn.TensorQuantizer() for _ in range(3))

        def forward(self, q, k, v):
            return super().forward(self.q_bmm_quantizer(q), self.k_bmm_quantizer(k), self.v_bmm_quantizer(v))

    mtq.register(original_cls=Attention, quantized_cls=QuantAttention)
    try:
        model = nn.ModuleList([Attention(), Attention()]).cuda()
        g = torch.Generator(device=DEV).manual_seed(7)

        def data(n, size):
            q, k, v = (torch.randn(n, h, dim, generator=g, device=DEV) for h in (heads * group, heads, heads))
            return [t.bfloat16().float() for t in (q, k * size, v * size)]

        calibration = [data(50, 1.0 + i) for i in range(2)]
        mtq.quantize(model, copy.deepcopy(mtq.NVFP4_KV_CFG), lambda m: [m[i](*calibration[i]) for i in range(2)])
        cache = mtq.NVFP4KVCache.from_quantizers([(m.k_bmm_quantizer, m.v_bmm_quantizer) for m in model], num_pages=20,
                                                 kv_heads=heads, head_dim=dim, max_requests=1, page_size=16)
        for i, m in enumerate(model):
            for name, at in (("k", 1), ("v", 2)):
                amax = calibration[i][at].abs().max()
                assert abs(float(cache.layers[i][1 + at] / amax * 2688) - 1) < 2.0 ** -22
        step = cache.step(_int32([90]), 90)
        cache.check()
        for i, m in enumerate(model):
            q, k, v = data(90, (1.0 + i) * 1.5)
            cache.append(i, k.bfloat16(), v.bfloat16(), step)
            out = cache.attend(i, q.bfloat16(), step).double()
            K, V = m.k_bmm_quantizer(k), m.v_bmm_quantizer(v)
            assert torch.isfinite(K).all() and torch.isfinite(V).all() and float(k.abs().max()) > float(calibration[i][1].abs().max())
            K, V, Q = K.double(), V.double(), q.double().view(90, heads, group, dim)
            want = Attention.forward(m, q.double(), K, V)
            p_abs = Attention.forward(m, q.double(), K, V.abs())
            big = torch.einsum("ihgd,nhd->hgin", Q.abs(), K.abs()).max() * dim ** -0.5
            rel = 2.0 ** -11 + 2 * (dim + 12) * 2.0 ** -23 * float(big) + 2.0 ** -20
            tol = (2.0 ** -8 * want.abs() + rel * p_abs + 90 * 2.0 ** -25 * V.abs().max()) * 1.01
            assert float(((out - want).abs() - tol).max()) <= 0
    finally:
        mtq.unregister(Attention)


@pytest.mark.parametrize("name,n,k,packed,dequantised", [
    ("INT4_BLOCKWISE_WEIGHT_ONLY_CFG", 512, 512, [1, 32], [33, 64, 128]),
    ("INT4_BLOCKWISE_WEIGHT_ONLY_CFG", 2048, 2048, [32, 33, 64], [65, 128]),
    ("INT4_BLOCKWISE_WEIGHT_ONLY_CFG", 5120, 5120, [64, 65, 128], [129]),
    ("NVFP4_MLP_WEIGHT_ONLY_CFG", 2048, 2048, [1, 32], [33])])
def test_rows_that_take_several_launches_need_a_large_layer(name, n, k, packed, dequantised):
    """Several launches of the packed product only where the weight is large enough to pay for them."""
    import b200q as mtq
    from b200q import ops

    class Layer(nn.Module):
        def __init__(self):
            super().__init__()
            self.mlp = nn.Linear(k, n, bias=False)

    model = Layer().bfloat16().cuda()
    mtq.quantize(model, copy.deepcopy(getattr(mtq, name)), lambda m: None)
    mtq.compress(model, {"weight_only_gemm": True})
    calls, real = [], ops._w4_linear
    try:
        ops._w4_linear = lambda *a, **kw: (calls.append(a[0]), real(*a, **kw))[1]
        for rows in packed + dequantised:
            x = torch.randn(rows, k, device=DEV, dtype=torch.bfloat16)
            calls.clear()
            with torch.no_grad():
                got = model.mlp(x)
                assert len(calls) == (rows in packed), rows
                want = F.linear(x, model.mlp.weight_quantizer.dequantize(model.mlp.weight))
            size = x.float().abs() @ model.mlp.weight_quantizer.dequantize(model.mlp.weight).float().abs().t()
            # weights rounded to bf16 on one side, outputs on both
            assert float(((got.float() - want.float()).abs() - 3 * 2.0 ** -8 * size).max()) <= 0
    finally:
        ops._w4_linear = real
