"""The paged NVFP4 KV cache: page tables and slots of a step, the append, and attention over the cache, each
against a plain implementation in 64 bits (or in whole numbers), at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


# --------------------------------------------------------------------------------- kv_step ----

def _step_reference(lens, new, free, taken, table, page, tokens):
    """The step in whole numbers, request by request."""
    table = [row[:] for row in table]
    slots, positions = [-1] * tokens, [0] * tokens
    cu, lens_out, status, exhausted = [0], [], 0, False
    for b, (n, m) in enumerate(zip(lens, new)):
        first = cu[-1]
        cu.append(first + max(m, 0))
        have, want = -(-n // page), -(-(n + max(m, 0)) // page)
        bad = 0
        if n < 0 or m < 0 or n + m > 2 ** 31 - 1:
            bad = 4
        elif want > len(table[b]):
            bad = 2
        elif cu[-1] > tokens:
            bad = 8
        elif want > have and (exhausted or taken + want - have > len(free)):
            bad, exhausted = 1, True
        status |= bad
        if bad:
            lens_out.append(n)
            continue
        for i in range(have, want):
            table[b][i] = free[taken]
            taken += 1
        for i in range(m):
            pos = n + i
            positions[first + i] = pos
            slots[first + i] = table[b][pos // page] * page + pos % page
        lens_out.append(n + m)
    return table, slots, positions, [min(c, tokens) for c in cu], lens_out, taken, status


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _run_step(lens, new, free, taken, table, page, tokens):
    from b200q import ops

    wide = torch.full((len(lens), len(table[0]) + 3), -7, dtype=torch.int32, device=DEV)   # guard columns
    view = wide[:, : len(table[0])]
    view.copy_(_i32(table))
    args = (_i32(lens), _i32(new), _i32(free), _i32([taken]), view, page, tokens)
    for _ in range(2):                                   # repeating the call changes nothing
        st = ops.kv_step(*args)
    want = _step_reference(lens, new, free, taken, table, page, tokens)
    assert view.tolist() == want[0]
    assert (wide[:, len(table[0]):] == -7).all()
    assert st.slots.tolist() == want[1] and st.positions.tolist() == want[2]
    assert st.cu_new.tolist() == want[3] and st.lens.tolist() == want[4]
    assert st.taken.tolist() == [want[5]] and st.status.tolist() == [want[6]]
    return want[6]


def _make_step(b, page, hi, new_hi, seed, spare=4):
    import random
    r = random.Random(seed)
    lens = [r.randint(0, hi) for _ in range(b)]
    new = [r.randint(0, new_hi) for _ in range(b)]
    width = max(-(-(n + m) // page) for n, m in zip(lens, new)) + 1
    held = [-(-n // page) for n in lens]
    total = sum(-(-(n + m) // page) for n, m in zip(lens, new)) + spare
    free = r.sample(range(total), total)
    at, table = 0, []
    for h in held:
        table.append(free[at:at + h] + [-1] * (width - h))
        at += h
    return lens, new, free, at, table


@pytest.mark.parametrize("b,page,hi,new_hi", [(1, 64, 0, 1), (1, 16, 500, 300), (7, 128, 300, 1), (64, 64, 2000, 1),
                                             (33, 48, 90, 40), (257, 16, 40, 33), (1000, 32, 100, 3)])
def test_step_matches_whole_number_reference(b, page, hi, new_hi):
    lens, new, free, taken, table = _make_step(b, page, hi, new_hi, seed=b)
    assert _run_step(lens, new, free, taken, table, page, sum(new) + b % 5) == 0


def test_step_largest_number_of_requests():
    lens, new, free, taken, table = _make_step(8192, 16, 20, 2, seed=3)
    assert _run_step(lens, new, free, taken, table, 16, sum(new)) == 0


@pytest.mark.parametrize("spare", [0, -1, -3, -10])
def test_step_refuses_in_order_when_pages_run_out(spare):
    lens, new, free, taken, table = _make_step(20, 16, 50, 40, seed=9, spare=0)
    free = free if spare == 0 else free[:spare]
    assert _run_step(lens, new, free, taken, table, 16, sum(new)) == (0 if spare == 0 else 1)


def test_step_refuses_malformed_requests_and_serves_the_others():
    lens, new = [5, -1, 30, 7, 3, 2 ** 31 - 2, 9], [3, 4, 40, -2, 1, 5, 50]
    table = [[0, -1, -1], [-1] * 3, [1, 2, -1], [3, -1, -1], [4, -1, -1], [-1] * 3, [5, -1, -1]]
    status = _run_step(lens, new, [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10], 6, table, 16, 60)
    assert status == 4 | 2                               # the last one too: ceil(59 / 16) = 4 pages, three columns
    # 13 new tokens for 10 rows: the request that crosses the end is refused
    assert _run_step([5, 9, 2], [4, 4, 5], [0, 1, 2, 3], 3, [[0, -1], [1, -1], [2, -1]], 16, 10) == 8
    # a count of taken pages that lies outside the list serves nobody who needs a page
    assert _run_step([16, 3], [1, 1], [0, 1, 2], 5, [[0, -1], [1, -1]], 16, 2) == 1


def test_step_without_rows_and_with_zero_tokens():
    assert _run_step([16, 0], [0, 0], [0, 1], 1, [[0], [-1]], 16, 0) == 0


# --------------------------------------------------------------------------------- append ----

def _cache(pages, heads, page, dim, fill=0):
    codes = torch.full((pages, heads, page, dim // 2), fill, dtype=torch.uint8, device=DEV)
    scales = torch.full((pages, heads, page, dim // 16), fill, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    return codes, scales


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 16, 16), (3, 2, 64, 16), (130, 8, 128, 64), (17, 3, 80, 48),
                                                  (5, 1, 256, 128), (4096, 4, 64, 32)])
def test_append_writes_what_the_quantiser_gives(dtype, tokens, heads, dim, page):
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(tokens + dim)
    qkv = torch.randn(tokens, 3, heads, dim, generator=g, device=DEV) * 3
    qkv[0, 1, 0, :16] = 0                                # a block of zeros
    qkv = qkv.to(dtype)
    k, v = qkv[:, 1], qkv[:, 2]                          # strided views
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens]
    kc, vc = _cache(pages, heads, page, dim, 0x5a), _cache(pages, heads, page, dim, 0xa5)
    before = [c.view(torch.uint8).clone() for c in (*kc, *vc)]
    k2, v2 = torch.tensor(7.31 / 2688, device=DEV), torch.tensor(20.7 / 2688, device=DEV)   # K is exceeded: saturates
    if tokens > 2:
        slots[1], slots[2] = -1, pages * page            # skipped rows
    kv, vv = ops.nvfp4_kv_append(k, v, slots, kc, vc, k2, v2, return_values=True)
    for x, cache, s2, old, values in ((k, kc, k2, before[:2], kv), (v, vc, v2, before[2:], vv)):
        packed, scales, _ = ops.nvfp4_quantize(x.contiguous(), scale2=s2, saturate_scales=True)
        assert torch.equal(values, ops.nvfp4_dequantize(packed, scales, s2, dtype))
        for got, new, was in ((cache[0], packed, old[0]), (cache[1].view(torch.uint8), scales.view(torch.uint8), old[1])):
            want = was.clone()
            for t in range(tokens) if tokens < 200 else range(0, tokens, 37):
                s = int(slots[t])
                if 0 <= s < pages * page:
                    assert torch.equal(got[s // page, :, s % page], new[t]), (t, s)
            written = torch.zeros(pages * page, dtype=torch.bool, device=DEV)
            written[slots[(slots >= 0) & (slots < pages * page)]] = True
            keep = ~written.view(pages, 1, page, 1)
            assert torch.equal(got * keep, want * keep)  # nothing else was touched


def test_append_saturates_infinities_and_keeps_nan_in_its_block():
    from b200q import ops

    x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    x[0, 0, 3], x[0, 0, 20] = math.inf, math.nan
    kc, vc = _cache(1, 1, 16, 64), _cache(1, 1, 16, 64)
    s2 = torch.tensor(1.0 / 448, device=DEV)
    k, _ = ops.nvfp4_kv_append(x, x, torch.zeros(1, dtype=torch.int64, device=DEV), kc, vc, s2, s2, return_values=True)
    k = k.float().flatten()
    assert k[3] == 6 and torch.isnan(k[16:32]).all()
    assert torch.isfinite(k[:16]).all() and torch.isfinite(k[32:]).all()


def test_append_of_nothing_and_of_unaligned_views():
    from b200q import ops

    kc, vc = _cache(1, 1, 16, 64), _cache(1, 1, 16, 64)
    s2 = torch.tensor(4.0 / 2688, device=DEV)
    none = torch.empty(0, 1, 64, dtype=torch.float16, device=DEV)
    k, v = ops.nvfp4_kv_append(none, none, torch.empty(0, dtype=torch.int64, device=DEV), kc, vc, s2, s2, return_values=True)
    assert k.shape == v.shape == (0, 1, 64) and not kc[0].any()
    wide = torch.randn(4, 1, 65, device=DEV).half()
    x = wide[:, :, 1:]                                   # rows that start at odd elements
    slots = torch.arange(4, device=DEV)
    got, _ = ops.nvfp4_kv_append(x, x, slots, kc, vc, s2, s2, return_values=True)
    packed, scales, _ = ops.nvfp4_quantize(x.contiguous(), scale2=s2, saturate_scales=True)
    assert torch.equal(got, ops.nvfp4_dequantize(packed, scales, s2, torch.float16))


def test_empty_tables_and_lists():
    """A table without columns and an empty free list: every request with tokens is refused, none sees anything."""
    from b200q import ops

    table = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    st = ops.kv_step(_i32([3, 0]), _i32([1, 0]), _i32([]), _i32([0]), table, 16, 2)
    assert st.slots.tolist() == [-1, -1] and int(st.status) == 2 and st.lens.tolist() == [3, 0] and int(st.taken) == 0
    q = torch.randn(2, 4, 64, device=DEV).half()
    kc, vc, s2 = _cache(1, 1, 16, 64), _cache(1, 1, 16, 64), torch.tensor(0.1, device=DEV)
    out, lse = ops.nvfp4_kv_attention(q, kc, vc, s2, s2, table, _i32([5, 0]), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = ops.nvfp4_kv_attention(q, kc, vc, s2, s2, table, _i32([5, 0]), cu_q=_i32([1, 1, 1]), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()              # no request has a row


# ------------------------------------------------------------------------------ attention ----

def _dequantised(cache, s2):
    from b200q import ops

    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    codes, scales = cache
    pair = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)
    return (pair.unflatten(-1, (-1, 16)) * scales.float().double().unsqueeze(-1) * s2.double()).flatten(-2)


def _reference(q, k_cache, v_cache, k2, v2, table, lens, q_lens, scale):
    """(out, lse, tolerance) in 64 bits.  The tolerance counts what the kernel rounds: P to fp16 (2^-11 of each
    weight, 2^-25 absolute below fp16's normal range), scores in fp32 (D + 8 additions and products, each off by
    2^-23 of the sum of magnitudes, twice in a weight's ratio to the sum), the result to its type (below its
    smallest normal number t a type is a grid of spacing eps t, so half a step is eps / 2 * max(|result|, t))."""
    K, V = _dequantised(k_cache, k2), _dequantised(v_cache, v2)
    page, heads, dim = K.shape[2], K.shape[1], K.shape[3]
    group = q.shape[1] // heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    at = 0
    for b, (n, m) in enumerate(zip(lens, q_lens)):
        ids = table[b, : -(-n // page)].long()
        ok = (ids >= 0) & (ids < K.shape[0])
        k = K[ids.clamp(0, K.shape[0] - 1)].transpose(0, 1).flatten(1, 2)[:, :n]        # [heads, n, dim]
        v = V[ids.clamp(0, K.shape[0] - 1)].transpose(0, 1).flatten(1, 2)[:, :n]
        there = ok.repeat_interleave(page)[:n]
        for i in range(m):
            see = there & (torch.arange(n, device=DEV) <= n - m + i)
            if not bool(see.any()):
                continue
            kk, vv = k[:, see], v[:, see]
            for h in range(heads):
                for j in range(group):
                    row = q[at + i, h * group + j].double()
                    z = scale * (kk[h] @ row)
                    p = torch.softmax(z, 0)
                    o = p @ vv[h]
                    big = abs(scale) * (kk[h].abs() @ row.abs()).max()
                    rel = 2.0 ** -11 + 2 * (dim + 8) * 2.0 ** -23 * big + 2.0 ** -20
                    out[at + i, h * group + j], lse[at + i, h * group + j] = o, torch.logsumexp(z, 0)
                    tol[at + i, h * group + j] = (torch.finfo(q.dtype).eps / 2 * o.abs().clamp(min=torch.finfo(q.dtype).tiny) + rel * (p @ vv[h].abs())
                                                  + kk.shape[1] * 2.0 ** -25 * vv[h].abs().amax(0)) * 1.01
                    ltol[at + i, h * group + j] = (dim + 8) * 2.0 ** -23 * big + 2.0 ** -20 * (1 + lse[at + i, h * group + j].abs())
        at += m
    return out, lse, tol, ltol


def _attention_case(lens, q_lens, heads, group, dim, page, dtype, seed=0, garbage=True, q_scale=1.3):
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    # what no token was written to holds NaN scales and arbitrary codes
    kc, vc = (_cache(pages, heads, page, dim, 0xff if garbage else 0) for _ in range(2))
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32, device=DEV)
    at, slots = 0, []
    for b, (n, c) in enumerate(zip(lens, need)):
        table[b, :c] = ids[at:at + c]
        t = torch.arange(n, device=DEV)
        slots.append(table[b, t // page].long() * page + t % page)
        at += c
    slots = torch.cat(slots)
    k2, v2 = torch.tensor(11.3 / 2688, device=DEV), torch.tensor(4.9 / 2688, device=DEV)
    if slots.numel():
        k = torch.randn(slots.numel(), heads, dim, generator=g, device=DEV) * torch.linspace(0.2, 3, dim, device=DEV)
        v = torch.randn(slots.numel(), heads, dim, generator=g, device=DEV) + 0.3
        ops.nvfp4_kv_append(k, v, slots, kc, vc, k2, v2)
    q = (torch.randn(sum(q_lens), heads * group, dim, generator=g, device=DEV) * q_scale).to(dtype)
    cu = _i32([0, *torch.tensor(q_lens).cumsum(0).tolist()])
    return q, kc, vc, k2, v2, table, _i32(lens), cu


def _check_attention(lens, q_lens, heads, group, dim, page, dtype, scale=None, **kw):
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, cu = _attention_case(lens, q_lens, heads, group, dim, page, dtype, **kw)
    one = all(m == 1 for m in q_lens)
    out, lse = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=None if one else cu, scale=scale, return_lse=True)
    kz, vz = ((c[0], torch.where(torch.isnan(c[1].float()), 0.0, c[1].float()).to(torch.float8_e4m3fn)) for c in (kc, vc))
    ref, rlse, tol, ltol = _reference(q, kz, vz, k2, v2, table, lens, q_lens, dim ** -0.5 if scale is None else scale)
    assert float(((out.double() - ref).abs() - tol).max()) <= 0
    empty = rlse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool(empty.all()) or float(((lse.double() - rlse).abs() - ltol)[~empty].max()) <= 0
    return q, kc, vc, k2, v2, table, ln, cu, out


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 127, 300, 1000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(2, 4, 16), (1, 1, 64), (3, 8, 48), (1, 5, 128)])
def test_attention_single_tokens(dtype, dim, heads, group, page):
    _check_attention(LENS, [1] * len(LENS), heads, group, dim, page, dtype, seed=dim + group)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [9, 16, 33])
def test_attention_groups_of_more_than_eight_heads(dim, group):
    _check_attention([0, 5, 200, 77], [1, 1, 1, 1], 2, group, dim, 16, torch.bfloat16, seed=group)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_attention_several_queries_are_causal(dtype, dim, group):
    # more queries than tokens too: the first of them see nothing
    _check_attention([20, 3, 64, 0, 130, 33], [4, 5, 1, 2, 19, 33], 2, group, dim, 16, dtype, seed=group)


def test_attention_requests_without_queries():
    _check_attention([50, 40, 30], [0, 3, 0], 1, 4, 128, 16, torch.bfloat16)


def test_attention_one_long_request_is_split_over_the_gpu():
    _check_attention([40000], [1], 1, 2, 128, 64, torch.bfloat16)
    _check_attention([9000], [3], 1, 4, 64, 16, torch.float16)
    _check_attention([5000], [1], 1, 1, 256, 32, torch.float16)


def test_attention_many_short_requests():
    lens = [(7 * i) % 40 for i in range(700)]
    _check_attention(lens, [1] * 700, 1, 2, 64, 16, torch.bfloat16)


@pytest.mark.parametrize("q_scale", [1e-30, 1e4, 3e30])
def test_attention_query_magnitudes(q_scale):
    # bf16 queries far outside fp16's range; the scale brings the scores back
    _check_attention([100, 33], [1, 1], 2, 4, 128, 16, torch.bfloat16, scale=0.05 / q_scale, q_scale=q_scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_many_small_weights_beside_a_large_one(dim):
    """One token whose weight is 1 and very many of 2^-26 to 2^-24 each: together they are part of the output.  The
    values' average shows what is lost: V is 1 for the one, -400 for the others.  Enough requests (of the same pages)
    that each is handled in one piece."""
    from b200q import ops

    page, tokens, b = 64, 40000, 1000
    pages = -(-tokens // page)
    kc, vc = _cache(pages, 1, page, dim), _cache(pages, 1, page, dim)
    k, v = torch.zeros(tokens, 1, dim, device=DEV), torch.full((tokens, 1, dim), -400.0, device=DEV)
    k[0, 0, 0], v[0] = 6, 1
    k2, v2 = torch.tensor(1 / 448, device=DEV), torch.tensor(1 / 4, device=DEV)
    ops.nvfp4_kv_append(k, v, torch.arange(tokens, device=DEV), kc, vc, k2, v2)
    q = torch.zeros(b, 1, dim, dtype=torch.float16, device=DEV)
    q[:, 0, 0] = 1
    table, lens = torch.arange(pages, dtype=torch.int32, device=DEV).expand(b, pages), _i32([tokens] * b)
    z = _dequantised(kc, k2).flatten(0, 2)[:tokens, 0]
    for bits in (24.5, 25.5):
        scale = bits * math.log(2) / float(z[0])
        p = torch.softmax(z * scale, 0)
        ref = p @ _dequantised(vc, v2).flatten(0, 2)[:tokens]
        out = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, lens, scale=scale)[:, 0].double()
        # the output's half step; 2^-11 of each weight, 2^-36 of the largest where that is less; the exponent's rounding (25 * 2^-23 and the scale's 2^-24), the
        # sums in fp32 (chains of 40000 / 128 steps of a warp, each with two products of 16 tokens: below 1000 additions)
        size = p @ _dequantised(vc, v2).flatten(0, 2)[:tokens].abs()
        tol = 2.0 ** -11 * ref.abs() + size * (2.0 ** -11 + 25 * 2.0 ** -22 + 1000 * 2.0 ** -23) + tokens * 400 * 2.0 ** -36
        assert float(((out - ref).abs() - tol).max()) <= 0


def test_attention_scale_may_be_negative():
    _check_attention([70, 9], [1, 2], 1, 4, 64, 16, torch.float16, scale=-0.2)


def test_attention_absent_pages_hide_their_tokens():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([100, 64], [1, 1], 2, 4, 64, 16, torch.bfloat16)
    table[0, 2], table[0, 4] = -1, kc[0].shape[0]            # outside the cache on either side
    table[1] = -5
    out = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    kz, vz = ((c[0], torch.where(torch.isnan(c[1].float()), 0.0, c[1].float()).to(torch.float8_e4m3fn)) for c in (kc, vc))
    ref, _, tol, _ = _reference(q, kz, vz, k2, v2, table, [100, 64], [1, 1], 64 ** -0.5)
    assert float(((out.double() - ref).abs() - tol).max()) <= 0
    assert (out[1] == 0).all()


def test_attention_lengths_beyond_the_table_are_cut():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([64], [1], 1, 4, 64, 16, torch.bfloat16)
    table = table[:, :4].contiguous()
    want = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    assert torch.equal(ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln + 1000), want)
    assert (ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln - 100) == 0).all()
    assert (ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table[:, :0], ln) == 0).all()


def test_attention_nan_values_reach_only_the_queries_that_see_them():
    from b200q import ops

    lens, q_lens = [40, 21], [6, 20]
    q, kc, vc, k2, v2, table, ln, cu = _attention_case(lens, q_lens, 2, 3, 128, 16, torch.bfloat16, garbage=False)
    clean = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu)
    # token 37 of request 0 (seen by its queries 3, 4, 5), block 2 of head 1; token 5 of request 1 (queries 4 ...)
    vc[1].view(torch.uint8)[int(table[0, 2]), 1, 5, 2] = 0x7f
    vc[1].view(torch.uint8)[int(table[1, 0]), 0, 5, 7] = 0xff
    out = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu)
    want = clean.clone().float()
    want[3:6, 3:6, 32:48] = math.nan
    want[6 + 4:, 0:3, 112:128] = math.nan
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.equal(out.float()[fine], want[fine])


def test_attention_infinite_query_makes_its_own_row_nan_only():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([40, 40], [1, 1], 1, 4, 64, 16, torch.bfloat16, garbage=False)
    clean = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    q[0, 1, 7], q[1, 3, 0] = math.nan, math.inf
    out = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    assert torch.isnan(out[0, 1]).all() and torch.isnan(out[1, 3]).all()
    keep = torch.ones(2, 4, dtype=torch.bool, device=DEV)
    keep[0, 1] = keep[1, 3] = False
    assert torch.equal(out[keep], clean[keep])


def test_attention_rows_behind_the_last_request():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, cu = _attention_case([40, 21], [3, 2], 1, 4, 64, 16, torch.bfloat16)
    qp = torch.cat([q, torch.full((4, 4, 64), math.nan, dtype=q.dtype, device=DEV)])
    want = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu)
    out, lse = ops.nvfp4_kv_attention(qp, kc, vc, k2, v2, table, ln, cu_q=cu, return_lse=True)
    assert torch.equal(out[:5], want) and (out[5:] == 0).all() and (lse[5:] == -math.inf).all()
    # rows in front of the first request as well
    front, flse = ops.nvfp4_kv_attention(torch.cat([qp[5:], q]), kc, vc, k2, v2, table, ln, cu_q=cu + 4, return_lse=True)
    assert torch.equal(front[4:], want) and (front[:4] == 0).all() and (flse[:4] == -math.inf).all()
    buf = torch.full_like(qp, 7)
    assert ops.nvfp4_kv_attention(qp, kc, vc, k2, v2, table, ln, cu_q=cu, out=buf) is buf
    assert torch.equal(buf[:5], want) and (buf[5:] == 7).all()


def test_attention_strided_queries_and_shared_tables():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([40], [1], 2, 4, 128, 16, torch.float16)
    want = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    wide = torch.zeros(1, 3, 8, 128, dtype=q.dtype, device=DEV)
    wide[:, 1] = q
    assert torch.equal(ops.nvfp4_kv_attention(wide[:, 1], kc, vc, k2, v2, table, ln), want)
    odd = torch.zeros(1, 8, 129, dtype=q.dtype, device=DEV)
    odd[..., 1:] = q
    assert torch.equal(ops.nvfp4_kv_attention(odd[..., 1:], kc, vc, k2, v2, table, ln), want)
    # several requests over the same pages, by an expanded table
    many = ops.nvfp4_kv_attention(q.expand(5, -1, -1), kc, vc, k2, v2, table.expand(5, -1), ln.repeat(5))
    assert all(torch.equal(many[i], want[0]) for i in range(5))


def test_attention_offsets_beyond_32_bits():
    from b200q import ops

    page, heads, dim = 64, 8, 128
    pages = (1 << 31) // (heads * page * dim // 2) + 300          # codes of more than 2^31 bytes
    kc, vc = ((torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device=DEV),
               torch.empty(pages, heads, page, dim // 16, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)) for _ in range(2))
    small = _attention_case([200], [1], heads, 2, dim, page, torch.bfloat16)
    q, skc, svc, k2, v2, table, ln, _ = small
    far = table.clone()
    for i in range(4):
        src, dst = int(table[0, i]), pages - 1 - 60 * i
        far[0, i] = dst
        for big, sm in ((kc, skc), (vc, svc)):
            big[0][dst], big[1].view(torch.uint8)[dst] = sm[0][src], sm[1].view(torch.uint8)[src]
    assert torch.equal(ops.nvfp4_kv_attention(q, kc, vc, k2, v2, far, ln), ops.nvfp4_kv_attention(q, skc, svc, k2, v2, table, ln))
    # and the append reaches there too
    x = torch.randn(1, heads, dim, device=DEV).bfloat16()
    slot = torch.tensor([pages * page - 1], device=DEV)
    ops.nvfp4_kv_append(x, x, slot, kc, vc, k2, v2)
    packed, _, _ = ops.nvfp4_quantize(x, scale2=k2, saturate_scales=True)
    assert torch.equal(kc[0][-1, :, -1], packed[0])


def test_attention_is_deterministic():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([4000, 3, 900], [1, 1, 1], 2, 4, 128, 64, torch.bfloat16)
    first = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    for _ in range(5):
        assert torch.equal(ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln), first)


def test_attention_captured_and_replayed_with_other_lengths():
    from b200q import ops

    a = _attention_case([400, 30], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=1)
    b = _attention_case([77, 3000], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=2)
    width = b[5].shape[1]
    q, table, ln = torch.zeros_like(a[0]), torch.full((2, width), -1, dtype=torch.int32, device=DEV), _i32([0, 0])
    caches = [tuple(torch.zeros_like(x) for x in b[i]) for i in (1, 2)]

    def load(case):
        q.copy_(case[0])
        table.fill_(-1)
        table[:, : case[5].shape[1]] = case[5]
        ln.copy_(case[6])
        for dst, src in zip(caches, (case[1], case[2])):
            for d, s in zip(dst, src):
                d.view(torch.uint8)[: s.shape[0]] = s.view(torch.uint8)

    def step():
        return ops.nvfp4_kv_attention(q, caches[0], caches[1], a[3], a[4], table, ln)

    step()
    graphs = []
    for _ in range(2):                                            # two graphs of the same call
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for case in (a, b, a):
        load(case)
        want = ops.nvfp4_kv_attention(case[0], case[1], case[2], case[3], case[4], case[5], case[6])
        for gr, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert torch.equal(out, want)


def test_attention_on_two_streams_at_once():
    from b200q import ops

    cases = [_attention_case([3000, 50], [1, 1], 2, 4, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [ops.nvfp4_kv_attention(*c[:7]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.nvfp4_kv_attention(*c[:7]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_operators_on_a_device_that_is_not_current():
    from b200q import ops

    c = _attention_case([100, 3], [1, 1], 1, 4, 64, 16, torch.bfloat16)
    want = ops.nvfp4_kv_attention(*c[:7])
    other = [tuple(x.to("cuda:1") for x in t) if isinstance(t, tuple) else t.to("cuda:1") for t in c[:7]]
    assert torch.equal(ops.nvfp4_kv_attention(*other).cpu(), want.cpu())


# --------------------------------------------------------------------------------- together ----

def test_steps_of_a_growing_cache_agree_with_dense_attention():
    """Prompts of several lengths, then tokens one by one and a few at a time: step, append, attention."""
    from b200q import ops

    g = torch.Generator(device=DEV).manual_seed(5)
    b, heads, group, dim, page, pages = 3, 2, 4, 64, 16, 24
    kc, vc = _cache(pages, heads, page, dim, 0xff), _cache(pages, heads, page, dim, 0xff)
    k2, v2 = torch.tensor(4.1 / 2688, device=DEV), torch.tensor(4.3 / 2688, device=DEV)
    table = torch.full((b, 8), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pages, generator=g, device=DEV).int()
    lens, taken = _i32([0] * b), _i32([0])
    keys, values = [[] for _ in range(b)], [[] for _ in range(b)]
    for new in ([17, 1, 40], [1, 1, 1], [1, 0, 1], [3, 2, 1], [0, 16, 4]):
        t = sum(new) + 2
        x = torch.randn(t, heads * (group + 2), dim, generator=g, device=DEV).bfloat16()
        q, k, v = x.split([heads * group, heads, heads], 1)
        st = ops.kv_step(lens, _i32(new), free, taken, table, page, t)
        kv, vv = ops.nvfp4_kv_append(k, v, st.slots, kc, vc, k2, v2, return_values=True)
        out = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, st.lens, cu_q=st.cu_new)
        lens, taken = st.lens, st.taken
        assert int(st.status) == 0
        at = 0
        for r, m in enumerate(new):
            keys[r].append(kv[at:at + m].double())
            values[r].append(vv[at:at + m].double())
            K, V = torch.cat(keys[r]), torch.cat(values[r])
            n = K.shape[0]
            assert int(lens[r]) == n
            for i in range(m):
                see = n - m + i + 1
                z = torch.einsum("hgd,nhd->hgn", q[at + i].double().view(heads, group, dim), K[:see]) * dim ** -0.5
                want = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), V[:see]).reshape(heads * group, dim)
                # kv / vv are the cached values rounded to bf16: 2^-8 of each, in the scores (|z| below 8) and the sum
                assert ((out[at + i].double() - want).abs() <= 2.0 ** -8 * (1 + 2 * 8 + 2) * V[:see].abs().amax()).all()
            at += m
        assert (out[at:] == 0).all()


# ---------------------------------------------------------------------------------- refusals ----

def test_operators_refuse_what_they_do_not_cover():
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, cu = _attention_case([40, 21], [3, 2], 1, 4, 64, 16, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.nvfp4_kv_attention(q.float(), kc, vc, k2, v2, table, ln, cu_q=cu)
    for bad in (dict(cu_q=None), dict(cu_q=cu[:-1]), dict(cu_q=cu.long()), dict(cu_q=cu, out=torch.empty_like(q).half()), dict(cu_q=cu, out=q)):
        with pytest.raises(ValueError):
            ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, **bad)
    for args in ((q[:, :3, :32], kc, vc, k2, v2, table, ln), (q, (kc[0], kc[1][:, :, :8]), vc, k2, v2, table, ln),
                 (q, kc, (vc[0][:1], vc[1][:1]), k2, v2, table, ln), (q, kc, vc, k2, v2, table.long(), ln),
                 (q, kc, vc, k2, v2, table[:1], ln), (q, kc, vc, k2, v2, table, ln.long()),
                 (q, kc, vc, torch.ones(2, device=DEV), v2, table, ln), (q, kc, vc, k2, v2, table.t(), ln)):
        with pytest.raises(ValueError):
            ops.nvfp4_kv_attention(*args, cu_q=cu)
    odd = _cache(4, 1, 8, 64)
    with pytest.raises(ValueError):
        ops.nvfp4_kv_attention(q, odd, odd, k2, v2, table, ln, cu_q=cu)       # pages of 8
    x = torch.randn(2, 1, 64, device=DEV).half()
    slots = torch.arange(2, device=DEV)
    for args in ((x, x[:1], slots), (x, x.float(), slots), (x, x, slots.int()), (x, x, slots[:1]), (x[..., :32], x[..., :32], slots)):
        with pytest.raises(ValueError):
            ops.nvfp4_kv_append(*args, kc, vc, k2, v2)
    with pytest.raises(TypeError):
        ops.nvfp4_kv_append(x.double(), x.double(), slots, kc, vc, k2, v2)
    one = _i32([1])
    for args in ((one, _i32([1, 1]), one, one, table[:1]), (one, one, one, _i32([0, 0]), table[:1]), (one, one, one, one, table),
                 (one.long(), one, one, one, table[:1]), (ln, ln, one, one, table[:1].expand(2, -1))):
        with pytest.raises(ValueError):
            ops.kv_step(*args, 16, 1)
    for page, tokens in ((0, 1), (16, -1), (2 ** 32 + 16, 1), (16, 2 ** 32 + 1)):
        with pytest.raises(ValueError):
            ops.kv_step(one, one, one, one, table[:1], page, tokens)
    many = torch.zeros(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        ops.kv_step(many, many, one, one, torch.zeros(8193, 1, dtype=torch.int32, device=DEV), 16, 1)


# ------------------------------------------------------------------- segments of a single tile ----

@pytest.mark.parametrize("dim,page,several", [(64, 16, False), (128, 64, False), (128, 48, True), (256, 32, True)])
def test_attention_shares_that_begin_with_requests_of_one_tile(dim, page, several):
    """Requests of at most one tile (128 tokens): a block handles several segments, and its two fetches ahead already
    lie in different ones.  A segment of one tile is never split, so each request alone gives the same bits."""
    from b200q import ops

    lens = [1 + (37 * i) % 128 for i in range(600)]
    q_lens = [1 + i % 3 if several else 1 for i in range(600)]
    q, kc, vc, k2, v2, table, ln, cu = _attention_case(lens, q_lens, 3, 2, dim, page, torch.bfloat16, seed=page)
    out, lse = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu if several else None, return_lse=True)
    for _ in range(3):
        assert torch.equal(ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu if several else None), out)
    first = cu.tolist()
    for b in range(0, 600, 7):
        rows = slice(first[b], first[b + 1])
        alone, alse = ops.nvfp4_kv_attention(q[rows], kc, vc, k2, v2, table[b:b + 1], ln[b:b + 1],
                                             cu_q=_i32([0, q_lens[b]]) if several else None, return_lse=True)
        assert torch.equal(alone, out[rows]) and torch.equal(alse, lse[rows])


def test_step_numbers_of_requests_around_the_default_shared_memory():
    """The scans of 4090 to 4095 requests fit the 48 KB a kernel has by default only without its own 72 bytes.  In a
    process of its own, the smaller numbers first: a larger call raises the limit for the rest of the process."""
    import subprocess
    import sys

    code = """
import sys
sys.path[:0] = %r
import torch
from b200q import ops
for b in (4089, 4090, 4092, 4095, 4096, 4097):
    lens = torch.arange(b, dtype=torch.int32, device="cuda") %% 5
    one = torch.ones(b, dtype=torch.int32, device="cuda")
    table = torch.full((b, 1), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(b, dtype=torch.int32, device="cuda").flip(0)
    held = lens > 0
    table[held, 0] = free[:int(held.sum())]
    st = ops.kv_step(lens, one, free, held.sum().int().view(1), table, 16, b)
    assert int(st.status) == 0 and int(st.taken) == b and torch.equal(st.lens, lens + 1), b
    assert torch.equal(st.slots, table[:, 0].long() * 16 + lens) and sorted(table[:, 0].tolist()) == list(range(b)), b
""" % sys.path
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_log_sums_of_rows_without_a_request_when_out_is_given():
    """``out`` keeps its rows in front of the first request and behind the last one; the log-sums are a fresh buffer and
    say -inf there, whatever its memory held before."""
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, cu = _attention_case([40, 21], [3, 2], 1, 4, 64, 16, torch.bfloat16)
    want, wlse = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln, cu_q=cu, return_lse=True)
    qp = torch.cat([q.new_full((3, 4, 64), math.nan), q, q.new_full((4, 4, 64), math.nan)])
    for _ in range(3):
        torch.full((12, 4), 3.0, dtype=torch.float32, device=DEV)              # freed memory that is no -inf
        buf = torch.full_like(qp, 7)
        out, lse = ops.nvfp4_kv_attention(qp, kc, vc, k2, v2, table, ln, cu_q=cu + 3, out=buf, return_lse=True)
        assert out is buf and torch.equal(buf[3:8], want) and (buf[:3] == 7).all() and (buf[8:] == 7).all()
        assert torch.equal(lse[3:8], wlse) and (lse[:3] == -math.inf).all() and (lse[8:] == -math.inf).all()


def test_step_says_what_a_request_sees():
    """``seen``: the length after the step, 0 for a request that was refused, whatever the reason."""
    from b200q import ops

    lens, new = [5, -1, 30, 7, 3, 2 ** 31 - 2, 9, 4], [3, 4, 40, -2, 1, 5, 50, 0]
    table = _i32([[0, -1, -1], [-1] * 3, [1, 2, -1], [3, -1, -1], [4, -1, -1], [-1] * 3, [5, -1, -1], [6, -1, -1]])
    st = ops.kv_step(_i32(lens), _i32(new), _i32(list(range(7))), _i32([7]), table, 16, 60)
    # 103 rows are asked for and 60 there: requests behind the end are refused, the last one, without any row, among them
    assert len(st) == 6 and st.seen.tolist() == [8, 0, 0, 0, 4, 0, 0, 0]
    st = ops.kv_step(_i32([16, 3, 16]), _i32([1, 1, 0]), _i32([0, 1, 2]), _i32([3]), _i32([[0, -1], [1, -1], [2, -1]]), 16, 2)
    assert int(st.status) == 1 and st.seen.tolist() == [0, 4, 16]
    st = ops.kv_step(_i32([5, 9, 2]), _i32([4, 4, 5]), _i32([0, 1, 2, 3]), _i32([3]), _i32([[0, -1], [1, -1], [2, -1]]), 16, 10)
    assert int(st.status) == 8 and st.seen.tolist() == [9, 13, 0]


def test_out_and_queries_of_one_storage():
    """Two ranges of one arena are fine; ranges that overlap are refused, by a single element too."""
    from b200q import ops

    q, kc, vc, k2, v2, table, ln, _ = _attention_case([40, 21], [1, 1], 1, 4, 64, 16, torch.bfloat16)
    want = ops.nvfp4_kv_attention(q, kc, vc, k2, v2, table, ln)
    n = q.numel()
    arena = torch.zeros(3 * n, dtype=q.dtype, device=DEV)
    arena[n:2 * n] = q.flatten()
    mine = arena[n:2 * n].view_as(q)
    for at in (0, 2 * n):
        out = arena[at:at + n].view_as(q)
        assert ops.nvfp4_kv_attention(mine, kc, vc, k2, v2, table, ln, out=out) is out and torch.equal(out, want)
    assert torch.equal(mine, q)
    for at in (8, n - 8, n, n + 8, 2 * n - 8):
        with pytest.raises(ValueError, match="share"):
            ops.nvfp4_kv_attention(mine, kc, vc, k2, v2, table, ln, out=arena[at:at + n].view_as(q))
    # strided queries reach as far as their last element
    wide = torch.zeros(2, 3, 4, 64, dtype=q.dtype, device=DEV)
    wide[:, 0] = q
    flat = wide.view(-1)
    with pytest.raises(ValueError, match="share"):
        ops.nvfp4_kv_attention(wide[:, 0], kc, vc, k2, v2, table, ln, out=flat[n // 2:n // 2 + n].view_as(q))
    out = flat[2 * n:3 * n].view_as(q)                       # behind the last query
    assert torch.equal(ops.nvfp4_kv_attention(wide[:, 0], kc, vc, k2, v2, table, ln, out=out), want)
