"""What one decoding step of a 4-bit model reads and writes, as cases that can be measured:

* ``kv_step``    page tables and slots of a paged KV cache, built on the GPU from request lengths
* ``kv_append``  new keys and values quantised to NVFP4 and written into the cache's pages
* ``kv_attention``  attention of the new tokens over the NVFP4 cache, grouped heads, ragged lengths
* ``w4_linear``  products of a few rows with 4-bit weights (INT4 with group scales, NVFP4)

Each has a plain form in elementary torch operations (``own`` false), the library's entry points
(``own`` true) and its definition in 64 bits (``exact``).
"""
import math
import random

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------- cases ----

def listed():
    return [
        # the start of a decoding step of a busy server: every request gets one token
        dict(name="step_decode_64", op="kv_step", requests=64, lo=1, hi=8192, new_lo=1, new_hi=1, page=64, pad=0, lens_seed=1),
        # admission of many prompts at once, some of them continued, with rows of padding behind the last one
        dict(name="step_prompts_512", op="kv_step", requests=512, lo=0, hi=300, new_lo=1, new_hi=511, page=16, pad=100, lens_seed=2),
        # the decoding step's own keys and values
        dict(name="append_decode_64", op="kv_append", tokens=64, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # a long prompt, read out of a fused qkv projection's output
        dict(name="append_prompt_32k", op="kv_append", tokens=32768, kv_heads=8, dim=128, page=16, dtype="fp16"),
        # a small server: few short conversations, heads of 64
        dict(name="attn_small_d64", op="kv_attention", requests=4, lo=1, hi=509, q_lo=1, q_hi=1, kv_heads=2, group=7, dim=64, page=16, dtype="fp16", lse=False, lens_seed=3),
        # the ordinary decoding batch: ragged contexts, grouped heads
        dict(name="attn_decode_64", op="kv_attention", requests=64, lo=17, hi=8192, q_lo=1, q_hi=1, kv_heads=8, group=4, dim=128, page=64, dtype="bf16", lse=False, lens_seed=4),
        # few very long contexts
        dict(name="attn_long_8x64k", op="kv_attention", requests=8, lo=65536, hi=65536, q_lo=1, q_hi=1, kv_heads=8, group=8, dim=128, page=64, dtype="bf16", lse=False, lens_seed=5),
        # draft tokens to verify: several queries a request, heads of 256, the log-sum for a merge
        dict(name="attn_verify_d256", op="kv_attention", requests=16, lo=9, hi=4099, q_lo=1, q_hi=8, kv_heads=4, group=2, dim=256, page=32, dtype="bf16", lse=True, lens_seed=6),
        # one token through an attention projection with INT4 weights
        dict(name="int4_1x4096x4096", op="w4_linear", fmt="int4", rows=1, n=4096, k=4096, block=128, bias=False, dtype="bf16"),
        # a decoding batch through a large down projection
        dict(name="int4_16x8192x28672", op="w4_linear", fmt="int4", rows=16, n=8192, k=28672, block=128, bias=False, dtype="bf16"),
        # one token through a large up projection with NVFP4 weights
        dict(name="nvfp4_1x28672x8192", op="w4_linear", fmt="nvfp4", rows=1, n=28672, k=8192, block=16, bias=False, dtype="bf16"),
        # odd sizes, with a bias
        dict(name="nvfp4_5x4099x2080", op="w4_linear", fmt="nvfp4", rows=5, n=4099, k=2080, block=16, bias=True, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv_step", "kv_append", "kv_attention", "kv_attention", "w4_linear", "w4_linear"])
    seed = rng.randrange(1 << 30)
    dtype = rng.choice(["bf16", "fp16"])
    if op == "kv_step":
        b = _log(rng, 1, 512)
        one = rng.random() < 0.5
        return dict(op=op, requests=b, lo=0, hi=_log(rng, 2, 8192), new_lo=1 if one else 0,
                    new_hi=1 if one else max(1, _log(rng, 2, 131072) // b), page=rng.choice([16, 32, 64, 128]),
                    pad=rng.choice([0, 0, 7, 64]), lens_seed=seed)
    if op == "kv_append":
        return dict(op=op, tokens=_log(rng, 1, 32768), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64, 128]), dtype=dtype, slots_seed=seed)
    if op == "kv_attention":
        heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        b = _log(rng, 1, 64)
        hi = _log(rng, 2, max(2, min(65536, 8 * 65536 * 8 * 128 // (b * heads * dim) // 2)))
        return dict(op=op, requests=b, lo=rng.choice([0, 1, max(1, hi // 2)]), hi=hi, q_lo=1,
                    q_hi=rng.choice([1, 1, 1, 4]), kv_heads=heads, group=rng.choice([1, 2, 4, 5, 8, 16]), dim=dim,
                    page=rng.choice([16, 32, 64, 128]), dtype=dtype, lse=rng.random() < 0.3, lens_seed=seed)
    fmt = rng.choice(["int4", "nvfp4"])
    block = rng.choice([32, 64, 128, 128]) if fmt == "int4" else 16
    unit = max(32, block)
    return dict(op=op, fmt=fmt, rows=_log(rng, 1, 16), n=_log(rng, 64, 8192), k=unit * _log(rng, 2, 28672 // unit),
                block=block, bias=rng.random() < 0.3, dtype=dtype)


def _lens(case):
    """(tokens a request holds, tokens it adds or asks with) of a case: the case's own, whatever the seed of its inputs."""
    r = random.Random(case["lens_seed"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["requests"])]
    lo, hi = (case["new_lo"], case["new_hi"]) if case["op"] == "kv_step" else (case["q_lo"], case["q_hi"])
    new = [r.randint(lo, hi) for _ in range(case["requests"])]
    return lens, new


def _up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------- NVFP4 values ----

def _quantize(x, s2):
    """x [..., D] -> (codes uint8 [..., D/2], low nibble first; block scales float8_e4m3fn [..., D/16]) in fp32:
    scale = e4m3(amax / (6 s2)) at most 448 (1 for a block of zeros), code = nearest E2M1 of x / (scale s2), ties to even."""
    xb = x.float().reshape(*x.shape[:-1], -1, 16)
    amax = xb.abs().amax(-1)
    t = amax / (6.0 * s2)
    t = torch.where(t == 0, torch.ones_like(t), t).clamp(max=448.0)
    s8 = t.to(torch.float8_e4m3fn)
    q = xb / (s8.float() * s2).unsqueeze(-1)
    a = q.abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (mag | ((q < 0).to(torch.uint8) << 3)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), s8


def _values(codes, s8, s2):
    """fp32 values of codes and block scales."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    pair = torch.stack((lut[(codes & 15).int()], lut[(codes >> 4).int()]), -1)
    v = pair.reshape(*codes.shape[:-1], -1, 16)
    return (v * (s8.float() * s2).unsqueeze(-1)).reshape(*codes.shape[:-1], -1)


def _values64(codes, s8, s2):
    """The same in 64 bits, from the formats' bit fields."""
    def e2m1(c):
        e, m = ((c >> 1) & 3).double(), (c & 1).double()
        v = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.exp2(e - 1))
        return torch.where((c & 8) != 0, -v, v)

    b = s8.view(torch.uint8)
    e, m = ((b >> 3) & 15).double(), (b & 7).double()
    s = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e - 7)) * torch.where(b >= 128, -1.0, 1.0)
    pair = torch.empty(*codes.shape, 2, dtype=torch.float64, device=codes.device)
    pair[..., 0], pair[..., 1] = e2m1(codes & 15), e2m1(codes >> 4)
    return (pair.reshape(*s.shape, 16) * s.unsqueeze(-1) * s2.double()).reshape(*codes.shape[:-1], -1)



# ----------------------------------------------------------------------------------- prepare ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"kv_step": _prepare_step, "kv_append": _prepare_append, "kv_attention": _prepare_attention,
            "w4_linear": _prepare_linear}[case["op"]](case, g)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_step(case, g):
    lens, new = _lens(case)
    page, b = case["page"], case["requests"]
    have = [_up(n, page) for n in lens]
    total = sum(_up(n + m, page) for n, m in zip(lens, new)) + 8
    width = max(_up(n + m, page) for n, m in zip(lens, new)) + 1
    pages = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < _int32(have)[:, None]
    table[held] = pages[: sum(have)]
    return dict(case=case, lens=_int32(lens), new=_int32(new), free=pages, taken=_int32([sum(have)]), table=table,
                tokens=sum(new) + case["pad"])


def _prepare_append(case, g):
    t, h, d, page, dtype = case["tokens"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    # keys and values as views of a fused projection's output [t, 3 h d]; some key channels carry outliers
    qkv = torch.randn(t, 3 * h * d, generator=g, device="cuda")
    qkv[:, h * d:h * d + 4] *= 8
    qkv = qkv.to(dtype)
    k, v = (qkv[:, i * h * d:(i + 1) * h * d].unflatten(1, (h, d)) for i in (1, 2))
    pages = _up(t, page) + 3                                   # the last one is no request's
    slots = torch.randperm((pages - 1) * page, generator=g, device="cuda")[:t]
    if t > 1:
        slots[t // 2] = -1                                     # a row of padding

    def cache():
        return (torch.zeros(pages, h, page, d // 2, dtype=torch.uint8, device="cuda"),
                torch.zeros(pages, h, page, d // 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn))

    # amax / (6 * 448) with the amax of a percentile calibration: exceeded now and then, and no value of the data itself
    # (the ratio of two 16-bit values puts block scales on rounding borders, where 32 and 64 bits part)
    return dict(case=case, k=k, v=v, slots=slots, k_cache=cache(), v_cache=cache(),
                k_scale2=torch.tensor(30.51731 / 2688, device="cuda"), v_scale2=torch.tensor(4.32917 / 2688, device="cuda"))


def _prepare_attention(case, g):
    lens, new = _lens(case)
    h, d, page, dtype = case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    new = [min(n, m) if n else m for n, m in zip(lens, new)]   # a request's queries are its last tokens
    need = [_up(n, page) for n in lens]
    pages, width = sum(need) + 3, max(max(need), 1)
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda")[None, :] < _int32(need)[:, None]] = ids[: sum(need)]
    ks2, vs2 = torch.tensor(12.0 / 2688, device="cuda"), torch.tensor(4.7 / 2688, device="cuda")
    channel = 1 + 2 * torch.rand(h, 1, d, generator=g, device="cuda") ** 4

    def cache(s2, scale):
        codes = torch.empty(pages, h, page, d // 2, dtype=torch.uint8, device="cuda")
        s8 = torch.empty(pages, h, page, d // 16, dtype=torch.float8_e4m3fn, device="cuda")
        step = max(1, (1 << 25) // (h * page * d))
        for i in range(0, pages, step):
            n = min(step, pages - i)
            codes[i:i + n], s8[i:i + n] = _quantize(torch.randn(n, h, page, d, generator=g, device="cuda") * scale, s2)
        return codes, s8

    k_cache, v_cache = cache(ks2, channel), cache(vs2, 1.0)
    q = (torch.randn(sum(new), h * case["group"], d, generator=g, device="cuda") * 1.3).to(dtype)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(_int32(new), 0)
    return dict(case=case, q=q, k_cache=k_cache, v_cache=v_cache, k_scale2=ks2, v_scale2=vs2, table=table, lens=_int32(lens),
                cu_q=None if case["q_hi"] == 1 else cu, host=(lens, new))


def _prepare_linear(case, g):
    m, n, k, block, dtype = case["rows"], case["n"], case["k"], case["block"], DTYPES[case["dtype"]]
    x = torch.randn(m, k, generator=g, device="cuda")
    x[:, :: 97] *= 20                                          # activations have outlier channels
    x = x.to(dtype)
    bias = (torch.randn(n, generator=g, device="cuda")).to(dtype) if case["bias"] else None
    if case["fmt"] == "nvfp4":
        codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(n, k // 16, dtype=torch.float8_e4m3fn, device="cuda")
        s2 = torch.tensor(0.11 / 2688, device="cuda")
    else:
        codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(n * (k // block), 1, dtype=dtype, device="cuda")
        s2 = None
    step = max(1, (1 << 25) // k)
    for i in range(0, n, step):
        w = torch.randn(min(step, n - i), k, generator=g, device="cuda") * 0.02
        if s2 is not None:
            codes[i:i + step], scales[i:i + step] = _quantize(w, s2)
            continue
        wb = w.to(dtype).float().reshape(-1, block)
        s = (7.0 / wb.abs().amax(-1, keepdim=True)).to(dtype)
        c = (torch.round(wb * s.float()).clamp(-8, 7) + 8).to(torch.uint8).reshape(w.shape)
        codes[i:i + step] = (c[:, 0::2] << 4) | c[:, 1::2]
        scales[i * (k // block): i * (k // block) + s.shape[0]] = s
    return dict(case=case, x=x, codes=codes, scales=scales, scale2=s2, bias=bias)


# --------------------------------------------------------------------------------------- run ----

def run(state):
    return {"kv_step": _run_step, "kv_append": _run_append, "kv_attention": _run_attention,
            "w4_linear": _run_linear}[state["case"]["op"]](state)


def _run_step(s):
    page, tokens = s["case"]["page"], s["tokens"]
    if own:
        ops = _ops()
        step = ops.kv_step(s["lens"], s["new"], s["free"], s["taken"], s["table"], page, tokens)
        return dict(table=s["table"], slots=step.slots, positions=step.positions, cu=step.cu_new, lens=step.lens,
                    taken=step.taken, status=step.status)
    lens, new, table = s["lens"].long(), s["new"].long(), s["table"]
    b, width = table.shape
    have, want = (lens + page - 1) // page, (lens + new + page - 1) // page
    need = want - have
    base = s["taken"] + torch.cumsum(need, 0) - need
    col = torch.arange(width, device="cuda")
    fresh = (col >= have[:, None]) & (col < want[:, None])
    source = (base[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][source], table))
    cu = torch.zeros(b + 1, dtype=torch.int32, device="cuda")
    cu[1:] = torch.cumsum(new, 0)
    token = torch.arange(tokens, device="cuda", dtype=torch.int32)
    row = torch.searchsorted(cu[1:], token, right=True).clamp(max=b - 1)
    real = token < cu[-1]
    pos = torch.where(real, lens[row] + token - cu[row], 0)
    slots = torch.where(real, table[row, (pos // page).clamp(max=width - 1)].long() * page + pos % page, -1)
    return dict(table=table, slots=slots, positions=pos.int(), cu=cu, lens=(lens + new).int(),
                taken=(s["taken"] + need.sum()).int(), status=torch.zeros(1, dtype=torch.int32, device="cuda"))


def _run_append(s):
    if own:
        ops = _ops()
        k, v = ops.nvfp4_kv_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale2"], s["v_scale2"],
                                   return_values=True)
        return dict(k=k, v=v)
    page, slots = s["case"]["page"], s["slots"]
    out = {}
    for name in ("k", "v"):
        codes, s8 = _quantize(s[name], s[name + "_scale2"])
        to = torch.where(slots >= 0, slots, s["k_cache"][0].shape[0] * page - 1)   # rows of padding: to the page that is no request's
        p, i = to // page, to % page
        s[name + "_cache"][0][p, :, i] = codes
        s[name + "_cache"][1].view(torch.uint8)[p, :, i] = s8.view(torch.uint8)
        out[name] = _values(codes, s8, s[name + "_scale2"]).to(s[name].dtype)
    return out


def _gather(pages, table):
    """[P, H, page, X] by a table [B, W] -> [B, H, W page, X]; absent pages read page 0."""
    x = pages[table.clamp(min=0)]
    return x.transpose(1, 2).flatten(2, 3)


def _run_attention(s):
    c = s["case"]
    if own:
        ops = _ops()
        r = ops.nvfp4_kv_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale2"], s["v_scale2"], s["table"], s["lens"],
                                   cu_q=s["cu_q"], return_lse=c["lse"])
        return dict(out=r[0], lse=r[1]) if c["lse"] else dict(out=r)
    q, table, lens = s["q"], s["table"], s["lens"].long()
    b, h, group, d = c["requests"], c["kv_heads"], c["group"], c["dim"]
    k = _values(_gather(s["k_cache"][0], table), _gather(s["k_cache"][1].view(torch.uint8), table).view(torch.float8_e4m3fn), s["k_scale2"])
    v = _values(_gather(s["v_cache"][0], table), _gather(s["v_cache"][1].view(torch.uint8), table).view(torch.float8_e4m3fn), s["v_scale2"])
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(b + 1, device="cuda")
    qn = cu[1:] - cu[:-1]
    most = c["q_hi"]
    i = torch.arange(most, device="cuda")
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)         # [b, most]
    qb = q[at].float().reshape(b, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, most * group, d)
    scores = (qb @ k.transpose(-1, -2)) * d ** -0.5            # [b, h, most group, L]
    last = lens[:, None] - qn[:, None] + i                     # the last position a query sees
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    seen &= torch.arange(k.shape[2], device="cuda") < lens[:, None, None]
    seen = seen.repeat_interleave(group, 1)[:, None]           # [b, 1, most group, L]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    lse = torch.log(total) + top
    token = torch.arange(q.shape[0], device="cuda")
    row = torch.searchsorted(cu[1:], token, right=True)
    rows = row * most + token - cu[row]
    out = out.reshape(b, h, most, group, d).permute(0, 2, 1, 3, 4).reshape(b * most, h * group, d)[rows].to(q.dtype)
    lse = lse.reshape(b, h, most, group).permute(0, 2, 1, 3).reshape(b * most, h * group)[rows]
    return dict(out=out, lse=lse) if c["lse"] else dict(out=out)


def _run_linear(s):
    c = s["case"]
    if own:
        ops = _ops()
        if c["fmt"] == "int4":
            return ops.int4_linear(s["x"], s["codes"], s["scales"], c["block"], s["bias"])
        return ops.nvfp4_linear(s["x"], s["codes"], s["scales"], s["scale2"], s["bias"])
    if c["fmt"] == "int4":
        codes = torch.stack((s["codes"] >> 4, s["codes"] & 15), -1)
        w = (codes.float() - 8).reshape(-1, c["block"]) / s["scales"].float()
        w = w.reshape(c["n"], c["k"])
    else:
        w = _values(s["codes"], s["scales"], s["scale2"])
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _ops():
    import sys
    if "tensorrt-model-optimizer_b200" not in sys.path:
        sys.path.insert(0, "tensorrt-model-optimizer_b200")
    from b200q import ops
    return ops


# -------------------------------------------------------------------------------------- work ----

def work(case):
    op = case["op"]
    if op == "kv_step":
        lens, new = _lens(case)
        fresh = sum(_up(n + m, case["page"]) - _up(n, case["page"]) for n, m in zip(lens, new))
        return {"bytes": 8 * fresh + 4 * 4 * case["requests"] + 12 * (sum(new) + case["pad"]), "flops": 0}
    if op == "kv_append":
        n = case["tokens"] * case["kv_heads"] * case["dim"] * 2
        return {"bytes": n * (2 + 0.5 + 1 / 16 + 2) + 8 * case["tokens"], "flops": 0}
    if op == "kv_attention":
        lens, new = _lens(case)
        new = [min(n, m) if n else m for n, m in zip(lens, new)]
        heads = case["kv_heads"] * case["group"]
        seen = sum(sum(max(0, n - m + i + 1) for i in range(m)) for n, m in zip(lens, new))
        return {"bytes": sum(lens) * case["kv_heads"] * case["dim"] * 2 * (0.5 + 1 / 16) + sum(new) * heads * case["dim"] * 4,
                "flops": 4 * seen * heads * case["dim"]}
    m, n, k = case["rows"], case["n"], case["k"]
    per = 0.5 + (1 / 16 if case["fmt"] == "nvfp4" else 2 / case["block"])
    return {"bytes": n * k * per + 2 * m * (n + k), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------- exact ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"kv_step": lambda s: None, "kv_append": _exact_append, "kv_attention": _exact_attention,
            "w4_linear": _exact_linear}[case["op"]](s)


def _exact_append(s):
    out = {}
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    for name in ("k", "v"):
        s2 = s[name + "_scale2"].double()
        x = s[name].double().unflatten(-1, (-1, 16))
        t = x.abs().amax(-1, keepdim=True) / (6 * s2)
        step = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
        scale = torch.where(t == 0, 1.0, (torch.round(t / step) * step).clamp(max=448.0))
        q = x / (scale * s2)
        a = q.abs().clamp(max=6.0)
        exp = torch.floor(torch.log2(a.clamp(min=1.0)))
        unit = torch.exp2(exp - 1)                             # E2M1: one bit behind the leading one
        a = (torch.round(a / unit) * unit).clamp(max=6.0)
        assert bool(torch.isin(a[:1].flatten(), grid).all())
        out[name] = (torch.copysign(a, q) * scale * s2).flatten(-2)
    return out


def _exact_attention(s):
    c, (lens, new) = s["case"], s["host"]
    h, group, d, page = c["kv_heads"], c["group"], c["dim"], c["page"]
    outs, lses, at = [], [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        q = s["q"][at:at + m].double().reshape(m, h, group, d)
        at += m
        out = torch.zeros(m, h, group, d, dtype=torch.float64, device="cuda")
        lse = torch.full((m, h, group), -math.inf, dtype=torch.float64, device="cuda")
        ids = s["table"][b, :_up(n, page)].long()
        for j in range(h if n else 0):
            k, v = (_values64(cc[0][ids, j].flatten(0, 1)[:n], cc[1].view(torch.uint8)[ids, j].flatten(0, 1)[:n].view(torch.float8_e4m3fn), s2)
                    for cc, s2 in ((s["k_cache"], s["k_scale2"]), (s["v_cache"], s["v_scale2"])))
            for i in range(m):
                seen = n - m + i + 1
                if seen <= 0:
                    continue
                z = (q[i, j] @ k[:seen].t()) / math.sqrt(d)
                lse[i, j] = torch.logsumexp(z, -1)
                out[i, j] = torch.softmax(z, -1) @ v[:seen]
        outs.append(out.reshape(m, h * group, d))
        lses.append(lse.reshape(m, h * group))
    r = dict(out=torch.cat(outs))
    return dict(r, lse=torch.cat(lses)) if c["lse"] else r


def _exact_linear(s):
    c, x = s["case"], s["x"].double()
    y = torch.empty(c["rows"], c["n"], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // c["k"])
    for i in range(0, c["n"], step):
        codes = s["codes"][i:i + step]
        if c["fmt"] == "int4":
            w = torch.empty(codes.shape[0], c["k"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (codes >> 4).double() - 8, (codes & 15).double() - 8
            per = c["k"] // c["block"]
            w = w.unflatten(1, (per, -1)) / s["scales"].reshape(c["n"], per)[i:i + step].double().unsqueeze(-1)
            w = w.flatten(1)
        else:
            w = _values64(codes, s["scales"][i:i + step], s["scale2"])
        y[:, i:i + step] = x @ w.t()
    return y if s["bias"] is None else y + s["bias"].double()
