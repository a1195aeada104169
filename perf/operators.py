"""The operators of an 8-bit decoder layer with block scales, in their plain form and through the calls a user makes.

  linear   `ops.fp8_linear_block`: e4m3 activations with a scale for each token and 128 inputs, e4m3 weights with a scale
           for each block of 128 x 128
  norm     `glue.rmsnorm_fp8_block`: residual addition, RMS norm and the e4m3 activations that such a layer reads
  plan     `paged_cache.plan_step`: pages and slots of a step's new tokens, from the requests' lengths
  append   `paged_cache.kv8_append`: rotated keys, and values, into a paged cache of 8 bits, a scale for each page and head
  attend   `paged_cache.attn_decode_kv8`: attention of the newest tokens over that cache

Sizes are those of the Qwen2-0.5B / 1.5B / 7B layers of the benchmark and the tests, plus odd ones in between.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
F8 = torch.float8_e4m3fn
FLOOR = 1e-12                     # least maximum of a quantization group


def listed():
    return [
        # the smallest call: one token through the gate projection of the smallest model
        {"name": "linear_m1", "kind": "linear", "M": 1, "N": 4864, "K": 896, "bias": True, "dtype": "fp16"},
        # decode of a batch: the widest layer of the largest model
        {"name": "linear_m64", "kind": "linear", "M": 64, "N": 37888, "K": 3584, "bias": False, "dtype": "bf16"},
        # prompts: the layer with the longest sums
        {"name": "linear_m4096", "kind": "linear", "M": 4096, "N": 3584, "K": 18944, "bias": False, "dtype": "bf16"},
        # one norm of a decode step
        {"name": "norm_m64", "kind": "norm", "M": 64, "H": 3584, "residual": True, "dtype": "bf16"},
        # one norm over prompts, an odd number of tokens
        {"name": "norm_m8191", "kind": "norm", "M": 8191, "H": 3584, "residual": True, "dtype": "fp16"},
        # a decode step of a batch: a page is needed by one request in sixteen
        {"name": "plan_b64", "kind": "plan", "B": 64, "page": 16, "context": 8192, "new": 1, "tokens": 64},
        # prompts arrive beside running requests
        {"name": "plan_prompts", "kind": "plan", "B": 333, "page": 64, "context": 4096, "new": 700, "tokens": 131072},
        # one layer's new tokens of a decode step
        {"name": "append_b64", "kind": "append", "B": 64, "new": 1, "page": 64, "Hkv": 4, "d": 128, "cache": "e4m3",
         "rotary": True, "dtype": "bf16"},
        # one layer's keys and values of prompts, whose pages end anywhere
        {"name": "append_prompts", "kind": "append", "B": 13, "new": 2500, "page": 32, "Hkv": 4, "d": 128, "cache": "int8",
         "rotary": True, "dtype": "fp16"},
        # decode of a few short sequences, the smallest model's heads
        {"name": "attend_b5", "kind": "attend", "B": 5, "Sq": 1, "Hq": 14, "Hkv": 2, "d": 64, "longest": 300, "page": 16,
         "cache": "int8", "rotary": True, "softcap": 0.0, "dtype": "fp16"},
        # decode of a ragged batch
        {"name": "attend_b64", "kind": "attend", "B": 64, "Sq": 1, "Hq": 28, "Hkv": 4, "d": 128, "longest": 6000, "page": 64,
         "cache": "e4m3", "rotary": True, "softcap": 0.0, "dtype": "bf16"},
        # one long sequence, two tokens at a time (a draft beside the newest token)
        {"name": "attend_long", "kind": "attend", "B": 1, "Sq": 2, "Hq": 28, "Hkv": 4, "d": 128, "longest": 131072, "page": 128,
         "cache": "e4m3", "rotary": True, "softcap": 0.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "plan", "append", "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "linear":
        N, K = _log(rng, 40, 40000), 16 * _log(rng, 4, 1200)
        M = _log(rng, 1, max(1, min(4096, 278_000_000_000 // (N * K))))
        return {"kind": kind, "M": M, "N": N, "K": K, "bias": rng.random() < 0.5, "dtype": dtype}
    if kind == "norm":
        H = 8 * _log(rng, 8, 1024)
        return {"kind": kind, "M": _log(rng, 1, min(8192, 29_000_000 // H)), "H": H, "residual": rng.random() < 0.7, "dtype": dtype}
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        B, new = _log(rng, 1, 1000), rng.choice([1, _log(rng, 2, 4000)])
        new = min(new, max(1, 200_000 // B))
        return {"kind": kind, "B": B, "page": page, "context": _log(rng, 1, 8192), "new": new,
                "tokens": rng.choice([B * new, B * new + 100, max(1, B * new // 2)])}
    cache = rng.choice(["e4m3", "int8"])
    if kind == "append":
        Hkv, d = rng.choice([(4, 128), (2, 128), (2, 64), (3, 64), (8, 128)])
        B, new = _log(rng, 1, 256), rng.choice([1, _log(rng, 2, 4000)])
        new = min(new, max(1, 32_000 * 512 // (B * Hkv * d)))
        return {"kind": kind, "B": B, "new": new, "page": page, "Hkv": Hkv, "d": d, "cache": cache, "rotary": rng.random() < 0.7,
                "dtype": dtype}
    Hq, Hkv, d = rng.choice([(28, 4, 128), (12, 2, 128), (14, 2, 64), (4, 4, 64), (32, 2, 128), (8, 8, 128)])
    B, Sq = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 3, 5])
    longest = _log(rng, Sq, max(Sq, min(131072, 131072 * 512 // (B * Hkv * d))))
    return {"kind": kind, "B": B, "Sq": Sq, "Hq": Hq, "Hkv": Hkv, "d": d, "longest": longest, "page": page, "cache": cache,
            "rotary": rng.random() < 0.7, "softcap": rng.choice([0.0, 0.0, 30.0]), "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _ints(g, lo, hi, n):
    """n whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _tables(rows, d):
    """cos and sin of pos * 1e6^(-2i/d), fp32 [rows, d/2]; the angles in 64 bits."""
    f = 1e6 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _shuffled_pages(g, n):
    return torch.randperm(n, generator=g, device="cuda").int()


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = dict(case)
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        kb = -(-K // 128)
        x = _randn(g, M, K)
        x[:, torch.randint(0, K, (max(1, K // 200),), generator=g, device="cuda")] *= 20.0      # channels with outliers
        pad = torch.zeros(M, kb * 128, device="cuda")
        pad[:, :K] = x
        sa = pad.view(M, kb, 128).abs().amax(2).clamp_min(FLOOR) / 448.0
        s["a"] = (pad.view(M, kb, 128) / sa[:, :, None]).view(M, -1)[:, :K].contiguous().to(F8)
        s["a_scale"] = sa
        w = torch.empty(N, K, device="cuda", dtype=F8)
        for n0 in range(0, N, 4096):
            w[n0:n0 + 4096] = (_randn(g, min(4096, N - n0), K) * 110.0).clamp_(-448.0, 448.0).to(F8)
        s["w"] = w
        s["w_scale"] = torch.rand(-(-N // 128), kb, generator=g, device="cuda") * 2e-4 + 1e-4
        s["bias"] = _randn(g, N).to(DTYPES[case["dtype"]]) if case["bias"] else None
    elif kind == "norm":
        M, H, dt = case["M"], case["H"], DTYPES[case["dtype"]]
        s["x"] = (_randn(g, M, H) * 3.0).to(dt)
        s["r"] = _randn(g, M, H).to(dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.3 * _randn(g, H)).to(dt)
    elif kind == "plan":
        B, page, new = case["B"], case["page"], case["new"]
        s["context"] = _ints(g, 0, case["context"], B)
        # running requests have one new token, arriving ones many; some have none
        s["new_lens"] = _ints(g, 0, 1, B) if new == 1 else torch.where(_ints(g, 0, 1, B) > 0, _ints(g, 0, 2 * new, B), 1).int()
        have = (s["context"] + page - 1) // page
        width = -(-(case["context"] + 2 * new) // page)
        pool = B * width
        order = _shuffled_pages(g, pool)
        col = torch.arange(width, device="cuda")[None, :]
        first = have.cumsum(0) - have
        used = int(have.sum())
        at = (first[:, None] + col).clamp_max(pool - 1)
        s["table"] = torch.where(col < have[:, None], order[at], -1).int()
        s["free"] = torch.cat([order[used:], order[:used]]).contiguous()       # a stack: its top is the last of the free ones
        s["count"] = torch.tensor([pool - used], dtype=torch.int32, device="cuda")
        s["left"] = torch.zeros_like(s["count"])
    elif kind == "append":
        B, new, page, Hkv, d, dt = case["B"], case["new"], case["page"], case["Hkv"], case["d"], DTYPES[case["dtype"]]
        lens = _ints(g, 0, 3 * page, B)                                        # what each request holds already
        news = torch.ones_like(lens) if new == 1 else _ints(g, 1, new, B)
        ends = lens + news
        pages = (ends + page - 1) // page
        first = pages.cumsum(0) - pages
        P = B * (3 + -(-new // page)) + 3                                      # (as many for every seed)
        order = _shuffled_pages(g, P).long()
        b = torch.repeat_interleave(torch.arange(B, device="cuda"), news.long())
        i = torch.arange(b.numel(), device="cuda") - (news.cumsum(0) - news)[b]
        pos = lens[b] + i
        s["slots"] = order[(first[b] + pos // page).long()] * page + pos % page
        s["positions"] = pos.int()
        T = b.numel()
        row = _randn(g, T, 3, Hkv, d).to(dt)                                   # slices of a fused projection's rows
        s["k"], s["v"] = row[:, 1], row[:, 2]
        s["k_scale"], s["v_scale"] = (_page_scales(g, case["cache"], P, Hkv) for _ in range(2))
        s["k_cache"], s["v_cache"] = (_codes(g, case["cache"], P, Hkv, page, d) for _ in range(2))
        s["cos"], s["sin"] = _tables(int(ends.max()), d) if case["rotary"] else (None, None)
    else:
        B, Sq, Hq, Hkv, d, page, longest = (case[k] for k in ("B", "Sq", "Hq", "Hkv", "d", "page", "longest"))
        lens = _ints(g, max(Sq, longest // 8), longest, B)
        lens[0] = longest
        width = -(-longest // page)
        pages = (lens + page - 1) // page
        P = int(pages.sum()) + 1
        order = _shuffled_pages(g, P)
        col = torch.arange(width, device="cuda")[None, :]
        at = ((pages.cumsum(0) - pages)[:, None] + col).clamp_max(P - 1)
        s["table"] = torch.where(col < pages[:, None], order[at], -1).int()
        s["lens"] = lens
        row = _randn(g, B, Sq, Hq + 2 * Hkv, d).to(DTYPES[case["dtype"]])
        s["q"] = row[:, :, :Hq]
        s["k_scale"], s["v_scale"] = (_page_scales(g, case["cache"], P, Hkv) for _ in range(2))
        s["k_cache"], s["v_cache"] = (_codes(g, case["cache"], P, Hkv, page, d) for _ in range(2))
        s["cos"], s["sin"] = _tables(longest, d) if case["rotary"] else (None, None)
    return s


def _page_scales(g, cache, P, Hkv):
    """Scales of pages whose values are about normal: powers of two for e4m3, a maximum / 127 for int8."""
    if cache == "e4m3":
        return torch.exp2(torch.randint(-7, -5, (P, Hkv), generator=g, device="cuda").float())
    return (torch.rand(P, Hkv, generator=g, device="cuda") + 3.5) / 127.0


def _codes(g, cache, P, Hkv, page, d):
    out = torch.empty(P, Hkv, page, d, device="cuda", dtype=CACHES[cache])
    step = max(1, (1 << 26) // (Hkv * page * d))
    for p in range(0, P, step):
        x = _randn(g, min(step, P - p), Hkv, page, d)
        out[p:p + step] = (x * 90.0).clamp_(-448.0, 448.0).to(F8) if cache == "e4m3" else (x * 32.0).round_().clamp_(-127, 127).to(torch.int8)
    return out


# ---- the passes --------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if own:
        return _run_own(s)
    return {"linear": _linear, "norm": _norm, "plan": _plan, "append": _append, "attend": _attend}[kind](s)


def _run_own(s):
    from llmqrt_b200 import glue, ops, paged_cache
    kind = s["kind"]
    if kind == "linear":
        return ops.fp8_linear_block(s["a"], s["w"], s["bias"], s["a_scale"], s["w_scale"], DTYPES[s["dtype"]], static_weight=True)
    if kind == "norm":
        q, scale, h = glue.rmsnorm_fp8_block(s["x"], s["weight"], 1e-6, residual=s["r"])
        return {"q": q, "scale": scale, "h": h} if h is not None else {"q": q, "scale": scale}
    if kind == "plan":
        seq, cu, slots, positions = paged_cache.plan_step(s["context"], s["new_lens"], s["table"], s["free"], s["count"], s["page"],
                                                          s["tokens"], free_left=s["left"])
        return {"table": s["table"], "left": s["left"], "seq": seq, "cu": cu, "slots": slots, "positions": positions}
    if kind == "append":
        paged_cache.kv8_append(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["k"], s["v"], s["slots"], s["cos"],
                               s["sin"], s["positions"])
        return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return paged_cache.attn_decode_kv8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lens"],
                                       s["longest"], softcap=s["softcap"], cos=s["cos"], sin=s["sin"])


def _spread(scale, rows, cols, of_rows):
    """A scale for each block of of_rows x 128 as one for each element of [rows, cols]."""
    return scale.repeat_interleave(of_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _linear(s):
    M, N, K = s["M"], s["N"], s["K"]
    y = (s["a"].float() * _spread(s["a_scale"], M, K, 1)) @ (s["w"].float() * _spread(s["w_scale"], N, K, 128)).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["dtype"]])


def _norm(s):
    M, H, dt = s["M"], s["H"], DTYPES[s["dtype"]]
    h = s["x"].float()
    out = {}
    if s["r"] is not None:
        out["h"] = (h + s["r"].float()).to(dt)
        h = out["h"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
    kb = -(-H // 128)
    pad = torch.zeros(M, kb * 128, device=y.device)
    pad[:, :H] = y
    top = pad.view(M, kb, 128).abs().amax(2).clamp_min(FLOOR)
    out["scale"] = top / torch.full_like(top, 448.0)
    q = pad.view(M, kb, 128) * (torch.full_like(top, 448.0) / top)[:, :, None]
    out["q"] = q.clamp(-448.0, 448.0).view(M, -1)[:, :H].to(F8)
    return out


def _plan(s):
    page, most = s["page"], s["tokens"]
    ctx, new, table = s["context"].long(), s["new_lens"].long(), s["table"]
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    have = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page - have
    fits = (cu[1:] <= most) & (have + need <= table.shape[1])
    need = torch.where(fits, need, 0)
    upto = need.cumsum(0)
    fits &= (need == 0) | (upto <= s["count"].long())
    need = torch.where(fits, need, 0)
    # pages from the top of the stack, in the order of the requests
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    j = col - have[:, None]
    fresh = (j >= 0) & (j < need[:, None])
    at = s["count"].long() - 1 - ((upto - need)[:, None] + j)
    table.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], table))
    s["left"].copy_(s["count"] - need.sum().int())
    t = torch.arange(most, device=table.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    inside = b < ctx.numel()
    b = b.clamp_max(ctx.numel() - 1)
    inside &= fits[b]
    pos = ctx[b] + t - cu[b]
    slot = table[b, (pos // page).clamp(0, table.shape[1] - 1)].long() * page + pos % page
    return {"table": table, "left": s["left"], "seq": torch.where(fits, ctx + new, ctx).int(), "cu": cu.int(),
            "slots": torch.where(inside, slot, -1), "positions": torch.where(inside, pos, 0).int()}


def _rotated(x, cos, sin):
    """Half-split pairing; x [..., d], cos and sin broadcast over [..., d/2]."""
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)


def _append(s):
    page, slots = s["page"], s["slots"]
    page_of, row_of = slots // page, slots % page
    pages, group = torch.unique_consecutive(page_of, return_inverse=True)
    first = torch.full_like(pages, page).scatter_reduce_(0, group, row_of, "amin")
    last = torch.zeros_like(pages).scatter_reduce_(0, group, row_of, "amax")
    k, v = s["k"].float(), s["v"].float()
    if s["cos"] is not None:
        at = s["positions"].long()
        k = _rotated(k, s["cos"][at][:, None], s["sin"][at][:, None])
    rows = torch.arange(page, device=slots.device)[None, None, :, None]
    before, inside = rows < first[:, None, None, None], (rows >= first[:, None, None, None]) & (rows <= last[:, None, None, None])
    for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        most = 448.0 if cache.dtype == F8 else 127.0
        new = torch.zeros(pages.numel(), page, *x.shape[1:], device=x.device)
        new[group, row_of] = x
        new = new.transpose(1, 2)                                              # [pages, Hkv, page, d]
        top = new.abs().amax((2, 3)).clamp_min(FLOOR)
        want = top / torch.full_like(top, most)
        if cache.dtype == F8:                                                  # the least power of two that holds it
            m, e = torch.frexp(want)
            want = torch.ldexp(torch.ones_like(want), e - (m == 0.5).int())
        old = torch.where(first[:, None] > 0, scale[pages], 0.0)
        got = torch.maximum(old, want)
        was = cache[pages].float()
        ratio = (old / got)[:, :, None, None]
        kept = torch.where(before, was * ratio, was)
        put = new * (torch.ones_like(got) / got)[:, :, None, None]
        q = torch.where(inside, put, kept)
        q = q.clamp(-448.0, 448.0).to(F8) if cache.dtype == F8 else q.round().clamp(-127, 127).to(torch.int8)
        cache[pages] = torch.where(before | inside, q.float(), was).to(cache.dtype)
        scale[pages] = got
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _attend(s):
    B, Sq, Hq, Hkv, d, page = (s[k] for k in ("B", "Sq", "Hq", "Hkv", "d", "page"))
    lens, table = s["lens"].long(), s["table"].long().clamp_min(0)
    L = table.shape[1] * page
    q = s["q"].float()
    if s["cos"] is not None:
        at = lens[:, None] - Sq + torch.arange(Sq, device=q.device)
        q = _rotated(q, s["cos"][at][:, :, None], s["sin"][at][:, :, None])
    q = q.view(B, Sq, Hkv, Hq // Hkv, d).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, d)
    k, v = ((c[table].float() * sc[table][..., None, None]).transpose(1, 2).reshape(B, Hkv, L, d)
            for c, sc in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
    logit = q @ k.transpose(2, 3) * d ** -0.5
    if s["softcap"]:
        logit = s["softcap"] * torch.tanh(logit / s["softcap"])
    sees = lens[:, None] - Sq + 1 + torch.arange(Sq, device=q.device)           # keys that a query token sees
    hidden = torch.arange(L, device=q.device) >= sees[..., None]                # [B, Sq, L]
    logit = logit.masked_fill(hidden.repeat_interleave(Hq // Hkv, 1)[:, None], float("-inf"))
    e = torch.exp(logit - logit.amax(3, keepdim=True))
    o = e @ v / e.sum(3, keepdim=True)
    return o.view(B, Hkv, Sq, Hq // Hkv, d).permute(0, 2, 1, 3, 4).reshape(B, Sq, Hq, d).to(s["q"].dtype)


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        kb, nb = -(-K // 128), -(-N // 128)
        return {"bytes": M * K + N * K + 4 * (M + nb) * kb + 2 * M * N + 2 * N * case["bias"], "flops": 2 * M * N * K}
    if kind == "norm":
        M, H = case["M"], case["H"]
        return {"bytes": M * H * (7 if case["residual"] else 3) + 4 * M * -(-H // 128) + 2 * H, "flops": 6 * M * H}
    if kind == "plan":                    # lengths in and out, a slot and a position for each token, the pages of the tokens twice
        B, T = case["B"], case["tokens"]
        return {"bytes": 16 * B + 12 * T + 8 * (B + T // case["page"]), "flops": 4 * T}
    Hkv, d = case["Hkv"], case["d"]
    if kind == "append":                  # (lengths are even over 1 .. new)
        T = case["B"] * (1 if case["new"] == 1 else (1 + case["new"]) / 2)
        return {"bytes": T * (Hkv * d * 2 * 3 + 12 + (4 * d if case["rotary"] else 0)) + 16 * (T // case["page"] + case["B"]) * Hkv,
                "flops": 8 * T * Hkv * d}
    B, Sq, longest = case["B"], case["Sq"], case["longest"]
    keys = longest + (B - 1) * (longest + max(Sq, longest // 8)) / 2            # (lengths are even over their range)
    return {"bytes": keys * Hkv * (2 * d + 8 / case["page"]) + 4 * keys / case["page"] + 4 * B * Sq * case["Hq"] * d,
            "flops": 4 * keys * Sq * case["Hq"] * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _to_e4m3(x):
    """The e4m3 value nearest to x (ties to the even one), within +-448."""
    m, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)           # spacing of e4m3 around x
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    f = torch.float64
    if kind == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        y = torch.zeros(M, N, dtype=f, device="cuda")
        n_block = torch.arange(N, device="cuda") // 128
        for g in range(-(-K // 128)):
            k = slice(128 * g, min(K, 128 * g + 128))
            y += (s["a"][:, k].to(f) @ s["w"][:, k].to(f).t()) * s["a_scale"][:, g:g + 1].to(f) * s["w_scale"][n_block, g].to(f)
        return y if s["bias"] is None else y + s["bias"].to(f)
    if kind == "norm":
        dt, H = DTYPES[case["dtype"]], case["H"]
        h, out = s["x"].to(f), {}
        if case["residual"]:
            h = h + s["r"].to(f)
            out["h"] = h.clone()
            h = h.to(dt).to(f)                                                  # the norm is of what is stored
        y = h * s["weight"].to(f) / torch.sqrt(h.square().sum(1, keepdim=True) / H + 1e-6)
        parts, scales = [], []
        for k in range(0, H, 128):
            p = y[:, k:k + 128]
            sc = p.abs().amax(1, keepdim=True).clamp_min(FLOOR) / 448
            parts.append(_to_e4m3(p / sc))
            scales.append(sc)
        out["q"], out["scale"] = torch.cat(parts, 1), torch.cat(scales, 1)
        return out
    if kind == "plan":
        return None                                                             # whole numbers
    if kind == "append":
        out = {}
        page, slots = case["page"], s["slots"].tolist()
        starts = [0] + [t for t in range(1, len(slots)) if slots[t] // page != slots[t - 1] // page] + [len(slots)]
        if len(starts) * 2 > 9000:
            return None
        k, v = s["k"].to(f), s["v"].to(f)
        if s["cos"] is not None:
            c, sn = (t.to(f)[s["positions"].long()][:, None, :] for t in (s["cos"], s["sin"]))
            half = case["d"] // 2
            k = torch.cat([k[..., :half] * c - k[..., half:] * sn, k[..., half:] * c + k[..., :half] * sn], -1)
        for name, x in (("k", k), ("v", v)):
            held, scale = s[name + "_cache"].to(f), s[name + "_scale"].to(f)
            for a, b in zip(starts[:-1], starts[1:]):
                p, r0 = slots[a] // page, slots[a] % page
                part = x[a:b].transpose(0, 1)                                   # [Hkv, n, d]
                top = part.abs().amax((1, 2)).clamp_min(FLOOR)
                if case["cache"] == "e4m3":
                    m, e = torch.frexp(top / 448)
                    want = torch.ldexp(torch.ones_like(top), e - (m == 0.5).to(e.dtype))
                else:
                    want = top / 127
                got = torch.maximum(want, scale[p]) if r0 else want
                rounded = _to_e4m3 if case["cache"] == "e4m3" else torch.round
                if r0:
                    held[p, :, :r0] = rounded(held[p, :, :r0] * (scale[p] / got)[:, None, None])
                held[p, :, r0:r0 + b - a] = rounded(part / got[:, None, None])
                scale[p] = got
            out[name + "_cache"] = held if case["cache"] == "e4m3" else None    # int8 codes are whole numbers
            out[name + "_scale"] = scale
        return out
    B, Sq, Hq, Hkv, d, page = (case[k] for k in ("B", "Sq", "Hq", "Hkv", "d", "page"))
    out = torch.zeros(B, Sq, Hq, d, dtype=f, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        ids = s["table"][b, : -(-n // page)].long()
        k, v = ((c[ids].to(f) * sc[ids].to(f)[:, :, None, None]).permute(1, 0, 2, 3).reshape(Hkv, -1, d)[:, :n]
                for c, sc in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
        for i in range(Sq):
            at = n - Sq + i
            q = s["q"][b, i].to(f)
            if s["cos"] is not None:
                c, sn = s["cos"][at].to(f), s["sin"][at].to(f)
                q = torch.cat([q[:, : d // 2] * c - q[:, d // 2:] * sn, q[:, d // 2:] * c + q[:, : d // 2] * sn], 1)
            z = torch.einsum("hrd,hkd->hrk", q.view(Hkv, -1, d), k[:, : at + 1]) / math.sqrt(d)
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            out[b, i] = torch.einsum("hrk,hkd->hrd", torch.softmax(z, 2), v[:, : at + 1]).reshape(Hq, d)
    return out
