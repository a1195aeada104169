"""Paged 8-bit cache: pages and slots, writes, attention, against plain implementations in 64 bits."""
import math

import pytest
import torch

from tests.util import bits_equal, rel_fro

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
CACHE = {"e4m3": F8, "int8": torch.int8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- pages and slots -----------------------------------------------------------------------------------
def _plan(ctx, new, table, free, count, page, most):
    """The rule, request by request.  table: list of lists, changed in place."""
    width, cu, wanted, taken = len(table[0]) if table else 0, [0], 0, 0
    seq, slots, pos = [], [-1] * most, [0] * most
    count = min(max(count, 0), len(free))
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        first = cu[-1]
        cu.append(first + n)
        have, all_ = -(-c // page), -(-(c + n) // page)
        need, fits = all_ - have, cu[-1] <= most and all_ <= width
        if fits:
            wanted += need
            fits = need == 0 or wanted <= count
        if fits:
            for j in range(need):
                table[b][have + j] = free[count - 1 - (wanted - need) - j]
            taken += need
            for i in range(n):
                p = table[b][(c + i) // page]
                slots[first + i], pos[first + i] = (p * page + (c + i) % page if p >= 0 else -1), c + i
        seq.append(c + n if fits else c)
    return seq, cu, slots, pos, count - taken


def _plan_case(B, page, top_ctx, top_new, width, pool, g):
    ctx = torch.randint(0, top_ctx + 1, (B,), generator=g).tolist()
    new = torch.randint(0, top_new + 1, (B,), generator=g).tolist()
    free = torch.randperm(pool, generator=g).tolist()
    table, n = [], 0
    for c in ctx:                                            # contexts hold pages of their own, behind the pool's numbers
        k = min(-(-c // page), width)
        table.append([pool + n + j for j in range(k)] + [-1] * (width - k))
        n += k
    return ctx, new, free, table


@pytest.mark.parametrize("B,page,top_ctx,top_new,width,pool,count,most", [
    (1, 16, 0, 1, 1, 1, 1, 1),
    (1, 16, 15, 1, 2, 1, 0, 1),                              # nothing left in the stack
    (7, 16, 40, 0, 5, 3, 3, 0),                              # nothing new
    (7, 32, 40, 1, 5, 30, 30, 9),
    (64, 16, 300, 1, 25, 40, 17, 64),
    (64, 64, 1000, 500, 40, 400, 400, 40000),
    (64, 64, 1000, 500, 40, 400, 150, 40000),                # the stack runs out
    (64, 128, 1000, 500, 9, 400, 390, 40000),                # the table is too narrow for some
    (64, 16, 100, 50, 40, 400, 390, 777),                    # too few tokens
    (511, 16, 50, 3, 8, 900, 900, 2000),
    (513, 16, 50, 3, 8, 900, 200, 2000),
    (2000, 32, 90, 40, 10, 5000, 4000, 50000),
    (8192, 16, 5, 2, 2, 20, 15, 9000),
])
def test_plan_step(B, page, top_ctx, top_new, width, pool, count, most):
    from llmqrt_b200.paged_cache import plan_step
    g = torch.Generator().manual_seed(B * 1000 + page + most)
    ctx, new, free, table = _plan_case(B, page, top_ctx, top_new, width, pool, g)
    if B > 5:
        ctx[1], new[2] = -3, -5                              # count as none
        table[1] = [-1] * width
    dev_ctx, dev_new, dev_free = _i32(ctx), _i32(new), _i32(free)
    wide = torch.full((B, width + 3), 7, dtype=torch.int32, device="cuda")
    wide[:, :width] = _i32(table)
    dev_table = wide[:, :width]                              # rows of a wider table
    dev_count = _i32([count])
    left = torch.full((1,), -9, dtype=torch.int32, device="cuda")
    got = plan_step(dev_ctx, dev_new, dev_table, dev_free, dev_count, page, most, free_left=left)
    seq, cu, slots, pos, rest = _plan(ctx, new, table, free, count, page, most)
    for have, want in zip(got, (seq, cu, slots, pos)):
        assert have.tolist() == want
    assert dev_table.tolist() == table and (wide[:, width:] == 7).all()
    assert left.tolist() == [rest] and dev_count.tolist() == [count] and dev_ctx.tolist() == ctx
    # in place, what a captured step does
    wide[:, :width] = _i32([[-1 if j >= -(-max(c, 0) // page) else t for j, t in enumerate(r)] for c, r in zip(ctx, table)])
    again = plan_step(dev_ctx, dev_new, dev_table, dev_free, dev_count, page, most, seq_lens=dev_ctx)
    assert again[0].data_ptr() == dev_ctx.data_ptr() and dev_ctx.tolist() == seq and dev_count.tolist() == [rest]
    assert again[2].tolist() == slots and dev_table.tolist() == table


@pytest.mark.parametrize("B,most", [(128, 256), (128, 257), (129, 256), (512, 1500), (513, 700), (1024, 1500), (1025, 1500), (8191, 9000), (8192, 30000)])
def test_plan_step_at_the_borders_of_its_forms(B, most):
    test_plan_step(B, 16, 50, 3, 8, 9000, B // 2, most)


def test_plan_step_without_requests():
    from llmqrt_b200.paged_cache import plan_step
    e, table, count = _i32([]), torch.zeros(0, 4, dtype=torch.int32, device="cuda"), _i32([2])
    seq, cu, slots, pos = plan_step(e, e, table, _i32([5, 6]), count, 16, 3)
    assert seq.numel() == 0 and cu.tolist() == [0] and slots.tolist() == [-1] * 3 and pos.tolist() == [0] * 3 and count.tolist() == [2]


@pytest.mark.parametrize("count", [-4, 9])
def test_plan_step_keeps_within_the_pool(count):
    """A count outside the pool is taken as the nearest one inside."""
    from llmqrt_b200.paged_cache import plan_step
    table, c = torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), _i32([count])
    seq, _, slots, _ = plan_step(_i32([0, 0]), _i32([16, 17]), table, _i32([4, 2, 9]), c, 16, 33)
    if count < 0:
        assert seq.tolist() == [0, 0] and c.tolist() == [0] and (slots == -1).all()
    else:
        assert seq.tolist() == [16, 17] and c.tolist() == [0] and table.tolist() == [[9, -1, -1], [2, 4, -1]]


@pytest.mark.parametrize("B,page", [(1, 16), (6, 32), (700, 16)])
def test_release_pages(B, page):
    from llmqrt_b200.paged_cache import release_pages
    g = torch.Generator().manual_seed(B)
    width, lens = 5, torch.randint(0, 5 * page + 1, (B,), generator=g).tolist()
    done = (torch.rand(B, generator=g) < 0.4).tolist()
    table = [[b * width + j for j in range(width)] for b in range(B)]
    free = [-7] * (B * width + 2)
    free[0], free[1] = 900001, 900002
    dl, df, dc = _i32(lens), _i32(free), _i32([2])
    release_pages(torch.tensor(done, device="cuda"), dl, _i32(table), df, dc, page)
    want = free[:2] + [table[b][j] for b in range(B) if done[b] for j in range(-(-lens[b] // page))]
    assert dc.tolist() == [len(want)] and df.tolist()[:len(want)] == want and (df[len(want):] == -7).all()
    assert dl.tolist() == [0 if d else n for n, d in zip(lens, done)]
    release_pages(torch.tensor(done, device="cuda"), dl, _i32(table), df, dc, page)      # they hold nothing any more
    assert dc.tolist() == [len(want)]


# ---- writes --------------------------------------------------------------------------------------------
def _e4m3(x):
    """The e4m3 value nearest to x (64 bits, ties to the even one), within +-448; NaN stays."""
    m, e = torch.frexp(x.clamp(-448, 448))
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)
    return torch.where(x.isnan(), x, (x.clamp(-448, 448) / step).round() * step)


def _append(kind, lo, hi, scale, x, slots):
    """The rule, run by run, in 64 bits.  lo, hi (code values) and scale are changed in place; a code written may be anything
    from lo to hi, which lie apart where the definition's value is next to a border: fp32 arithmetic moves it by at most 8 * 2^-24
    of the page's maximum (two products and a sum of a rotation, each of at most twice the maximum: 4; reciprocal and
    product 2; the scale 2)."""
    P, Hkv, page, d = lo.shape
    most = 448 if kind == "e4m3" else 127
    q = _e4m3 if kind == "e4m3" else (lambda v: torch.where(v.isnan(), 0.0, v).clamp(-127, 127).round())
    slack = 8 * 2.0 ** -24 * most
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < P * page:
            t += 1
            continue
        p, r, n = slots[t] // page, slots[t] % page, 1
        while t + n < len(slots) and r + n < page and slots[t + n] == slots[t] + n:
            n += 1
        part = x[t:t + n].transpose(0, 1)                     # [Hkv, n, d]
        top = torch.where(part.isnan(), 0.0, part).abs().amax((1, 2)).clamp(1e-12, 3e38)
        if kind == "e4m3":
            m, e = torch.frexp(top / 448)
            new = torch.ldexp(torch.ones_like(top), e - (m == 0.5).to(e.dtype))
        else:
            new = top / 127
        s = torch.maximum(new, scale[p]) if r else new
        for cache, sign in ((lo, -1), (hi, 1)):
            if r:
                f = (scale[p] / s)[:, None, None]
                cache[p, :, :r] = torch.where(f == 1, cache[p, :, :r], q(cache[p, :, :r] * f + sign * slack * (f < 1)))
            cache[p, :, r:r + n] = q(part / s[:, None, None] + sign * slack)
        scale[p] = s
        t += n


def _random_codes(g, kind, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * 90).clamp(-448, 448).to(F8) if kind == "e4m3" else (x * 40).round().clamp(-127, 127).to(torch.int8)


def _check_append(kind, dt, page, Hkv, d, slots, g, rotary=True, P=None, x=None, stale_scale=1.0):
    from llmqrt_b200 import glue
    from llmqrt_b200.paged_cache import kv8_append
    T = len(slots)
    P = P or max(slots + [0]) // page + 2
    kc, vc = (_random_codes(g, kind, (P, Hkv, page, d)) for _ in range(2))
    ks, vs = (torch.rand(P, Hkv, generator=g, device="cuda") * 0.02 * stale_scale + 1e-4 for _ in range(2))
    if kind == "e4m3":
        ks, vs = (torch.exp2(s.log2().round()) for s in (ks, vs))
    if x is None:
        x = torch.randn(T, 3, Hkv, d, generator=g, device="cuda").to(dt)
        x[:, 1] *= 3.0
    k, v = x[:, 1], x[:, 2]
    pos = torch.randint(0, 700, (T,), generator=g, device="cuda", dtype=torch.int32)
    cos, sin = glue.rope_tables(d, 600, 1e4, "cuda") if rotary else (None, None)      # (some positions lie behind the tables)
    kk = k.double()
    if rotary:
        at = pos.clamp_max(599).long()
        c, s = cos[at].double()[:, None], sin[at].double()[:, None]
        lo, hi = kk.chunk(2, -1)
        kk = torch.where((pos < 600)[:, None, None], torch.cat([lo * c - hi * s, lo * s + hi * c], -1), kk)
    want = []
    for cache, scale, new in ((kc, ks, kk), (vc, vs, v.double())):
        lo, hi, s = cache.float().double(), cache.float().double(), scale.double()
        _append(kind, lo, hi, s, new, slots)
        want.append((lo, hi, s))
    before = [t.clone() for t in (kc, vc)]
    kv8_append(kc, vc, ks, vs, k, v, torch.tensor(slots, dtype=torch.int64, device="cuda"), cos, sin, pos)
    for i, (cache, scale) in enumerate(((kc, ks), (vc, vs))):
        lo, hi, s = want[i]
        # a scale is one fp32 division of a maximum that, rotated, three fp32 roundings made
        assert ((scale.double() - s).abs() <= 6 * 2.0 ** -24 * s).all()
        got = cache.float().double()
        assert ((got >= lo) & (got <= hi) | got.isnan() & lo.isnan()).all()
        written = torch.zeros(P, page, dtype=torch.bool, device="cuda")
        for t in slots:
            if 0 <= t < P * page:
                written[t // page, :t % page + 1] = True
        assert bits_equal(cache.transpose(1, 2)[~written], before[i].transpose(1, 2)[~written])
    return kc, vc, ks, vs


def _slots_of(page, spans):
    """Slots of requests that hold `have` tokens and get `new`, in pages handed out in a scattered order."""
    out, nxt = [], 0
    for have, new in spans:
        n = -(-(have + new) // page)
        pages = [(nxt + j) * 7 % 401 for j in range(n)]       # (distinct: fewer than 401 in all)
        nxt += n
        out += [pages[i // page] * page + i % page for i in range(have, have + new)]
    return out


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("page,Hkv,d", [(16, 4, 128), (32, 1, 64), (64, 3, 128), (128, 2, 64)])
def test_append(kind, dt, page, Hkv, d):
    g = _gen(page + Hkv + d)
    for spans in ([(0, 1)], [(5, 1)], [(page - 1, 1)], [(page, 1)], [(0, page)], [(3, 2 * page + 1), (0, page + 1), (page - 1, 2)],
                  [(i, 1) for i in range(9)], [(2 * i % page, 40) for i in range(4)]):
        _check_append(kind, DT[dt], page, Hkv, d, _slots_of(page, spans), g)
    # a large call takes wider windows
    _check_append(kind, DT[dt], page, Hkv, d, _slots_of(page, [(7, 1300), (page - 3, 1100)] if page > 32 else [(7, 1300), (page - 3, 20), (0, 780)]), g, rotary=False)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_skips_and_keeps(kind):
    g = _gen(3)
    page = 16
    # tokens without a slot, slots outside the cache, a page begun in the middle although it was never written
    _check_append(kind, torch.float16, page, 2, 64, [-1, 5, 6, -1, 7 * page, 100000, -5, 33, -1, -1], g, P=7, stale_scale=50.0)
    # an old scale that stays the greater one: the rows ahead keep their codes
    kc, vc, ks, vs = _check_append(kind, torch.float16, page, 2, 64, [9, 10, 11], g, P=3, stale_scale=5000.0)
    assert (ks[0] > 0.1).all()
    from llmqrt_b200.paged_cache import kv8_append
    empty = torch.empty(0, 2, 64, device="cuda", dtype=torch.float16)
    was = kc.clone()
    kv8_append(kc, vc, ks, vs, empty, empty, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert bits_equal(kc, was)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_append_special_values(kind, dt):
    """Zeros, infinities (the greatest code), NaN (NaN, as int8 0), and values below the scale's floor."""
    from llmqrt_b200.paged_cache import kv8_append
    x = torch.zeros(4, 1, 64, device="cuda", dtype=DT[dt])
    x[1, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.0], dtype=DT[dt])
    x[2, 0, 0] = float("nan")
    x[2, 0, 1] = 3.0
    x[3] = 1e-20
    kc, vc = (torch.zeros(4, 1, 16, 64, dtype=torch.int8, device="cuda").view(CACHE[kind]) for _ in range(2))
    ks, vs = (torch.full((4, 1), 7.0, device="cuda") for _ in range(2))
    kv8_append(kc, vc, ks, vs, x, x, torch.tensor([0, 16, 32, 48], device="cuda"))
    top, c = (448.0, kc.float()[:, 0, 0]) if kind == "e4m3" else (127.0, kc.float()[:, 0, 0])
    assert bits_equal(kc, vc) and torch.equal(ks, vs) and torch.isfinite(ks).all() and (ks > 0).all()
    assert (c[0] == 0).all() and (c[3] == 0).all()
    assert c[1, 0] == top and c[1, 1] == -top and c[1, 3] == 0
    for v in (c[1, 2], c[2, 0]):
        assert v.isnan() if kind == "e4m3" else v == 0
    assert abs(float(c[2, 1] * ks[2]) - 3.0) <= 3.0 * 2.0 ** -4


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_token_by_token(kind):
    """A page that fills token by token.  Its scale is that of all its tokens at once; what is off is one rounding (e4m3: codes
    equal but for values that became subnormal) or one for each time the scale grew (int8: half a step of the scale
    of the time, and scales only grow)."""
    from llmqrt_b200.paged_cache import kv8_append
    g = _gen(5)
    page, Hkv, d, T = 32, 3, 128, 32
    x = (torch.randn(T, Hkv, d, generator=g, device="cuda") * torch.linspace(0.2, 5, T, device="cuda")[:, None, None]).half()
    caches = [torch.zeros(2, Hkv, page, d, dtype=torch.int8, device="cuda").view(CACHE[kind]) for _ in range(4)]
    scales = [torch.zeros(2, Hkv, device="cuda") for _ in range(4)]
    slots = torch.arange(T, device="cuda") + page
    kv8_append(*caches[:2], *scales[:2], x, x, slots)
    grew = torch.zeros(Hkv, device="cuda")
    for t in range(T):
        was = scales[2][1].clone()
        kv8_append(*caches[2:], *scales[2:], x[t:t + 1], x[t:t + 1], slots[t:t + 1])
        grew += (scales[2][1] > was).float()
    assert torch.equal(scales[0][1], scales[2][1])
    want = x.transpose(0, 1).double()
    got = caches[2][1].float().double() * scales[2][1][:, None, None].double()
    if kind == "int8":
        assert ((got - want).abs() <= (grew * scales[2][1] * 0.5 * (1 + 2.0 ** -20))[:, None, None]).all()
    else:
        once = caches[0][1].float().double() * scales[0][1][:, None, None].double()
        small = want.abs() < 2.0 ** -6 * scales[0][1][:, None, None].double()
        assert torch.equal(got[~small], once[~small])
        assert ((got - want).abs()[small] <= (2.0 ** -9 * scales[0][1][:, None, None].double()).expand_as(want)[small]).all()


# ---- attention -----------------------------------------------------------------------------------------
def _attend(q, kc, vc, ks, vs, table, lens, top, softcap, cos, sin):
    """One sequence at a time in 64 bits.  q [B, Sq, Hq, d]; a page outside the cache has no keys."""
    B, Sq, Hq, d = q.shape
    P, Hkv, page, _ = kc.shape
    out = torch.zeros(B, Sq, Hq, d, dtype=torch.float64, device="cuda")
    kd, vd = ((c.float().double() * s[:, :, None, None].double()) for c, s in ((kc, ks), (vc, vs)))
    for b, n_raw in enumerate(lens):
        n = min(n_raw, top, table.shape[1] * page)
        for s in range(Sq):
            m = min(n, n_raw - Sq + 1 + s)
            if m <= 0:
                continue
            ids = table[b, : -(-m // page)].tolist()
            keep = torch.tensor([i for i in range(m) if 0 <= ids[i // page] < P], dtype=torch.long, device="cuda")
            if not len(keep):
                continue
            idx = torch.tensor([i if 0 <= i < P else 0 for i in ids], device="cuda")
            k, v = (c[idx].transpose(1, 2).reshape(-1, Hkv, d)[keep] for c in (kd, vd))
            x, at = q[b, s].double(), n_raw - Sq + s
            if cos is not None and 0 <= at < cos.shape[0]:
                lo, hi = x.chunk(2, -1)
                c, sn = cos[at].double(), sin[at].double()
                x = torch.cat([lo * c - hi * sn, lo * sn + hi * c], -1)
            z = torch.einsum("hrd,khd->hrk", x.view(Hkv, -1, d), k) / math.sqrt(d)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            out[b, s] = torch.einsum("hrk,khd->hrd", z.softmax(-1), v).reshape(Hq, d)
    return out


def _cache(g, kind, P, Hkv, page, d):
    kc, vc = (_random_codes(g, kind, (P, Hkv, page, d)) for _ in range(2))
    if kind == "e4m3":
        ks, vs = (torch.exp2(torch.randint(-8, -4, (P, Hkv), generator=g, device="cuda").float()) for _ in range(2))
    else:
        ks, vs = ((torch.rand(P, Hkv, generator=g, device="cuda") + 0.2) * 0.03 for _ in range(2))
    return kc, vc, ks, vs


def _tables(g, lens, page, width, P):
    table, perm, n = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), torch.randperm(P, generator=g, device="cuda"), 0
    for b, m in enumerate(lens):
        k = min(-(-max(m, 0) // page), width)
        table[b, :k] = perm[n:n + k].int()
        n += k
    return table


def _check_attend(lens, page, Hq, Hkv, d, Sq, kind, dt, softcap=0.0, rotary=True, top=None, seed=0, width=None):
    from llmqrt_b200 import glue
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(seed + len(lens) + max(lens))
    width = width or max(1, -(-max(lens) // page))
    P = sum(-(-max(n, 0) // page) for n in lens) + 2
    kc, vc, ks, vs = _cache(g, kind, P, Hkv, page, d)
    table = _tables(g, lens, page, width, P)
    row = torch.randn(len(lens), Sq, Hq + 2 * Hkv, d, generator=g, device="cuda").to(dt)
    q = row[:, :, :Hq]
    cos, sin = glue.rope_tables(d, max(max(lens) - 1, 1), 1e4, "cuda") if rotary else (None, None)      # (the newest of all stands behind them)
    top = width * page if top is None else top
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), top, softcap, cos, sin)
    want = _attend(q, kc, vc, ks, vs, table, lens, top, softcap, cos, sin)
    assert out.dtype == dt and out.shape == q.shape
    # fp16: the result's rounding alone, 2^-11 (P and Q keep 22 bits), and 2^-16 for the fp32 arithmetic;
    # bf16: 2^-8, P in fp16 2^-11, and rotated Q in fp16, which moves scores of at most about eight by 2^-11 of them
    tol = 2.0 ** -11 + 2.0 ** -16 if dt == torch.float16 else 2.0 ** -8 + 9 * 2.0 ** -11
    assert rel_fro(out, want) < tol
    dead = want.abs().amax(-1) == 0
    assert (out[dead] == 0).all()
    return q, kc, vc, ks, vs, table, out


@pytest.mark.parametrize("lens,page", [([1], 16), ([15, 16, 17, 0, 1], 16), ([64], 64), ([127, 128, 129, 3], 128), ([500, 33, 64, 65], 32),
                                       ([2000, 1, 700], 16), ([300] * 70, 64)])
@pytest.mark.parametrize("Hq,Hkv,d", [(28, 4, 128), (14, 2, 64), (4, 4, 128), (16, 1, 64)])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_attend(lens, page, Hq, Hkv, d, kind, dt):
    _check_attend(lens, page, Hq, Hkv, d, 1, kind, DT[dt])


@pytest.mark.parametrize("Sq", [2, 3, 7, 16])
@pytest.mark.parametrize("Hq,Hkv,d", [(28, 4, 128), (6, 6, 64), (32, 2, 64)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_attend_several_tokens(Sq, Hq, Hkv, d, dt):
    """Query tokens see the keys up to their own; sequences shorter than the queries leave the first of them without a key."""
    _check_attend([100, Sq, 1, 0, 900, 17], 16, Hq, Hkv, d, Sq, "e4m3", DT[dt])


@pytest.mark.parametrize("lens,top,width", [([9000, 20, 8200], None, None), ([5000] * 40, None, None), ([33000], None, None),
                                            ([900, 300], 500, None), ([900, 300], 100000, 80), ([70], 0, None), ([40, 3], None, 4000)])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_attend_splits(lens, top, width, kind):
    """Splits merged by a cluster and by a second kernel, lengths beyond the bound, tables wider than the lengths."""
    _check_attend(lens, 16, 14, 2, 64, 1, kind, torch.float16, top=top, width=width)


def test_attend_long_blocks():
    """So many query rows that a block takes more keys than it holds page numbers for at a time."""
    _check_attend([9000] + [10] * 63, 16, 32, 2, 64, 16, "e4m3", torch.float16, rotary=False, top=40000, width=2500)


@pytest.mark.parametrize("softcap", [5.0, 30.0])
def test_attend_softcap(softcap):
    _check_attend([100, 700], 32, 28, 4, 128, 1, "int8", torch.float16, softcap=softcap)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_attend_scales_far_apart(kind, dt):
    """Pages whose scales differ by many orders, queries near the type's ends."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(8)
    kc, vc, ks, vs = _cache(g, kind, 12, 2, 16, 64)
    vs *= torch.logspace(-9, 9, 12, device="cuda")[:, None]
    ks[:] = 1e-3
    q = torch.randn(1, 8, 64, generator=g, device="cuda")
    q[0, 0] *= 1e-7 if dt == "fp16" else 1e-30
    q[0, 1] *= 2e3
    q = q.to(DT[dt])
    table = torch.arange(12, dtype=torch.int32, device="cuda")[None]
    want = _attend(q[:, None], kc, vc, ks, vs, table, [190], 192, 0.0, None, None)[:, 0]
    keep = want.abs().amax(-1) < 6e4 if dt == "fp16" else torch.ones(1, 8, dtype=torch.bool, device="cuda")
    if dt == "fp16":                                         # values that fp16 holds
        vs *= 1e-9
        want = want * 1e-9
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([190]), 192)
    # (scores of up to 2e3 standard ones: their fp32 roundings move P by 2^-24 * 2000 * 8)
    assert rel_fro(out, want) < (2.0 ** -11 if dt == "fp16" else 2.0 ** -8 + 2.0 ** -11) + 2e-3
    assert keep is not None and torch.isfinite(out).all()


def test_attend_pages_outside_the_cache():
    """Table entries that name no page are not read; their tokens get no weight, a sequence of none but them gives zeros."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    for Sq in (1, 2):
        g = _gen(11)
        kc, vc, ks, vs = _cache(g, "e4m3", 9, 2, 16, 128)
        q = torch.randn(3, Sq, 8, 128, generator=g, device="cuda").half()
        table = torch.tensor([[0, -1, 3, 9, 4], [-1, -5, 2 ** 31 - 1, -2 ** 31, 9], [8, 7, 6, 5, 2]], dtype=torch.int32, device="cuda")
        lens = [80, 70, 77]
        out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), 80)
        want = _attend(q, kc, vc, ks, vs, table, lens, 80, 0.0, None, None)
        assert rel_fro(out, want) < 2.0 ** -11 + 2.0 ** -16 and (out[1] == 0).all()


def test_attend_does_not_read_behind_the_last_key():
    """Rows behind the last token and pages behind the last one hold NaN."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(12)
    kc, vc, ks, vs = _cache(g, "e4m3", 6, 2, 32, 64)
    q = torch.randn(1, 4, 64, generator=g, device="cuda").half()
    table = torch.tensor([[2, 5, 1, 3]], dtype=torch.int32, device="cuda")
    clean = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([45]), 128)
    for c in (kc, vc):
        c.view(torch.uint8)[5, :, 13:] = 0x7F
        c.view(torch.uint8)[[0, 1, 3, 4]] = 0xFF
    ks[[0, 1, 3, 4]] = float("nan")
    assert bits_equal(attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([45]), 128), clean)


@pytest.mark.parametrize("lens,Hq,Hkv,Sq,top", [([1, 0, 0, 2, 0], 4, 1, 1, 20000), ([0] * 300 + [1, 64, 65, 5000] + [0] * 9, 2, 1, 1, 9000),
                                               ([3000] + [1] * 130 + [129], 8, 8, 1, 40000), ([200, 70, 0, 64], 256, 256, 1, 9000),
                                               ([777, 64], 512, 256, 16, 9000), ([6000, 5, 6001], 32, 2, 16, 9000),
                                               ([300, 64, 0], 1024, 1024, 1, 9000), ([130, 1], 1024, 64, 16, 9000)])
def test_attend_shares(lens, Hq, Hkv, Sq, top):
    """Fewer keys than blocks, sequences without keys between others, heads that fill the machine by themselves."""
    _check_attend(lens, 16, Hq, Hkv, 64, Sq, "int8", torch.float16, top=top, width=-(-top // 16))


@pytest.mark.parametrize("lens,Sq,top", [([700, 64, 2000, 1, 1300] * 13, 1, 9000), ([40000], 2, 40000), ([90, 300], 3, 512)])
def test_attend_gives_the_same_bits_again(lens, Sq, top):
    """Clusters' and blocks' parts are added up in one order, whoever is first."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    q, kc, vc, ks, vs, table, out = _check_attend(lens, 32, 14, 2, 128, Sq, "e4m3", torch.bfloat16, rotary=False, top=top, width=-(-top // 32))
    for _ in range(5):
        assert bits_equal(attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), top), out)


def test_attend_many_sequences():
    """So many sequences that their keys, laid end to end, pass what 32-bit products hold; all of them share the same pages."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(17)
    B, n = 60000, 1900
    kc, vc, ks, vs = _cache(g, "int8", 119, 1, 16, 64)
    table = torch.randperm(119, generator=g, device="cuda").int().expand(B, 119)[:, :119]
    table = table.contiguous()
    lens = torch.randint(1, n + 1, (B,), generator=g, device="cuda").int()
    lens[::3] = n
    lens[[5, 4000, B - 2]] = 0
    q = torch.randn(B, 2, 64, generator=g, device="cuda").half()
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, lens, 9000)
    some = torch.cat([torch.arange(0, B, 997, device="cuda"), torch.tensor([5, 4000, B - 2, B - 1], device="cuda")])
    want = _attend(q[some][:, None], kc, vc, ks, vs, table[some], lens[some].tolist(), 9000, 0.0, None, None)[:, 0]
    assert rel_fro(out[some], want) < 2.0 ** -11 + 2.0 ** -16 and (out[[5, 4000, B - 2]] == 0).all()
    # (what a call of a part of them gives, whose blocks cut the sequences elsewhere: each off by its own rounding, 2^-11)
    parts = torch.cat([attn_decode_kv8(q[i:i + 7000], kc, vc, ks, vs, table[i:i + 7000], lens[i:i + 7000], n) for i in range(0, B, 7000)])
    assert rel_fro(out, parts) < 2 * (2.0 ** -11 + 2.0 ** -16)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 1), (16, 2), (24, 2)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_attend_keeps_nan_with_the_rows_that_see_it(d, Hq, Hkv, dt):
    """A NaN in a later token's value or key is not seen by the earlier ones; a NaN in a query stays in its row."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(15)
    kc, vc, ks, vs = _cache(g, "e4m3", 8, Hkv, 16, d)
    q = torch.randn(2, 4, Hq, d, generator=g, device="cuda").to(DT[dt])
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = [40, 63]
    clean = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), 64)
    vc.view(torch.uint8)[2, 0, 6, 5] = 0x7F                   # sequence 0's key 38: its last two tokens see it
    kc.view(torch.uint8)[7, Hkv - 1, 14, 3] = 0xFF            # sequence 1's key 62: the last token alone
    q[1, 0, 1, 7] = float("nan")
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), 64)
    bad = torch.zeros_like(out, dtype=torch.bool)
    rep = Hq // Hkv
    bad[0, 2:, :rep, 5] = True
    bad[1, 3, -rep:] = True
    bad[1, 0, 1] = True
    assert torch.isnan(out[bad]).all() and bits_equal(torch.where(bad, torch.zeros_like(out), out), torch.where(bad, torch.zeros_like(out), clean))


def test_attend_keeps_a_bad_scale_with_the_rows_that_see_it():
    """A page whose scales are NaN and that only the last token sees."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(16)
    kc, vc, ks, vs = _cache(g, "int8", 4, 2, 16, 64)
    q = torch.randn(1, 3, 8, 64, generator=g, device="cuda").half()
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    clean = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([49]), 64)
    ks[3], vs[3] = float("nan"), float("nan")
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([49]), 64)
    assert torch.isnan(out[0, 2]).all() and bits_equal(out[0, :2], clean[0, :2])


def test_attend_beyond_32_bits():
    """A cache whose pages lie more than 2^32 bytes apart."""
    from llmqrt_b200.paged_cache import attn_decode_kv8, kv8_append
    g = _gen(13)
    P, Hkv, page, d = 5 * 2 ** 30 // (4 * 128 * 128) + 3, 4, 128, 128
    kc, vc = (torch.empty(P, Hkv, page, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(P, Hkv, device="cuda") for _ in range(2))
    ids = [P - 1, 1, P - 2]
    x = torch.randn(300, 2, Hkv, d, generator=g, device="cuda").half()
    slots = torch.tensor([ids[i // page] * page + i % page for i in range(300)], device="cuda")
    kv8_append(kc, vc, ks, vs, x[:, 0], x[:, 1], slots)
    q, table = torch.randn(1, 28, d, generator=g, device="cuda").half(), _i32([ids])
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([300]), 300)
    small = [t[torch.tensor(ids, device="cuda")] for t in (kc, vc, ks, vs)]
    want = _attend(q[:, None], *small, _i32([[0, 1, 2]]), [300], 300, 0.0, None, None)[:, 0]
    assert rel_fro(out, want) < 2.0 ** -11 + 2.0 ** -16
    got = (small[0].double() * small[2][:, :, None, None]).transpose(1, 2).reshape(-1, Hkv, d)[:300]
    assert ((got - x[:, 0].double()).abs() <= 0.5001 * small[2].repeat_interleave(page, 0)[:300, :, None]).all()


def test_views_of_a_cache():
    """A cache that is a view: every other page, heads of a wider one."""
    from llmqrt_b200.paged_cache import attn_decode_kv8, kv8_append
    g = _gen(14)
    big = [torch.zeros(12, 5, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    view = [t[::2, 1:3] for t in big]
    flat = [torch.zeros(6, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
    x = torch.randn(40, 2, 2, 64, generator=g, device="cuda").half()
    slots = torch.tensor([s + (32 if s >= 16 else 0) for s in range(3, 43)], device="cuda")
    q, table = torch.randn(1, 4, 64, generator=g, device="cuda").half(), _i32([[0, 3, 4]])
    outs = []
    for kc, vc in (view, flat):
        ks, vs = (torch.ones(6, 2, device="cuda") for _ in range(2))
        kv8_append(kc, vc, ks, vs, x[:, 0], x[:, 1], slots)
        outs.append(attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([43]), 48))
    assert bits_equal(outs[0], outs[1]) and all(bits_equal(a.contiguous(), b) for a, b in zip(view, flat))
    assert not any(t[1::2].any() or t[:, :1].any() or t[:, 3:].any() for t in big)


# ---- together ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(kind, graph):
    """Prompts, then steps of one token with requests that come and go, against attention over what the cache stands for
    and over what was put in; the decode step as it is captured and replayed."""
    from llmqrt_b200 import glue
    from llmqrt_b200.paged_cache import PagedKVCache8
    B, Hq, Hkv, d, page, layers = 5, 8, 2, 64, 16, 2
    g = _gen(21)
    cache = PagedKVCache8(layers, 60, page, Hkv, d, B, 200, "cuda", CACHE[kind])
    cos, sin = glue.rope_tables(d, 200, 1e4, "cuda")
    told = [[torch.zeros(0, Hkv, d, dtype=torch.float64, device="cuda") for _ in range(B)] for _ in range(2 * layers)]
    lens = [0] * B

    def record(new, kv):
        n = 0
        for b, m in enumerate(new):
            for layer in range(layers):
                k, v = (kv[layer][n:n + m, i].double() for i in range(2))
                pos = torch.arange(lens[b], lens[b] + m, device="cuda")
                c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
                lo, hi = k.chunk(2, -1)
                k = torch.cat([lo * c - hi * s, lo * s + hi * c], -1)
                told[2 * layer][b], told[2 * layer + 1][b] = torch.cat([told[2 * layer][b], k]), torch.cat([told[2 * layer + 1][b], v])
            lens[b] += m
            n += m

    def check(q, outs):
        for layer in range(layers):
            want = _attend(q[:, None], cache.k[layer], cache.v[layer], cache.k_scale[layer], cache.v_scale[layer], cache.block_table,
                           lens, 200, 0.0, cos, sin)[:, 0]
            assert rel_fro(outs[layer], want) < 2.0 ** -11 + 2.0 ** -16
            for b in range(B):                                   # and what was put in: codes are off by at most 2^-4 (e4m3), 1/254 (int8; twice requantized 3/254)
                if not lens[b]:
                    assert (outs[layer][b] == 0).all()
                    continue
                kk, vv = (c[cache.block_table[b, : -(-lens[b] // page)].long()].float() for c in (cache.k[layer], cache.v[layer]))
                for codes, scale, put in ((kk, cache.k_scale, told[2 * layer][b]), (vv, cache.v_scale, told[2 * layer + 1][b])):
                    s = scale[layer][cache.block_table[b, : -(-lens[b] // page)].long()]
                    got = (codes * s[:, :, None, None]).transpose(1, 2).reshape(-1, Hkv, d)[:lens[b]].double()
                    step = s.repeat_interleave(page, 0)[:lens[b], :, None].double()
                    assert ((got - put).abs() <= (put.abs() * 2.0 ** -4 + step * 2.0 ** -9 if kind == "e4m3" else step * 0.5 * page)).all()

    prompt = [20, 0, 33, 1, 16]
    T = sum(prompt) + 6                                          # (a padded batch: the last tokens have no slot)
    kv = [torch.randn(T, 2, Hkv, d, generator=g, device="cuda").half() for _ in range(layers)]
    step = cache.plan(_i32(prompt), T)
    for layer in range(layers):
        cache.append(layer, kv[layer][:, 0], kv[layer][:, 1], step, cos, sin)
    record(prompt, kv)
    assert cache.seq_lens.tolist() == lens and step.cu_new.tolist() == [0, 20, 20, 53, 54, 70]

    new, q = _i32([0] * B), torch.zeros(B, Hq, d, dtype=torch.float16, device="cuda")
    kv = [torch.zeros(B, 2, Hkv, d, dtype=torch.float16, device="cuda") for _ in range(layers)]

    def decode():
        step = cache.plan(new, B)
        outs = []
        for layer in range(layers):
            cache.append(layer, kv[layer][:, 0], kv[layer][:, 1], step, cos, sin)
            outs.append(cache.attend(layer, q, cos=cos, sin=sin))
        return outs

    run = decode
    if graph:
        saved = [t.clone() for t in (cache.seq_lens, cache.free_count, cache.block_table)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode()
        torch.cuda.current_stream().wait_stream(side)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            held = decode()
        for t, s in zip((cache.seq_lens, cache.free_count, cache.block_table), saved):
            t.copy_(s)

        def run():
            cg.replay()
            return held

    for i in range(20):
        live = [1, int(i > 3), int(i % 5 > 0), 1, int(i < 9)]
        new.copy_(_i32(live))
        q.copy_(torch.randn(B, Hq, d, generator=g, device="cuda"))
        for t in kv:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        outs = run()
        record(live, kv)
        assert cache.seq_lens.tolist() == lens
        check(q, outs)
        if i == 12:
            cache.release(torch.tensor([False, False, True, False, True], device="cuda"))
            for b in (2, 4):
                lens[b] = 0
                for t in told:
                    t[b] = t[b][:0]
    used = cache.block_table[cache.block_table >= 0]
    live_pages = torch.cat([cache.block_table[b, : -(-lens[b] // page)] for b in range(B)])
    assert live_pages.unique().numel() == live_pages.numel() and used.numel() > 0
    assert int(cache.free_count) + live_pages.numel() == 60
    rest = torch.cat([live_pages, cache.free_pages[: int(cache.free_count)]])
    assert rest.sort().values.tolist() == list(range(60))


def test_runs_on_the_current_stream():
    from llmqrt_b200.paged_cache import attn_decode_kv8, kv8_append
    g = _gen(31)
    kc, vc, ks, vs = _cache(g, "int8", 40, 2, 16, 64)
    x, q = torch.randn(600, 2, 2, 64, generator=g, device="cuda").half(), torch.randn(1, 4, 64, generator=g, device="cuda").half()
    slots, table = torch.arange(600, device="cuda"), torch.arange(38, dtype=torch.int32, device="cuda")[None]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        x2 = x * 1.0
        kv8_append(kc, vc, ks, vs, x2[:, 0], x2[:, 1], slots)
        out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([600]), 608)
    torch.cuda.current_stream().wait_stream(side)
    assert rel_fro(out, _attend(q[:, None], kc, vc, ks, vs, table, [600], 608, 0.0, None, None)[:, 0]) < 2.0 ** -11 + 2.0 ** -16


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("top", [112, 9000])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_attend_scores_far_below_zero(d, top, kind):
    """Scores of -1e31 and less: the greatest of them gets the weight all the same."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(19)
    kc, vc, ks, vs = _cache(g, kind, 7, 2, 16, d)
    codes = torch.randint(2, 16, (7, 2, 16, 1), generator=g, device="cuda").expand(7, 2, 16, d)
    kc.copy_(-codes.float())
    kc[4, 0, 5], kc[1, 1, 15] = -1.0, -1.0
    ks[:] = 1e13
    q = torch.full((1, 2, d), 1e18, device="cuda").bfloat16()
    table = torch.full((1, -(-top // 16)), -1, dtype=torch.int32, device="cuda")
    table[0, :7] = torch.arange(7)
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([105]), top)
    want = torch.stack([vc[4, 0, 5].float() * vs[4, 0], vc[1, 1, 15].float() * vs[1, 1]])
    # (one weight of 1: the result's own rounding, 2^-8)
    assert ((out[0].float() - want).abs() <= want.abs() * 2.0 ** -8).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_greatest_values(kind):
    """bf16's greatest numbers are finite ones: within half a step of their codes."""
    from llmqrt_b200.paged_cache import kv8_append
    top = torch.finfo(torch.bfloat16).max
    x = torch.linspace(-1, 1, 64, device="cuda").mul(top).bfloat16().clamp(-top, top)[None, None]
    kc, vc = (torch.zeros(1, 1, 16, 64, dtype=torch.int8, device="cuda").view(CACHE[kind]) for _ in range(2))
    ks, vs = (torch.zeros(1, 1, device="cuda") for _ in range(2))
    kv8_append(kc, vc, ks, vs, x, x, torch.tensor([0], device="cuda"))
    want = x[0, 0].double()
    for codes, s in ((kc, ks), (vc, vs)):
        got = codes[0, 0, 0].float().double() * s.double()[0, 0]
        # (half a step: 2^-4 of an e4m3 value, 1/254 of the greatest int8 one; three fp32 roundings, 2^-24 each)
        tol = want.abs() * 2.0 ** -4 + 2.0 ** -10 * s.double() if kind == "e4m3" else torch.full_like(want, top / 254)
        assert ((got - want).abs() <= tol + 3 * 2.0 ** -24 * top).all()


@pytest.mark.parametrize("lens,Hq,Hkv,Sq,d", [([10000], 1024, 1024, 1, 64), ([14000, 30, 0], 1024, 1024, 1, 128), ([24000], 1024, 512, 4, 128),
                                              ([12000], 1024, 64, 16, 64), ([9000, 4097], 1024, 64, 16, 128), ([30000, 5], 512, 32, 16, 64)])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_attend_shares_longer_than_a_span(lens, Hq, Hkv, Sq, d, kind, dt):
    """So many heads that a block takes more than 4096 keys of a sequence, whose page numbers and scales it fetches again and again: each
    row against the definition."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    rows = Sq * Hq // Hkv
    columns = Hkv * (-(-rows // 16) if rows > 8 else 1)
    # (four blocks an SM and four waves of them, the most there are: the keys of a block's share, less what beginning sequences counts)
    blocks = 4 * 4 * torch.cuda.get_device_properties(0).multi_processor_count // columns
    assert sum(lens) // blocks > 4096 + 640 * len(lens)
    g = _gen(max(lens) + Hkv)
    P = sum(-(-n // 32) for n in lens) + 1
    kc, vc, ks, vs = _cache(g, kind, P, Hkv, 32, d)
    table = _tables(g, lens, 32, 1000, P)
    q = torch.randn(len(lens), Sq, Hq, d, generator=g, device="cuda").to(DT[dt])
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32(lens), 32000)
    assert torch.isfinite(out).all()
    # the result's rounding (and bf16's P in fp16), and a warp's sums of up to 24000 / 64 steps of two roundings each, 2^-23 as tensor cores cut
    # off: 2^-13.4 of a row at most
    tol = (2.0 ** -11 if dt == "fp16" else 2.0 ** -8 + 2.0 ** -11) + 2.0 ** -13.4
    for h in range(0, Hq, 128):                                  # (some heads at a time: 64 bits take room)
        k0, k1 = h * Hkv // Hq, (h + 128) * Hkv // Hq
        want = _attend(q[:, :, h:h + 128], kc[:, k0:k1], vc[:, k0:k1], ks[:, k0:k1], vs[:, k0:k1], table, lens, 32000, 0.0, None, None)
        assert ((out[:, :, h:h + 128].double() - want).norm(dim=-1) <= tol * want.norm(dim=-1)).all()
