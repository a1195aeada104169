"""Attention over a paged 8-bit cache whose pages' value scales lie far apart, against the formula in 64 bits, row by row: a page's
scale is for the rows that see it and for the products of its own keys alone."""
import math

import pytest
import torch

from tests.test_gpu_paged_cache import CACHE, DT, _attend, _cache, _gen, _i32

pytestmark = pytest.mark.gpu

# fp16: the result's rounding alone (P and Q keep 22 bits) and 2^-16 for the fp32 arithmetic; bf16, Q not rotated and so exact in
# fp16: the result's 2^-8 and P's 2^-11.  Each holds element by element of P and of the result, hence for each row's norm.
TOL = {"fp16": 2.0 ** -11 + 2.0 ** -16, "bf16": 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16}


def _off(out, want):
    """The greatest relative error of a row's norm."""
    assert torch.isfinite(out).all()
    return float(((out.double() - want).norm(dim=-1) / want.norm(dim=-1)).max())


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), 2.0 ** 100, -2.0 ** 100, float("nan")])
@pytest.mark.parametrize("d,Hq,Hkv", [(64, 2, 1), (128, 4, 2), (64, 24, 2), (128, 16, 1)])
@pytest.mark.parametrize("top", [64, 9000])                      # (parts merged by a cluster, and shared out to all blocks)
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_a_scale_stays_with_the_rows_that_see_it(scale, d, Hq, Hkv, top, kind, dt):
    """The last page is seen by the last of three tokens alone."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(16)
    kc, vc, ks, vs = _cache(g, kind, 4, Hkv, 16, d)
    q = torch.randn(1, 3, Hq, d, generator=g, device="cuda").to(DT[dt])
    table = torch.full((1, -(-top // 16)), -1, dtype=torch.int32, device="cuda")
    table[0, :4] = torch.arange(4)
    vs[3] = scale
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([49]), top)
    clean = vs.clone()
    clean[3] = 1.0
    want = _attend(q, kc, vc, ks, clean, table, [49], top, 0.0, None, None)
    assert _off(out[:, :2], want[:, :2]) < TOL[dt]
    if math.isfinite(scale) and dt == "bf16":
        assert _off(out, _attend(q, kc, vc, ks, vs, table, [49], top, 0.0, None, None)) < TOL[dt]
    elif not math.isfinite(scale):
        assert not torch.isfinite(out[0, 2]).any()


@pytest.mark.parametrize("d,Hq,Hkv", [(64, 2, 1), (128, 4, 2), (64, 24, 2), (128, 16, 1)])
@pytest.mark.parametrize("scale", [2.0 ** -30, 2.0 ** 60])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_nan_on_a_page_of_distant_scale(d, Hq, Hkv, scale, dt):
    """A NaN among the values of a page whose scale is far from the others': for the rows that see its key, not for those that see others of its page."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(17)
    kc, vc, ks, vs = _cache(g, "e4m3", 8, Hkv, 16, d)
    q = torch.randn(1, 3, Hq, d, generator=g, device="cuda").to(DT[dt])
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    vs[7] = scale
    if scale > 1:                                                # (its values are zeros)
        vc.view(torch.uint8)[7] = 0
    want = _attend(q, kc, vc, ks, vs, table, [116], 128, 0.0, None, None)
    vc.view(torch.uint8)[7, 0, 3, 5] = 0x7F                      # key 115, the last
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([116]), 128)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 2, : Hq // Hkv, 5] = True
    assert torch.isnan(out[bad]).all()
    assert _off(torch.where(bad, torch.zeros_like(out), out), torch.where(bad, torch.zeros_like(want), want)) < TOL[dt]


@pytest.mark.parametrize("d,Hq,Hkv", [(64, 4, 2), (128, 24, 2)])
@pytest.mark.parametrize("top", [2048, 9000])                    # (a warp takes several pages)
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_an_infinity_stays_in_its_column(d, Hq, Hkv, top, kind, dt):
    """An infinity among the values that are written makes its page's scale as great as it goes; the other columns of later queries keep
    what the other pages hold."""
    from llmqrt_b200.paged_cache import attn_decode_kv8, kv8_append
    g = _gen(23)
    T, P = 1100, 69
    kc, vc, ks, vs = _cache(g, kind, P, Hkv, 16, d)
    x = torch.randn(T, 2, Hkv, d, generator=g, device="cuda").to(DT[dt])
    x[37, 1, 1, 5] = float("inf")
    kv8_append(kc, vc, ks, vs, x[:, 0], x[:, 1], torch.arange(T, device="cuda"))
    q = torch.randn(1, 1, Hq, d, generator=g, device="cuda").to(DT[dt])
    table = torch.full((1, -(-top // 16)), -1, dtype=torch.int32, device="cuda")
    table[0, :P] = torch.arange(P)
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([T]), top)
    want = _attend(q, kc, vc, ks, vs, table, [T], top, 0.0, None, None)
    there, rest = out[0, 0, Hq // Hkv:, 5].clone(), want[0, 0, Hq // Hkv:, 5].clone()
    out[0, 0, Hq // Hkv:, 5], want[0, 0, Hq // Hkv:, 5] = 0, 0
    assert _off(out, want) < TOL[dt]
    if dt == "fp16":
        assert (there == float("inf")).all()
    else:
        assert ((there.double() - rest).abs() <= TOL[dt] * rest).all()


@pytest.mark.parametrize("apart", [0, 7, 8, 9, 15, 24, 40, 60, 90])
@pytest.mark.parametrize("great", ["first", "between", "last"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_weight_on_pages_of_small_scale(apart, great, d, kind, dt):
    """Pages whose value scale is 2^apart times the others', whose keys get a weight so small that they hardly count."""
    from llmqrt_b200.paged_cache import attn_decode_kv8
    g = _gen(31)
    P, page = 128, 16                                            # (a cluster of eight blocks: a warp has every fourth page of sixteen neighbours)
    kc, vc, ks, vs = _cache(g, kind, P, 2, page, d)
    q = torch.randn(1, 1, 2, d, generator=g, device="cuda").to(DT[dt])
    vs[:] = 2.0 ** -8
    at = {"first": 0, "between": 4, "last": 12}[great]
    ids = [i for i in range(P) if at <= i % 16 < at + 4]
    vs[ids] = 2.0 ** (apart - 8)
    # keys of these pages (a quarter of all) point away from the query: a score of -(12 + apart ln 2), against a few of the other pages'
    ks[:] = 2.0 ** -8
    for h in range(2):
        away = -(12 + apart * math.log(2)) * math.sqrt(d) * q[0, 0, h].float() / q[0, 0, h].float().square().sum()
        top = float(away.abs().max())
        ks[ids, h] = top / 100
        codes = away / (top / 100)
        kc[ids, h] = (codes.round().to(torch.int8) if kind == "int8" else codes.to(torch.float8_e4m3fn)).expand(len(ids), page, d)
    table = torch.arange(P, dtype=torch.int32, device="cuda")[None]
    out = attn_decode_kv8(q, kc, vc, ks, vs, table, _i32([P * page - 3]), P * page)
    want = _attend(q, kc, vc, ks, vs, table, [P * page - 3], P * page, 0.0, None, None)
    # (scores of up to 12 + 62 in fp32: 2^-24 of them, ten roundings, is what moves the small weights; those count by e^-12 at most)
    assert _off(out, want) < TOL[dt]
