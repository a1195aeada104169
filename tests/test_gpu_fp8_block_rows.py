"""e4m3 activations with a scale for each token and 128 features: the quantizer and the RMS norm ahead of it, against the
definition in 64 bits."""
import pytest
import torch

from tests.util import bits_equal

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _e4m3(x):
    m, e = torch.frexp(x.clamp(-448, 448))
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)
    return (x.clamp(-448, 448) / step).round() * step


def _groups(y):
    """y [M, K] (64 bits) -> codes before rounding, scales."""
    M, K = y.shape
    G = -(-K // 128)
    pad = torch.zeros(M, G * 128, dtype=y.dtype, device=y.device)
    pad[:, :K] = y
    scale = pad.view(M, G, 128).abs().amax(2).clamp_min(1e-12) / 448
    return (pad.view(M, G, 128) / scale[:, :, None]).view(M, G * 128)[:, :K], scale


def _check(q, scale, y, roundings):
    """roundings: how many fp32 ones, of 2^-24 each, stand between the definition's values and the codes."""
    code, s = _groups(y)
    assert q.dtype == F8 and q.shape == y.shape and scale.dtype == torch.float32 and scale.shape == s.shape
    assert ((scale.double() - s).abs() <= (roundings + 4) * 2.0 ** -24 * s).all()
    got = q.float().double()
    # a code rounds to the nearest of what lies within those roundings of the definition's value
    lo, hi = (_e4m3(code * (1 + f * roundings * 2.0 ** -24)) for f in (-1, 1))
    assert ((got - lo) * (got - hi) <= 0).all()


@pytest.mark.parametrize("M,K", [(1, 8), (1, 128), (3, 136), (5, 896), (17, 120), (333, 1536), (2, 18944), (4096, 1000), (0, 256)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_quantize(M, K, dt):
    from llmqrt_b200.ops import quantize_fp8_block
    g = torch.Generator(device="cuda").manual_seed(M + K)
    wide = (torch.randn(M, K + 24, generator=g, device="cuda") * 3).to(DT[dt])
    for x in (wide[:, 8:8 + K], wide[:, 8:8 + K].contiguous(), wide[:, 3:3 + K]):      # rows of a wider matrix, of their own, misaligned
        q, scale = quantize_fp8_block(x)
        _check(q, scale, x.double(), 3)
    y = wide[:, :K].contiguous().view(1, M, K) if M else wide[:, :K].contiguous()
    assert bits_equal(quantize_fp8_block(y)[0], quantize_fp8_block(y.reshape(M, K))[0])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_quantize_special_values(dt):
    from llmqrt_b200.ops import quantize_fp8_block
    x = torch.zeros(4, 256, dtype=DT[dt], device="cuda")
    x[1, 3], x[1, 200] = float("nan"), 5.0
    x[1, 5] = 2.0
    x[2, :] = torch.finfo(DT[dt]).tiny
    x[3, 7], x[3, 8] = float("inf"), 1.0
    q, s = quantize_fp8_block(x)
    v = q.float()
    assert (v[0] == 0).all() and torch.isfinite(s[0]).all() and (s[0] > 0).all()
    assert v[1, 3].isnan() and v[1, 5] == 448 and v[1, 200] == 448 and not v[1, 4].isnan() and abs(s[1, 0] - 2 / 448) < 1e-8
    _check(q[2:3], s[2:3], x[2:3].double(), 3)
    assert (v[3, :128] * s[3, 0])[7].isnan() and torch.isfinite(v[3, 128:] * s[3, 1]).all()


@pytest.mark.parametrize("M,H", [(1, 8), (1, 128), (2, 136), (64, 896), (333, 1536), (64, 3584), (700, 3584), (5, 8200), (300, 16384), (7, 32768),
                                 (0, 128)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("residual", [True, False])
def test_rmsnorm(M, H, dt, residual):
    from llmqrt_b200.glue import rmsnorm_fp8_block
    g = torch.Generator(device="cuda").manual_seed(M + H)
    wide = torch.randn(M, 2 * H + 16, generator=g, device="cuda").to(DT[dt])
    x, r = wide[:, 8:8 + H], wide[:, 8 + H:8 + 2 * H]
    w = (1 + 0.3 * torch.randn(H, generator=g, device="cuda")).to(DT[dt])
    q, scale, h = rmsnorm_fp8_block(x, w, 1e-6, r if residual else None)
    want = x
    if residual:
        want = (x.float() + r.float()).to(DT[dt])
        assert bits_equal(h, want)
    else:
        assert h is None
    y = want.double()
    if M:
        y = y * w.double() / (y.square().mean(1, keepdim=True) + 1e-6).sqrt()
    # codes: the group's factor and the product; scales: the mean (a butterfly over 32 after at most 8 * 8 sums), root, products
    code, s = _groups(y)
    assert ((scale.double() - s).abs() <= (8 + 5 + 8 + 6) * 2.0 ** -24 * s).all()
    got = q.float().double()
    lo, hi = (_e4m3(code * (1 + f * 3 * 2.0 ** -24)) for f in (-1, 1))
    assert ((got - lo) * (got - hi) <= 0).all()
    # every row has the same bits alone
    for m in {0, M // 2, M - 1} if M else ():
        q1, s1, _ = rmsnorm_fp8_block(x[m:m + 1], w, 1e-6, r[m:m + 1] if residual else None)
        assert bits_equal(q1[0], q[m]) and torch.equal(s1[0], scale[m])


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_rmsnorm_special_values(dt):
    from llmqrt_b200.glue import rmsnorm_fp8_block
    x = torch.ones(4, 256, dtype=DT[dt], device="cuda")
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 130] = float("inf")
    w = torch.ones(256, dtype=DT[dt], device="cuda")
    w[128:] = 0
    q, s, _ = rmsnorm_fp8_block(x, w, 1e-6)
    v = q.float() * s.repeat_interleave(128, 1)
    assert (v[0] == 0).all() and v[1, :128].isnan().all() and v[2, 130].isnan()
    assert (v[3, 128:] == 0).all() and ((v[3, :128] - 1).abs() < 2e-3).all()
    tiny = torch.full((1, 128), 1e-4, dtype=DT[dt], device="cuda")     # a group of less than the scale's floor
    q, s, _ = rmsnorm_fp8_block(tiny, torch.full((128,), 1e-7 if dt == "fp16" else 1e-9, dtype=DT[dt], device="cuda"), 1e12)
    assert torch.allclose(s, torch.tensor([[1e-12 / 448]], device="cuda")) and torch.isfinite(q.float()).all()


def test_rows_refuse():
    from llmqrt_b200 import glue, ops
    x = torch.ones(2, 128, device="cuda").half()
    for bad, error in ((x[:, :12], RuntimeError), (x.float(), RuntimeError), (x.int(), TypeError), (torch.ones(2, 40000, device="cuda").half(), RuntimeError),
                       (x.cpu(), RuntimeError)):
        with pytest.raises(error):
            ops.quantize_fp8_block(bad)
        with pytest.raises((error, TypeError)):
            glue.rmsnorm_fp8_block(bad, torch.ones(bad.shape[-1], dtype=bad.dtype, device=bad.device), 1e-6)
    with pytest.raises(RuntimeError):
        glue.rmsnorm_fp8_block(x, x[0, :64], 1e-6)
    with pytest.raises(RuntimeError):
        glue.rmsnorm_fp8_block(x, x[0], 1e-6, x[:1])
    with pytest.raises(TypeError):
        glue.rmsnorm_fp8_block(x, x[0].float(), 1e-6)


@pytest.mark.parametrize("M,K", [(4096, 3584), (4097, 3584), (10000, 1000), (1300, 8200), (300, 32768), (600, 18944), (100000, 136)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_quantize_many_rows(M, K, dt):
    """So many features that a thread takes four units of them: the bits of the same rows a few at a time, and the definition's codes."""
    from llmqrt_b200.ops import quantize_fp8_block
    g = torch.Generator(device="cuda").manual_seed(M + K)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.logspace(-3, 3, M, device="cuda")[:, None]).to(DT[dt])
    x[M // 2] = 0
    x[M // 3, K // 2:] = float("inf")
    x[M // 3, 0] = float("nan")
    assert M * K // 8 >= torch.cuda.get_device_properties(0).multi_processor_count * 2048 * 4
    q, scale = quantize_fp8_block(x)
    rows = torch.cat([torch.arange(0, 70), torch.arange(M // 3 - 9, M // 3 + 9), torch.arange(M // 2 - 9, M // 2 + 9), torch.arange(M - 70, M)]).unique().cuda()
    few = quantize_fp8_block(x[rows])
    assert bits_equal(q[rows], few[0]) and bits_equal(scale[rows], few[1])
    ok = torch.arange(M, device="cuda") != M // 3
    for part in torch.arange(M, device="cuda")[ok].split(20_000_000 // K):
        _check(q[part], scale[part], x[part].double(), 3)
