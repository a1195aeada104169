"""FP8 linear layers with a scale for each block of 128, against the definition in 64 bits."""
import pytest
import torch

from tests.util import bits_equal

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _inputs(M, N, K, g, bias_dtype=None):
    kb, nb = -(-K // 128), -(-N // 128)
    a = (torch.randn(M, K, generator=g, device="cuda") * 60).clamp(-448, 448).to(F8)
    w = (torch.randn(N, K, generator=g, device="cuda") * 60).clamp(-448, 448).to(F8)
    a_s = torch.rand(M, kb, generator=g, device="cuda") * 3e-3 + 1e-3
    w_s = torch.exp2(torch.randn(nb, kb, generator=g, device="cuda") * 2) * 1e-4      # blocks of very different sizes
    bias = torch.randn(N, generator=g, device="cuda").to(bias_dtype) if bias_dtype else None
    return a, w, bias, a_s, w_s


def _reference(a, w, bias, a_s, w_s):
    """(value, sum of magnitudes) in 64 bits."""
    M, K = a.shape
    N = w.shape[0]
    y, mag = (torch.zeros(M, N, dtype=torch.float64, device="cuda") for _ in range(2))
    nb = torch.arange(N, device="cuda") // 128
    for i in range(-(-K // 128)):
        x, v = a[:, 128 * i:128 * i + 128].double(), w[:, 128 * i:128 * i + 128].double()
        f = a_s[:, i:i + 1].double() * w_s[nb, i].double()
        y += (x @ v.t()) * f
        mag += (x.abs() @ v.abs().t()) * f
    if bias is not None:
        y += bias.double()
        mag += bias.double().abs()
    return y, mag


def _check(out, a, w, bias, a_s, w_s):
    y, mag = _reference(a, w, bias, a_s, w_s)
    # the result's rounding (half a step), and fp32 sums of 128 products, of the blocks' scaled sums and the bias
    adds = 128 + 3 * a_s.shape[1] + 2
    tol = y.abs() * (torch.finfo(out.dtype).eps / 2) * 1.001 + adds * 2.0 ** -24 * mag + 2.0 ** -25
    assert out.shape == y.shape and ((out.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("M", [1, 7, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256, 300, 700])
@pytest.mark.parametrize("N,K", [(16, 16), (128, 128), (130, 144), (333, 1040), (896, 4864), (4864, 896), (257, 2064), (3584, 3584)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_linear(M, N, K, dt):
    from llmqrt_b200 import _lib, ops
    g = torch.Generator(device="cuda").manual_seed(M * 7 + N + K)
    bias_dtype = {0: None, 1: DT[dt], 2: torch.float32}[(M + N) % 3]
    args = _inputs(M, N, K, g, bias_dtype)
    out = ops.fp8_linear_block(*args, DT[dt])
    assert out.dtype == DT[dt]
    _check(out, *args)
    assert bits_equal(out, ops.fp8_linear_block(*args, DT[dt], static_weight=True))       # and the same bits again
    assert _lib.kernel_status(out.device) == 0


@pytest.mark.parametrize("M,N,K", [(64, 37888, 3584), (1, 18944, 3584), (4096, 1000, 2000), (2500, 4864, 896), (1100, 897, 18944), (5000, 8, 128)])
def test_large(M, N, K):
    from llmqrt_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(M + N)
    args = _inputs(M, N, K, g, torch.bfloat16)
    _check(ops.fp8_linear_block(*args, torch.bfloat16), *args)


@pytest.mark.parametrize("M,N,K", [(33, 37000, 272), (64, 37888, 384), (64, 19072, 1024), (48, 37761, 16), (50, 56000, 144)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_wide_layers_of_few_tokens(M, N, K, dt):
    """More tiles of weight rows than SMs, an odd number of them among these."""
    from llmqrt_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(M * N + K)
    args = _inputs(M, N, K, g, DT[dt])
    _check(ops.fp8_linear_block(*args, DT[dt]), *args)


@pytest.mark.parametrize("M", [1, 50, 130, 600])
@pytest.mark.parametrize("N,pad", [(200, 8), (200, 3), (129, 1)])
def test_rows_of_wider_matrices(M, N, pad):
    """Operands whose rows lie in wider matrices; an output whose pitch is wider than it: nothing else is written."""
    from llmqrt_b200 import _lib as L
    from llmqrt_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(M + N)
    a, w, bias, a_s, w_s = _inputs(M, N, 400, g)
    want = ops.fp8_linear_block(a, w, bias, a_s, w_s, torch.float16)
    wide = [torch.full((t.shape[0], 640), 3.0, device="cuda").to(F8) for t in (a, w)]
    for t, v in zip(wide, (a, w)):
        t[:, 32:432] = v
    assert bits_equal(ops.fp8_linear_block(wide[0][:, 32:432], wide[1][:, 32:432], bias, a_s, w_s, torch.float16), want)
    odd = [torch.full((t.shape[0], 641), 3.0, device="cuda").to(F8) for t in (a, w)]        # rows that are not aligned: copied
    for t, v in zip(odd, (a, w)):
        t[:, 5:405] = v
    assert bits_equal(ops.fp8_linear_block(odd[0][:, 5:405], odd[1][:, 5:405], bias, a_s, w_s, torch.float16), want)
    out = torch.full((M + 2, N + pad), -77.0, device="cuda", dtype=torch.float16)
    L.call("llmqrt_fp8_linear_block", L.ptr(a), a.stride(0), L.ptr(w), w.stride(0), None, 0, L.ptr(a_s), L.ptr(w_s), L.ptr(out[1]), L.F16,
           out.stride(0), M, N, 400, L.ptr(L.workspace(out.device)), L.stream(out.device), 0)
    assert bits_equal(out[1:M + 1, :N].contiguous(), want)
    assert (out[0] == -77).all() and (out[M + 1] == -77).all() and (out[:, N:] == -77).all()


def test_special_values():
    """A NaN or an infinite scale stays in its token's row, a zero scale silences a block."""
    from llmqrt_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    for M in (20, 200):
        a, w, bias, a_s, w_s = _inputs(M, 300, 512, g)
        a.view(torch.uint8)[3, 7] = 0x7F
        a_s[5, 1] = float("inf")
        w_s[:, 2] = 0
        out = ops.fp8_linear_block(a, w, bias, a_s, w_s, torch.bfloat16)
        assert out[3].isnan().all() and not torch.isfinite(out[5]).any()
        keep = [m for m in range(M) if m not in (3, 5)]
        _check(out[keep], a[keep], w, bias, a_s[keep], w_s)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("bias", [True, False])
def test_module(dt, M, bias):
    """FP8BlockLinear against the 16-bit layer it was made from, and against its own parts."""
    from llmqrt_b200 import ops
    from llmqrt_b200.linear import FP8BlockLinear, get_concrete_linear_module
    assert get_concrete_linear_module("fp8_block_quant") is FP8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(M)
    src = torch.nn.Linear(1040, 333, bias=bias, device="cuda", dtype=DT[dt])
    layer = FP8BlockLinear.from_linear(src, init_only=False, dtype=DT[dt])
    x = torch.randn(2, M, 1040, generator=g, device="cuda").to(DT[dt])
    y = layer(x)
    assert y.shape == (2, M, 333) and y.dtype == DT[dt]
    q, s = ops.quantize_fp8_block(x)
    assert bits_equal(layer.forward_quantized(q, s), y.view(-1, 333))
    _check(y.view(-1, 333), q, layer.weight.data, layer.bias.data if bias else None, s, layer.weight_scale.data)
    # a weight and an activation are off by at most 2^-4 of themselves: their product by twice that, and so their sums
    want = x.double() @ src.weight.double().t() + (src.bias.double() if bias else 0)
    assert (y.double() - want).norm() / want.norm() < 2 * 2.0 ** -4
    wq = layer.weight.data.float() * layer.weight_scale.data.repeat_interleave(128, 0)[:333].repeat_interleave(128, 1)[:, :1040]
    step = layer.weight_scale.data.repeat_interleave(128, 0)[:333].repeat_interleave(128, 1)[:, :1040]
    assert ((wq - src.weight.float()).abs() <= src.weight.float().abs() * 2.0 ** -4 * 1.01 + step * 2.0 ** -9).all()
    assert layer(x[:, :0]).shape == (2, 0, 333) and layer(x[0, 0]).shape == (333,)
    state = FP8BlockLinear(1040, 333, bias, dtype=DT[dt])
    state.load_state_dict(layer.state_dict())
    assert bits_equal(state(x), y)


def test_graph_and_stream():
    from llmqrt_b200.linear import FP8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(2)
    src = torch.nn.Linear(896, 640, device="cuda", dtype=torch.bfloat16)
    layer = FP8BlockLinear.from_linear(src, init_only=False)
    for M in (3, 60, 400):
        x = torch.randn(M, 896, generator=g, device="cuda").bfloat16()
        want = layer(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(10_000_000)
            y = layer(x * 1.0)
        torch.cuda.current_stream().wait_stream(side)
        assert bits_equal(y, want)
        held = torch.zeros_like(x)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            y = layer(held)
        for _ in range(2):
            held.copy_(x)
            cg.replay()
            assert bits_equal(y, want)
            held.zero_()


@pytest.mark.parametrize("M", [3, 80, 300])
def test_norm_into_linear(M):
    """The RMS norm's 8-bit output as the layer takes it, residual stream carried on."""
    from llmqrt_b200 import glue
    from llmqrt_b200.linear import FP8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(M)
    layer = FP8BlockLinear.from_linear(torch.nn.Linear(1536, 2048, device="cuda", dtype=torch.float16), init_only=False, dtype=torch.float16)
    x, r = (torch.randn(M, 1536, generator=g, device="cuda").half() for _ in range(2))
    w = torch.ones(1536, device="cuda").half()
    q, s, h = glue.rmsnorm_fp8_block(x, w, 1e-6, residual=r)
    y = layer.forward_quantized(q, s)
    _check(y, q, layer.weight.data, layer.bias.data, s, layer.weight_scale.data)
    n = h.double() / (h.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    plain = layer(n.half())                                   # normed in 64 bits, quantized by the layer: codes may round the other way
    assert (plain.double() - y.double()).norm() / y.double().norm() < 2.0 ** -4


@pytest.mark.parametrize("K", [32768, 32784, 53248])
@pytest.mark.parametrize("M", [1, 3, 700])
def test_module_of_many_inputs(M, K):
    """Layers of more inputs than one block of the quantizer takes: the codes are those of the row in pieces."""
    from llmqrt_b200 import ops
    from llmqrt_b200.linear import FP8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(K + M)
    layer = FP8BlockLinear(K, 200, True, dtype=torch.float16)
    a, w, bias, a_s, w_s = _inputs(1, 200, K, g, torch.float16)
    for p, v in ((layer.weight, w), (layer.weight_scale, w_s), (layer.bias, bias)):
        p.data.copy_(v)
    x = (torch.randn(M, K + 8, generator=g, device="cuda") * 1e-3).half()[:, :K]
    y = layer(x)
    pieces = [ops.quantize_fp8_block(x[:, i:i + 16384]) for i in range(0, K, 16384)]
    q, s = torch.cat([p[0].view(torch.uint8) for p in pieces], 1).view(F8), torch.cat([p[1] for p in pieces], 1)
    assert bits_equal(layer.forward_quantized(q, s), y)
    _check(y, q, w, bias, s, w_s)


def test_module_moved_and_converted():
    from llmqrt_b200.linear import FP8BlockLinear
    src = torch.nn.Linear(272, 130, bias=False)
    layer = FP8BlockLinear.from_linear(src, init_only=False, dtype=torch.float16)
    x = torch.randn(5, 272, device="cuda").half()
    y = layer.cuda()(x)
    assert bits_equal(torch.nn.Sequential(layer).half()(x), y) and bits_equal(layer.bfloat16().cpu().to("cuda")(x), y)
