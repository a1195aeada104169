"""What the block-scaled fp8 layer refuses, before anything is launched (on CPU tensors: shapes and types are checked first)."""
import pytest
import torch

F8 = torch.float8_e4m3fn


def _call(M=4, N=200, K=256, **kw):
    from llmqrt_b200 import ops
    f8 = lambda *s: torch.zeros(s, dtype=torch.uint8).view(F8)  # noqa: E731
    a = dict(a=f8(M, K), w=f8(N, K), bias=None, a_scale=torch.ones(M, -(-K // 128)), w_scale=torch.ones(-(-N // 128), -(-K // 128)),
             out_dtype=torch.float16)
    return ops.fp8_linear_block(**(a | kw))


@pytest.mark.parametrize("kw,error,match", [
    (dict(), RuntimeError, "CUDA device"),
    (dict(a=torch.zeros(4, 256).half()), TypeError, "float8_e4m3fn"),
    (dict(a=torch.zeros(4, 256, dtype=torch.uint8).view(torch.float8_e5m2)), TypeError, "float8_e4m3fn"),
    (dict(w=torch.zeros(200, 256).half()), TypeError, "float8_e4m3fn"),
    (dict(w=torch.zeros(200, 128, dtype=torch.uint8).view(F8)), RuntimeError, "weight must be"),
    (dict(w=torch.zeros(256, 200, dtype=torch.uint8).view(F8).t()), RuntimeError, "weight must be"),
    (dict(a_scale=torch.ones(4, 1)), RuntimeError, "a's scales"),
    (dict(a_scale=torch.ones(2, 4).t()), RuntimeError, "a's scales"),
    (dict(a_scale=torch.ones(4, 2).half()), TypeError, "fp32"),
    (dict(w_scale=torch.ones(1, 2)), RuntimeError, "weight's scales"),
    (dict(w_scale=torch.ones(2, 2).double()), TypeError, "fp32"),
    (dict(bias=torch.zeros(128).half()), RuntimeError, "bias"),
    (dict(out_dtype=torch.int32), TypeError, "dtype"),
    (dict(out_dtype="fp16"), TypeError, "dtype"),
])
def test_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        _call(**kw)


def test_the_library_refuses():
    """Sizes and pointers that the kernels do not take come back as a status; nothing is launched."""
    from llmqrt_b200 import _lib

    def call(M=1, N=1, K=128, lda=128, ldw=128, ldo=1, out=0, bias=None, bd=0, p=64, flags=0):
        return _lib._lib.llmqrt_fp8_linear_block(p, lda, p, ldw, bias, bd, p, p, p, out, ldo, M, N, K, None, None, flags)
    for kw in (dict(K=120), dict(K=0), dict(N=0), dict(M=-1), dict(lda=112), dict(ldw=136), dict(ldo=0), dict(out=2), dict(bias=64, bd=3), dict(p=None),
               dict(p=8), dict(flags=2), dict(M=2 ** 31)):
        assert call(**kw) == -1, kw
    assert call(M=0) == 0

    def rows(K=128, ldx=128, dt=0, p=64, M=1):
        return _lib._lib.llmqrt_quantize_fp8_block(p, dt, M, K, ldx, p, p, None)
    for kw in (dict(K=12), dict(K=0), dict(ldx=120), dict(ldx=132), dict(dt=2), dict(p=None), dict(p=68), dict(K=40000, ldx=40000), dict(M=-1)):
        assert rows(**kw) == -1, kw
    norm = lambda res, h: _lib._lib.llmqrt_rmsnorm_fp8_block(64, 128, res, 128, h, 64, 1e-6, 64, 64, 0, 1, 128, None)  # noqa: E731
    assert norm(64, None) == -1 and norm(None, 64) == -1


def test_module_refuses():
    from llmqrt_b200.linear import FP8BlockLinear
    with pytest.raises(ValueError):
        FP8BlockLinear(200, 8, False, dev="cpu")
    layer = FP8BlockLinear(160, 130, True, dev="cpu")
    assert layer.weight.shape == (130, 160) and layer.weight_scale.shape == (2, 2) and layer.bias.shape == (130,)
    with pytest.raises(AssertionError):
        FP8BlockLinear.from_linear(torch.nn.Linear(32, 32), group_size=64)


def test_quantized_blocks():
    """A weight's codes and scales, on the CPU: within half a step of e4m3 of the weight, absmax at the greatest code."""
    from llmqrt_b200.linear.linear_fp8 import quantize_blocks
    w = torch.randn(300, 400, generator=torch.Generator().manual_seed(0))
    w[:128, :128] *= 100
    w[130:140] = 0
    q, s = quantize_blocks(w)
    assert q.shape == w.shape and q.dtype == F8 and s.shape == (3, 4)
    full = s.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :400]
    err = (q.float() * full - w).abs()
    assert (err <= w.abs() * 2.0 ** -4 * 1.001 + full * 2.0 ** -10 * 1.001).all() and (q.float().abs().amax() == 448)


def _layers(outs, k=160, bias=(True, False, True)):
    from llmqrt_b200.linear import FP8BlockLinear
    g, layers = torch.Generator().manual_seed(1), []
    for n, b in zip(outs, bias):
        m = torch.nn.Linear(k, n, bias=b)
        m.weight.data.copy_(torch.randn(n, k, generator=g))
        layers.append(FP8BlockLinear.from_linear(m, init_only=False, dtype=torch.float16))
    return layers


def test_fused_projections():
    """Rows of codes and of scales one below the other; a layer without a bias counts as one of zeros."""
    from llmqrt_b200.fused_utils import FusedGateUpMLP, fuse_linears, fuse_qkv
    layers = _layers((256, 128, 72))
    w = torch.cat([l.weight.data.float() for l in layers])
    s = torch.cat([l.weight_scale.data for l in layers])
    bias = torch.cat([layers[0].bias.data, torch.zeros(128).half(), layers[2].bias.data])
    fused = fuse_qkv(torch.nn.Module(), *layers)
    assert fused.out_features == 456 and torch.equal(fused.weight.data.float(), w) and torch.equal(fused.weight_scale.data, s)
    assert torch.equal(fused.bias.data, bias) and not hasattr(layers[0], "weight")
    odd = _layers((200, 128, 72))
    assert fuse_qkv(torch.nn.Module(), *odd) == tuple(odd)               # a row of scales would serve two layers
    with pytest.raises(ValueError, match="128"):
        fuse_linears(odd)
    gate, up, down = _layers((192, 192, 64), bias=(False, False, False))
    assert FusedGateUpMLP(gate, up, down).gate_up is None


@pytest.mark.parametrize("change", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.bfloat16),
                                    lambda m: m.type(torch.float16), lambda m: m.to("cpu"), lambda m: m.share_memory()])
def test_conversions_keep_codes_and_scales(change):
    """A module's conversions to other types reach the layer's bias alone."""
    layer = _layers((200,))[0]
    layer.weight.data.view(torch.uint8)[3, 5] = 0x7F             # (a NaN and a scale that no 16-bit type holds)
    layer.weight_scale.data[0, 0] = 1e-9
    w, s = layer.weight.data.view(torch.uint8).clone(), layer.weight_scale.data.clone()
    names = [n for n, _ in layer.named_parameters()]
    whole = change(torch.nn.Sequential(layer, torch.nn.Linear(4, 4)))
    assert whole[0] is layer and [n for n, _ in layer.named_parameters()] == names and isinstance(layer.weight, torch.nn.Parameter)
    assert layer.weight.dtype == F8 and torch.equal(layer.weight.data.view(torch.uint8), w) and not layer.weight.requires_grad
    assert layer.weight_scale.dtype == torch.float32 and torch.equal(layer.weight_scale.data, s)
    assert layer.bias.dtype in (whole[1].weight.dtype, torch.float16)


def test_layer_without_storage():
    from llmqrt_b200.linear import FP8BlockLinear
    layer = FP8BlockLinear(160, 130, True, dev="meta").half().to_empty(device="cpu")
    assert layer.weight.dtype == F8 and layer.weight.shape == (130, 160) and layer.weight.device.type == "cpu"
    assert layer.weight_scale.dtype == torch.float32 and layer.weight_scale.shape == (2, 2)


def _dequantized(state):
    w, s = state["weight"].float(), state["weight_scale"]
    return w * s.repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]


def _state(n, k, bias, seed):
    from llmqrt_b200.linear import FP8BlockLinear
    g = torch.Generator().manual_seed(seed)
    m = torch.nn.Linear(k, n, bias=bias)
    for p in m.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g))
    return FP8BlockLinear.from_linear(m, init_only=False, dtype=torch.float16).state_dict()


def test_tensor_parallel_shards():
    """Shards of a layer are the layer's own values, fit the layer class, and make up the whole."""
    from llmqrt_b200 import tp
    from llmqrt_b200.linear import FP8BlockLinear
    state = _state(700, 400, True, 3)                            # (last blocks of 60 outputs and 16 inputs)
    full = _dequantized(state)
    cuts = [(0, 256), (256, 384), (384, 700)]
    parts = [tp.shard_linear_state(state, "fp8_block_quant", "column", c) for c in cuts]
    assert torch.equal(torch.cat([_dequantized(p) for p in parts]), full) and torch.equal(torch.cat([p["bias"] for p in parts]), state["bias"])
    for p, (a, b) in zip(parts, cuts):
        FP8BlockLinear(400, b - a, True, dev="cpu", dtype=torch.float16).load_state_dict(p)
    cuts = [(0, 128), (128, 400)]
    parts = [tp.shard_linear_state(state, "fp8_block_quant", "row", c, keep_bias=i == 0) for i, c in enumerate(cuts)]
    assert torch.equal(torch.cat([_dequantized(p) for p in parts], 1), full)
    assert torch.equal(parts[0]["bias"], state["bias"]) and not parts[1]["bias"].any()
    picked = tp.shard_linear_state(state, "fp8_block_quant", "column", list(range(512, 640)) + list(range(0, 128)))
    assert torch.equal(_dequantized(picked), torch.cat([full[512:640], full[:128]]))
    for mode, sel in (("column", (0, 64)), ("column", (64, 192)), ("column", (640, 690)), ("row", (0, 200)), ("column", list(range(640, 700)) + list(range(128)))):
        with pytest.raises(ValueError, match="128"):
            tp.shard_linear_state(state, "fp8_block_quant", mode, sel)


@pytest.mark.parametrize("world", [1, 2, 4])
@pytest.mark.parametrize("inter", [1024, 1040])
def test_tensor_parallel_decoder_layer(world, inter):
    from llmqrt_b200 import tp
    H, heads, kv, d = 512, 8, 4, 128
    layer = {n: _state(o, i, b, s) for s, (n, o, i, b) in enumerate([("q_proj", heads * d, H, True), ("k_proj", kv * d, H, True), ("v_proj", kv * d, H, True),
             ("o_proj", H, heads * d, False), ("gate_proj", inter, H, False), ("up_proj", inter, H, False), ("down_proj", H, inter, False)])}
    ranks = [tp.shard_decoder_layer(layer, "fp8_block_quant", heads, kv, d, world, r) for r in range(world)]
    for name, state in layer.items():
        axis = 1 if name in ("o_proj", "down_proj") else 0
        assert torch.equal(torch.cat([_dequantized(r[name]) for r in ranks], axis), _dequantized(state)), name


def test_conversion_of_a_layer_with_other_types():
    """Parameters that are not the layer's own types (a state dict assigned as it was) are converted like any."""
    layer = _layers((200,))[0]
    layer.weight_scale = torch.nn.Parameter(layer.weight_scale.data.half(), requires_grad=False)
    layer.weight = torch.nn.Parameter(layer.weight.data.float(), requires_grad=False)
    layer.bfloat16()
    assert layer.weight_scale.dtype == layer.weight.dtype == torch.bfloat16 and layer.weight.shape == (200, 160)
