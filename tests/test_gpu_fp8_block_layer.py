"""An 8-bit decoder layer's operators as they are used together: norm, block-scaled linear layers, paged 8-bit cache, attention; eager
and as a captured graph, each stage against its own formula on what the stage before it left."""
import pytest
import torch

from tests.test_gpu_paged_cache import _attend, _i32
from tests.util import rel_fro

pytestmark = pytest.mark.gpu


def _times(q, scale):
    """Values of codes with a scale for each row and 128 columns, in 64 bits."""
    return q.float().double() * scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]


class Layer:
    def __init__(self, dt, H=512, I=640, Hq=8, Hkv=2, d=64, B=6, page=16, top=300):
        from llmqrt_b200 import glue
        from llmqrt_b200.linear import FP8BlockLinear
        from llmqrt_b200.paged_cache import PagedKVCache8
        g = torch.Generator(device="cuda").manual_seed(5)
        self.g, self.dt, self.B, self.H, self.I, self.Hq, self.Hkv, self.d, self.top = g, dt, B, H, I, Hq, Hkv, d, top

        def linear(n, k, bias):
            m = torch.nn.Linear(k, n, bias=bias, device="cuda")
            m.weight.data.copy_(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
            return FP8BlockLinear.from_linear(m, init_only=False, dtype=dt)
        self.qkv, self.o = linear((Hq + 2 * Hkv) * d, H, True), linear(H, Hq * d, False)
        self.gate_up, self.down = linear(2 * I, H, False), linear(H, I, False)
        self.norms = [(1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(dt) for _ in range(2)]
        self.cache = PagedKVCache8(1, 80, page, Hkv, d, B, top, "cuda")
        self.cos, self.sin = glue.rope_tables(d, top, 1e4, "cuda")

    def step(self, x, new):
        """x [T, H], the new tokens of all requests back to back; from the attention on, every request's newest of them (one without a
        new token goes along with another's row).  Returns what each stage left."""
        from llmqrt_b200 import glue, ops
        T = x.shape[0]
        plan = self.cache.plan(new, T)
        n1, s1, _ = glue.rmsnorm_fp8_block(x, self.norms[0], 1e-6)
        row = self.qkv.forward_quantized(n1, s1).view(T, self.Hq + 2 * self.Hkv, self.d)
        self.cache.append(0, row[:, self.Hq:self.Hq + self.Hkv], row[:, self.Hq + self.Hkv:], plan, self.cos, self.sin)
        newest = (plan.cu_new[1:] - 1).clamp_min(0).long()
        q = row[newest, :self.Hq]
        a = self.cache.attend(0, q, cos=self.cos, sin=self.sin)
        aq, sa = ops.quantize_fp8_block(a.view(self.B, -1))
        o = self.o.forward_quantized(aq, sa)
        h0 = x[newest]
        n2, s2, h = glue.rmsnorm_fp8_block(o, self.norms[1], 1e-6, h0)
        gu = self.gate_up.forward_quantized(n2, s2)
        act, _, _ = glue.silu_mul(gu)
        out = self.down(act)
        return dict(n1=n1, s1=s1, row=row, q=q, a=a, aq=aq, sa=sa, o=o, h0=h0, n2=n2, s2=s2, h=h, gu=gu, act=act, out=out)

    def check(self, x, z, lens):
        half = torch.finfo(self.dt).eps / 2
        live = torch.tensor([n > 0 for n in lens], device="cuda")

        def normed(v, w, q, scale):
            y = v.double() * w.double() / (v.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
            # a code is off by 2^-4 of its value at most, by half the least step, 2^-10 of the scale, below e4m3's normal numbers
            assert ((_times(q, scale) - y).abs() <= y.abs() * (2.0 ** -4 + 2.0 ** -20) + scale.double().repeat_interleave(128, 1)[:, :y.shape[1]] * 2.0 ** -9).all()

        def linear(m, q, scale, y):
            w = m.weight.float().double() * m.weight_scale.double().repeat_interleave(128, 0)[:m.out_features].repeat_interleave(128, 1)[:, :m.in_features]
            want = _times(q, scale) @ w.T + (m.bias.double() if m.bias is not None else 0)
            assert rel_fro(y, want) < half + 2.0 ** -16          # the result's rounding, and the fp32 sums'
        normed(x, self.norms[0], z["n1"], z["s1"])
        linear(self.qkv, z["n1"], z["s1"], z["row"].reshape(x.shape[0], -1))
        c = self.cache
        want = _attend(z["q"][:, None], c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], c.block_table, lens, self.top, 0.0, self.cos, self.sin)[:, 0]
        # fp16: the result's rounding; bf16: P and the rotated Q in fp16 as well, which moves scores of about eight by 2^-11 of them
        assert rel_fro(z["a"], want) < (half + 2.0 ** -16 if self.dt == torch.float16 else half + 9 * 2.0 ** -11)
        assert (z["a"][~live] == 0).all()
        y = z["a"].reshape(self.B, -1).double()
        assert ((_times(z["aq"], z["sa"]) - y).abs() <= y.abs() * (2.0 ** -4 + 2.0 ** -20) + z["sa"].double().repeat_interleave(128, 1)[:, :y.shape[1]] * 2.0 ** -9).all()
        linear(self.o, z["aq"], z["sa"], z["o"])
        assert torch.equal(z["h"], z["o"] + z["h0"])
        normed(z["h"], self.norms[1], z["n2"], z["s2"])
        linear(self.gate_up, z["n2"], z["s2"], z["gu"])
        g, u = z["gu"].double().chunk(2, -1)
        assert rel_fro(z["act"], g * torch.sigmoid(g) * u) < 3 * half    # (silu is rounded before the product)
        act = z["act"].double()
        w = self.down.weight.float().double() * self.down.weight_scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
        # quantized activations: each off by 2^-4 at most, which the products' Frobenius norm cannot exceed
        assert ((z["out"].double() - act @ w.T).abs() <= (act.abs() @ w.abs().T) * (2.0 ** -4 + 2.0 ** -6) + 1e-3).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_layer(dt):
    """A ragged batch's prompts, then decode steps replayed from a graph with requests that come and go; a second graph of
    the same layer, captured before the first has run, shares the workspace."""
    layer = Layer(dt)
    B, H, g = layer.B, layer.H, layer.g
    prompt, lens = [40, 0, 129, 1, 16, 77], [40, 0, 129, 1, 16, 77]
    x = torch.randn(sum(prompt) + 9, H, generator=g, device="cuda").to(dt)      # (a padded batch)
    z = layer.step(x, _i32(prompt))
    assert layer.cache.seq_lens.tolist() == lens
    layer.check(x, z, lens)

    x, new = torch.zeros(B, H, dtype=dt, device="cuda"), _i32([0] * B)
    saved = [t.clone() for t in (layer.cache.seq_lens, layer.cache.free_count, layer.cache.block_table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, new)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            graphs.append((cg, layer.step(x, new)))
    for t, s in zip((layer.cache.seq_lens, layer.cache.free_count, layer.cache.block_table), saved):
        t.copy_(s)
    for i in range(6):
        now = [1, int(i > 2), 1, int(i % 2), 1, int(i < 4)]
        x.copy_(torch.randn(B, H, generator=g, device="cuda"))
        new.copy_(_i32(now))
        cg, z = graphs[i % 2]
        cg.replay()
        lens = [n + m for n, m in zip(lens, now)]
        assert layer.cache.seq_lens.tolist() == lens
        layer.check(x, z, lens)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_fused_projections(dt, T):
    """Projections of one input as one layer: each output as its own layer gives it, but for the order of the fp32 sums."""
    from llmqrt_b200.fused_utils import FusedGateUpMLP, fuse_qkv
    from llmqrt_b200.linear import FP8BlockLinear
    g = torch.Generator(device="cuda").manual_seed(T)

    def linear(n, k, bias):
        m = torch.nn.Linear(k, n, bias=bias, device="cuda")
        m.weight.data.copy_(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
        return FP8BlockLinear.from_linear(m, init_only=False, dtype=dt)
    x = torch.randn(1, T, 512, generator=g, device="cuda").to(dt)
    parts = [linear(n, 512, True) for n in (512, 128, 128)]
    apart = torch.cat([l(x) for l in parts], -1)
    half = torch.finfo(dt).eps / 2
    assert rel_fro(fuse_qkv(torch.nn.Module(), *parts)(x), apart) < 2 * (half + 2.0 ** -16)      # (each off by its own rounding)
    gate, up, down = linear(640, 512, False), linear(640, 512, False), linear(512, 640, False)
    a, b = gate(x).double(), up(x).double()
    w = down.weight.float().double() * down.weight_scale.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    act = a * torch.sigmoid(a) * b
    mlp = FusedGateUpMLP(gate, up, down)
    assert mlp.gate_up is not None
    # codes of the activations off by 2^-4 at most, and 2^-6 for their own roundings
    assert ((mlp(x).double() - act @ w.T).abs() <= (act.abs() @ w.abs().T) * (2.0 ** -4 + 2.0 ** -6) + 1e-3).all()
