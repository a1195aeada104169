"""What the paged cache's calls refuse, before anything is launched (on CPU tensors: shapes and types are checked first)."""
import pytest
import torch

F8 = torch.float8_e4m3fn


def _cache(P=3, Hkv=2, page=16, d=64, dtype=torch.int8):
    return [torch.zeros(P, Hkv, page, d, dtype=torch.int8).view(dtype) for _ in range(2)] + [torch.ones(P, Hkv) for _ in range(2)]


def _append(**kw):
    from llmqrt_b200.paged_cache import kv8_append
    kc, vc, ks, vs = _cache()
    a = dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, k=torch.zeros(4, 2, 64).half(), v=torch.zeros(4, 2, 64).half(),
             slots=torch.zeros(4, dtype=torch.int64))
    kv8_append(**(a | kw))


def _attend(**kw):
    from llmqrt_b200.paged_cache import attn_decode_kv8
    kc, vc, ks, vs = _cache()
    a = dict(q=torch.zeros(2, 4, 64).half(), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs,
             block_table=torch.zeros(2, 3, dtype=torch.int32), seqlens=torch.ones(2, dtype=torch.int32), max_seqlen=48)
    return attn_decode_kv8(**(a | kw))


def _plan(**kw):
    from llmqrt_b200.paged_cache import plan_step
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    a = dict(context_lens=i(2), new_lens=i(2), block_table=i(2, 3), free_pages=i(5), free_count=i(1), page_size=16, max_tokens=4)
    return plan_step(**(a | kw))


@pytest.mark.parametrize("call", [_append, _attend, _plan])
def test_there_is_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="CUDA device"):
        call()


@pytest.mark.parametrize("kw,error,match", [
    (dict(k_cache=torch.zeros(3, 2, 16, 64).half()), TypeError, "int8 or both float8"),
    (dict(k_cache=_cache(dtype=F8)[0]), TypeError, "int8 or both float8"),
    (dict(v_cache=_cache(P=4)[0]), RuntimeError, "pages, Hkv, page, d"),
    (dict(k_cache=_cache(d=128)[0][..., ::2]), RuntimeError, "pages, Hkv, page, d"),
    (dict(k_scale=torch.ones(3, 2).half()), TypeError, "fp32"),
    (dict(v_scale=torch.ones(3, 3)), RuntimeError, r"\[pages, Hkv\]"),
    (dict(v_scale=torch.ones(2, 3).t()), RuntimeError, r"\[pages, Hkv\]"),
])
def test_caches(kw, error, match):
    for call in (_append, _attend):
        with pytest.raises(error, match=match):
            call(**kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(k=torch.zeros(4, 2, 64)), TypeError, "one dtype"),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.int32), v=torch.zeros(4, 2, 64, dtype=torch.int32)), TypeError, "dtype"),
    (dict(k=torch.zeros(5, 2, 64).half()), RuntimeError, "k and v"),
    (dict(k=torch.zeros(4, 3, 64).half(), v=torch.zeros(4, 3, 64).half()), RuntimeError, "k and v"),
    (dict(slots=torch.zeros(4, dtype=torch.int32)), TypeError, "int64"),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), RuntimeError, "slots"),
    (dict(cos=torch.zeros(9, 32)), RuntimeError, "cos and sin"),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32)), TypeError, "positions"),
    (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64), positions=torch.zeros(4, dtype=torch.int32)), RuntimeError, "rotary"),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=torch.zeros(3, dtype=torch.int32)), RuntimeError, "positions"),
    (dict(cos=torch.zeros(9, 32).half(), sin=torch.zeros(9, 32).half(), positions=torch.zeros(4, dtype=torch.int32)), TypeError, "fp32"),
])
def test_append(kw, error, match):
    with pytest.raises(error, match=match):
        _append(**kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=torch.zeros(2, 4, 128).half()), RuntimeError, "q must be"),
    (dict(q=torch.zeros(4, 64).half()), RuntimeError, "q must be"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.int32)), TypeError, "dtype"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), TypeError, "block_table"),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32)), RuntimeError, "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), RuntimeError, "block_table"),
    (dict(seqlens=torch.zeros(2, dtype=torch.int64)), TypeError, "seqlens"),
    (dict(seqlens=torch.zeros(1, dtype=torch.int32)), RuntimeError, "seqlens"),
    (dict(max_seqlen=-1), RuntimeError, "max_seqlen"),
    (dict(sin=torch.zeros(9, 32)), RuntimeError, "cos and sin"),
])
def test_attend(kw, error, match):
    with pytest.raises(error, match=match):
        _attend(**kw)


@pytest.mark.parametrize("kw,error,match", [
    (dict(context_lens=torch.zeros(2, dtype=torch.int64)), TypeError, "context_lens"),
    (dict(new_lens=torch.zeros(3, dtype=torch.int32)), RuntimeError, "new_lens"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), RuntimeError, "block_table"),
    (dict(free_count=torch.zeros(2, dtype=torch.int32)), RuntimeError, "free_count"),
    (dict(free_left=torch.zeros(1, dtype=torch.int64)), TypeError, "free_left"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), RuntimeError, "seq_lens"),
    (dict(max_tokens=-1), RuntimeError, "max_tokens"),
])
def test_plan(kw, error, match):
    with pytest.raises(error, match=match):
        _plan(**kw)


def _status(name, *args):
    from llmqrt_b200 import _lib
    return getattr(_lib._lib, name)(*args)


def test_the_library_refuses():
    """Sizes that the kernels do not take come back as a status; nothing is launched (there is no device here to launch on)."""
    from llmqrt_b200 import _lib

    def plan(B=1, width=1, pool=1, page=16, most=1, p=64):
        return _status("llmqrt_plan_step", p, p, p, width, p, p, p, p, p, p, p, B, width, pool, page, most, None, None)
    for kw in (dict(page=8), dict(page=48), dict(page=256), dict(B=8193), dict(B=-1), dict(width=2 ** 28), dict(most=-1), dict(p=None)):
        assert plan(**kw) == -1, kw

    def append(type=_lib.E4M3, dt=0, T=1, page=16, d=64, Hkv=1, ps=1024, hs=1024, ts=64, p=64, cos=None):
        return _status("llmqrt_kv8_append", p, p, p, p, type, ps, hs, p, ts, p, ts, dt, p, cos, cos, 0, p, T, 4, page, Hkv, d, None)
    for kw in (dict(type=0), dict(dt=2), dict(page=20), dict(d=96), dict(Hkv=0), dict(hs=1000), dict(ps=512), dict(ts=60), dict(p=72), dict(p=None),
               dict(cos=64), dict(T=-1)):
        assert append(**kw) == -1, kw

    def attend(type=_lib.I8, dt=1, B=1, Sq=1, Hq=4, Hkv=2, d=64, page=16, ps=2048, hs=1024, most=16, p=64, ts=256):
        return _status("llmqrt_attn_decode_kv8", p, ts, ts, p, p, type, ps, hs, p, p, p, 1, 1, p, None, None, 0, p, dt, B, Sq, Hq, Hkv, d, 4, page,
                       most, 0.0, None, None)
    for kw in (dict(type=1), dict(dt=3), dict(Sq=17), dict(Hq=5), dict(Hq=34, Hkv=2), dict(d=80), dict(page=0), dict(ps=1024), dict(hs=100),
               dict(most=-1), dict(p=None), dict(p=8), dict(ts=100), dict(B=65536)):
        assert attend(**kw) == -1, kw
    assert attend(B=0) == 0 and attend(Sq=0) == 0


def test_cache_object_refuses():
    from llmqrt_b200.paged_cache import PagedKVCache8
    ok = dict(num_layers=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, max_requests=2, max_seqlen=40, device="cpu")
    c = PagedKVCache8(**ok)
    assert c.max_seqlen == 48 and c.block_table.shape == (2, 3) and c.free_pages.tolist() == [3, 2, 1, 0]
    with pytest.raises(TypeError):
        PagedKVCache8(**ok, dtype=torch.float16)
    for kw in (dict(page_size=24), dict(head_dim=96), dict(num_pages=0), dict(max_requests=9000), dict(max_requests=0)):
        with pytest.raises(ValueError):
            PagedKVCache8(**(ok | kw))
