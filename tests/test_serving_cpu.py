"""Serving operators without a GPU: what the calls refuse, and the rotary frequencies against their formulas."""
import ctypes
import math

import pytest
import torch

from conftest import PKG_DIR  # noqa: F401  (puts the package on sys.path)


def append_args(**change):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k=torch.zeros(3, 2, 64, dtype=torch.bfloat16), v=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
             k_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16), v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16),
             positions=torch.zeros(3, dtype=torch.int64), slots=torch.zeros(3, dtype=torch.int64), inv_freq=torch.ones(32, dtype=torch.float64))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(3, 4, 64, dtype=torch.int32)), dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(3, 2, 64)), dict(v=torch.zeros(3, 1, 64, dtype=torch.bfloat16)), dict(k_cache=torch.zeros(5, 3, 16, 64, dtype=torch.bfloat16)),
    dict(v_cache=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)), dict(v_cache=torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16).expand(5, 2, 16, 64)),
    dict(positions=torch.zeros(3, dtype=torch.int32)), dict(slots=torch.zeros(4, dtype=torch.int64)), dict(inv_freq=torch.ones(32)),
    dict(inv_freq=torch.ones(33, dtype=torch.float64)), dict(q_out=torch.zeros(3, 4, 32, dtype=torch.bfloat16)),
    dict(q_out=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64)), dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
])
def test_rope_append_refuses(change):
    from mxfp4 import rope_append
    with pytest.raises(ValueError):
        rope_append(**append_args(**change))


def test_rope_append_has_no_cpu_path():
    from mxfp4 import rope_append
    with pytest.raises(RuntimeError, match="CUDA"):
        rope_append(**append_args())


def attention_args(**change):
    a = dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16),
             v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16), block_tables=torch.zeros(3, 2, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(k_cache=torch.zeros(5, 2, 16, 64, dtype=torch.float16)),
    dict(v_cache=torch.zeros(5, 2, 32, 64, dtype=torch.bfloat16)), dict(block_tables=torch.zeros(3, 2, dtype=torch.int64)),
    dict(seq_lens=torch.ones(2, dtype=torch.int32)), dict(seq_lens=torch.ones(3, dtype=torch.int64)), dict(prefix_pages=torch.zeros(1, dtype=torch.int32)),
    dict(prefix_len=torch.zeros(1, dtype=torch.int32)), dict(prefix_pages=torch.zeros(1, dtype=torch.int32), prefix_len=torch.zeros(2, dtype=torch.int32)),
    dict(q_starts=torch.zeros(3, dtype=torch.int32)), dict(out=torch.zeros(3, 4, 64)), dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), dict(out=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64)),
])
def test_paged_attention_refuses(change):
    from mxfp4 import paged_attention
    with pytest.raises(ValueError):
        paged_attention(**attention_args(**change))


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 9, dtype=torch.float64)), dict(logits=torch.zeros(9)), dict(logits=torch.zeros(2, 0)), dict(uniforms=torch.zeros(3)),
    dict(uniforms=torch.zeros(2, dtype=torch.float64)), dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5), dict(min_p=-0.1),
    dict(top_k=torch.zeros(2)), dict(top_p=torch.zeros(3)),
])
def test_sample_tokens_refuses(change):
    from mxfp4 import sample_tokens
    a = dict(logits=torch.zeros(2, 9), uniforms=torch.zeros(2))
    a.update(change)
    with pytest.raises(ValueError):
        sample_tokens(a.pop("logits"), a.pop("uniforms"), **a)


def test_library_refuses_sizes_before_any_launch():
    from mxfp4 import _capi
    L = _capi.load()
    a = _capi.PagedAttentionArgs()
    a.dtype, a.batch, a.tokens, a.num_pages, a.table_pages, a.heads, a.kv_heads, a.head_dim, a.page_size = 0, 2, 2, 4, 2, 4, 2, 64, 16
    ask = lambda: L.mxfp4_paged_attention_workspace_bytes(ctypes.byref(a))  # noqa: E731
    assert ask() == -1                                     # no scale given
    a.scale = 0.125
    assert ask() > 0
    for name, bad, code in [("dtype", 2, -1), ("head_dim", 96, -4), ("page_size", 24, -4), ("page_size", 8, -4), ("page_size", 2048, -4), ("kv_heads", 3, -2),
                            ("heads", 0, -2), ("tokens", 3, -2), ("batch", -1, -2), ("table_pages", 1 << 30, -2), ("scale", 0.0, -1), ("scale", -1.0, -1), ("scale", float("nan"), -1), ("scale", float("inf"), -1)]:
        good = getattr(a, name)
        setattr(a, name, bad)
        assert ask() == -1
        assert L.mxfp4_paged_attention(ctypes.byref(a), None) == code, name
        setattr(a, name, good)
    assert L.mxfp4_paged_attention(ctypes.byref(a), None) == -1                    # null pointers
    for f in ("q", "out", "seq_lens", "block_tables", "k_cache", "v_cache", "workspace"):
        setattr(a, f, 0x1000)
    a.q_stride, a.out_stride, a.k_cache_stride, a.v_cache_stride = (256, 64), (256, 64), (2048, 1024, 64), (2048, 1024, 64)
    assert L.mxfp4_paged_attention(ctypes.byref(a), None) == -7                    # no workspace given
    a.q_stride = (260, 64)
    assert L.mxfp4_paged_attention(ctypes.byref(a), None) == -3
    r = _capi.RopeAppendArgs()
    r.dtype, r.tokens, r.heads, r.kv_heads, r.head_dim, r.rotary, r.page_size, r.num_pages = 0, 1, 2, 2, 64, 64, 16, 4
    for name, bad, code in [("dtype", 7, -1), ("rotary", 63, -2), ("rotary", 66, -2), ("page_size", 0, -2), ("tokens", -1, -2), ("tokens", 1, -1)]:
        good = getattr(r, name)
        setattr(r, name, bad)
        assert L.mxfp4_rope_append(ctypes.byref(r), None) == code, name
        setattr(r, name, good)
    s = _capi.SampleArgs()
    s.dtype, s.rows, s.vocab, s.ld = 0, 1, 100, 100
    for name, bad, code in [("dtype", 7, -1), ("ld", 99, -2), ("vocab", 0, -2), ("rows", -1, -2), ("rows", 1, -1)]:
        good = getattr(s, name)
        setattr(s, name, bad)
        assert L.mxfp4_sample(ctypes.byref(s), None) == code, name
        setattr(s, name, good)


def test_cache_refuses_shapes():
    from mxfp4 import PagedKVCache
    for bad in [dict(page_size=24), dict(page_size=8), dict(head_dim=80), dict(num_pages=0), dict(dtype=torch.float32)]:
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(num_pages=2, page_size=16, kv_heads=1, head_dim=64, device="cpu"), **bad})


def test_slots_follow_the_block_table():
    from mxfp4 import PagedKVCache
    c = PagedKVCache(8, 16, 1, 32, device="cpu")
    table = torch.tensor([[3, 7], [5, 0]], dtype=torch.int32)
    assert c.slots(table, torch.tensor([[0, 15, 16], [1, 17, 31]])).tolist() == [[48, 63, 112], [81, 1, 15]]
    assert c.slots(table, torch.tensor([[32], [-1]])).tolist() == [[128], [128]]          # outside the table: behind the cache's end


def test_rotary_frequencies_follow_their_formulas():
    from mxfp4 import rope_frequencies
    d, base, n = 64, 10000.0, 4096
    plain, one = rope_frequencies(d, base)
    want = [base ** (-2 * i / d) for i in range(d // 2)]
    # one power and one division in 64 bits: a few units in the last place
    assert one == 1.0 and plain.dtype == torch.float64 and torch.allclose(plain, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)
    linear, _ = rope_frequencies(d, base, {"type": "linear", "factor": 4.0})
    assert torch.allclose(linear, plain / 4, rtol=1e-14, atol=0)
    ntk, _ = rope_frequencies(d, base, {"type": "ntk", "factor": 8.0})
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12)
    l3, _ = rope_frequencies(d, base, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                       "original_max_position_embeddings": n})
    for i, f in enumerate(want):
        turns = n * f / (2 * math.pi)
        blend = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        assert math.isclose(l3[i], f * blend + f / 8 * (1 - blend), rel_tol=1e-12)
    ya, factor = rope_frequencies(d, base, {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": n})
    assert math.isclose(factor, 0.1 * math.log(16) + 1)
    assert ya[0] == plain[0] and math.isclose(ya[-1], plain[-1] / 16, rel_tol=1e-12) and bool((ya[1:] <= ya[:-1]).all())
    for i, f in enumerate(want):
        turns = n * f / (2 * math.pi)
        if turns > 45:
            assert math.isclose(ya[i], f, rel_tol=1e-12)
        if turns < 0.7:
            assert math.isclose(ya[i], f / 16, rel_tol=1e-12)
    for bad in [{"type": "dynamic", "factor": 2.0}, {"type": "longrope", "factor": 2.0}, {"type": "linear"}, {"type": "linear", "factor": 0.5}]:
        with pytest.raises(ValueError):
            rope_frequencies(d, base, bad)
    with pytest.raises(ValueError):
        rope_frequencies(63)
