"""What a decoder needs between its linear layers when keys and values live in a paged cache: rotary positions with the
append to the cache, attention over the cache (with a prefix that the whole batch shares), and sampling of the next token.

The reference has no counterpart: in its Llama scenario the model's own PyTorch code runs these steps.  The arithmetic is in
libmxfp4_b200.so (mxfp4_rope_append, mxfp4_paged_attention, mxfp4_sample); this module checks shapes, types and devices,
allocates outputs and a workspace per call, and enqueues on the tensors' device's current stream.  Nothing is kept from one
call for the next, so calls may run on several streams, be captured into CUDA graphs and be replayed side by side.

Values that only the device knows (lengths, offsets, slots, pages) cannot be refused by the call.  The kernels clamp them, skip
what lies outside the cache and report through a status word, which check_status() reads.
"""
import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from . import _capi

_status = {}                     # device index -> int32 status word of the serving kernels
_DT16 = {torch.bfloat16: 0, torch.float16: 1}


def _status_word(device: torch.device) -> torch.Tensor:
    st = _status.get(device.index)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            raise _capi.MXFP4BackendError("mxfp4: the first serving call on a device allocates its status word; make one call before the capture")
        st = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()      # other streams may use the word from here on
        st = _status.setdefault(device.index, st)
    return st


def check_status(device=None):
    """Synchronises and raises if a serving kernel on `device` met lengths, offsets, slots or pages outside its arguments,
    or a bounded wait that ran out."""
    for idx, st in list(_status.items()):
        if device is not None and torch.device(device).index not in (None, idx):
            continue
        torch.cuda.synchronize(idx)
        code = int(st.item())
        if code != 0:
            st.zero_()
            what = {-1: "a slot or page outside the cache", -2: "lengths or offsets outside the tables or the query rows",
                    -6: "a device-side wait timed out"}.get(code, "unknown")
            raise _capi.MXFP4BackendError(f"mxfp4 serving kernel reported status {code} ({what})")


def _need(ok, message):
    if not ok:
        raise ValueError("mxfp4: " + message)


def _on(t: torch.Tensor, device, dtype, shape, name):
    _need(isinstance(t, torch.Tensor) and t.device == device, f"{name} must be a tensor on {device}")
    _need(t.dtype == dtype, f"{name} must be {dtype} (got {t.dtype})")
    _need(tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)} (got {tuple(t.shape)})")
    return t if t.is_contiguous() else t.contiguous()


def _strides(t: torch.Tensor):
    """Element strides of all dimensions but the last; one that steps over a single entry takes part in no address."""
    return tuple(s if n > 1 else 8 for s, n in zip(t.stride()[:-1], t.shape[:-1]))


def _no_overlap(t: torch.Tensor, name):
    _need(all(s != 0 for s, n in zip(t.stride(), t.shape) if n > 1), f"{name} is written and must not be a broadcast view")


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """Angle per position of every pair of a rotated width, float64 [rotary_dim / 2], and the factor on sines and cosines.

    scaling: None, or a dict with "type" and "factor" as model configurations have them:
      "linear"   positions divided by the factor
      "ntk"      the base raised by factor^(d / (d - 2)), which stretches the slowest pair by the factor and leaves the fastest
      "llama3"   pairs whose wavelength exceeds original_max_position_embeddings / low_freq_factor divided by the factor, those
                 under original / high_freq_factor left, a linear blend in between
      "yarn"     pairs by their number of turns over original_max_position_embeddings: divided by the factor below beta_slow (1)
                 turns, left above beta_fast (32), a linear ramp over the pair's index in between; sines and cosines times
                 attention_factor (0.1 ln(factor) + 1)
    Scalings that depend on the current length ("dynamic", "longrope") are refused."""
    _need(rotary_dim > 0 and rotary_dim % 2 == 0, f"rotary_dim {rotary_dim} must be positive and even")
    half = rotary_dim // 2
    base = float(base)
    _need(base > 0, "base must be positive")
    i = torch.arange(half, dtype=torch.float64)
    freq = base ** (-i / half)
    attention = 1.0
    kind = None if scaling is None else scaling.get("type", scaling.get("rope_type"))
    if kind not in (None, "default"):
        factor = float(scaling["factor"]) if "factor" in scaling else 0.0
        if kind not in ("linear", "ntk", "llama3", "yarn"):
            raise ValueError(f"mxfp4: rotary scaling of type {kind!r} (linear, ntk, llama3 or yarn)")
        _need(factor >= 1.0, f"rotary scaling needs a factor of at least 1 (got {factor})")
        if kind == "linear":
            freq = freq / factor
        elif kind == "ntk":
            _need(half > 1, "ntk scaling needs at least two pairs")
            freq = (base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-i / half)
        elif kind == "llama3":
            low, high, original = (float(scaling[k]) for k in ("low_freq_factor", "high_freq_factor", "original_max_position_embeddings"))
            _need(0 < low < high and original > 0, "llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
            turns = original * freq / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            freq = freq * (keep + (1 - keep) / factor)
        else:
            original = float(scaling["original_max_position_embeddings"])
            fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)
            _need(0 < slow < fast and original > 0 and base > 1, "yarn scaling needs 0 < beta_slow < beta_fast and a base above 1")
            pair = lambda turns: half * math.log(original / (turns * 2 * math.pi)) / math.log(base)  # noqa: E731
            first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary_dim - 1)
            ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / factor * ramp
            given = scaling.get("attention_factor")
            attention = float(given) if given is not None else 0.1 * math.log(factor) + 1.0
    return freq.to(device) if device is not None else freq, attention


class PagedKVCache:
    """Keys and values of one layer on pages: k and v are [num_pages, kv_heads, page_size, head_dim].  Which pages belong to
    which sequence is the caller's: block tables for paged_attention, slots (page * page_size + offset) for rope_append."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device=None):
        _need(dtype in _DT16, f"a paged cache is bfloat16 or float16 (got {dtype})")
        _need(16 <= page_size <= 1024 and page_size & (page_size - 1) == 0, f"page_size {page_size} must be a power of two from 16 to 1024")
        _need(head_dim in (32, 64, 128), f"head_dim {head_dim} must be 32, 64 or 128")
        _need(num_pages > 0 and kv_heads > 0, "a paged cache needs pages and heads")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = num_pages, page_size, kv_heads, head_dim
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        self.k = torch.zeros(num_pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)

    def slots(self, block_tables: torch.Tensor, places: torch.Tensor) -> torch.Tensor:
        """Slots of the places [batch, n] (0 is a sequence's first own token) through block tables [batch, pages]."""
        page = torch.div(places, self.page_size, rounding_mode="floor")
        return block_tables.long().gather(1, page.long()) * self.page_size + places.long() % self.page_size


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, positions: torch.Tensor,
                slots: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False, scaling: float = 1.0,
                q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns q [tokens, heads, D] and k [tokens, kv_heads, D] by their positions, stores the turned k and the v at `slots` of
    the caches [pages, kv_heads, page_size, D], and returns the turned q (in q_out, which may be q itself).

    Pair i of the first 2 * len(inv_freq) elements of a head turns by positions * inv_freq[i] (float64, see rope_frequencies);
    pairs are (i, i + half), or (2i, 2i + 1) when interleaved; `scaling` multiplies the turned elements, the others stay as they
    are.  positions and slots are int64 [tokens]; a negative slot stores nothing; the slots of a call must differ.  q, k and v
    may be views of one projection's output; any strides, the last dimension contiguous.  bfloat16, float16 or float32."""
    dev = q.device
    dt = _capi.DT.get(q.dtype)
    _need(dt is not None, f"rope_append takes bfloat16, float16 or float32 (got {q.dtype})")
    _need(q.dim() == 3 and k.dim() == 3 and k_cache.dim() == 4, "q and k must be [tokens, heads, head_dim], the caches [pages, kv_heads, page_size, head_dim]")
    n, heads, dim = q.shape
    kv = k.shape[1]
    pages, page_size = k_cache.shape[0], k_cache.shape[2]
    _need(k.shape == (n, kv, dim) and v.shape == k.shape, f"k and v must be [{n}, kv_heads, {dim}]")
    _need(k_cache.shape == (pages, kv, page_size, dim) and v_cache.shape == k_cache.shape, f"the caches must be [pages, {kv}, page_size, {dim}]")
    if q_out is None:
        q_out = torch.empty(n, heads, dim, dtype=q.dtype, device=dev)
    else:
        _need(q_out.shape == q.shape, "q_out must have q's shape")
        _no_overlap(q_out, "q_out")
    for t, name in ((k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"), (q_out, "q_out")):
        _need(t.dtype == q.dtype and t.device == dev, f"{name} must be {q.dtype} on {dev}")
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"), (q_out, "q_out")):
        _need(dim <= 1 or t.stride(-1) == 1, f"the last dimension of {name} must be contiguous")
    _no_overlap(k_cache, "k_cache")
    _no_overlap(v_cache, "v_cache")
    _need(inv_freq.dim() == 1 and 2 * inv_freq.shape[0] <= dim, f"inv_freq must be one value per pair of at most {dim} elements")
    positions, slots = _on(positions, dev, torch.int64, (n,), "positions"), _on(slots, dev, torch.int64, (n,), "slots")
    inv_freq = _on(inv_freq, dev, torch.float64, inv_freq.shape, "inv_freq")
    _capi.require_cuda(q, "rope_append")
    if n == 0:
        return q_out
    a = _capi.RopeAppendArgs()
    a.dtype, a.tokens, a.heads, a.kv_heads, a.head_dim = dt, n, heads, kv, dim
    a.num_pages, a.page_size, a.rotary, a.interleaved, a.scaling = pages, page_size, 2 * inv_freq.shape[0], bool(interleaved), scaling
    a.q, a.k, a.v, a.q_out, a.k_cache, a.v_cache = (t.data_ptr() for t in (q, k, v, q_out, k_cache, v_cache))
    a.q_stride, a.k_stride, a.v_stride, a.q_out_stride = _strides(q), _strides(k), _strides(v), _strides(q_out)
    a.k_cache_stride, a.v_cache_stride = _strides(k_cache), _strides(v_cache)
    a.positions, a.slots, a.inv_freq = positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr()
    with _capi.on_device(dev):
        a.status_dev = _status_word(dev).data_ptr()
        _capi.check(_capi.load().mxfp4_rope_append(ctypes.byref(a), _capi.stream_ptr(dev)), "mxfp4_rope_append")
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, *,
                    q_starts: Optional[torch.Tensor] = None, prefix_pages: Optional[torch.Tensor] = None, prefix_len: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of q [tokens, heads, D] over the caches [pages, kv_heads, page_size, D]: out, or (out, lse) with return_lse.

    Sequence b owns seq_lens[b] keys on the pages block_tables[b] and has the query rows q_starts[b] .. q_starts[b + 1] (None: one
    row each); they are its last tokens, so its i-th of n rows sees its first seq_lens[b] - n + i + 1 keys.  In front of them
    every row sees the prefix_len[0] keys on prefix_pages, which the whole batch shares and which are read once for all where
    sequences have few rows.  A row that sees nothing gives zeros and a log-sum of -inf.  Head h reads key head h // (heads //
    kv_heads).  scale defaults to D ** -0.5.  seq_lens, q_starts, prefix_len ([1]) and the tables are int32 on the device: they
    may change between replays of a captured call.  Keys and values that a sequence owns must be finite.

    Rows outside q_starts[0] .. q_starts[-1] stay as they are in a given `out` (their lse undefined) and are zeros (lse -inf) in
    a fresh one.  bfloat16 or float16; D of 32, 64 or 128; page_size a power of two from 16 to 1024."""
    dev = q.device
    dt = _DT16.get(q.dtype)
    _need(dt is not None, f"paged_attention takes bfloat16 or float16 (got {q.dtype})")
    _need(q.dim() == 3 and k_cache.dim() == 4 and block_tables.dim() == 2,
          "q must be [tokens, heads, head_dim], the caches [pages, kv_heads, page_size, head_dim], block_tables [batch, pages]")
    n, heads, dim = q.shape
    pages, kv, page_size, cache_dim = k_cache.shape
    batch, table_pages = block_tables.shape
    _need(cache_dim == dim and v_cache.shape == k_cache.shape, f"the caches must be [pages, kv_heads, page_size, {dim}]")
    _need(k_cache.dtype == q.dtype and v_cache.dtype == q.dtype and k_cache.device == dev and v_cache.device == dev, f"the caches must be {q.dtype} on {dev}")
    _need(block_tables.dtype == torch.int32 and block_tables.device == dev, f"block_tables must be int32 on {dev}")
    _need((prefix_pages is None) == (prefix_len is None), "prefix_pages and prefix_len come together")
    seq_lens = _on(seq_lens, dev, torch.int32, (batch,), "seq_lens")
    if table_pages > 1 and block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    fresh = out is None
    if fresh:
        out = torch.empty(n, heads, dim, dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev, f"out must be {q.dtype} [{n}, {heads}, {dim}] on {dev}")
        _need(out.stride(-1) == 1, "the last dimension of out must be contiguous")
        _no_overlap(out, "out")
    for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(t.stride(-1) == 1, f"the last dimension of {name} must be contiguous")
    lse = torch.empty(n, heads, dtype=torch.float32, device=dev) if return_lse else None
    a = _capi.PagedAttentionArgs()
    a.dtype, a.batch, a.tokens, a.num_pages, a.table_pages = dt, batch, n, pages, table_pages
    a.heads, a.kv_heads, a.head_dim, a.page_size = heads, kv, dim, page_size
    a.scale = dim ** -0.5 if scale is None else float(scale)
    a.q, a.out, a.k_cache, a.v_cache = q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.q_stride, a.out_stride, a.k_cache_stride, a.v_cache_stride = _strides(q), _strides(out), _strides(k_cache), _strides(v_cache)
    a.block_tables, a.table_stride, a.seq_lens = block_tables.data_ptr(), block_tables.stride(0), seq_lens.data_ptr()
    if return_lse:
        a.lse = lse.data_ptr()
    if q_starts is not None:
        q_starts = _on(q_starts, dev, torch.int32, (batch + 1,), "q_starts")
        a.q_starts, a.fill_rest = q_starts.data_ptr(), fresh
    if prefix_pages is not None:
        _need(prefix_pages.dim() == 1, "prefix_pages must be one list of pages")
        prefix_pages = _on(prefix_pages, dev, torch.int32, prefix_pages.shape, "prefix_pages")
        prefix_len = _on(prefix_len, dev, torch.int32, (1,), "prefix_len")
        a.prefix_pages, a.prefix_len, a.prefix_table_pages = prefix_pages.data_ptr(), prefix_len.data_ptr(), prefix_pages.shape[0]
    _capi.require_cuda(q, "paged_attention")
    L = _capi.load()
    if n > 0:
        with _capi.on_device(dev):
            nbytes = L.mxfp4_paged_attention_workspace_bytes(ctypes.byref(a))
            if nbytes < 0:
                _capi.check(int(nbytes), "mxfp4_paged_attention")
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes, a.status_dev = workspace.data_ptr(), nbytes, _status_word(dev).data_ptr()
            _capi.check(L.mxfp4_paged_attention(ctypes.byref(a), _capi.stream_ptr(dev)), "mxfp4_paged_attention")
    return (out, lse) if return_lse else out



def _setting(value, rows, dev, dtype, name, low, high):
    """(pointer or None, number, the tensor to keep alive) of a per-row tensor or one number for all rows."""
    if isinstance(value, torch.Tensor):
        t = _on(value, dev, dtype, (rows,), name)
        return t.data_ptr(), 0, t
    _need(low <= value <= high, f"{name} must lie between {low} and {high} (got {value})")
    return None, value, None


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, *, temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
                  top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0, return_logprobs: bool = False):
    """The next token of every row of logits [rows, vocab]: int64 [rows], or (tokens, logprobs float32) with return_logprobs.

    With weights exp((l - max) / temperature) and the tokens in descending order of their logits (equal ones: the lower index
    first), top_k keeps the first k (0: all), top_p the shortest beginning whose weight reaches p times what top_k left, min_p the
    tokens whose weight is at least min_p times the largest.  The row's token is the first whose cumulative weight exceeds
    uniforms[row] (float32 in [0, 1)) times the kept weight; its log-probability is that among the kept ones.  temperature 0 takes
    the lowest index of the maximum, as does a row whose maximum is infinite; NaN logits count as -inf.  Each setting is a number
    or a tensor with one value per row (float32; top_k int32).  Logits in bfloat16, float16 or float32, rows of any pitch."""
    dev = logits.device
    dt = _capi.DT.get(logits.dtype)
    _need(dt is not None, f"sample_tokens takes bfloat16, float16 or float32 logits (got {logits.dtype})")
    _need(logits.dim() == 2 and logits.shape[1] > 0, "logits must be [rows, vocab]")
    rows, vocab = logits.shape
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    uniforms = _on(uniforms, dev, torch.float32, (rows,), "uniforms")
    a = _capi.SampleArgs()
    a.logits, a.dtype, a.rows, a.vocab, a.ld, a.uniforms = logits.data_ptr(), dt, rows, vocab, logits.stride(0) if rows > 1 else vocab, uniforms.data_ptr()
    a.temperature, a.temperature_value, t = _setting(temperature, rows, dev, torch.float32, "temperature", 0.0, math.inf)
    a.top_k, a.top_k_value, k = _setting(top_k, rows, dev, torch.int32, "top_k", 0, 2 ** 62)
    a.top_p, a.top_p_value, p = _setting(top_p, rows, dev, torch.float32, "top_p", 0.0, 1.0)
    a.min_p, a.min_p_value, m = _setting(min_p, rows, dev, torch.float32, "min_p", 0.0, 1.0)
    _capi.require_cuda(logits, "sample_tokens")
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
    a.tokens = tokens.data_ptr()
    if return_logprobs:
        a.logprobs = logprobs.data_ptr()
    with _capi.on_device(dev):
        _capi.check(_capi.load().mxfp4_sample(ctypes.byref(a), _capi.stream_ptr(dev)), "mxfp4_sample")
    return (tokens, logprobs) if return_logprobs else tokens
