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
import struct
from typing import Optional, Tuple, Union

import torch

from . import _capi

_status = {}                     # device index -> int32 status word of the serving kernels
_DT16 = {torch.bfloat16: 0, torch.float16: 1}
_workspace_bytes = {}            # device and sizes of a paged_attention call -> bytes of its workspace

# The argument structures as one pack() each: setting forty ctypes fields one by one costs more than a small kernel runs.
# Fields in the order of the C structs, with the compiler's own padding ("x"); sizes are compared on import.
_ROPE = struct.Struct("@i4xP2qP2qP2qP2qP3qP3qPPPdqqiiiiiiP")
_ATTN = struct.Struct("@i4xP2qP2qPP3qP3qPqPPPPqqqqqiiiidi4xPqP")
_SAMPLE = struct.Struct("@Pi4xqqqPPdPqPdPdPP")
assert (_ROPE.size, _ATTN.size, _SAMPLE.size) == tuple(ctypes.sizeof(t) for t in (_capi.RopeAppendArgs, _capi.PagedAttentionArgs, _capi.SampleArgs))


def _status_pointer(device: torch.device) -> int:
    st = _status.get(device.index)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            raise _capi.MXFP4BackendError("mxfp4: the first serving call on a device allocates its status word; make one call before the capture")
        st = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()      # other streams may use the word from here on
        st = _status.setdefault(device.index, st)
    return st.data_ptr()


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
    if t.dtype != dtype or t.device != device or t.shape != shape:
        raise ValueError(f"mxfp4: {name} must be {dtype} of shape {tuple(shape)} on {device} (got {t.dtype}, {tuple(t.shape)}, {t.device})")
    return t if t.is_contiguous() else t.contiguous()


def _strides(t: torch.Tensor, shape, name, written=False):
    """Element strides of all dimensions but the last, which must be contiguous."""
    st = t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"mxfp4: the last dimension of {name} must be contiguous")
    if written and 0 in st and any(x == 0 and n > 1 for x, n in zip(st, shape)):
        raise ValueError(f"mxfp4: {name} must not be a broadcast view")
    return st[:-1]


def _match(t: torch.Tensor, shape, dtype, device, name):
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"mxfp4: {name} must be {dtype} of shape {tuple(shape)} on {device} (got {t.dtype}, {tuple(t.shape)}, {t.device})")


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
        """Slots of the places [batch, n] (0 is a sequence's first own token) through block tables [batch, pages].  A place outside
        its table gets the slot behind the cache's end, which rope_append reports."""
        places = places.long()
        page = torch.div(places, self.page_size, rounding_mode="floor")
        inside = (page >= 0) & (page < block_tables.shape[1])
        slots = block_tables.long().gather(1, torch.where(inside, page, 0)) * self.page_size + places % self.page_size
        return torch.where(inside, slots, self.num_pages * self.page_size)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, positions: torch.Tensor,
                slots: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False, scaling: float = 1.0,
                q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns q [tokens, heads, D] and k [tokens, kv_heads, D] by their positions, stores the turned k and the v at `slots` of
    the caches [pages, kv_heads, page_size, D], and returns the turned q (in q_out, which may be q itself).

    Pair i of the first 2 * len(inv_freq) elements of a head turns by positions * inv_freq[i] (float64, see rope_frequencies);
    pairs are (i, i + half), or (2i, 2i + 1) when interleaved; `scaling` multiplies the turned elements, the others stay as they
    are.  positions and slots are int64 [tokens]; a negative slot stores nothing; the slots of a call must differ.  q, k and v
    may be views of one projection's output; any strides, the last dimension contiguous.  bfloat16, float16 or float32."""
    dev, dtype = q.device, q.dtype
    dt = _capi.DT.get(dtype)
    if dt is None:
        raise ValueError(f"mxfp4: rope_append takes bfloat16, float16 or float32 (got {dtype})")
    shape, k_shape, cache = q.shape, k.shape, k_cache.shape
    if len(shape) != 3 or len(k_shape) != 3 or len(cache) != 4:
        raise ValueError("mxfp4: q and k must be [tokens, heads, head_dim], the caches [pages, kv_heads, page_size, head_dim]")
    n, heads, dim = shape
    kv, pages, page_size, rotary = k_shape[1], cache[0], cache[2], 2 * inv_freq.numel()
    _match(k, (n, kv, dim), dtype, dev, "k")
    _match(v, k_shape, dtype, dev, "v")
    _match(k_cache, (pages, kv, page_size, dim), dtype, dev, "k_cache")
    _match(v_cache, cache, dtype, dev, "v_cache")
    if q_out is None:
        q_out = torch.empty(shape, dtype=dtype, device=dev)
    else:
        _match(q_out, shape, dtype, dev, "q_out")
    if rotary > dim:
        raise ValueError(f"mxfp4: inv_freq must be one value per pair of at most {dim} elements")
    positions, slots = _on(positions, dev, torch.int64, (n,), "positions"), _on(slots, dev, torch.int64, (n,), "slots")
    inv_freq = _on(inv_freq, dev, torch.float64, (rotary // 2,), "inv_freq")
    q_st, k_st, v_st, o_st = _strides(q, shape, "q"), _strides(k, k_shape, "k"), _strides(v, k_shape, "v"), _strides(q_out, shape, "q_out", True)
    kc_st, vc_st = _strides(k_cache, cache, "k_cache", True), _strides(v_cache, cache, "v_cache", True)
    _capi.require_cuda(q, "rope_append")
    if n == 0:
        return q_out
    args = _ROPE.pack(dt, q.data_ptr(), *q_st, k.data_ptr(), *k_st, v.data_ptr(), *v_st, q_out.data_ptr(), *o_st, k_cache.data_ptr(), *kc_st,
                      v_cache.data_ptr(), *vc_st, positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr(), scaling, n, pages, heads, kv, dim,
                      rotary, bool(interleaved), page_size, _status_pointer(dev))
    with _capi.on_device(dev):
        _capi.check(_capi.load().mxfp4_rope_append(args, _capi.stream_ptr(dev)), "mxfp4_rope_append")
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
    dev, dtype = q.device, q.dtype
    dt = _DT16.get(dtype)
    if dt is None:
        raise ValueError(f"mxfp4: paged_attention takes bfloat16 or float16 (got {dtype})")
    shape, cache, tables = q.shape, k_cache.shape, block_tables.shape
    if len(shape) != 3 or len(cache) != 4 or len(tables) != 2:
        raise ValueError("mxfp4: q must be [tokens, heads, head_dim], the caches [pages, kv_heads, page_size, head_dim], block_tables [batch, pages]")
    n, heads, dim = shape
    pages, kv, page_size, _ = cache
    batch, table_pages = tables
    _match(k_cache, (pages, kv, page_size, dim), dtype, dev, "k_cache")
    _match(v_cache, cache, dtype, dev, "v_cache")
    _match(block_tables, tables, torch.int32, dev, "block_tables")
    seq_lens = _on(seq_lens, dev, torch.int32, (batch,), "seq_lens")
    table_st = block_tables.stride()
    if table_pages > 1 and table_st[1] != 1:
        block_tables = block_tables.contiguous()
        table_st = block_tables.stride()
    starts_ptr = pre_ptr = pre_len_ptr = pre_pages = lse_ptr = 0
    fill = False
    if q_starts is not None:
        q_starts = _on(q_starts, dev, torch.int32, (batch + 1,), "q_starts")
        starts_ptr, fill = q_starts.data_ptr(), out is None
    if prefix_pages is not None or prefix_len is not None:
        if prefix_pages is None or prefix_len is None or prefix_pages.dim() != 1:
            raise ValueError("mxfp4: prefix_pages (one list of pages) and prefix_len come together")
        pre_pages = prefix_pages.shape[0]
        prefix_pages, prefix_len = _on(prefix_pages, dev, torch.int32, (pre_pages,), "prefix_pages"), _on(prefix_len, dev, torch.int32, (1,), "prefix_len")
        pre_ptr, pre_len_ptr = prefix_pages.data_ptr(), prefix_len.data_ptr()
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    else:
        _match(out, shape, dtype, dev, "out")
    q_st, o_st = _strides(q, shape, "q"), _strides(out, shape, "out", True)
    k_st, v_st = _strides(k_cache, cache, "k_cache", True), _strides(v_cache, cache, "v_cache", True)
    _capi.require_cuda(q, "paged_attention")
    lse = None
    if return_lse:
        lse = torch.empty(n, heads, dtype=torch.float32, device=dev)
        lse_ptr = lse.data_ptr()
    if n > 0:
        L = _capi.load()
        fixed = (dt, q.data_ptr(), *q_st, out.data_ptr(), *o_st, lse_ptr, k_cache.data_ptr(), *k_st, v_cache.data_ptr(), *v_st, block_tables.data_ptr(),
                 table_st[0], seq_lens.data_ptr(), starts_ptr, pre_ptr, pre_len_ptr, batch, n, pages, table_pages, pre_pages, heads, kv, dim, page_size,
                 dim ** -0.5 if scale is None else scale, fill)
        with _capi.on_device(dev):
            sizes = (dev.index, batch, n, pages, table_pages, pre_pages, heads, kv, dim, page_size, starts_ptr != 0, pre_ptr != 0)
            nbytes = _workspace_bytes.get(sizes)
            if nbytes is None:
                nbytes = L.mxfp4_paged_attention_workspace_bytes(_ATTN.pack(*fixed, 0, 0, 0))
                if nbytes < 0:
                    _capi.check(int(nbytes), "mxfp4_paged_attention")
                if len(_workspace_bytes) >= 4096:
                    _workspace_bytes.clear()
                _workspace_bytes[sizes] = nbytes
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            _capi.check(L.mxfp4_paged_attention(_ATTN.pack(*fixed, workspace.data_ptr(), nbytes, _status_pointer(dev)), _capi.stream_ptr(dev)),
                        "mxfp4_paged_attention")
    return (out, lse) if return_lse else out


def _setting(value, rows, dev, dtype, name, high):
    """(pointer, number, the tensor to keep alive) of a per-row tensor or one number for all rows."""
    if isinstance(value, torch.Tensor):
        t = _on(value, dev, dtype, (rows,), name)
        return t.data_ptr(), 0, t
    if not 0 <= value <= high:
        raise ValueError(f"mxfp4: {name} must lie between 0 and {high} (got {value})")
    return 0, value, None


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
    if dt is None:
        raise ValueError(f"mxfp4: sample_tokens takes bfloat16, float16 or float32 logits (got {logits.dtype})")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError("mxfp4: logits must be [rows, vocab]")
    rows, vocab = logits.shape
    pitch, step = logits.stride()
    if (vocab > 1 and step != 1) or (rows > 1 and pitch < vocab):
        logits = logits.contiguous()
        pitch = vocab
    uniforms = _on(uniforms, dev, torch.float32, (rows,), "uniforms")
    heat = _setting(temperature, rows, dev, torch.float32, "temperature", math.inf)
    most = _setting(top_k, rows, dev, torch.int32, "top_k", 2 ** 62)
    mass = _setting(top_p, rows, dev, torch.float32, "top_p", 1.0)
    least = _setting(min_p, rows, dev, torch.float32, "min_p", 1.0)
    _capi.require_cuda(logits, "sample_tokens")
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev) if return_logprobs else None
    args = _SAMPLE.pack(logits.data_ptr(), dt, rows, vocab, pitch if rows > 1 else vocab, uniforms.data_ptr(), heat[0], heat[1], most[0], int(most[1]),
                        mass[0], mass[1], least[0], least[1], tokens.data_ptr(), logprobs.data_ptr() if return_logprobs else 0)
    with _capi.on_device(dev):
        _capi.check(_capi.load().mxfp4_sample(args, _capi.stream_ptr(dev)), "mxfp4_sample")
    return (tokens, logprobs) if return_logprobs else tokens
