"""Quantized key/value cache for the attention of a language model (the text encoder's: grouped heads), and attention to it.

Keys and values are stored per token and KV head as 8-bit codes with one fp32 scale, in the arithmetic of the row quantizers
(`quantizers.quant_rows_i8` / `quant_rows`), in pages that sequences of any length share out among themselves:

    cache = kv_cache.alloc(pages=512, kv_heads=8, head_dim=128, page=64, kind="int8")
    rows = kv_cache.Rows(table, lens, starts)             # which rows of a call belong to which sequence, see Rows
    kv_cache.write(cache, k, v, rows)                     # quantize new tokens into their pages
    out = kv_cache.attention(q, cache, rows)              # their attention to everything their sequences hold
    out = kv_cache.attention_shared(q, cache, rows, prefix, n)   # behind one prefix that all sequences share
    k, v = kv_cache.read(cache, rows, total)              # back as bf16 rows

Nothing here has a backward pass: what `read` and the attentions return carries no gradient, whatever their inputs require.
`lens`, `starts` and the page table stay on the device and are read there, so a captured call follows them. The tensors of a call are on
the cache's device, and the work goes to that device's current stream. Everything is CUDA; there is no fallback.
"""
import struct
import threading
from dataclasses import dataclass

import torch

from . import _lib

FP8 = torch.float8_e4m3fn
PAGES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_KINDS = {"int8": (torch.int8, 0), "fp8": (FP8, 1)}

# rh3_kv_attn_args and rh3_kv_rows_args: the two tensors (pointer, token and head stride), the cache, the batch, then what the call adds
_TENSORS, _CACHE, _BATCH = struct.Struct("@PqqPqq"), struct.Struct("@PPPPqqqq"), struct.Struct("@PqqPPq")
_ATTN, _ROWS = struct.Struct("@qqPqqfiii"), struct.Struct("@qii")


class KVCache:
    """Codes k, v [pages, kv_heads, page, head_dim] (int8, or float8_e4m3fn) and scales k_scale, v_scale fp32 [pages, kv_heads, page],
    contiguous, on one CUDA device. page: 16, 32, 64 or 128 tokens; head_dim: 64 or 128. Codes are numbers (`write` stores no NaN of e4m3: rows that
    are not finite have codes 0). The tensors' contents may change, the tensors of an object may not: calls go by their addresses."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page", "head_dim", "kind", "device", "_index", "_args")

    def __init__(self, k, v, k_scale, v_scale):
        _lib.require_cuda(k, v, k_scale, v_scale)
        if k.ndim != 4 or k.dtype not in (torch.int8, FP8):
            raise RuntimeError(f"k: expected int8 or e4m3 codes [pages, kv_heads, page, head_dim], got {tuple(k.shape)} {k.dtype}")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise RuntimeError("v must have the shape and type of k")
        pages, kv_heads, page, head_dim = k.shape
        if page not in PAGES or head_dim not in HEAD_DIMS or pages < 1 or not 1 <= kv_heads <= 1024:
            raise RuntimeError(f"page must be one of {PAGES}, head_dim one of {HEAD_DIMS}: got a cache of {tuple(k.shape)}")
        for t in (k_scale, v_scale):
            if t.dtype != torch.float32 or t.shape != k.shape[:3]:
                raise RuntimeError("scales must be fp32 [pages, kv_heads, page]")
        for t in (k, v, k_scale, v_scale):
            if not t.is_contiguous() or t.data_ptr() % 16 or t.device != k.device:
                raise RuntimeError("the cache's tensors must be contiguous, 16-byte aligned and on one device")
        args = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        for name, x in zip(self.__slots__, (k, v, k_scale, v_scale, *k.shape, 0 if k.dtype == torch.int8 else 1, k.device, k.get_device(), args)):
            object.__setattr__(self, name, x)

    def __setattr__(self, name, value):
        if name in KVCache.__slots__ and value is not getattr(self, name):   # it is for `cache.v_scale *= 2`
            raise AttributeError(f"cannot assign {name}: calls go by the addresses of the tensors that the cache was made of")
        object.__setattr__(self, name, value)

    def __reduce__(self):   # a copy has its own tensors' addresses
        return type(self), (self.k, self.v, self.k_scale, self.v_scale)


def alloc(pages, kv_heads, head_dim=128, page=64, kind="int8", device="cuda"):
    """An empty cache of `pages` pages of `page` tokens; kind "int8" or "fp8" (e4m3)."""
    if kind not in _KINDS:
        raise RuntimeError(f"kind must be one of {tuple(_KINDS)}, got {kind!r}")
    shape = (pages, kv_heads, page, head_dim)
    k, v = (torch.zeros(shape, device=device, dtype=_KINDS[kind][0]) for _ in range(2))
    return KVCache(k, v, *(torch.zeros(shape[:3], device=device, dtype=torch.float32) for _ in range(2)))


@dataclass(frozen=True)
class Rows:
    """Which rows of a call belong to which sequence, int32 on the cache's device:
    table [B, P] the pages of each sequence in order (rows may be strided); lens [B] the tokens each sequence holds, the call's own
    among them; starts [B + 1], ascending: rows starts[b] .. starts[b + 1] - 1 of the call are the last tokens of sequence b,
    row t at position lens[b] - (starts[b + 1] - t).

    The values are not looked at on the host. Rows at or behind starts[B] (a padded batch) are left as they were; tokens that lie
    nowhere (before position 0, beyond the table, in a page the cache does not have) are not written, read as zeros and are
    masked, and a page the cache does not have is reported by `_lib.check_status()`. So are starts that do not ascend, by attention, which
    then computes nothing; which rows write and read take for a sequence's is open then."""
    table: torch.Tensor
    lens: torch.Tensor
    starts: torch.Tensor

    def __post_init__(self):
        table, lens, starts = self.table, self.lens, self.starts
        _lib.require_cuda(table, lens, starts)
        if not table.dtype == lens.dtype == starts.dtype == torch.int32:
            raise RuntimeError("table, lens and starts must be int32")
        if table.ndim != 2 or lens.ndim != 1 or starts.ndim != 1 or len(lens) != len(table) or len(starts) != len(lens) + 1 or len(lens) == 0:
            raise RuntimeError(f"expected table [B, P], lens [B], starts [B + 1] with B > 0, got {tuple(table.shape)}, {tuple(lens.shape)}, {tuple(starts.shape)}")
        if not (lens.is_contiguous() and starts.is_contiguous()) or (table.shape[1] > 1 and table.stride(1) != 1):
            raise RuntimeError("lens, starts and the rows of table must be contiguous")
        if (table.shape[0] > 1 and table.stride(0) < table.shape[1]) or not table.device == lens.device == starts.device:
            raise RuntimeError("the rows of table must not overlap, and all three must be on one device")
        object.__setattr__(self, "_index", table.get_device())
        object.__setattr__(self, "_sizes", (table.shape[1], len(lens)))
        object.__setattr__(self, "_args", _BATCH.pack(table.data_ptr(), max(table.stride(0), table.shape[1]), table.shape[1], lens.data_ptr(),
                                                      starts.data_ptr(), len(lens)))

    def __reduce__(self):   # as KVCache
        return type(self), (self.table, self.lens, self.starts)


# What the attention kernels need beside their arguments, per (device, stream), where only calls that cannot overlap share it: the counters,
# which are 0 between calls, and a workspace for calls that need little (for most, allocating one takes as long as the kernel).
_SCRATCH = {}
_lib.on_failed_status.append(_SCRATCH.clear)   # a call that was given up may leave its counters at anything
_KEPT_BYTES = 4 << 20
_KEPT_STREAMS = 64   # so many streams have them; behind these, the ones kept for longest are dropped (their memory goes back to their stream's)
_LAUNCH = threading.Lock()   # a call's kernels go to the stream together: another thread's would use the same workspace between them
_NEED = {}


def _scratch(device, index, stream, need):
    """(counters, workspace of `need` bytes) for a call on `stream`. A captured call gets its own, the counters cleared by the graph: a graph
    may be replayed on any stream."""
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.zeros(1024, device=device, dtype=torch.int32), torch.empty(need, device=device, dtype=torch.uint8)
    kept = _SCRATCH.get((index, stream))
    if kept is None:
        kept = torch.zeros(1024, device=device, dtype=torch.int32), torch.empty(_KEPT_BYTES, device=device, dtype=torch.uint8)
        with _LAUNCH:
            kept = _SCRATCH.setdefault((index, stream), kept)
            while len(_SCRATCH) > _KEPT_STREAMS:
                _SCRATCH.pop(next(iter(_SCRATCH), None), None)
    return kept if need <= _KEPT_BYTES else (kept[0], torch.empty(need, device=device, dtype=torch.uint8))


_PATHS = (None, False, True, "apart")


def use_wide(use):
    """Which kernel attention runs on: None (the default) the cheaper one for a call's sizes, False the one for few rows per sequence, True the one
    on 128-row tensor-core tiles; "apart": as False, and a shared prefix always has a pass of its own. For the whole process; returns
    the previous setting."""
    if not any(use is x for x in _PATHS[:3]) and use != "apart":
        raise RuntimeError(f"expected one of {_PATHS}, got {use!r}")
    before = _lib.lib().rh3_kv_attn_use_wide(_PATHS.index(use) - 1)
    _NEED.clear()
    return _PATHS[before + 1]


def _plan(*sizes):
    """(workspace bytes, kernels) of an attention call."""
    need = _NEED.get(sizes)
    if need is None:
        if len(_NEED) > 4096:
            _NEED.clear()
        need = _NEED[sizes] = _lib.lib().rh3_kv_attn_workspace_bytes(*sizes), _lib.lib().rh3_kv_attn_launches(*sizes)
    return need


def _run(index, fn):
    """fn() with device `index` current: the library works on the current device and its stream."""
    if index == torch._C._cuda_getDevice():
        return fn()
    with torch.cuda.device(index):
        return fn()


def _check_batch(cache, rows):
    if rows._index != cache._index:
        raise RuntimeError("the batch must be on the cache's device")


def _check_rows(x, name, cache, heads, types):
    """(pointer, token stride, head stride) of x [T, heads, head_dim]."""
    if x.get_device() != cache._index:
        raise RuntimeError(f"{name} must be a CUDA tensor on the cache's device; there is no CPU path")
    shape = x.shape
    if len(shape) != 3 or x.dtype not in types or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise RuntimeError(f"{name}: expected [T, {heads or 'heads'}, {cache.head_dim}] of {', '.join(str(t) for t in types)}, got {tuple(shape)} {x.dtype}")
    st, sh, unit = x.stride()
    ptr = x.data_ptr()
    per16 = 16 // x.element_size()
    if (unit != 1 or st % per16 or sh % per16 or ptr % 16) and x.numel():
        raise RuntimeError(f"{name}: the last dim must be contiguous and every row start on a 16-byte boundary")
    return ptr, st, sh


def _rows_overlap(t, heads, d, st, sh):
    """Whether two rows of d elements of a [t, heads] grid with these strides (not negative) share an element."""
    if t == 1 or heads == 1:
        return t * heads > 1 and (st if heads == 1 else sh) < d
    if sh >= d and st >= (heads - 1) * sh + d or st >= d and sh >= (t - 1) * st + d:   # rows of a token, or of a head, lie together
        return False
    if st < d or sh < d:
        return True
    # the token nearest to `far` is the one before it or the one behind
    return any(abs(i * st - far) < d for far in range(sh, heads * sh, sh) for i in (far // st, far // st + 1) if i < t)


def write(cache, k, v, rows):
    """Quantize k, v [T, kv_heads, head_dim] (bf16, fp16 or fp32, any token and head strides of whole 16 bytes) into the pages of
    their sequences. A row with a NaN or an infinity reads back as NaN. Sequences that share a page must not write the same token."""
    _check_batch(cache, rows)
    at = (*_check_rows(k, "k", cache, cache.kv_heads, tuple(_DTYPES)), *_check_rows(v, "v", cache, cache.kv_heads, (k.dtype,)))
    shape = k.shape
    if v.shape != shape:
        raise RuntimeError("k and v must have the same number of rows")
    t = shape[0]
    if t == 0:
        return
    args = _TENSORS.pack(*at) + cache._args + rows._args + _ROWS.pack(t, cache.kind, _DTYPES[k.dtype])
    _run(cache._index, lambda: _lib.call("rh3_kv_write", args, _lib.stream()))


def read(cache, rows, total, dtype=torch.bfloat16, out=None):
    """(k, v) [total, kv_heads, head_dim] of `dtype`: codes x scales of the tokens `rows` names, rounded once. Rows that no sequence
    has hold what `out` (a pair of contiguous tensors) held, or anything."""
    _check_batch(cache, rows)
    if dtype not in _DTYPES:
        raise RuntimeError(f"dtype must be one of {tuple(_DTYPES)}, got {dtype}")
    shape = (total, cache.kv_heads, cache.head_dim)
    if out is None:
        k, v = cache.k.new_empty(shape, dtype=dtype), cache.k.new_empty(shape, dtype=dtype)
    else:
        k, v = out
        for t in (k, v):
            if t.shape != shape or t.dtype != dtype or t.device != cache.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise RuntimeError(f"out: expected two contiguous, 16-byte aligned {dtype} tensors {shape} on the cache's device")
    if total == 0:
        return k, v
    args = _TENSORS.pack(k.data_ptr(), 0, 0, v.data_ptr(), 0, 0) + cache._args + rows._args + _ROWS.pack(total, cache.kind, _DTYPES[dtype])
    _run(cache._index, lambda: _lib.call("rh3_kv_read", args, _lib.stream()))
    return k, v


def _attend(q, cache, rows, prefix, prefix_len, scale, causal, out):
    _check_batch(cache, rows)
    at = _check_rows(q, "q", cache, None, (torch.bfloat16, torch.float16))
    t, heads, d = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise RuntimeError(f"{heads} query heads are not a multiple of the cache's {cache.kv_heads}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise RuntimeError("the softmax scale must be positive and finite")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        to = out.data_ptr(), heads * d, d
    else:
        to = _check_rows(out, "out", cache, heads, (q.dtype,))
        if out.shape != q.shape:
            raise RuntimeError("out must have the shape of q")
        if t and _rows_overlap(t, heads, d, to[1], to[2]):
            raise RuntimeError(f"out: rows must not overlap, got strides {out.stride()}")
    if t == 0:
        return out
    group = heads // cache.kv_heads
    pre, pre_pages = (0, 0) if prefix is None else (prefix.data_ptr(), prefix.numel())
    args = (_TENSORS.pack(*at, *to) + cache._args + rows._args
            + _ATTN.pack(t, group, pre, pre_pages, prefix_len, scale, cache.kind, _DTYPES[q.dtype], bool(causal)))

    def launch():
        stream = _lib.stream()
        need, kernels = _plan(cache.kv_heads, group, cache.page, d, *rows._sizes, t, prefix_len)
        counters, work = _scratch(q.device, cache._index, stream, need)
        with _LAUNCH:
            _lib.call("rh3_kv_attn", args, work.data_ptr(), need, counters.data_ptr(), stream, launches=kernels)

    _run(cache._index, launch)
    return out


def attention(q, cache, rows, scale=None, causal=True, out=None):
    """softmax(scale * q . k) v of new tokens q [T, heads, head_dim] (bf16 or fp16) over what their sequences hold in the cache.

    heads: a multiple of the cache's kv_heads (head h reads KV head h // group). causal: a token sees the tokens up to itself (the
    last one of its sequence sees all), else every token sees all of its sequence. A token that sees nothing gives 0. The call's own
    tokens are among what is seen: write them first. scale: 1 / sqrt(head_dim) unless given; out: a tensor like q to write to, whose rows do not overlap (q itself will do)."""
    return _attend(q, cache, rows, None, 0, scale, causal, out)


def attention_shared(q, cache, rows, prefix, prefix_len, scale=None, causal=True, out=None):
    """`attention` of a batch whose sequences all continue one cached prefix: its first `prefix_len` tokens lie in the pages `prefix`
    (int32, on the cache's device) and are seen by every token. `rows` describes the own parts alone (a length of 0 is a sequence
    that has nothing of its own). The prefix is read and multiplied once for the whole batch."""
    _lib.require_cuda(prefix)
    if prefix.dtype != torch.int32 or prefix.ndim != 1 or not prefix.is_contiguous() or prefix.device != cache.device:
        raise RuntimeError("prefix must be contiguous int32 [pages] on the cache's device")
    prefix_len = int(prefix_len)
    if not 0 <= prefix_len <= prefix.numel() * cache.page:
        raise RuntimeError(f"a prefix of {prefix_len} tokens does not fit {prefix.numel()} pages of {cache.page}")
    return _attend(q, cache, rows, prefix, prefix_len, scale, causal, out)
