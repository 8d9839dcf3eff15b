"""A paged 4-bit key/value cache: appending to it, attention over it, eviction from it.

For serving, where the cache is what a step reads: keys and values are held in 4 bits with a
scale and a zero for every 32, 64 or 128 channels, a quarter to a third of their 16-bit size.

    cache = KV4Cache.empty(num_pages=4096, heads=8, page_size=64, group=64)
    kv4_append(cache, k, v, page_table, lengths)           # prompt or new token, [B, T, H, 128]
    lengths = lengths + T
    o = kv4_attention(q, cache, page_table, lengths, decay=1.0)   # [B, T, heads_q, 128]
    src, lengths = kv4_evict_select(cache, page_table, lengths, keep, recent=256, seen=seen)
    kv4_evict_move(cache, page_table, src)

Slot i of sequence b is in page page_table[b, i // page_size]; lengths[b] slots hold tokens. Both
are int32 tensors on the cache's device that the caller keeps: the layers of a model share them,
so no call changes them. A prompt is appended and attended to with all of its tokens in one call,
causal among them; kv4_expand gives a range of the cache in 16 bits to whatever else needs it.

As with attention_forward, calls only enqueue work on the current stream, and the arithmetic is
the library's own kernels. What the device tensors may hold wrong (a page outside the pool, a
length past the table) cannot be seen before the launch: the kernels skip it and report it
through device_status() (include/llm_fa_b200.h names the codes).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from .attention import HEAD_DIM, _strides3

PAGE_SIZES = (16, 32, 64, 128, 256)
GROUPS = (32, 64, 128)
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_DTYPES = {torch.bfloat16: _lib.LLMFA_BF16, torch.float16: _lib.LLMFA_FP16}


def page_bytes(page_size: int, group: int) -> int:
    """Bytes of one page of one head."""
    return _size("llmfa_kv4_page_bytes", int(page_size), int(group))


class KV4Cache:
    """The pool: `pages` uint8 [num_pages, heads, page_bytes], `positions` int32 and `weights`
    fp32 [num_pages, heads, page_size], all contiguous on one device.

    positions holds where a token was appended, weights the attention weight that it has
    accumulated (kv4_attention with decay); eviction reads both.
    """

    def __init__(self, pages: torch.Tensor, positions: torch.Tensor, weights: torch.Tensor, *,
                 page_size: int = 64, group: int = 64):
        if page_size not in PAGE_SIZES:
            raise RuntimeError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if group not in GROUPS:
            raise RuntimeError(f"group must be one of {GROUPS}, got {group}")
        if pages.dim() != 3 or pages.dtype != torch.uint8 or 0 in pages.shape:
            raise RuntimeError("pages must be uint8 [num_pages, heads, page_bytes], got "
                               f"{pages.dtype} {tuple(pages.shape)}")
        if pages.shape[2] != page_bytes(page_size, group):
            raise RuntimeError(f"a page of {page_size} tokens with group {group} has "
                               f"{page_bytes(page_size, group)} bytes, got {pages.shape[2]}")
        want = (*pages.shape[:2], page_size)
        for t, nm, dt in ((positions, "positions", torch.int32), (weights, "weights", torch.float32)):
            if t.shape != want or t.dtype != dt:
                raise RuntimeError(f"{nm} must be {dt} {want}, got {t.dtype} {tuple(t.shape)}")
        for t, nm in ((pages, "pages"), (positions, "positions"), (weights, "weights")):
            if not t.is_cuda or t.device != pages.device:
                raise RuntimeError(f"{nm} must be a CUDA tensor on the pool's device "
                                   "(there is no CPU path)")
            if not t.is_contiguous():
                raise RuntimeError(f"{nm} must be contiguous")
        # read-only from here on: the C struct holds their addresses
        self._pages, self._positions, self._weights = pages, positions, weights
        self.page_size, self.group = page_size, group
        self._device, self._index = pages.device, pages.get_device()
        self._heads = pages.shape[1]
        self._c = _lib.Kv4Cache(pages.data_ptr(), positions.data_ptr(), weights.data_ptr(),
                                pages.shape[0], pages.shape[1], page_size, group)

    @classmethod
    def empty(cls, num_pages: int, heads: int, *, page_size: int = 64, group: int = 64,
              device: torch.device | int | str | None = None) -> "KV4Cache":
        """A pool of zeros on `device` (default: the current one)."""
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else (
            torch.device("cuda", device) if isinstance(device, int) else torch.device(device))
        shape = (num_pages, heads)
        return cls(torch.zeros(*shape, page_bytes(page_size, group), dtype=torch.uint8, device=dev),
                   torch.zeros(*shape, page_size, dtype=torch.int32, device=dev),
                   torch.zeros(*shape, page_size, dtype=torch.float32, device=dev),
                   page_size=page_size, group=group)

    @property
    def pages(self) -> torch.Tensor:
        return self._pages

    @property
    def positions(self) -> torch.Tensor:
        return self._positions

    @property
    def weights(self) -> torch.Tensor:
        return self._weights

    @property
    def device(self) -> torch.device:
        return self._device

    @property
    def heads(self) -> int:
        return self._heads


# A step of a small batch costs a few microseconds on the GPU, so the checks below read each
# property of a tensor once.

def _ints(t: torch.Tensor, name: str, cache: KV4Cache, batch: int) -> int:
    if t.dtype != torch.int32 or t.dim() != 1 or t.size(0) != batch or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous int32 of shape ({batch},), got {t.dtype} "
                           f"{tuple(t.shape)}")
    if t.get_device() != cache._index:
        raise RuntimeError(f"{name} is on {t.device}, expected {cache._device}")
    return t.data_ptr()


def _seqs(cache: KV4Cache, page_table: torch.Tensor, lengths: torch.Tensor | None) -> _lib.Kv4Seqs:
    shape = page_table.shape
    if len(shape) != 2 or page_table.dtype != torch.int32 or 0 in shape:
        raise RuntimeError("page_table must be int32 [batch, max_pages], got "
                           f"{page_table.dtype} {tuple(shape)}")
    if page_table.get_device() != cache._index:
        raise RuntimeError(f"page_table is on {page_table.device}, expected {cache._device}")
    batch, width = shape
    row, col = page_table.stride()
    if width > 1 and col != 1:
        raise RuntimeError("page_table rows must be contiguous (stride 1)")
    if batch > 1 and row < width:
        raise RuntimeError("page_table rows must not overlap")
    return _lib.Kv4Seqs(page_table.data_ptr(), row, width,
                        None if lengths is None else _ints(lengths, "lengths", cache, batch), batch)


def _rows(t: torch.Tensor, name: str, cache: KV4Cache, batch: int, heads: int | None,
          like: torch.Tensor | None = None):
    """Checks one [batch, tokens, heads, 128] tensor of 16-bit values; (shape, strides)."""
    shape, stride = t.shape, t.stride()
    if t.get_device() != cache._index:
        raise RuntimeError(f"{name} is on {t.device}, expected {cache._device}")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    if len(shape) != 4 or shape[3] != HEAD_DIM or shape[0] != batch or (
            heads is not None and shape[2] != heads):
        raise RuntimeError(f"{name} must be [{batch}, tokens, {heads or 'heads'}, {HEAD_DIM}], got "
                           f"shape {tuple(shape)}")
    if shape[1] == 0 or shape[2] == 0:
        raise RuntimeError(f"empty {name} is not supported")
    if stride[3] != 1:
        raise RuntimeError(f"{name} head dim must be contiguous (stride 1)")
    if like is not None and (shape != like.shape or t.dtype != like.dtype):
        raise RuntimeError(f"{name} must be {like.dtype} {tuple(like.shape)}, got {t.dtype} "
                           f"{tuple(shape)}")
    return shape, _strides3(stride)


def _call(cache: KV4Cache, name: str, *args) -> None:
    """One library call on the cache's device and its current stream (the last argument)."""
    index = cache._index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch.cuda.current_device() == index:
        rc = getattr(_lib.lib(), name)(cache._c, *args, stream)
    else:  # the library launches on the current device
        with torch.cuda.device(index):
            rc = getattr(_lib.lib(), name)(cache._c, *args, stream)
    if rc != _lib.LLMFA_OK:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=256)
def _size(name: str, *args: int) -> int:
    """A workspace size of the library."""
    out = ctypes.c_uint64(0)
    _lib.check(getattr(_lib.lib(), name)(*args, ctypes.byref(out)), name)
    return int(out.value)


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               lengths: torch.Tensor, *, counts: torch.Tensor | None = None,
               seen: torch.Tensor | None = None) -> None:
    """Quantise k, v [batch, tokens, heads, 128] into slots lengths[b] .. of each sequence.

    counts (int32 [batch], default: tokens) says how many of its rows are real; the rest are not
    read. seen (int32 [batch], default: lengths) is the position of the first new token, which
    differs from lengths once tokens were evicted. lengths itself is not changed.
    """
    seqs = _seqs(cache, page_table, lengths)
    B = seqs.batch
    shape, ks = _rows(k, "k", cache, B, cache._heads)
    _, vs = _rows(v, "v", cache, B, cache._heads, like=k)
    _call(cache, "llmfa_kv4_append", seqs, k.data_ptr(), ks, v.data_ptr(), vs,
          None if counts is None else _ints(counts, "counts", cache, B),
          None if seen is None else _ints(seen, "seen", cache, B), shape[1], _DTYPES[k.dtype])


def kv4_expand(cache: KV4Cache, page_table: torch.Tensor, start: torch.Tensor, tokens: int, *,
               counts: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
               out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """(k, v) [batch, tokens, heads, 128] of slots start[b] .. start[b] + counts[b] - 1 (counts
    default: tokens); rows past a count are zeros. With `out`, fills and returns that pair, which
    may share no element."""
    seqs = _seqs(cache, page_table, start)
    B = seqs.batch
    if out is None:
        if dtype not in _DTYPES or tokens < 1:
            raise RuntimeError("kv4_expand needs tokens >= 1 and bfloat16 or float16, got "
                               f"{tokens}, {dtype}")
        k = torch.empty(B, tokens, cache._heads, HEAD_DIM, dtype=dtype, device=cache._device)
        v = torch.empty_like(k)
        ks = vs = _strides3(k.stride())
    else:
        k, v = out
        shape, ks = _rows(k, "k", cache, B, cache._heads)
        _, vs = _rows(v, "v", cache, B, cache._heads, like=k)
        if shape[1] != tokens:
            raise RuntimeError(f"out holds {shape[1]} tokens, expected {tokens}")
    _call(cache, "llmfa_kv4_expand", seqs, k.data_ptr(), ks, v.data_ptr(), vs,
          None if counts is None else _ints(counts, "counts", cache, B), tokens, _DTYPES[k.dtype])
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, page_table: torch.Tensor,
                  lengths: torch.Tensor, *, counts: torch.Tensor | None = None,
                  causal: bool = True, softmax_scale: float | None = None,
                  decay: float | None = None, out: torch.Tensor | None = None,
                  return_lse: bool = False):
    """softmax(q k^T * softmax_scale) v of the last tokens of each sequence over its cache.

    q is [batch, tokens, heads_q, 128], heads_q a multiple of the cache's heads; lengths counts
    the new tokens, which were appended before. counts (int32 [batch], default: tokens) says how
    many of its rows are real: they are the last counts[b] tokens of the sequence. With causal,
    each sees the slots up to its own, otherwise all. A row that sees nothing gives zeros and an
    lse of -inf. Rows past a count are left as they were in `out`; without `out` they are zeros.
    `out` may share a tensor with q, as another slice of it, but no element.

    decay (0 to 1) also tracks the weight that each token received: cache.weights becomes
    decay * cache.weights + the softmax weights of this call, summed over the new tokens and the
    query heads that share a key head. 1.0 accumulates; 0.0 stores this call's sums alone. The
    sequences of such a call share no pages: their sums would overwrite one another.

    softmax_scale defaults to 1/sqrt(128). With return_lse, returns (O, lse): the natural-log
    log-sum-exp of every row, fp32 [batch, heads_q, tokens].
    """
    seqs = _seqs(cache, page_table, lengths)
    B = seqs.batch
    shape, qs = _rows(q, "q", cache, B, None)
    T, Hq = shape[1], shape[2]
    if Hq % cache._heads != 0:
        raise RuntimeError(f"q has {Hq} heads, not a multiple of the cache's {cache._heads}")
    if decay is None:
        decay = -1.0
    elif not 0.0 <= decay <= 1.0:
        raise RuntimeError(f"decay must be between 0 and 1, got {decay}")
    n = None if counts is None else _ints(counts, "counts", cache, B)
    fill = 0 if counts is None else _lib.LLMFA_KV4_FILL_LSE
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = _strides3(out.stride())
        fill |= _lib.LLMFA_KV4_FILL_OUT
    else:
        _, os = _rows(out, "out", cache, B, Hq, like=q)
        if out.data_ptr() == q.data_ptr():
            raise RuntimeError("out must not be q itself")
    nbytes = _size("llmfa_kv4_attention_workspace_size", B, cache._heads, Hq, T,
                   0 if decay < 0 else seqs.max_pages * cache.page_size)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cache._device)
    lse = ls = None
    if return_lse:
        lse = torch.empty(B, Hq, T, dtype=torch.float32, device=cache._device)
        ls = _lib.strides2((Hq * T, T))
    _call(cache, "llmfa_kv4_attention", seqs, q.data_ptr(), qs, out.data_ptr(), os,
          lse.data_ptr() if return_lse else None, ls, n, Hq, T, bool(causal),
          _SCALE if softmax_scale is None else float(softmax_scale), decay, fill,
          _DTYPES[q.dtype],
          ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out


def kv4_evict_select(cache: KV4Cache, page_table: torch.Tensor, lengths: torch.Tensor, keep: int,
                     *, recent: int = 0, seen: torch.Tensor | None = None):
    """What cutting every sequence to `keep` slots would leave where: (src, new_lengths).

    Of every head the lengths[b] - keep tokens of least weight go (lowest slot first among
    equals, NaN last), those at the `recent` latest positions after all others; seen (int32
    [batch], default: lengths) is how many tokens a sequence has been given in all. src (int32
    [batch, heads, keep]) names for each slot that stays the slot whose token it will hold, -1
    past the new length; freed slots take the survivors from above `keep` in order.
    """
    seqs = _seqs(cache, page_table, lengths)
    B = seqs.batch
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise RuntimeError(f"keep must be at least 1 and recent 0 to keep, got {keep}, {recent}")
    nbytes = _size("llmfa_kv4_evict_workspace_size", B, cache._heads, keep)
    src = torch.empty(B, cache._heads, keep, dtype=torch.int32, device=cache._device)
    new = torch.empty(B, dtype=torch.int32, device=cache._device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cache._device)
    _call(cache, "llmfa_kv4_evict_select", seqs,
          None if seen is None else _ints(seen, "seen", cache, B), keep, recent, src.data_ptr(),
          new.data_ptr(), ws.data_ptr(), nbytes)
    return src, new


def kv4_evict_move(cache: KV4Cache, page_table: torch.Tensor, src: torch.Tensor) -> None:
    """Make the moves that kv4_evict_select chose (codes, scales, positions and weights)."""
    seqs = _seqs(cache, page_table, None)
    shape = src.shape
    if len(shape) != 3 or shape[0] != seqs.batch or shape[1] != cache._heads or shape[2] == 0 \
            or src.dtype != torch.int32 or not src.is_contiguous():
        raise RuntimeError(f"src must be contiguous int32 [{seqs.batch}, {cache._heads}, keep], got "
                           f"{src.dtype} {tuple(shape)}")
    if src.get_device() != cache._index:
        raise RuntimeError(f"src is on {src.device}, expected {cache._device}")
    _call(cache, "llmfa_kv4_evict_move", seqs, src.data_ptr(), shape[2])
