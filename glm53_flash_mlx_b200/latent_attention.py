"""Latent attention over a paged cache, on B200.

The attention between a layer's block-FP8 projections (the latent projection
``[latent + rope, hidden]`` and the output projection that
``DSAOutputProjection`` runs): every token leaves one shared latent row and
one rotary row in a paged cache, and all heads read them.

    plan = plan_pages(cached, new, table, free_pages, free_count, page_size=64, tokens=T)
    q_rope = latent_cache_write(kv, cache, plan.slots, norm_weight=w, positions=plan.positions,
                                inv_freq=inv_freq, queries=q[..., 192:])
    out = latent_attention_absorbed(q_latent, q_rope, cache, table, plan.seq_lens, scale=scale,
                                    query_starts=plan.query_starts)          # decode
    out = latent_attention_expanded(q[..., :192], q_rope, kv_b[..., :192], cache_rope, kv_b[..., 192:],
                                    plan.query_starts, key_starts, scale=scale)   # prefill

Tensors are BF16 or FP16.  Scores, maxima, sums and results are FP32 until the
result is rounded; in between the tensor cores take the softmax weights in the
tensors' type, one rounding more each (their sum takes them unrounded), so the
error against exact results is up to 1.4 times that of a 32-bit form.
Lengths, tables and plans stay on the device: no call reads them back, so each
can be captured into a CUDA graph after one eager call of any of them on the
device.  Errors that only the device can see (a page id outside the cache, a
plan that does not fit) set a status word: the call leaves its documented safe
result and the next call of this module raises (``IndexError`` /
``RuntimeError``); ``check_latent_status()`` synchronises and raises at once.
A call under capture raises too, but leaves the word to the next eager one.
"""

from __future__ import annotations

import functools
import struct
from typing import NamedTuple

import torch

from . import _native as N
from .packed import StatusWord, _SYNC_STATUS, _raise_status

_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_FP16}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None

# device index -> (status word, its address, the mirror's address, the mirror)
_STATUS: dict[int, tuple] = {}


def _status(index: int) -> tuple:
    entry = _STATUS.get(index)
    if entry is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a latent-attention operator once on this device before capturing it")
        sw = StatusWord(torch.device("cuda", index))
        torch.cuda.current_stream(index).synchronize()  # cleared before a call on any stream sets it
        entry = _STATUS[index] = (sw, sw.word.data_ptr(), sw.host.data_ptr(), sw._host_word)
    return entry


def check_latent_status(device: torch.device | int | None = None) -> None:
    """Synchronise and raise for any device-side error of this module's calls so far."""
    if isinstance(device, int):
        index = device
    else:
        index = None if device is None else torch.device(device).index
    entry = _STATUS.get(torch.cuda.current_device() if index is None else index)
    if entry is not None:
        entry[0].check()


def _device(first: torch.Tensor, *rest: torch.Tensor | None) -> int:
    """The CUDA device index that all tensors share; raises as ``require_cuda`` does otherwise."""
    index = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        N.require_cuda(first, *rest)
        raise ValueError("tensors on different devices")
    return index


class _Entry:
    """One C-ABI entry point, called through ``glm53_latent_call``: a word per argument (``floats`` names the
    positions that hold floating-point values; 0 stands for NULL) costs a third of converting each of them."""

    def __init__(self, number: int, count: int, floats: tuple = ()):
        self.number = number
        # three more words: status, its mirror, the stream
        self.pack = struct.Struct("".join("d" if i in floats else "q" for i in range(count + 3))).pack

    def __call__(self, index: int, *args) -> None:
        """Call on the device's current stream with its status word, whatever the current device is."""
        sw, word, host, mirror = _status(index)
        if mirror.value:
            if torch.cuda.is_current_stream_capturing():
                _raise_status(mirror.value & 0xFFFFFFFF)  # a capture can neither wait for the device nor clear the word
            sw.raise_pending()
        lib = N._lib or N.lib()
        stream = _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream
        words = self.pack(*args, word, host, stream)
        if torch.cuda.current_device() == index:
            rc = lib.glm53_latent_call(self.number, words)
        else:
            with torch.cuda.device(index):
                rc = lib.glm53_latent_call(self.number, words)
        if rc:
            N.check(rc, "glm53_latent_call")
        if _SYNC_STATUS:
            sw.check()


_PLAN_PAGES = _Entry(0, 16)
_CACHE_WRITE = _Entry(1, 19, floats=(7,))
_ABSORBED = _Entry(2, 26, floats=(20,))
_EXPANDED = _Entry(3, 29, floats=(24,))


def _int32(t: torch.Tensor, name: str, count: int) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != count:
        raise ValueError(f"{name} must be int32 [{count}], got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be BF16 or FP16, got {t.dtype}")
    return code


def _same(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _pieces(t: torch.Tensor) -> tuple:
    """(tensor, address, strides but the last): `t` itself where its rows can be read in 16-byte pieces, else a
    contiguous copy."""
    *outer, last = t.stride()
    ptr = t.data_ptr()
    if last == 1 and not ptr & 15:
        for s in outer:
            if s <= 0 or s & 7:
                break
        else:
            return t, ptr, outer
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.stride()[:-1]


def _table(t: torch.Tensor, requests: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] != requests:
        raise ValueError(f"block_table must be int32 [{requests}, pages], got {t.dtype} {list(t.shape)}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses that `t`'s elements lie in."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _output(out: torch.Tensor | None, shape: tuple, like: torch.Tensor, *rest: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return like.new_empty(shape)
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    _same(out, "out", like.dtype, shape)
    a, b = _span(out)
    for t in (like, *rest):
        if t is not None:
            c, d = _span(t)
            if a < d and c < b:
                raise ValueError("out must not overlap an input")
    return out


@functools.lru_cache(maxsize=4096)
def _absorbed_bytes(T: int, H: int, R: int, index: int) -> int:
    with torch.cuda.device(index):
        return N.lib().glm53_latent_absorbed_workspace_bytes(T, H, R)


class PagePlan(NamedTuple):
    """Where a batch's new tokens go: ``slots`` int64 and ``positions`` int32 per token (slot -1 and
    position 0 behind the last), ``query_starts`` int32 [requests + 1], ``seq_lens`` int32 [requests]
    (cached + new) and ``free_count`` int32 [1], the free pages left."""

    slots: torch.Tensor
    positions: torch.Tensor
    query_starts: torch.Tensor
    seq_lens: torch.Tensor
    free_count: torch.Tensor


def plan_pages(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
               free_pages: torch.Tensor, free_count: torch.Tensor, *, page_size: int, tokens: int) -> PagePlan:
    """Give every request's new tokens their cache rows, in one launch.

    ``cached_lens`` / ``new_lens`` int32 [requests] (up to 8192); ``block_table``
    int32 [requests, width], updated in place with the pages that are taken, in
    request order, from the end of ``free_pages[:free_count]``; ``tokens`` is the
    length of the per-token outputs (a captured graph's padded batch).  A plan
    that does not fit plans nothing (every slot -1, every start 0, the table
    untouched) and sets the status word.  Pass the returned ``free_count`` to the
    next call; to release pages, write their ids behind it and add their number.
    """
    B = cached_lens.numel()
    cached_lens = _int32(cached_lens, "cached_lens", B)
    new_lens = _int32(new_lens, "new_lens", B)
    _table(block_table, B)
    width = block_table.shape[1]
    stride, step = block_table.stride()
    if width > 1 and step != 1:
        raise ValueError("block_table is updated in place: its rows must be contiguous")
    if B <= 1:
        stride = width
    elif stride < width:
        raise ValueError("block_table is updated in place: its rows must not overlap")
    pages = free_pages.numel()
    free_pages = _int32(free_pages, "free_pages", pages)
    free_count = _int32(free_count, "free_count", 1)
    if page_size < 1 or tokens < 0:
        raise ValueError(f"page_size {page_size} and tokens {tokens} must be positive")
    index = _device(cached_lens, new_lens, block_table, free_pages, free_count)
    slots = cached_lens.new_empty(tokens, dtype=torch.int64)
    words = cached_lens.new_empty(tokens + 2 * B + 2)
    positions, starts, lens, left = words.split_with_sizes([tokens, B + 1, B, 1])
    at = words.data_ptr()
    _PLAN_PAGES(index, cached_lens.data_ptr(), new_lens.data_ptr(), B, block_table.data_ptr(), stride,
          width, free_pages.data_ptr(), pages, free_count.data_ptr(), page_size, tokens, slots.data_ptr(), at,
          at + 4 * tokens, at + 4 * (tokens + B + 1), at + 4 * (tokens + 2 * B + 1))
    return PagePlan(slots, positions, starts, lens, left)


def latent_cache_write(kv: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, *, rope_dim: int = 64,
                       norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                       positions: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
                       interleaved: bool = False, queries: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store one row a token in the paged cache.

    ``kv`` [tokens, latent + rope] (rows may be strided) is the latent
    projection's output; its latent part is RMS-normalised with ``norm_weight``
    [latent] (None: as given) and its last ``rope_dim`` values are rotated by
    ``positions`` int32 [tokens] times ``inv_freq`` float64 [rope_dim / 2] (None:
    as given), pairing value i with i + rope_dim / 2, or neighbours when
    ``interleaved``.  Unlike ``rms_norm`` the row is rounded once, at its store.
    ``cache`` [pages, page_size, latent + rope] is contiguous; ``slots`` int64
    [tokens] (``PagePlan.slots``): a negative slot stores nothing, the others are
    distinct (a row that two tokens name can end with pieces of both).  ``kv`` and
    ``queries`` lie outside the cache.  ``queries`` [tokens, heads, rope_dim] are
    rotated likewise into a new tensor, which is returned (None without queries).
    """
    code = _dtype(kv, "kv")
    if kv.dim() != 2 or not 0 <= rope_dim < kv.shape[1]:
        raise ValueError(f"kv must be [tokens, latent + {rope_dim}], got {list(kv.shape)}")
    T, width = kv.shape
    latent = width - rope_dim
    if cache.dim() != 3 or cache.dtype != kv.dtype or cache.shape[2] != width or not cache.is_contiguous():
        raise ValueError(f"cache must be contiguous {kv.dtype} [pages, page_size, {width}], got {cache.dtype} "
                         f"{list(cache.shape)}")
    if slots.dtype is not torch.int64 or slots.shape != (T,):
        raise ValueError(f"slots must be int64 [{T}], got {slots.dtype} {list(slots.shape)}")
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq come together")
    wp = pp = fp = 0
    if norm_weight is not None:
        norm_weight, wp, _ = _pieces(_same(norm_weight, "norm_weight", kv.dtype, (latent,)))
    if positions is not None:
        positions = _int32(positions, "positions", T)
        inv_freq = _same(inv_freq, "inv_freq", torch.float64, (rope_dim // 2,)).contiguous()
        pp, fp = positions.data_ptr(), inv_freq.data_ptr()
    rotated = None
    qp = rp = heads = qt = qh = 0
    if queries is not None:
        if positions is None:
            raise ValueError("queries are rotated by positions and inv_freq, which are missing")
        if queries.dim() != 3 or queries.dtype is not kv.dtype or queries.shape[0] != T \
                or queries.shape[2] != rope_dim or queries.shape[1] < 1:
            raise ValueError(f"queries must be {kv.dtype} [{T}, heads, {rope_dim}], got {queries.dtype} "
                             f"{list(queries.shape)}")
    index = _device(kv, cache, slots, norm_weight, positions, inv_freq, queries)
    if queries is not None:
        heads = queries.shape[1]
        rotated = kv.new_empty((T, heads, rope_dim))
        rp = rotated.data_ptr()
        queries, qp, (qt, qh) = _pieces(queries)
    if T > 1 and kv.stride(0) < width:  # overlapping rows
        kv = kv.clone(memory_format=torch.contiguous_format)
    kv, kp, (kt,) = _pieces(kv)
    first = cache.data_ptr()
    end = first + 2 * cache.numel()
    if T and (kp < end and kp + 2 * ((T - 1) * kt + width) > first or heads and qp < end
              and qp + 2 * ((T - 1) * qt + (heads - 1) * qh + rope_dim) > first):
        raise ValueError("kv and queries must lie outside the cache")
    if T:
        if not slots.is_contiguous():
            slots = slots.contiguous()
        _CACHE_WRITE(index, kp, T, kt if kt > width else width, latent, rope_dim, code, wp, eps, pp, fp,
              interleaved, slots.data_ptr(), first, cache.shape[0] * cache.shape[1], qp, heads, qt, qh, rp)
    return rotated


def latent_attention_absorbed(q_latent: torch.Tensor, q_rope: torch.Tensor | None, cache: torch.Tensor,
                              block_table: torch.Tensor, seq_lens: torch.Tensor, *, scale: float,
                              query_starts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                              return_lse: bool = False):
    """Attention of latent-space queries over the cached rows themselves (the
    absorbed form, for decode): scores ``scale * (q_latent . c + q_rope . r)``,
    result ``softmax . c``.

    ``q_latent`` [tokens, heads, latent] (latent 128, 256, 384 or 512),
    ``q_rope`` [tokens, heads, 64] (None for a cache without a rotary part),
    ``cache`` [pages, page_size, latent (+ 64)] contiguous, page_size a multiple
    of 8, ``block_table`` int32 [requests, width] and ``seq_lens`` int32
    [requests].  ``query_starts`` int32 [requests + 1] bounds each request's
    tokens (None: one each); the last one sees every row, each earlier one a row
    less.  Returns ``out`` [tokens, heads, latent] and, with ``return_lse``, the
    FP32 log-sum-exp [tokens, heads].  A token that sees no row, or whose scores
    are all -inf, gives 0 and -inf.  Tokens behind ``query_starts[-1]`` give 0 in
    a new result, are left as they were in a given ``out``, and have the
    log-sum-exp -inf.
    """
    code = _dtype(q_latent, "q_latent")
    if q_latent.dim() != 3 or q_latent.shape[1] < 1:
        raise ValueError(f"q_latent must be [tokens, heads, latent], got {list(q_latent.shape)}")
    T, H, R = q_latent.shape
    if R not in (128, 256, 384, 512):
        raise ValueError(f"latent size {R} must be 128, 256, 384 or 512")
    rope = 0
    if q_rope is not None:
        rope = 64
        _same(q_rope, "q_rope", q_latent.dtype, (T, H, 64))
    if cache.dim() != 3 or cache.dtype != q_latent.dtype or cache.shape[2] != R + rope or not cache.is_contiguous():
        raise ValueError(f"cache must be contiguous {q_latent.dtype} [pages, page_size, {R + rope}], got {cache.dtype} "
                         f"{list(cache.shape)}")
    pages, page_size = cache.shape[:2]
    if page_size < 8 or page_size % 8:
        raise ValueError(f"page_size {page_size} must be a positive multiple of 8")
    B = seq_lens.numel()
    seq_lens = _int32(seq_lens, "seq_lens", B)
    _table(block_table, B)
    sp = 0
    if query_starts is not None:
        query_starts = _int32(query_starts, "query_starts", B + 1)
        sp = query_starts.data_ptr()
    elif T != B:
        raise ValueError(f"without query_starts there is one token a request: {T} tokens, {B} requests")
    index = _device(q_latent, q_rope, cache, block_table, seq_lens, query_starts, out)
    width = block_table.shape[1]
    stride, step = block_table.stride()
    if (width > 1 and step != 1) or (B > 1 and stride < width):
        block_table = block_table.clone(memory_format=torch.contiguous_format)
        stride = width
    if B <= 1:
        stride = width
    result = _output(out, (T, H, R), q_latent, q_rope, cache)
    lse = q_latent.new_empty((T, H), dtype=torch.float32) if return_lse else None
    if T:
        q_latent, lp, (lt, lh) = _pieces(q_latent)
        rp = rt = rh = 0
        if rope:
            q_rope, rp, (rt, rh) = _pieces(q_rope)
        nbytes = _absorbed_bytes(T, H, R, index)
        # from the caching allocator: ordered on this stream, private to a captured graph
        ws = q_latent.new_empty((nbytes + 1) // 2)
        _ABSORBED(index, lp, lt, lh, rp, rt, rh, T, H, R, rope, code, cache.data_ptr(), pages,
              page_size, block_table.data_ptr(), stride, width, seq_lens.data_ptr(), B, sp, scale, result.data_ptr(),
              0 if lse is None else lse.data_ptr(), out is None, ws.data_ptr(), nbytes)
    return (result, lse) if return_lse else result


def latent_attention_expanded(q_nope: torch.Tensor, q_rope: torch.Tensor | None, k_nope: torch.Tensor,
                              k_rope: torch.Tensor | None, values: torch.Tensor, query_starts: torch.Tensor,
                              key_starts: torch.Tensor, *, scale: float, causal: bool = True,
                              out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention over the expanded keys and values of a ragged batch (prefill).

    ``q_nope`` [queries, heads, nope], ``q_rope`` [queries, heads, 64], ``k_nope``
    [keys, heads, nope], ``k_rope`` [keys, 64] (shared by the heads; both rope
    tensors None without a rotary part) and ``values`` [keys, heads, value] may be
    views, as of ``kv_b``'s output and of the cache rows; nope and value are
    multiples of 64, nope + rope and value at most 256.  ``query_starts`` and
    ``key_starts`` int32 [requests + 1] bound each request's rows.  With
    ``causal``, query j of nq sees keys 0 .. nk - nq + j (earlier context first).
    Returns ``out`` [queries, heads, value], whose flattened rows are the output
    projection's input, and with ``return_lse`` the FP32 log-sum-exp
    [queries, heads]; rows without keys and rows outside every request as in
    ``latent_attention_absorbed``.  Starts that descend or leave the rows set the
    status word: a request between such key starts has no keys; one between such
    query starts, or that begins before a start ahead of its own, has no queries.
    """
    code = _dtype(q_nope, "q_nope")
    if q_nope.dim() != 3 or q_nope.shape[1] < 1:
        raise ValueError(f"q_nope must be [queries, heads, nope], got {list(q_nope.shape)}")
    if k_nope.dim() != 3 or values.dim() != 3:
        raise ValueError(f"k_nope and values must be [keys, heads, size], got {list(k_nope.shape)} and "
                         f"{list(values.shape)}")
    Tq, H, dn = q_nope.shape
    Tk, _, dv = values.shape
    _same(k_nope, "k_nope", q_nope.dtype, (Tk, H, dn))
    _same(values, "values", q_nope.dtype, (Tk, H, dv))
    if (q_rope is None) != (k_rope is None):
        raise ValueError("q_rope and k_rope come together")
    dr = 0
    if q_rope is not None:
        dr = 64
        _same(q_rope, "q_rope", q_nope.dtype, (Tq, H, 64))
        _same(k_rope, "k_rope", q_nope.dtype, (Tk, 64))
    if dn <= 0 or dn % 64 or dv <= 0 or dv % 64 or dn + dr > 256 or dv > 256:
        raise ValueError(f"nope {dn} and value {dv} must be multiples of 64, nope + rope and value at most 256")
    B = query_starts.numel() - 1
    if B < 0:
        raise ValueError("query_starts must hold requests + 1 entries")
    query_starts = _int32(query_starts, "query_starts", B + 1)
    key_starts = _int32(key_starts, "key_starts", B + 1)
    index = _device(q_nope, q_rope, k_nope, k_rope, values, query_starts, key_starts, out)
    result = _output(out, (Tq, H, dv), q_nope, q_rope, k_nope, k_rope, values)
    lse = q_nope.new_empty((Tq, H), dtype=torch.float32) if return_lse else None
    if Tq:
        q_nope, qp, (qt, qh) = _pieces(q_nope)
        k_nope, kp, (kt, kh) = _pieces(k_nope)
        values, vp, (vt, vh) = _pieces(values)
        qrp = krp = qrt = qrh = krt = 0
        if dr:
            q_rope, qrp, (qrt, qrh) = _pieces(q_rope)
            k_rope, krp, (krt,) = _pieces(k_rope)
        _EXPANDED(index, qp, qt, qh, qrp, qrt, qrh, kp, kt, kh, krp, krt, vp, vt, vh, Tq, Tk, H, dn,
              dr, dv, code, query_starts.data_ptr(), key_starts.data_ptr(), B, scale, causal, result.data_ptr(),
              0 if lse is None else lse.data_ptr(), out is None)
    return (result, lse) if return_lse else result
