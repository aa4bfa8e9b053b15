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

Tensors are BF16 or FP16; products, statistics and sums are FP32, rounded once
into the result.  Lengths, tables and plans stay on the device: no call reads
them back, so each can be captured into a CUDA graph after one eager call on
the device.  Errors that only the device can see (a page id outside the cache,
a plan that does not fit) set a status word: the call leaves its documented
safe result and the next call of this module raises (``IndexError`` /
``RuntimeError``); ``check_latent_status()`` synchronises and raises at once.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .packed import StatusWord, _SYNC_STATUS

_DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_FP16}
_STATUS: dict[int, StatusWord] = {}


def _status(dev: torch.device) -> StatusWord:
    sw = _STATUS.get(dev.index)
    if sw is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call a latent-attention operator once on this device before capturing it")
        sw = _STATUS[dev.index] = StatusWord(dev)
    return sw


def check_latent_status(device: torch.device | int | None = None) -> None:
    """Synchronise and raise for any device-side error of this module's calls so far."""
    index = torch.cuda.current_device() if device is None else torch.device("cuda", device).index \
        if isinstance(device, int) else torch.device(device).index
    sw = _STATUS.get(torch.cuda.current_device() if index is None else index)
    if sw is not None:
        sw.check()


def _call(name: str, dev: torch.device, *args) -> None:
    """One C-ABI call on `dev`'s current stream with its status word, whatever the current device is."""
    sw = _status(dev)
    sw.raise_pending()
    status = (sw.word.data_ptr(), sw.host.data_ptr(), N.stream(dev))
    fn = getattr(N.load_library(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, *status)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, *status)
    if rc:
        N.check(rc, name)
    if _SYNC_STATUS:
        sw.check()


def _int32(t: torch.Tensor, name: str, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be BF16 or FP16, got {t.dtype}")
    return code


def _same(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _pieces(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where its rows can be read in 16-byte pieces, else a contiguous copy."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0:
        for s in t.stride()[:-1]:
            if s <= 0 or s % 8:
                break
        else:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _output(out: torch.Tensor | None, like: torch.Tensor, shape: tuple) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    return _same(out, "out", like.dtype, shape)


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
    cached_lens = _int32(cached_lens, "cached_lens", (B,))
    new_lens = _int32(new_lens, "new_lens", (B,))
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be int32 [{B}, pages], got {block_table.dtype} {list(block_table.shape)}")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table is updated in place: its rows must be contiguous")
    width = block_table.shape[1]
    if B > 1 and block_table.stride(0) < width:
        raise ValueError("block_table is updated in place: its rows must not overlap")
    free_pages = _int32(free_pages, "free_pages", (free_pages.numel(),))
    free_count = _int32(free_count, "free_count", (1,))
    if page_size < 1 or tokens < 0:
        raise ValueError(f"page_size {page_size} and tokens {tokens} must be positive")
    dev = N.require_cuda(cached_lens, new_lens, block_table, free_pages, free_count)
    slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    words = torch.empty(tokens + 2 * B + 2, dtype=torch.int32, device=dev)
    positions, starts, lens, left = words.split([tokens, B + 1, B, 1])
    _call("glm53_plan_pages", dev, cached_lens.data_ptr(), new_lens.data_ptr(), B, block_table.data_ptr(),
          block_table.stride(0) if B > 1 else width, width, free_pages.data_ptr(), free_pages.numel(),
          free_count.data_ptr(), page_size, tokens, slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
          lens.data_ptr(), left.data_ptr())
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
    [tokens] (``PagePlan.slots``): a negative slot stores nothing; slots are
    distinct (of two tokens with one slot either row stays).  ``queries``
    [tokens, heads, rope_dim] are rotated likewise into a new tensor, which is
    returned (None without queries).
    """
    code = _dtype(kv, "kv")
    if kv.dim() != 2 or not 0 <= rope_dim < kv.shape[1]:
        raise ValueError(f"kv must be [tokens, latent + {rope_dim}], got {list(kv.shape)}")
    T, width = kv.shape
    latent = width - rope_dim
    if cache.dim() != 3 or cache.dtype != kv.dtype or cache.shape[2] != width or not cache.is_contiguous():
        raise ValueError(f"cache must be contiguous {kv.dtype} [pages, page_size, {width}], got {cache.dtype} "
                         f"{list(cache.shape)}")
    if slots.dtype != torch.int64 or tuple(slots.shape) != (T,):
        raise ValueError(f"slots must be int64 [{T}], got {slots.dtype} {list(slots.shape)}")
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq come together")
    if norm_weight is not None:
        norm_weight = _pieces(_same(norm_weight, "norm_weight", kv.dtype, (latent,)))
    if positions is not None:
        positions = _int32(positions, "positions", (T,))
        inv_freq = _same(inv_freq, "inv_freq", torch.float64, (rope_dim // 2,)).contiguous()
    rotated = None
    heads = qt = qh = 0
    if queries is not None:
        if positions is None:
            raise ValueError("queries are rotated by positions and inv_freq, which are missing")
        if queries.dim() != 3 or queries.dtype != kv.dtype or queries.shape[0] != T or queries.shape[2] != rope_dim \
                or queries.shape[1] < 1:
            raise ValueError(f"queries must be {kv.dtype} [{T}, heads, {rope_dim}], got {queries.dtype} "
                             f"{list(queries.shape)}")
    dev = N.require_cuda(kv, cache, slots, norm_weight, positions, inv_freq, queries)
    if queries is not None:
        queries = _pieces(queries)
        heads = queries.shape[1]
        qt, qh = queries.stride(0), queries.stride(1)
        rotated = torch.empty((T, heads, rope_dim), dtype=kv.dtype, device=dev)
    kv = _pieces(kv)
    slots = slots.contiguous()
    _call("glm53_latent_cache_write", dev, kv.data_ptr(), T, max(kv.stride(0), width), latent, rope_dim, code,
          N.ptr(norm_weight), eps, N.ptr(positions), N.ptr(inv_freq), interleaved, slots.data_ptr(), cache.data_ptr(),
          cache.shape[0] * cache.shape[1], N.ptr(queries), heads, qt, qh, N.ptr(rotated))
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
    FP32 log-sum-exp [tokens, heads].  A token that sees no row gives 0 and
    -inf.  Tokens behind ``query_starts[-1]`` give 0 in a new result and are
    left as they were in a given ``out``.
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
    seq_lens = _int32(seq_lens, "seq_lens", (B,))
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be int32 [{B}, pages], got {block_table.dtype} {list(block_table.shape)}")
    if query_starts is not None:
        query_starts = _int32(query_starts, "query_starts", (B + 1,))
    elif T != B:
        raise ValueError(f"without query_starts there is one token a request: {T} tokens, {B} requests")
    dev = N.require_cuda(q_latent, q_rope, cache, block_table, seq_lens, query_starts, out)
    width = block_table.shape[1]
    if (width > 1 and block_table.stride(1) != 1) or (B > 1 and block_table.stride(0) < width):
        block_table = block_table.clone(memory_format=torch.contiguous_format)
    result = _output(out, q_latent, (T, H, R))
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    if T:
        q_latent = _pieces(q_latent)
        qrt = qrh = 0
        if rope:
            q_rope = _pieces(q_rope)
            qrt, qrh = q_rope.stride(0), q_rope.stride(1)
        nbytes = N.load_library().glm53_latent_absorbed_workspace_bytes(T, H, R)
        # from the caching allocator: ordered on this stream, private to a captured graph
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _call("glm53_latent_absorbed", dev, q_latent.data_ptr(), q_latent.stride(0), q_latent.stride(1), N.ptr(q_rope),
              qrt, qrh, T, H, R, rope, code, cache.data_ptr(), pages, page_size, block_table.data_ptr(),
              block_table.stride(0) if B > 1 else width, width, seq_lens.data_ptr(), B, N.ptr(query_starts), scale,
              result.data_ptr(), N.ptr(lse), out is None, ws.data_ptr(), nbytes)
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
    ``latent_attention_absorbed``.
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
    query_starts = _int32(query_starts, "query_starts", (B + 1,))
    key_starts = _int32(key_starts, "key_starts", (B + 1,))
    dev = N.require_cuda(q_nope, q_rope, k_nope, k_rope, values, query_starts, key_starts, out)
    result = _output(out, q_nope, (Tq, H, dv))
    lse = torch.empty((Tq, H), dtype=torch.float32, device=dev) if return_lse else None
    if Tq:
        q_nope, k_nope, values = _pieces(q_nope), _pieces(k_nope), _pieces(values)
        qrt = qrh = krt = 0
        if dr:
            q_rope, k_rope = _pieces(q_rope), _pieces(k_rope)
            qrt, qrh, krt = q_rope.stride(0), q_rope.stride(1), k_rope.stride(0)
        _call("glm53_latent_expanded", dev, q_nope.data_ptr(), q_nope.stride(0), q_nope.stride(1), N.ptr(q_rope), qrt,
              qrh, k_nope.data_ptr(), k_nope.stride(0), k_nope.stride(1), N.ptr(k_rope), krt, values.data_ptr(),
              values.stride(0), values.stride(1), Tq, Tk, H, dn, dr, dv, code, query_starts.data_ptr(),
              key_starts.data_ptr(), B, scale, causal, result.data_ptr(), N.ptr(lse), out is None)
    return (result, lse) if return_lse else result
