"""8-bit paged KV cache for ragged batches, with its page tables on the device.

The 2 to 4 bit stores hold one length for all sequences and hand out pages on
the host.  A serving batch has requests of any lengths, and an 8-bit cache is
nearly lossless: this module holds K and V as int8 or float8 (e4m3) codes with
one fp32 scale per block of 16 tokens and head, and plans pages, slots and
positions on the GPU from the requests' lengths, so that a decode step (plan,
append, attention) runs without the host and can be captured into a graph.

Store formats (n = page_tokens = 64 << k; value = code * scale):

* ``kpool`` (P, H, n, d), ``vpool`` (P, H, n / 16, d, 16): codes, a V block's
  tokens innermost; ``kscale`` / ``vscale`` (P, H, n / 16) fp32.
* ``table`` (B, W) int32: token t of request b lies in page table[b, t // n],
  at slot page * n + t % n.
* ``free`` (P,) int32 with ``free_count`` (1,): the first free_count entries are
  free pages, taken from the end.
* ``shares`` (P,) int32, where requests share pages: a page's holders beyond the
  first.

Operators: :func:`plan_pages`, :func:`release_pages`, :func:`append_kv8`,
:func:`read_kv8`, :func:`attention_kv8`; for pages that requests share
:func:`fork_pages`, :func:`copy_pages`, :func:`compact_pages` and
:func:`attention_kv8_shared` (quashkv_amd.rotary turns rows by their positions).  :class:`PagedKV8Store` holds the
tensors and calls them; :class:`PagedKV8Engine` is the engine interface
(append / attention / clear over sequences of one length) on that store.
All calls run on the current stream of the tensors' device and never
synchronise.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N
from .paged import PAGE_SIZES, PAGE_TOKENS
from .quantizer import _default_device

BLOCK_TOKENS = 16
CODE_DTYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_FMT = {torch.int8: N.QKV_CODES_I8, torch.float8_e4m3fn: N.QKV_CODES_E4M3}


def _call(dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) on ``dev``, which is made the current device for it:
    launches go there, whatever device the stream belongs to."""
    if dev.index == torch.cuda.current_device():
        N.check(fn(*args, N.stream(dev)))
    else:
        with torch.cuda.device(dev):
            N.check(fn(*args, N.stream(dev)))


def _want(t: torch.Tensor, what: str, dtype: torch.dtype, shape: Optional[tuple] = None) -> None:
    if t.dtype is not dtype:
        raise ValueError(f"{what} must be {dtype}; got {t.dtype}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what} must have shape {shape}; got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


@dataclass
class PagePlan:
    """What :func:`plan_pages` found out about a step's rows (device tensors)."""
    q_start: torch.Tensor      # (B + 1,) int32: each request's first row
    q_lens: torch.Tensor       # (B,) int32: rows served, 0 where a request was refused
    kv_lens: torch.Tensor      # (B,) int32: cached tokens after the step
    slots: torch.Tensor        # (rows,) int64: a row's place in the pool, -1: none
    positions: torch.Tensor    # (rows,) int32: a row's token position, 0: none
    free_count: torch.Tensor   # (1,) int32: free pages left
    scratch: torch.Tensor      # (B,) int32 workspace
    max_q_len: int             # bound of q_lens, as far as the host knows

    @classmethod
    def empty(cls, B: int, rows: int, device, kv_lens: Optional[torch.Tensor] = None,
              free_count: Optional[torch.Tensor] = None,
              max_q_len: Optional[int] = None) -> "PagePlan":
        if rows < 0:
            raise ValueError(f"rows must not be negative; got {rows}")
        # one allocation for the int32 parts (without split's records for autograd, which
        # integers have not: 2.7 -> 1.5 us)
        q_start, q_lens, kv, positions, scratch, count = torch.empty(
            4 * B + rows + 2, dtype=torch.int32, device=device).unsafe_split_with_sizes(
                (B + 1, B, B, rows, B, 1))
        return cls(q_start, q_lens, kv if kv_lens is None else kv_lens,
                   torch.empty(rows, dtype=torch.int64, device=device), positions,
                   count if free_count is None else free_count, scratch,
                   rows if max_q_len is None else max_q_len)


def plan_pages(table: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor,
               free: torch.Tensor, free_count: torch.Tensor, rows: int, page_tokens: int,
               out: Optional[PagePlan] = None) -> PagePlan:
    """Pages, slots and positions of the tokens that B requests bring.

    Request b holds ``lens[b]`` tokens and brings ``new_lens[b]`` (negative
    counts as 0); the batch has ``rows`` rows, request b's behind those of
    request b - 1, and rows behind the last are padding.  New pages come from
    the end of ``free[:free_count]`` and are written into ``table``; every other
    result is in the plan, or in ``out``, whose ``kv_lens`` / ``free_count`` may be
    ``lens`` / ``free_count`` themselves.

    A request is served wholly or not at all (``q_lens`` 0, slots -1, its
    length kept): not, when its rows end behind ``rows``, its pages behind the
    table's width or its tokens behind 2^31 - 64, or when it needs pages and the pages needed up to it, in
    request order, exceed the free ones."""
    dev = _one_device("plan_pages", table, lens, new_lens, free, free_count)
    if table.dim() != 2:
        raise ValueError("page table must be a 2-D int32 tensor")
    B, width = table.shape
    _want(table, "page table", torch.int32)
    _want(lens, "lens", torch.int32, (B,))
    _want(new_lens, "new_lens", torch.int32, (B,))
    if free.dim() != 1:
        raise ValueError("free must be a 1-D int32 tensor")
    _want(free, "free", torch.int32)
    _want(free_count, "free_count", torch.int32, (1,))
    if out is None:
        out = PagePlan.empty(B, rows, dev)
    else:
        for name, dt, shape in (("q_start", torch.int32, (B + 1,)), ("q_lens", torch.int32, (B,)),
                                ("kv_lens", torch.int32, (B,)), ("slots", torch.int64, (rows,)),
                                ("positions", torch.int32, (rows,)),
                                ("free_count", torch.int32, (1,)),
                                ("scratch", torch.int32, (B,))):
            _want(getattr(out, name), f"out.{name}", dt, shape)
        _one_device("plan_pages", table, out.q_start, out.q_lens, out.kv_lens, out.slots,
                    out.positions, out.free_count, out.scratch)
    _call(dev, N.lib().qkv_page_plan, lens.data_ptr(), new_lens.data_ptr(), B, table.data_ptr(),
          width, free.data_ptr(), free.numel(), free_count.data_ptr(), page_tokens, rows,
          out.q_start.data_ptr(), out.q_lens.data_ptr(), out.kv_lens.data_ptr(),
          out.slots.data_ptr(), out.positions.data_ptr(), out.free_count.data_ptr(),
          out.scratch.data_ptr())
    return out


def release_pages(table: torch.Tensor, lens: torch.Tensor, done: torch.Tensor,
                  free: torch.Tensor, free_count: torch.Tensor, page_tokens: int,
                  shares: Optional[torch.Tensor] = None) -> None:
    """The pages of the requests with ``done`` ((B,) bool) go back to the free
    list and their lengths become 0, all in place.  With ``shares`` each of their
    table entries takes one holder away, and a page goes back with its last one, at the
    place of the last of the entries that name it."""
    dev = _one_device("release_pages", table, lens, done, free, free_count, shares)
    B, width, P = _check_books(table, lens, free, free_count, shares)
    _want(done, "done", torch.bool, (B,))
    if shares is None:
        _call(dev, N.lib().qkv_page_release, lens.data_ptr(), done.data_ptr(), B,
              table.data_ptr(), width, free.data_ptr(), P, free_count.data_ptr(), page_tokens)
    else:
        _call(dev, N.lib().qkv_page_release_shared, lens.data_ptr(), done.data_ptr(), B,
              table.data_ptr(), width, free.data_ptr(), P, free_count.data_ptr(),
              shares.data_ptr(), page_tokens)


def _check_books(table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor,
                 free_count: torch.Tensor, shares: Optional[torch.Tensor]) -> tuple[int, int, int]:
    """(requests, table width, pages) of the tensors that keep a pool's pages."""
    if table.dim() != 2:
        raise ValueError("page table must be a 2-D int32 tensor")
    B, width = table.shape
    _want(table, "page table", torch.int32)
    _want(lens, "lens", torch.int32, (B,))
    if free.dim() != 1:
        raise ValueError("free must be a 1-D int32 tensor")
    _want(free, "free", torch.int32)
    _want(free_count, "free_count", torch.int32, (1,))
    if shares is not None:
        _want(shares, "shares", torch.int32, (free.numel(),))
    return B, width, free.numel()


@dataclass
class ForkPlan:
    """What :func:`fork_pages` granted, and the pages that are to be copied (device tensors)."""
    granted: torch.Tensor      # (F,) int32: tokens that the fork holds, -1 where refused
    src_pages: torch.Tensor    # (F,) int32: a page in part filled, -1: none
    dst_pages: torch.Tensor    # (F,) int32: the fork's own page for its tokens
    copy_tokens: torch.Tensor  # (F,) int32: how many


def fork_pages(table: torch.Tensor, lens: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               tokens: Optional[torch.Tensor], free: torch.Tensor, free_count: torch.Tensor,
               shares: torch.Tensor, page_tokens: int) -> ForkPlan:
    """Requests ``dst`` ((F,) int32) go on from requests ``src``: fork i holds the first
    ``tokens[i]`` tokens (None: all; at most all, negative counts as 0) of ``src[i]``.

    Whole pages are shared (``shares``, (P,) int32, counts their holders beyond the
    first); a page in part filled gets a page of its own from the end of the free list, into
    which :func:`copy_pages` brings the plan's pages, in each layer's pools.  The table,
    lengths, free count and shares move on in place.

    All forks go by the lengths before the call.  A fork is granted wholly or refused
    (``granted`` -1): where src or dst is no request or both are the same, dst holds
    tokens, an earlier fork of the call (of two different requests) names the same dst, or it
    needs a page and the pages needed up to it, in fork order, exceed the free ones.  A
    copied block of 16 tokens keeps its scale for the fork's own tokens behind them."""
    dev = _one_device("fork_pages", table, lens, src, dst, tokens, free, free_count, shares)
    B, width, P = _check_books(table, lens, free, free_count, shares)
    if src.dim() != 1:
        raise ValueError("src must be a 1-D int32 tensor")
    F = src.numel()
    _want(src, "src", torch.int32)
    _want(dst, "dst", torch.int32, (F,))
    if tokens is not None:
        _want(tokens, "tokens", torch.int32, (F,))
    out = torch.empty(4 * F, dtype=torch.int32, device=dev)
    at = out.data_ptr()
    _call(dev, N.lib().qkv_page_fork, table.data_ptr(), lens.data_ptr(), B, width, src.data_ptr(),
          dst.data_ptr(), N.ptr(tokens), F, free.data_ptr(), P, free_count.data_ptr(),
          shares.data_ptr(), page_tokens, at, at + 4 * F, at + 8 * F, at + 12 * F)
    return ForkPlan(*out.unsafe_split_with_sizes((F, F, F, F)))


@dataclass
class CompactPlan:
    """What :func:`compact_pages` moves (device tensors)."""
    src_pages: torch.Tensor    # (P // 2,) int32: -1 behind the moves
    dst_pages: torch.Tensor    # (P // 2,) int32
    moves: torch.Tensor        # (1,) int32
    remap: torch.Tensor        # (P,) int32: a page's new place


def compact_pages(table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor,
                  free_count: torch.Tensor, page_tokens: int,
                  shares: Optional[torch.Tensor] = None) -> CompactPlan:
    """The U pages in use (those not on the free list, whoever holds them) move to places
    0 .. U - 1 of the pool: the i-th in use at U or above to the i-th free one below.  The
    table's entries within the requests' lengths, shares and free list (P - 1 down to U) follow
    in place; ``copy_pages(plan.src_pages, plan.dst_pages, ..., count=plan.moves)`` moves the
    tokens, in each layer's pools, and ``plan.remap`` serves tables of the caller's."""
    dev = _one_device("compact_pages", table, lens, free, free_count, shares)
    B, width, P = _check_books(table, lens, free, free_count, shares)
    src, dst, moves, remap = torch.empty(
        2 * (P // 2) + 1 + P, dtype=torch.int32, device=dev).unsafe_split_with_sizes(
            (P // 2, P // 2, 1, P))
    _call(dev, N.lib().qkv_page_compact, table.data_ptr(), lens.data_ptr(), B, width,
          free.data_ptr(), P, free_count.data_ptr(), N.ptr(shares), page_tokens, src.data_ptr(),
          dst.data_ptr(), moves.data_ptr(), remap.data_ptr())
    return CompactPlan(src, dst, moves, remap)


def copy_pages(src: torch.Tensor, dst: torch.Tensor, kpool: torch.Tensor, kscale: torch.Tensor,
               vpool: torch.Tensor, vscale: torch.Tensor, tokens: Optional[torch.Tensor] = None,
               count: Optional[torch.Tensor] = None) -> None:
    """Page ``src[i]`` to page ``dst[i]`` ((n,) int32) of the pools, codes and scales of all
    heads: the blocks that hold its first ``tokens[i]`` tokens ((n,) int32; None: the whole
    page), for the first ``count`` ((1,) int32) pairs (None: all).  Pairs with a page
    outside the pool, such as -1, are left out.  No page may be source and target in one
    call, or target twice."""
    dev = _one_device("copy_pages", src, dst, kpool, kscale, vpool, vscale, tokens, count)
    P, H, n, d, fmt = _check_pools(kpool, kscale, vpool, vscale)
    if src.dim() != 1:
        raise ValueError("src must be a 1-D int32 tensor")
    F = src.numel()
    _want(src, "src", torch.int32)
    _want(dst, "dst", torch.int32, (F,))
    if tokens is not None:
        _want(tokens, "tokens", torch.int32, (F,))
    if count is not None:
        _want(count, "count", torch.int32, (1,))
    _call(dev, N.lib().qkv_kv8_copy_pages, src.data_ptr(), dst.data_ptr(), N.ptr(tokens), F,
          N.ptr(count), H, d, fmt, kpool.data_ptr(), kscale.data_ptr(), vpool.data_ptr(),
          vscale.data_ptr(), P, n)


def _one_device(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """The tensors' HIP device; N.require_gpu's errors where they have not one."""
    i = first.get_device()
    if i < 0:
        N.require_gpu(first, what=what)
    for t in others:
        if t is not None and t.get_device() != i:
            N.require_gpu(first, *others, what=what)
    return first.device


def _check_pools(kpool: torch.Tensor, kscale: torch.Tensor, vpool: torch.Tensor,
                 vscale: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(pages, H, page tokens, d, code format) of the pools."""
    shape, dtype = kpool.shape, kpool.dtype
    if len(shape) != 4:
        raise ValueError("kpool must be (pages, kv heads, page_tokens, head_dim)")
    P, H, n, d = shape
    fmt = _FMT.get(dtype)
    if fmt is None:
        raise ValueError(f"kpool must be int8 or float8_e4m3fn; got {dtype}")
    if n not in PAGE_SIZES:
        raise ValueError(f"page_tokens {n} must be one of {PAGE_SIZES}")
    nb = n // BLOCK_TOKENS
    _want(kpool, "kpool", dtype)
    _want(vpool, "vpool", dtype, (P, H, nb, d, BLOCK_TOKENS))
    _want(kscale, "kscale", torch.float32, (P, H, nb))
    _want(vscale, "vscale", torch.float32, (P, H, nb))
    return P, H, n, d, fmt


def append_kv8(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, kpool: torch.Tensor,
               kscale: torch.Tensor, vpool: torch.Tensor, vscale: torch.Tensor) -> None:
    """Quantise rows k, v (rows, H, d; fp32, fp16 or bf16, any row and head
    strides) into the pools at ``slots`` ((rows,) int64, as plan_pages makes them:
    the rows of a block follow each other at consecutive slots, each slot once; -1
    skips a row).

    A block's scale covers its largest finite value.  Tokens that the block
    holds already keep their codes while the scale stands and are quantised anew
    where the new ones need a larger scale; NaN becomes 0, infinities the
    largest code."""
    dev = _one_device("append_kv8", k, v, slots, kpool, kscale, vpool, vscale)
    P, H, n, d, fmt = _check_pools(kpool, kscale, vpool, vscale)
    rows = k.shape[0] if k.dim() == 3 else -1
    if k.shape != v.shape or tuple(k.shape) != (rows, H, d) or k.dtype != v.dtype:
        raise ValueError(f"expected keys and values of shape (rows, {H}, {d}) and one type; got "
                         f"{tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    _want(slots, "slots", torch.int64, (rows,))
    # unit stride along the head_dim; the other strides are passed on
    k, v = (x if x.stride(2) == 1 else x.contiguous() for x in (k, v))
    _call(dev, N.lib().qkv_kv8_append, N.dtype_code(k.dtype), k.data_ptr(), k.stride(0),
          k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), rows, H, d, fmt,
          kpool.data_ptr(), kscale.data_ptr(), vpool.data_ptr(), vscale.data_ptr(), P, n)


def read_kv8(slots: torch.Tensor, kpool: torch.Tensor, kscale: torch.Tensor,
             vpool: torch.Tensor, vscale: torch.Tensor,
             out_dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """(keys, values) (rows, H, d) that the cache holds at ``slots`` ((rows,)
    int64, any order); rows whose slot is outside the pool become 0."""
    dev = _one_device("read_kv8", slots, kpool, kscale, vpool, vscale)
    P, H, n, d, fmt = _check_pools(kpool, kscale, vpool, vscale)
    rows = slots.numel()
    _want(slots, "slots", torch.int64, (rows,))
    dt = N.dtype_code(out_dtype)
    k = torch.empty(rows, H, d, dtype=out_dtype, device=dev)
    v = torch.empty_like(k)
    _call(dev, N.lib().qkv_kv8_read, slots.data_ptr(), rows, H, d, fmt, kpool.data_ptr(),
          kscale.data_ptr(), vpool.data_ptr(), vscale.data_ptr(), P, n, k.data_ptr(),
          v.data_ptr(), dt)
    return k, v


def _check_attention(q: torch.Tensor, H: int, d: int, table: torch.Tensor, kv_lens: torch.Tensor,
                     q_start: Optional[torch.Tensor], q_lens: Optional[torch.Tensor],
                     out_dtype: torch.dtype, out: Optional[torch.Tensor], dev: torch.device):
    """(rows, query heads, requests, table width, result) of an attention's arguments."""
    if q.dim() != 3:
        raise ValueError(f"queries must be (rows, heads, {d}); got {tuple(q.shape)}")
    rows, Hq, dq = q.shape
    if dq != d or Hq == 0 or Hq % H != 0:
        raise ValueError(f"queries {tuple(q.shape)} do not match the cache (rows, a multiple of "
                         f"{H} heads, {d})")
    if table.dim() != 2:
        raise ValueError("page table must be a 2-D int32 tensor")
    B, width = table.shape
    _want(table, "page table", torch.int32)
    _want(kv_lens, "kv_lens", torch.int32, (B,))
    if q_start is not None:
        _want(q_start, "q_start", torch.int32, (B + 1,))
    elif q_lens is not None:
        raise ValueError("q_lens needs q_start")
    elif B == 0 or rows % B != 0:
        raise ValueError(f"without q_start the rows ({rows}) must be a multiple of the "
                         f"requests ({B})")
    if q_lens is not None:
        _want(q_lens, "q_lens", torch.int32, (B,))
    if out is None:
        make = torch.empty if q_start is None else torch.zeros
        out = make(rows, Hq, d, dtype=out_dtype, device=dev)
    else:
        _want(out, "out", out.dtype, (rows, Hq, d))
    return rows, Hq, B, width, out


def attention_kv8(q: torch.Tensor, kpool: torch.Tensor, kscale: torch.Tensor,
                  vpool: torch.Tensor, vscale: torch.Tensor, table: torch.Tensor,
                  kv_lens: torch.Tensor, q_start: Optional[torch.Tensor] = None,
                  q_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  causal: bool = False, out_dtype: torch.dtype = torch.float32,
                  max_q_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of query rows (rows, Hq, d; fp32, fp16 or bf16, any row and head
    strides) over each request's first ``kv_lens[b]`` cached tokens.

    Request b's rows are ``q_start[b] ... + q_lens[b]`` (without q_lens up to the
    next request's, also where that lies behind the last row; without q_start the
    rows are split evenly).  ``causal``
    places query i of q_len at token kv_len - q_len + i.  Queries that see no
    token give 0; rows of no request keep what ``out`` holds (0 where this
    call makes it).  Head h reads kv head h // (Hq // H).

    Value scales of one request and head, other than 0, lie within 2^80 of each other
    (fp16 values always do), or the smaller ones' weights may be missing from the sum.

    Scores and sums are fp32; softmax weights reach the value product in 22 bits,
    or, for bf16 results of 16-bit queries where a request has more than 32 rows (of
    a kv head), in 11, which the result's 8 bits do not show.

    ``max_q_len``: the longest request's rows where the caller knows it (1 in a
    decode step); it picks the kernels, not the result (but for rounding).  ``workspace`` (uint8,
    :func:`attention_kv8_workspace_bytes`) must belong to one call at a time."""
    dev = _one_device("attention_kv8", q, kpool, kscale, vpool, vscale, table, kv_lens, q_start,
                      q_lens, out, workspace)
    P, H, n, d, fmt = _check_pools(kpool, kscale, vpool, vscale)
    rows, Hq, B, width, out = _check_attention(q, H, d, table, kv_lens, q_start, q_lens, out_dtype,
                                               out, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    longest = rows // max(B, 1) if q_start is None else rows
    if max_q_len is not None:
        longest = max(0, min(longest, int(max_q_len)))
    ts, hs, ls = q.stride()
    if ls != 1:
        q = q.contiguous()
        ts, hs, ls = q.stride()
    if workspace is None:
        nbytes = attention_kv8_workspace_bytes(B, rows, Hq, H, d, longest)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    else:
        _want(workspace, "workspace", torch.uint8)
        nbytes = workspace.numel()
    _call(dev, N.lib().qkv_kv8_attention, q.data_ptr(), N.dtype_code(q.dtype), ts, hs, rows,
          kpool.data_ptr(), kscale.data_ptr(), vpool.data_ptr(),
          vscale.data_ptr(), fmt, P, n, table.data_ptr(), width, N.ptr(q_start), N.ptr(q_lens),
          kv_lens.data_ptr(), B, Hq, H, d, longest, float(scale), 1 if causal else 0,
          out.data_ptr(), N.dtype_code(out.dtype), workspace.data_ptr(), nbytes)
    return out


def attention_kv8_workspace_bytes(B: int, rows: int, Hq: int, H: int, d: int,
                                  max_q_len: int) -> int:
    """Bytes of the workspace that attention_kv8 needs at these sizes."""
    return N.lib().qkv_kv8_attention_workspace_bytes(B, rows, Hq, H, d, max_q_len)


def attention_kv8_shared(q: torch.Tensor, kpool: torch.Tensor, kscale: torch.Tensor,
                         vpool: torch.Tensor, vscale: torch.Tensor, table: torch.Tensor,
                         kv_lens: torch.Tensor, group_start: torch.Tensor,
                         prefix_lens: torch.Tensor, q_start: Optional[torch.Tensor] = None,
                         q_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                         causal: bool = False, out_dtype: torch.dtype = torch.float32,
                         out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None, always: bool = False,
                         max_q_len: Optional[int] = None) -> torch.Tensor:
    """:func:`attention_kv8` of a batch in groups whose requests share a prefix, which is
    read once for all rows of a group.

    Requests ``group_start[g]`` up to ``group_start[g + 1]`` ((groups + 1,) int32, ascending;
    at most 2048 groups) hold the same first ``prefix_lens[g]`` ((groups,) int32) tokens, as
    :func:`fork_pages` makes them; whole steps of 64 of them are read from the first request
    of the group whose queries all see them.  Requests that do not (idle ones, chunks that
    begin inside the prefix) and those before the first or behind the last group go over
    all of their own tokens, and so do all where sharing would cost more than it saves (short
    prefixes, requests of many rows, small calls), unless ``always`` is set.  The rules know the
    lengths on the device alone: a call of many rows whose groups do not share is up to
    8 % slower than attention_kv8, and calls count as small by the table's width, so that
    it should have room for little more than the requests' tokens.

    Calls of 2^28 rows times query heads, or of 2^22 requests times kv heads, are refused.  So
    are, with ``always``, those over a table with room for so many tokens a request that times
    B + groups + rows * Hq / H / 64 they are about 2^36; without, they are attention_kv8's,
    as small calls are: ``max_q_len``, the longest request's rows, is for both.

    The other arguments and the result are attention_kv8's but for rounding.  (For bf16 results of
    16-bit queries the weights of requests of more than 32 rows of a kv head have 11 bits, over
    the prefix where all requests that share it are such ones; all others 22.)  ``workspace`` (uint8,
    :func:`attention_kv8_shared_workspace_bytes`) must belong to one call at a time."""
    dev = _one_device("attention_kv8_shared", q, kpool, kscale, vpool, vscale, table, kv_lens,
                      group_start, prefix_lens, q_start, q_lens, out, workspace)
    P, H, n, d, fmt = _check_pools(kpool, kscale, vpool, vscale)
    rows, Hq, B, width, out = _check_attention(q, H, d, table, kv_lens, q_start, q_lens, out_dtype,
                                               out, dev)
    if prefix_lens.dim() != 1:
        raise ValueError("prefix_lens must be a 1-D int32 tensor")
    groups = prefix_lens.numel()
    _want(prefix_lens, "prefix_lens", torch.int32)
    _want(group_start, "group_start", torch.int32, (groups + 1,))
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    ts, hs, ls = q.stride()
    if ls != 1:
        q = q.contiguous()
        ts, hs, ls = q.stride()
    if workspace is None:
        nbytes = attention_kv8_shared_workspace_bytes(B, groups, rows, Hq, H, d)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    else:
        _want(workspace, "workspace", torch.uint8)
        nbytes = workspace.numel()
    if (max_q_len is not None and not always
            and max_q_len < _shared_plain(B, groups, rows, Hq, H, d, width, n)):
        _call(dev, N.lib().qkv_kv8_attention, q.data_ptr(), N.dtype_code(q.dtype), ts, hs, rows,
              kpool.data_ptr(), kscale.data_ptr(), vpool.data_ptr(), vscale.data_ptr(), fmt, P, n,
              table.data_ptr(), width, N.ptr(q_start), N.ptr(q_lens), kv_lens.data_ptr(), B, Hq, H,
              d, max(0, int(max_q_len)), float(scale), 1 if causal else 0, out.data_ptr(),
              N.dtype_code(out.dtype), workspace.data_ptr(), nbytes)
        return out
    _call(dev, N.lib().qkv_kv8_attention_shared, q.data_ptr(), N.dtype_code(q.dtype), ts, hs, rows,
          kpool.data_ptr(), kscale.data_ptr(), vpool.data_ptr(), vscale.data_ptr(), fmt, P, n,
          table.data_ptr(), width, group_start.data_ptr(), prefix_lens.data_ptr(), groups,
          1 if always else 0, N.ptr(q_start), N.ptr(q_lens), kv_lens.data_ptr(), B, Hq, H, d, float(scale),
          1 if causal else 0, out.data_ptr(), N.dtype_code(out.dtype), workspace.data_ptr(),
          nbytes)
    return out


@functools.lru_cache(maxsize=256)
def attention_kv8_shared_workspace_bytes(B: int, groups: int, rows: int, Hq: int, H: int,
                                         d: int) -> int:
    """Bytes of the workspace that attention_kv8_shared needs at these sizes."""
    return N.lib().qkv_kv8_attention_shared_workspace_bytes(B, groups, rows, Hq, H, d)


@functools.lru_cache(maxsize=256)
def _shared_plain(B: int, groups: int, rows: int, Hq: int, H: int, d: int, width: int,
                  page_tokens: int) -> int:
    return N.lib().qkv_kv8_attention_shared_plain(B, groups, rows, Hq, H, d, width, page_tokens)


class PagedKV8Store:
    """Pools, page table and free list of a batch of B requests, on the device.

    A step::

        plan = store.plan(new_lens, rows)          # who gets how many tokens
        store.append(k, v, plan)                   # (rows, H, d)
        out = store.attention(q, plan)             # (rows, Hq, d), causal
        store.release(done)                        # finished requests' pages

    With ``sharing`` requests may go on from others' tokens (between steps)::

        store.fork(src, dst)                       # whole pages shared, not copied
        out = store.attention(q, plan, groups=(group_start, prefix_lens))

    ``code`` is "int8" or "fp8" (float8 e4m3).  Nothing here reads a length back
    to the host, so a step can be captured; :meth:`grow` adds pages.

    A plan's tokens count as cached from then on.  An append that refuses its rows
    (shape, type) has written nothing: append them with the same plan, before the
    next step reads the cache."""

    def __init__(self, B: int, H: int, d: int, num_pages: int, device,
                 page_tokens: int = PAGE_TOKENS, pages_per_seq: Optional[int] = None,
                 code: str = "int8", sharing: bool = False):
        if code not in CODE_DTYPES:
            raise ValueError(f"code {code!r} must be one of {tuple(CODE_DTYPES)}")
        if d not in (64, 96, 128):
            raise ValueError(f"the 8-bit cache runs head_dim 64, 96 or 128; got {d}")
        if page_tokens not in PAGE_SIZES:
            raise ValueError(f"page_tokens {page_tokens} must be one of {PAGE_SIZES}")
        if B < 1 or H < 1 or num_pages < 1:
            raise ValueError(f"need at least one request, head and page; got {B}, {H}, {num_pages}")
        self.B, self.H, self.d, self.pt, self.code = B, H, d, page_tokens, code
        dev, nb = torch.device(device), page_tokens // BLOCK_TOKENS
        self.kpool = torch.zeros(num_pages, H, page_tokens, d, dtype=torch.int8,
                                 device=dev).view(CODE_DTYPES[code])
        self.vpool = torch.zeros(num_pages, H, nb, d, BLOCK_TOKENS, dtype=torch.int8,
                                 device=dev).view(CODE_DTYPES[code])
        self.kscale = torch.zeros(num_pages, H, nb, dtype=torch.float32, device=dev)
        self.vscale = torch.zeros_like(self.kscale)
        self.table = torch.zeros(B, pages_per_seq or num_pages, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)
        # the lowest page is handed out first
        self.free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=dev)
        # a page's holders beyond the first; None: no page is ever shared
        self.shares = torch.zeros(num_pages, dtype=torch.int32, device=dev) if sharing else None
        self.device = self.lens.device

    @property
    def num_pages(self) -> int:
        return self.kpool.shape[0]

    @property
    def pages_per_seq(self) -> int:
        return self.table.shape[1]

    def pools(self) -> dict:
        return dict(kpool=self.kpool, kscale=self.kscale, vpool=self.vpool, vscale=self.vscale)

    def plan(self, new_lens: torch.Tensor, rows: int, max_q_len: Optional[int] = None,
             out: Optional[PagePlan] = None) -> PagePlan:
        """plan_pages for this step's ``new_lens`` ((B,) int32, device); the store's
        lengths, table and free list move on.  ``out`` takes the plan of an earlier
        step of the same ``rows`` (a captured step keeps one)."""
        if out is None:
            out = PagePlan.empty(self.B, rows, self.device, self.lens, self.free_count, max_q_len)
        elif out.kv_lens is not self.lens or out.free_count is not self.free_count:
            raise ValueError("out must be a plan that this store made")
        elif max_q_len is not None:
            out.max_q_len = max_q_len
        return plan_pages(self.table, self.lens, new_lens, self.free, self.free_count, rows,
                          self.pt, out=out)

    def append(self, k: torch.Tensor, v: torch.Tensor, plan: PagePlan) -> None:
        append_kv8(k, v, plan.slots, **self.pools())

    def read(self, slots: torch.Tensor, out_dtype: torch.dtype = torch.float32):
        return read_kv8(slots, **self.pools(), out_dtype=out_dtype)

    def attention(self, q: torch.Tensor, plan: PagePlan, scale: Optional[float] = None,
                  causal: bool = True, out_dtype: torch.dtype = torch.float32,
                  out: Optional[torch.Tensor] = None,
                  groups: Optional[tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
        """``groups``: (group_start, prefix_lens) of attention_kv8_shared, where requests
        share a prefix that is to be read once for all of a group."""
        if groups is not None:
            return attention_kv8_shared(q, **self.pools(), table=self.table, kv_lens=plan.kv_lens,
                                        group_start=groups[0], prefix_lens=groups[1],
                                        q_start=plan.q_start, q_lens=plan.q_lens, scale=scale,
                                        causal=causal, out_dtype=out_dtype, out=out,
                                        max_q_len=plan.max_q_len)
        return attention_kv8(q, **self.pools(), table=self.table, kv_lens=plan.kv_lens,
                             q_start=plan.q_start, q_lens=plan.q_lens, scale=scale, causal=causal,
                             out_dtype=out_dtype, max_q_len=plan.max_q_len, out=out)

    def release(self, done: Optional[torch.Tensor] = None) -> None:
        """Finished requests' pages back to the pool (all requests' without ``done``)."""
        if done is None:
            done = torch.ones(self.B, dtype=torch.bool, device=self.device)
        release_pages(self.table, self.lens, done, self.free, self.free_count, self.pt,
                      shares=self.shares)

    def fork(self, src: torch.Tensor, dst: torch.Tensor,
             tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Empty requests ``dst`` go on from the first ``tokens`` tokens of requests ``src``
        ((F,) int32 each; tokens None: all), see fork_pages; returns the tokens that each
        holds, -1 where refused.  A step's rows are appended before."""
        if self.shares is None:
            raise ValueError("fork needs a store made with sharing=True")
        p = fork_pages(self.table, self.lens, src, dst, tokens, self.free, self.free_count,
                       self.shares, self.pt)
        copy_pages(p.src_pages, p.dst_pages, **self.pools(), tokens=p.copy_tokens)
        return p.granted

    def compact(self) -> CompactPlan:
        """The pages in use move to the lowest places of the pool, see compact_pages.  Slots of
        plans made before are stale."""
        p = compact_pages(self.table, self.lens, self.free, self.free_count, self.pt,
                          shares=self.shares)
        copy_pages(p.src_pages, p.dst_pages, **self.pools(), count=p.moves)
        return p

    def shrink(self, num_pages: int) -> None:
        """A pool of ``num_pages`` pages, compacted (new tensors: a captured step has to be
        captured again).  Reads the free count back to the host; ValueError, with nothing
        changed, where more pages are in use."""
        old = self.num_pages
        used = old - int(self.free_count.item())
        if num_pages < 1 or num_pages > old or used > num_pages:
            raise ValueError(f"cannot shrink {old} pages, {used} of them in use, to {num_pages}")
        self.compact()
        for name in ("kpool", "vpool", "kscale", "vscale"):
            t = getattr(self, name)
            setattr(self, name, t.view(torch.uint8)[:num_pages].clone().view(t.dtype))
        self.free = self.free[old - num_pages:].clone()
        self.free_count -= old - num_pages
        if self.shares is not None:
            self.shares = self.shares[:num_pages].clone()

    def grow(self, num_pages: int, pages_per_seq: Optional[int] = None) -> None:
        """At least ``num_pages`` pages in the pool and ``pages_per_seq`` in the
        table (new tensors: a captured step has to be captured again)."""
        old, more = self.num_pages, num_pages - self.num_pages
        if more > 0:
            for name in ("kpool", "vpool", "kscale", "vscale"):
                t = getattr(self, name)
                new = torch.zeros(num_pages, *t.shape[1:], device=self.device,
                                  dtype=torch.int8 if t.element_size() == 1 else t.dtype)
                new = new.view(t.dtype)
                new[:old].view(torch.uint8).copy_(t.view(torch.uint8))
                setattr(self, name, new)
            # the new pages go under the free ones: [new pages, old free list]
            ids = torch.arange(num_pages - 1, old - 1, -1, dtype=torch.int32, device=self.device)
            self.free = torch.cat([ids, self.free])
            self.free_count += more
            if self.shares is not None:
                self.shares = torch.cat([self.shares, torch.zeros_like(ids)])
        if pages_per_seq is not None and pages_per_seq > self.pages_per_seq:
            pad = torch.zeros(self.B, pages_per_seq - self.pages_per_seq, dtype=torch.int32,
                              device=self.device)
            self.table = torch.cat([self.table, pad], 1)

    def to(self, device) -> None:
        self.device = torch.device(device)
        for name in ("kpool", "vpool", "kscale", "vscale", "table", "lens", "free", "free_count",
                     "shares"):
            if getattr(self, name) is not None:
                setattr(self, name, getattr(self, name).to(self.device))
        self.device = self.lens.device

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size()
                   for t in (self.kpool, self.kscale, self.vpool, self.vscale))


class PagedKV8Engine:
    """The engine interface (QuashKVEngine: append / attention / clear over B
    sequences of one length) on the 8-bit paged store.  No rotation, codebook or
    seed: ``key_bits`` and ``value_bits`` are 8."""

    def __init__(self, head_dim: int = 128, device=None, num_pages: int = 0,
                 page_tokens: int = PAGE_TOKENS, code: str = "int8"):
        if head_dim not in (64, 96, 128):
            raise ValueError(f"the 8-bit cache runs head_dim 64, 96 or 128; got {head_dim}")
        if code not in CODE_DTYPES:
            raise ValueError(f"code {code!r} must be one of {tuple(CODE_DTYPES)}")
        if page_tokens not in PAGE_SIZES:
            raise ValueError(f"page_tokens {page_tokens} must be one of {PAGE_SIZES}")
        self.head_dim, self.key_bits, self.value_bits = head_dim, 8, 8
        self.device = _default_device(device)
        self.initial_pages, self.page_tokens, self.code = num_pages, page_tokens, code
        self._store: Optional[PagedKV8Store] = None
        self._total_tokens = 0
        self._appends = 0

    def append(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Quantise (B, H, S, d) keys / values into the pages behind the cached ones."""
        dev = N.require_gpu(keys, values, what="PagedKV8Engine.append")
        if keys.dim() != 4 or keys.shape != values.shape or keys.shape[-1] != self.head_dim:
            raise ValueError(
                f"Expected keys and values of shape (batch, n_heads, seq_len, {self.head_dim}); "
                f"got {tuple(keys.shape)} and {tuple(values.shape)}")
        B, H, S, d = keys.shape
        n, T = self.page_tokens, self._total_tokens
        st = self._store
        if st is not None and ((st.B, st.H) != (B, H) or st.device != dev):
            if T:
                raise ValueError(f"append shape (B={B}, H={H}) on {dev} does not match the cache "
                                 f"(B={st.B}, H={st.H}) on {st.device}")
            st = self._store = None  # empty (cleared): any shape
        if B == 0 or H == 0:
            raise ValueError(f"need at least one sequence and head; got {tuple(keys.shape)}")
        need = -(-(T + S) // n)      # pages a sequence
        if st is None:
            st = self._store = PagedKV8Store(B, H, d, max(self.initial_pages, B * need, 1), dev, n,
                                             max(need, 1), self.code)
        if B * need > st.num_pages or need > st.pages_per_seq:
            st.grow(max(2 * st.num_pages, B * need) if B * need > st.num_pages else st.num_pages,
                    max(2 * st.pages_per_seq, need))
        if keys.dtype != values.dtype or keys.dtype not in (torch.float32, torch.float16,
                                                            torch.bfloat16):
            keys, values = keys.float(), values.float()
        if S > 0:
            k, v = (x.transpose(1, 2).reshape(B * S, H, d) for x in (keys, values))
            new = torch.full((B,), S, dtype=torch.int32, device=dev)
            st.append(k, v, st.plan(new, B * S, max_q_len=S))
        self._total_tokens += S
        self._appends += 1

    def attention(self, queries: torch.Tensor, scale: Optional[float] = None,
                  causal: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Attention of (B, Hq, Q, d) queries over every cached token, Hq a
        multiple of the kv heads; causal: query i sits at token T - Q + i."""
        if self._total_tokens == 0:
            raise ValueError("No compressed KV blocks in cache. Call append() first.")
        st = self._store
        N.require_gpu(queries, what="PagedKV8Engine.attention")
        if (queries.dim() != 4 or queries.shape[0] != st.B or queries.shape[3] != self.head_dim
                or queries.shape[1] % st.H != 0):
            raise ValueError(f"queries {tuple(queries.shape)} do not match the cache "
                             f"(B={st.B}, kv heads={st.H}, head_dim={self.head_dim})")
        B, Hq, Q, d = queries.shape
        q = queries.transpose(1, 2).reshape(B * Q, Hq, d)
        if q.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            q = q.float()
        out = attention_kv8(q, **st.pools(), table=st.table, kv_lens=st.lens, scale=scale,
                            causal=causal, out_dtype=out_dtype)
        return out.view(B, Q, Hq, d).transpose(1, 2).contiguous()

    def clear(self) -> None:
        if self._store is not None:
            self._store.release()
        self._total_tokens = self._appends = 0

    @property
    def store(self) -> Optional[PagedKV8Store]:
        return self._store

    @property
    def total_tokens(self) -> int:
        return self._total_tokens

    @property
    def num_blocks(self) -> int:
        return self._appends

    def compression_ratio(self, original_dtype: torch.dtype = torch.float16) -> float:
        """Bits of a token's K and V in ``original_dtype`` over those held: 8 a
        value and an fp32 scale for each half of a 16-token block."""
        if self._total_tokens == 0:
            return 1.0
        bits = 2 * (8 * self.head_dim + 32 / BLOCK_TOKENS)
        return 2 * self.head_dim * torch.finfo(original_dtype).bits / bits

    def actual_memory_bytes(self) -> int:
        """Bytes of the codes and scales of the cached tokens."""
        if self._total_tokens == 0:
            return 0
        T, st = self._total_tokens, self._store
        return st.B * st.H * 2 * (T * self.head_dim + 4 * (-(-T // BLOCK_TOKENS)))

    def to(self, device) -> "PagedKV8Engine":
        self.device = torch.device(device)
        if self._store is not None:
            self._store.to(device)
        return self

    def __repr__(self) -> str:
        pages = 0 if self._store is None else self._store.num_pages
        return (f"PagedKV8Engine(head_dim={self.head_dim}, code={self.code}, "
                f"cached_tokens={self._total_tokens}, pages={pages}, device={self.device})")
