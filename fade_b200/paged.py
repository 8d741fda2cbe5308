"""A serving step over a paged FP16/BF16 cache.

Prompts live uncompressed until their first tier reassignment.  For a
continuous batch of requests of different lengths this module keeps them in
pages of a shared pool and runs one step as three operators on the GPU, with
no host synchronisation:

* ``plan_step``: pages for the step's new tokens (block table, free list), the
  slot and position of every token, from the requests' lengths;
* ``rope_append``: rotary positions (one to four axes) of q and k, and the
  write of k and v to their slots (``rope_axes``: the rotation alone);
* ``chunk_attention``: every new token over its request's pages, from single
  tokens to long prompt chunks, causal and optionally windowed.

``PagedKVCache`` owns the pool, table and free list and strings the three
together; ``gather`` hands a request's K/V on to the tier quantisers:
``TieredDecoder.load_prompt``, and ``TieredKVCache.update`` for requests at text
positions (see there).

Serving only: results carry no gradient, whatever the inputs ask for.

The reference keeps one dense cache per batch and has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import Tensor

from fade_b200 import _lib

PAGE_SIZES = (16, 32, 64, 128)

_PLAN_ERRORS = {
    1: "the free list holds too few pages",
    2: "a request needs more pages than a row of the block table holds",
    3: "more new tokens than `total`",
    4: "a negative length, or a free count outside the free list",
}


_I32, _I64 = torch.int32, torch.int64


def _int32(t: Tensor, shape: tuple, what: str) -> int:
    if t.dtype is not _I32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _table(t: Tensor, rows: int) -> tuple[int, int, int]:
    shape, stride = t.shape, t.stride()
    if t.dtype is not _I32 or len(shape) != 2 or shape[0] != rows or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"block_table must be int32 [{rows}, pages per request] with contiguous rows, got {t.dtype} "
                         f"{tuple(shape)}")
    return t.data_ptr(), shape[1], stride[0]


@dataclass
class StepPlan:
    """What ``plan_step`` fills in (all on the device)."""

    cu_q: Tensor          # int32 [R + 1]: first token of each request, then the number of tokens
    kv_lens: Tensor       # int32 [R]: cached tokens, the new ones included
    positions: Tensor     # int32 [total]: position of each token in its request (0 for padding)
    slots: Tensor         # int64 [total]: cache slot of each token (-1 for padding)
    n_free: Tensor        # int32 [1]: pages left on the free list
    status: Tensor        # int32 [1]: 0, or why nothing was planned

    @classmethod
    def empty(cls, n_requests: int, total: int, device: torch.device | str = "cuda") -> "StepPlan":
        """Buffers for steps of `n_requests` requests and up to `total` tokens."""
        def i32(n):
            return torch.empty(n, dtype=torch.int32, device=device)

        return cls(i32(n_requests + 1), i32(n_requests), i32(total),
                   torch.empty(total, dtype=torch.int64, device=device), i32(1), i32(1))

    def check(self) -> None:
        """Raise if the step could not be planned (synchronises)."""
        code = int(self.status.item())
        if code:
            raise RuntimeError(f"plan_step: {_PLAN_ERRORS.get(code, f'status {code}')}")


def plan_step(new_lens: Tensor, kv_lens: Tensor, block_table: Tensor, free_pages: Tensor, n_free: Tensor,
              page_size: int, total: int, out: StepPlan | None = None) -> StepPlan:
    """Pages, slots and positions of one step's new tokens.

    new_lens / kv_lens: int32 [R], tokens to add and tokens cached so far;
    block_table: int32 [R, W], whose rows list the pages of the cached tokens
    and get the new pages appended in place; free_pages: int32 [F], a stack of
    free page ids of height ``n_free`` (int32 [1]).  ``total`` (host) is the
    length of the token arrays, at least the sum of new_lens; the rest of them
    is padding.  Requests take pages in order, from the top of the stack.

    Lengths and the free count are inputs only: the new ones are in the plan,
    so a repeated call plans the same step.  All or nothing: a step that does
    not fit leaves the table alone and is reported by ``StepPlan.check``."""
    if out is None:
        dev = _lib.same_device(new_lens, kv_lens, block_table, free_pages, n_free)
    else:
        dev = _lib.same_device(new_lens, kv_lens, block_table, free_pages, n_free, out.cu_q, out.kv_lens, out.positions,
                               out.slots, out.n_free, out.status)
    if dev != _lib._current():
        with _lib.on_device(dev):
            return plan_step(new_lens, kv_lens, block_table, free_pages, n_free, page_size, total, out)
    R, F = new_lens.numel(), free_pages.numel()
    total = int(total)
    if page_size < 1 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two of at most 2**20, got {page_size}")
    if total < 0:
        raise ValueError(f"total must not be negative, got {total}")
    if R > _lib.PLAN_MAX_ROWS:
        raise ValueError(f"at most {_lib.PLAN_MAX_ROWS} requests per step, got {R}")
    bt, width, stride = _table(block_table, R)
    if out is None:
        out = StepPlan.empty(R, total, new_lens.device)
    slots = out.slots
    if slots.dtype is not _I64 or slots.shape != (total,) or not slots.is_contiguous():
        raise ValueError(f"out.slots must be a contiguous int64 tensor of shape {(total,)}")
    kv_in, n_in = _int32(kv_lens, (R,), "kv_lens"), _int32(n_free, (1,), "n_free")
    kv_out, n_out = _int32(out.kv_lens, (R,), "out.kv_lens"), _int32(out.n_free, (1,), "out.n_free")
    if (kv_out == kv_in and R) or n_out == n_in:
        raise ValueError("out must not share kv_lens or n_free with the inputs")
    d = _lib.PACK_PLAN.pack(
        R, total, page_size, width, stride, F, _int32(new_lens, (R,), "new_lens"), kv_in, bt,
        _int32(free_pages, (F,), "free_pages"), n_in, _int32(out.cu_q, (R + 1,), "out.cu_q"), kv_out,
        _int32(out.positions, (total,), "out.positions"), slots.data_ptr(), n_out, _int32(out.status, (1,), "out.status"))
    code = _lib.load().fade_plan_step(d, _lib._stream(dev))
    if code:
        _lib.check(code, "plan_step")
    return out


def release_rows(rows: Tensor, kv_lens: Tensor, block_table: Tensor, page_size: int, free_pages: Tensor,
                 n_free: Tensor, status: Tensor | None = None) -> Tensor:
    """Give the pages of finished requests back to the free list, in place.

    rows: bool or uint8 [R], the requests to drop; their kv_lens become 0 and
    their pages go onto the stack in order.  Returns the device status (int32
    [1], 0 when done; nothing changes otherwise)."""
    dev = _lib.require_cuda(rows, kv_lens, block_table, free_pages, n_free, status)
    R, F = rows.numel(), free_pages.numel()
    if rows.dtype not in (torch.bool, torch.uint8) or rows.dim() != 1 or not rows.is_contiguous():
        raise ValueError("rows must be a contiguous bool or uint8 vector")
    if page_size < 1 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two of at most 2**20, got {page_size}")
    if R > _lib.PLAN_MAX_ROWS:
        raise ValueError(f"at most {_lib.PLAN_MAX_ROWS} requests per step, got {R}")
    bt, width, stride = _table(block_table, R)
    if status is None:
        status = torch.empty(1, dtype=torch.int32, device=dev)
    args = (_int32(kv_lens, (R,), "kv_lens"), _int32(free_pages, (F,), "free_pages"), _int32(n_free, (1,), "n_free"),
            _int32(status, (1,), "status"))
    with _lib.on_device(dev) as st:
        _lib.check(_lib.load().fade_release_rows(rows.data_ptr(), R, args[0], bt, width, stride, page_size, args[1], F,
                                                 args[2], args[3], st), "release_rows")
    return status


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def section_axes(sections, interleaved: bool = False) -> list[int]:
    """The axis of each frequency: ``sections[a]`` frequencies of axis a one
    after the other, or interleaved (frequency j of axis ``j % A`` while that
    axis has frequencies left, else of axis 0)."""
    A, half = len(sections), sum(sections)
    if interleaved:
        return [j % A if j % A and j < A * sections[j % A] else 0 for j in range(half)]
    return [a for a in range(A) for _ in range(sections[a])]


def _heads(t: Tensor, T: int, D: int, dtype: torch.dtype, what: str) -> tuple:
    """(tensor with contiguous channels, heads, token stride, head stride)"""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[0] != T or shape[2] != D or t.dtype is not dtype:
        raise ValueError(f"{what} must be [{T}, heads, {D}] in {dtype}, got {tuple(shape)} in {t.dtype}")
    if stride[2] != 1 and D > 1 and t.numel():
        t = t.contiguous()
        stride = t.stride()
    return t, shape[1], stride[0], stride[1]


def _rope_head(x: Tensor, T: int, D: int, positions: Tensor, inv_freq: Tensor, sections) -> tuple:
    """(positions, rot, axes, padded sections, pos_64, pos_stride) after the checks."""
    half = inv_freq.numel()
    sections = (half,) if sections is None else tuple(sections)
    A = len(sections)
    if not 1 <= A <= _lib.MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must list one to {_lib.MAX_AXES} counts, got {sections}")
    if inv_freq.dtype is not torch.float32 or not inv_freq.is_contiguous() or sum(sections) != half or 2 * half > D:
        raise ValueError(f"inv_freq must be contiguous float32 with sum(sections) = {sum(sections)} entries, at most "
                         f"half of head_dim {D}, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.shape != (A, T) or (positions.dtype is not _I32 and positions.dtype is not _I64):
        raise ValueError(f"positions must be int32 or int64 [{A}, {T}], got {positions.dtype} {tuple(positions.shape)}")
    ps, one = positions.stride()
    if one != 1:
        positions = positions.contiguous()
        ps = positions.stride(0)
    return (positions, 2 * half, A, sections + (0,) * (_lib.MAX_AXES - A), positions.dtype is _I64, ps)


def _out_heads(out: Tensor | None, x: Tensor, T: int, H: int, D: int) -> tuple:
    """(output, token stride, head stride)"""
    if out is None:
        return torch.empty((T, H, D), dtype=x.dtype, device=x.device), H * D, D
    stride = out.stride()
    if out.shape != (T, H, D) or out.dtype is not x.dtype or (D > 1 and stride[2] != 1):
        raise ValueError("out must match the input's shape and dtype, with contiguous channels")
    return out, stride[0], stride[1]


def rope_axes(x: Tensor, positions: Tensor, inv_freq: Tensor, sections=None, *, interleaved: bool = False,
              inverse: bool = False, round_tables: bool = False, out: Tensor | None = None) -> Tensor:
    """Rotary embedding with one to four position axes (time, height, width).

    x: [T, H, D] fp16, bf16 or fp32, any token and head strides; positions:
    integer [A, T] ([T] for one axis); inv_freq: float32 [rot/2] (a scheme's
    ``RopeScheme.axes_inv_freq``; its ``inv_freq`` belongs to its tables and
    differs for scaled positions and models without rotation); sections:
    frequencies per axis, see ``section_axes`` (default: all on one axis).  Channel j pairs with
    ``j + rot/2``; channels from rot on are copied.  ``inverse`` rotates back.
    Angles, cos and sin are fp32 and the result is rounded once;
    ``round_tables`` rounds cos and sin through x's dtype first, as the tables
    of ``MRope.compute_cos_sin`` are.  ``out`` may be x itself."""
    dev = _lib.same_device(x, positions, inv_freq) if out is None else _lib.same_device(x, positions, inv_freq, out)
    if dev != _lib._current():
        with _lib.on_device(dev):
            return rope_axes(x, positions, inv_freq, sections, interleaved=interleaved, inverse=inverse,
                             round_tables=round_tables, out=out)
    if x.dim() != 3:
        raise ValueError(f"expected a [tokens, heads, head_dim] tensor, got shape {tuple(x.shape)}")
    T, H, D = x.shape
    positions, rot, axes, sec, p64, ps = _rope_head(x, T, D, positions, inv_freq, sections)
    x, H, x_st, x_sh = _heads(x, T, D, x.dtype, "x")
    out, o_st, o_sh = _out_heads(out, x, T, H, D)
    d = _lib.PACK_ROPE.pack(
        _lib.dtype_code(x.dtype), T, H, 0, D, rot, axes, *sec, interleaved, inverse, round_tables, p64, ps,
        positions.data_ptr(), inv_freq.data_ptr(), x.data_ptr(), x_st, x_sh, out.data_ptr(), o_st, o_sh,
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    code = _lib.load().fade_rope_axes(d, _lib._stream(dev))
    if code:
        _lib.check(code, "rope_axes")
    return out


def _pool(t: Tensor, heads: int, D: int, dtype: torch.dtype, what: str) -> tuple:
    """(shape, pointer, page stride, head stride, token stride)"""
    shape, stride = t.shape, t.stride()
    if len(shape) != 4 or shape[1] != heads or shape[3] != D or t.dtype is not dtype or stride[3] != 1:
        raise ValueError(f"{what} must be [pages, {heads}, page size, {D}] in {dtype} with contiguous channels, got "
                         f"{tuple(shape)} in {t.dtype}")
    return shape, t.data_ptr(), stride[0], stride[1], stride[2]


def rope_append(q: Tensor, k: Tensor, v: Tensor, positions: Tensor, inv_freq: Tensor, sections, slots: Tensor,
                k_pool: Tensor, v_pool: Tensor, *, interleaved: bool = False, round_tables: bool = False,
                out: Tensor | None = None) -> Tensor:
    """Rotate q and k (see ``rope_axes``) and write the rotated k, and v, to
    their cache slots; returns the rotated q.

    q: [T, Hq, D]; k, v: [T, Hkv, D]; k_pool, v_pool: [n_pages, Hkv, page_size,
    D], any page, head and token strides; slots: int64 [T], page * page_size +
    offset (``StepPlan.slots``).  Tokens with a slot outside the pool (padding:
    -1) are rotated but not written.  ``out`` may be q itself."""
    dev = _lib.same_device(q, k, v, positions, inv_freq, slots, k_pool, v_pool, q if out is None else out)
    if dev != _lib._current():
        with _lib.on_device(dev):
            return rope_append(q, k, v, positions, inv_freq, sections, slots, k_pool, v_pool, interleaved=interleaved,
                               round_tables=round_tables, out=out)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [tokens, heads, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    T, Hq, D = q.shape
    dtype = q.dtype
    positions, rot, axes, sec, p64, ps = _rope_head(q, T, D, positions, inv_freq, sections)
    q, Hq, q_st, q_sh = _heads(q, T, D, dtype, "q")
    k, Hkv, k_st, k_sh = _heads(k, T, D, dtype, "k")
    v, Hv, v_st, v_sh = _heads(v, T, D, dtype, "v")
    if Hv != Hkv:
        raise ValueError(f"k and v must have the same heads, got {Hkv} and {Hv}")
    if slots.dtype is not _I64 or slots.shape != (T,) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of shape {(T,)}")
    shape, *kp = _pool(k_pool, Hkv, D, dtype, "k_pool")
    v_shape, *vp = _pool(v_pool, Hkv, D, dtype, "v_pool")
    page_size = shape[2]
    if page_size & (page_size - 1) or page_size < 1 or v_shape != shape:
        raise ValueError("k_pool and v_pool must have one shape and a page size that is a power of two")
    out, o_st, o_sh = _out_heads(out, q, T, Hq, D)
    d = _lib.PACK_ROPE.pack(
        _lib.dtype_code(dtype), T, Hq, Hkv, D, rot, axes, *sec, interleaved, 0, round_tables, p64, ps,
        positions.data_ptr(), inv_freq.data_ptr(), q.data_ptr(), q_st, q_sh, out.data_ptr(), o_st, o_sh,
        k.data_ptr(), k_st, k_sh, v.data_ptr(), v_st, v_sh, slots.data_ptr(), page_size, shape[0], *kp, *vp)
    code = _lib.load().fade_rope_axes(d, _lib._stream(dev))
    if code:
        _lib.check(code, "rope_append")
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
_WS: dict = {}          # (device, stream, head_dim) -> (workspace, address, bytes)


def chunk_attention(q: Tensor, k_pool: Tensor, v_pool: Tensor, block_table: Tensor, cu_q: Tensor, kv_lens: Tensor, *,
                    causal: bool = True, window: int | None = None, sm_scale: float | None = None,
                    out: Tensor | None = None, return_lse: bool = False) -> Tensor | dict:
    """Attention of a step's new tokens over their requests' paged caches.

    q: [T, Hq, D] fp16 or bf16, the requests' tokens one after the other
    (cu_q: int32 [R + 1]); k_pool, v_pool: [n_pages, Hkv, page_size, D];
    block_table: int32 [R, W]; kv_lens: int32 [R], cached tokens with the new
    ones included.  Query i of a request sits at position
    ``kv_len - q_len + i``; ``causal`` hides the keys after it, ``window`` those
    ``window`` or more before it.  Query head h reads kv head
    ``h // (Hq // Hkv)``; sm_scale defaults to 1/sqrt(D).

    Returns [T, Hq, D], zeros where no key is visible and for tokens past cu_q[R]
    (which a given `out` keeps); with ``return_lse`` a dict of that as "out" and
    the float32 [T, Hq] log of the sum of exponentials as "lse", -inf for those
    rows.  Head_dim 64 or 128, page size 16 to 128, Hq / Hkv up to 128.  What the
    pool holds past a request's kv_len is never used, and a NaN or infinity in a
    token's K or V reaches only the queries that see the token (a channel in which
    a query sees an infinity itself may be NaN).  `out` must not overlap q.

    Workspace is cached per (device, stream, head_dim), 39 MB at head_dim 128;
    calls on one stream, from any number of host threads, follow one another
    whole, so sharing it is safe.  A captured call's workspace belongs to its
    graph."""
    dev = _lib.same_device(q, k_pool, v_pool, block_table, cu_q, kv_lens, q if out is None else out)
    if dev != _lib._current():
        with _lib.on_device(dev):
            return chunk_attention(q, k_pool, v_pool, block_table, cu_q, kv_lens, causal=causal, window=window,
                                   sm_scale=sm_scale, out=out, return_lse=return_lse)
    if q.dim() != 3 or k_pool.dim() != 4:
        raise ValueError(f"q must be [tokens, heads, head_dim] and k_pool [pages, heads, page size, head_dim], got "
                         f"{tuple(q.shape)} and {tuple(k_pool.shape)}")
    T, Hq, D = q.shape
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"unsupported dtype {dtype}; expected float16 or bfloat16")
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    Hkv = k_pool.shape[1]
    shape, *kp = _pool(k_pool, Hkv, D, dtype, "k_pool")
    v_shape, *vp = _pool(v_pool, Hkv, D, dtype, "v_pool")
    n_pages, _, page_size, _ = shape
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page size must be one of {PAGE_SIZES}, got {page_size}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq > 128 * Hkv:
        raise ValueError(f"Hq={Hq} must be a multiple of Hkv={Hkv}, at most 128 times it")
    if v_shape != shape:
        raise ValueError(f"k_pool and v_pool must have one shape, got {tuple(shape)} and {tuple(v_shape)}")
    R = kv_lens.numel()
    bt, width, stride = _table(block_table, R)
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if not 1e-45 <= scale <= 1e30:
        raise ValueError(f"sm_scale must be 1e-45 (the least that fp32 tells from 0) to 1e30, got {sm_scale}")
    q_st, q_sh, one = q.stride()
    q_ptr = q.data_ptr()
    if one != 1 or q_st % 8 or q_sh % 8 or q_ptr % 16:   # rows must be 16-byte aligned for the kernel's loads
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        (q_st, q_sh, _), q_ptr = q.stride(), q.data_ptr()
    fresh = out is None
    out, o_st, o_sh = _out_heads(out, q, T, Hq, D)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    if R == 0:                                           # nothing is launched
        if fresh:
            out.zero_()
        if return_lse:
            lse.fill_(float("-inf"))
    d = _lib.PACK_CHUNK.pack(
        _lib.FADE_BF16 if dtype is torch.bfloat16 else _lib.FADE_F16, R, T, Hq, Hkv, D, page_size, n_pages, width, stride,
        causal, window or 0, fresh | bool(return_lse) << 1, scale, q_ptr, q_st, q_sh, out.data_ptr(), o_st, o_sh,
        0 if lse is None else lse.data_ptr(),
        *kp, *vp, bt, _int32(cu_q, (R + 1,), "cu_q"), _int32(kv_lens, (R,), "kv_lens"))
    lib = _lib.load()
    st = _lib._stream(dev)
    # a graph may be replayed beside anything, so its calls share no workspace with others'
    captured = _lib._capturing()
    ws = None if captured else _WS.get((dev, st, D))
    if ws is None:
        need = lib.fade_chunk_attn_workspace_size(d)
        if need == 0:
            raise ValueError(f"unsupported chunk attention sizes (R={R}, T={T}, n_pages={n_pages}, table width {width})")
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        ws = (ws, ws.data_ptr(), need)
        if not captured:
            ws = _WS.setdefault((dev, st, D), ws)     # another thread's, if it was first
    code = lib.fade_chunk_attn(d, ws[1], ws[2], st)
    if code:
        _lib.check(code, "chunk_attention")
    return {"out": out, "lse": lse} if return_lse else out


def check_device_errors(device: torch.device | str = "cuda") -> None:
    """Raise if a bounded device wait of a ``chunk_attention`` call on `device`
    gave up since this was last asked, in a replayed graph or not.  Synchronises
    the current stream; calls on others are covered once they have ended."""
    with _lib.on_device(torch.device(device)) as st:
        _lib.check(_lib.load().fade_chunk_attn_check(st), "chunk_attention")


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
class PagedKVCache:
    """Pages of K/V for up to `max_requests` requests, shared by all layers'
    tables: page ids are handed out once per step and index every layer's pool.

    Args:
        n_layers, n_kv_heads, head_dim, dtype: model shape.
        n_pages, page_size: pool size per layer (pages of 16 to 128 tokens).
        max_requests: rows of the block table.
        max_tokens: longest request (sets the table's width).
    """

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, max_requests: int,
                 max_tokens: int, page_size: int = 128, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page size must be one of {PAGE_SIZES}, got {page_size}")
        if not 1 <= max_requests <= _lib.PLAN_MAX_ROWS:
            raise ValueError(f"max_requests must be 1 to {_lib.PLAN_MAX_ROWS}, got {max_requests}")
        dev = torch.device(device)
        self.page_size, self.max_requests = page_size, max_requests
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=dev)
        self.v = torch.zeros(shape, dtype=dtype, device=dev)
        self.block_table = torch.zeros(max_requests, -(-max_tokens // page_size), dtype=torch.int32, device=dev)
        # pages are handed out in ascending order from a full pool
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self._state = torch.zeros(max_requests + 1, dtype=torch.int32, device=dev)
        self._state[-1] = n_pages
        self.kv_lens, self.n_free = self._state[:-1], self._state[-1:]
        # of the last release, and the worst since `check`
        self._released, self._release_status = torch.zeros(2, 1, dtype=torch.int32, device=dev)

    def plan(self, new_lens: Tensor, total: int, out: StepPlan | None = None) -> StepPlan:
        """Plan a step of ``new_lens`` (int32 [max_requests]) and take its
        pages: the cache's lengths and free count become the plan's."""
        if out is None:
            state = torch.empty_like(self._state)
            out = StepPlan.empty(0, int(total), state.device)
            out.cu_q = torch.empty_like(state)
            out.kv_lens, out.n_free = state[:-1], state[-1:]
        plan = plan_step(new_lens, self.kv_lens, self.block_table, self.free_pages, self.n_free, self.page_size, total,
                         out)
        self.kv_lens.copy_(plan.kv_lens)
        self.n_free.copy_(plan.n_free)
        return plan

    def append(self, layer: int, plan: StepPlan, q: Tensor, k: Tensor, v: Tensor, inv_freq: Tensor, sections=None,
               positions: Tensor | None = None, **kw) -> Tensor:
        """Rotate q and k and append k, v to `layer` (``rope_append``);
        positions default to the plan's."""
        return rope_append(q, k, v, plan.positions if positions is None else positions, inv_freq, sections, plan.slots,
                           self.k[layer], self.v[layer], **kw)

    def attend(self, layer: int, plan: StepPlan, q: Tensor, **kw):
        """``chunk_attention`` of the step's rotated queries over `layer`."""
        return chunk_attention(q, self.k[layer], self.v[layer], self.block_table, plan.cu_q, plan.kv_lens, **kw)

    def release(self, rows: Tensor) -> None:
        """Drop the requests of the bool [max_requests] mask `rows`.  A release
        that fails drops none of them; ``check`` raises on it, also after others."""
        release_rows(rows, self.kv_lens, self.block_table, self.page_size, self.free_pages, self.n_free, self._released)
        torch.maximum(self._release_status, self._released, out=self._release_status)

    def check(self) -> None:
        """Raise if a release failed or a device wait gave up since the last
        check (synchronises)."""
        code = int(self._release_status.item())
        if code:
            self._release_status.zero_()
            raise RuntimeError(f"release: {_PLAN_ERRORS.get(code, f'status {code}')}")
        check_device_errors(self._state.device)

    def gather(self, layer: int, rows, length: int) -> tuple[Tensor, Tensor]:
        """K, V [len(rows), n_kv_heads, length, head_dim] of the first `length`
        tokens of the given rows, contiguous: what the tier quantisers and
        ``TieredDecoder.load_prompt`` take.

        K comes as it was rotated.  ``TieredDecoder`` keeps it so, whatever its
        positions were.  ``TieredKVCache`` un-rotates what an eviction leaves, and
        has one position per token for it, counted from 0: hand it only requests
        that were appended at the plan's own positions (no ``positions``), not those
        with image or video tokens on several axes."""
        pages = self.block_table[rows, :-(-length // self.page_size)].long()
        return tuple(p[layer][pages].transpose(1, 2).flatten(2, 3)[:, :, :length].contiguous()
                     for p in (self.k, self.v))


__all__ = [
    "PAGE_SIZES",
    "PagedKVCache",
    "StepPlan",
    "check_device_errors",
    "chunk_attention",
    "plan_step",
    "release_rows",
    "rope_append",
    "rope_axes",
    "section_axes",
]
