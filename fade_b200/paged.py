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
together; ``gather`` hands a request's K/V on to the tier quantisers
(``TieredDecoder.load_prompt``, ``TieredKVCache.update``).

The reference keeps one dense cache per batch and has no counterpart.
"""

from __future__ import annotations

import ctypes
import math
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


def _int32(t: Tensor, shape: tuple, what: str) -> int:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {tuple(shape)}, got {t.dtype} "
                         f"{tuple(t.shape)}")
    return t.data_ptr()


def _table(t: Tensor, rows: int) -> tuple[int, int, int]:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != rows or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{rows}, pages per request] with contiguous rows, got {t.dtype} "
                         f"{tuple(t.shape)}")
    return t.data_ptr(), t.shape[1], t.stride(0)


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
    dev = _lib.require_cuda(new_lens, kv_lens, block_table, free_pages, n_free)
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
        out = StepPlan.empty(R, total, dev)
    else:
        _lib.require_cuda(new_lens, out.cu_q, out.kv_lens, out.positions, out.slots, out.n_free, out.status)
        if out.slots.dtype != torch.int64 or out.slots.shape != (total,) or not out.slots.is_contiguous():
            raise ValueError(f"out.slots must be a contiguous int64 tensor of shape {(total,)}")
        if out.kv_lens.data_ptr() == kv_lens.data_ptr() and R or out.n_free.data_ptr() == n_free.data_ptr():
            raise ValueError("out must not share kv_lens or n_free with the inputs")
    d = _lib.PlanDesc(
        R, total, page_size, width, stride, F,
        _int32(new_lens, (R,), "new_lens"), _int32(kv_lens, (R,), "kv_lens"), bt,
        _int32(free_pages, (F,), "free_pages"), _int32(n_free, (1,), "n_free"), _int32(out.cu_q, (R + 1,), "out.cu_q"),
        _int32(out.kv_lens, (R,), "out.kv_lens"), _int32(out.positions, (total,), "out.positions"),
        out.slots.data_ptr(), _int32(out.n_free, (1,), "out.n_free"), _int32(out.status, (1,), "out.status"))
    st = _lib.bind(dev)
    _lib.check(_lib.load().fade_plan_step(ctypes.byref(d), st), "plan_step")
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
    st = _lib.bind(dev)
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


def _heads(t: Tensor, T: int, D: int, dtype: torch.dtype, what: str) -> Tensor:
    if t.dim() != 3 or t.shape[0] != T or t.shape[2] != D or t.dtype != dtype:
        raise ValueError(f"{what} must be [{T}, heads, {D}] in {dtype}, got {tuple(t.shape)} in {t.dtype}")
    return t if t.stride(2) == 1 or D == 1 or t.numel() == 0 else t.contiguous()


def _rope_head(x: Tensor, positions: Tensor, inv_freq: Tensor, sections) -> tuple:
    """(positions, rot, padded sections, pos_64, pos_stride) after the checks."""
    sections = tuple(int(s) for s in sections)
    A, T = len(sections), x.shape[0]
    if not 1 <= A <= _lib.MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must list one to {_lib.MAX_AXES} counts, got {sections}")
    half = inv_freq.numel()
    if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or sum(sections) != half or 2 * half > x.shape[2]:
        raise ValueError(f"inv_freq must be contiguous float32 with sum(sections) = {sum(sections)} entries, at most "
                         f"half of head_dim {x.shape[2]}, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.shape != (A, T) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64 [{A}, {T}], got {positions.dtype} {tuple(positions.shape)}")
    if positions.stride(1) != 1:
        positions = positions.contiguous()
    return (positions, 2 * half, sections + (0,) * (_lib.MAX_AXES - A), positions.dtype == torch.int64,
            positions.stride(0))


def rope_axes(x: Tensor, positions: Tensor, inv_freq: Tensor, sections=None, *, interleaved: bool = False,
              inverse: bool = False, round_tables: bool = False, out: Tensor | None = None) -> Tensor:
    """Rotary embedding with one to four position axes (time, height, width).

    x: [T, H, D] fp16, bf16 or fp32, any token and head strides; positions:
    integer [A, T] ([T] for one axis); inv_freq: float32 [rot/2] (a
    ``RopeScheme.inv_freq``); sections: frequencies per axis, see
    ``section_axes`` (default: all on one axis).  Channel j pairs with
    ``j + rot/2``; channels from rot on are copied.  ``inverse`` rotates back.
    Angles, cos and sin are fp32 and the result is rounded once;
    ``round_tables`` rounds cos and sin through x's dtype first, as the tables
    of ``MRope.compute_cos_sin`` are.  ``out`` may be x itself."""
    dev = _lib.require_cuda(x, positions, inv_freq, out)
    if x.dim() != 3:
        raise ValueError(f"expected a [tokens, heads, head_dim] tensor, got shape {tuple(x.shape)}")
    T, H, D = x.shape
    positions, rot, sec, p64, ps = _rope_head(x, positions, inv_freq, sections or (inv_freq.numel(),))
    axes = len(sections or (0,))
    x = _heads(x, T, D, x.dtype, "x")
    if out is None:
        out = torch.empty((T, H, D), dtype=x.dtype, device=dev)
    elif out.shape != x.shape or out.dtype != x.dtype or (D > 1 and out.stride(2) != 1):
        raise ValueError("out must match x's shape and dtype, with contiguous channels")
    d = _lib.RopeDesc(_lib.dtype_code(x.dtype), T, H, 0, D, rot, axes, *sec, interleaved, inverse, round_tables, p64, ps,
                      positions.data_ptr(), inv_freq.data_ptr(), x.data_ptr(), x.stride(0), x.stride(1),
                      out.data_ptr(), out.stride(0), out.stride(1))
    st = _lib.bind(dev)
    _lib.check(_lib.load().fade_rope_axes(ctypes.byref(d), st), "rope_axes")
    return out


def _pool(t: Tensor, heads: int, D: int, dtype: torch.dtype, what: str) -> tuple:
    if t.dim() != 4 or t.shape[1] != heads or t.shape[3] != D or t.dtype != dtype or t.stride(3) != 1:
        raise ValueError(f"{what} must be [pages, {heads}, page size, {D}] in {dtype} with contiguous channels, got "
                         f"{tuple(t.shape)} in {t.dtype}")
    return t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)


def rope_append(q: Tensor, k: Tensor, v: Tensor, positions: Tensor, inv_freq: Tensor, sections, slots: Tensor,
                k_pool: Tensor, v_pool: Tensor, *, interleaved: bool = False, round_tables: bool = False,
                out: Tensor | None = None) -> Tensor:
    """Rotate q and k (see ``rope_axes``) and write the rotated k, and v, to
    their cache slots; returns the rotated q.

    q: [T, Hq, D]; k, v: [T, Hkv, D]; k_pool, v_pool: [n_pages, Hkv, page_size,
    D], any page, head and token strides; slots: int64 [T], page * page_size +
    offset (``StepPlan.slots``).  Tokens with a slot outside the pool (padding:
    -1) are rotated but not written.  ``out`` may be q itself."""
    dev = _lib.require_cuda(q, k, v, positions, inv_freq, slots, k_pool, v_pool, out)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [tokens, heads, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    T, Hq, D = q.shape
    Hkv, dtype = k.shape[1], q.dtype
    positions, rot, sec, p64, ps = _rope_head(q, positions, inv_freq, sections or (inv_freq.numel(),))
    axes = len(sections or (0,))
    q, k, v = _heads(q, T, D, dtype, "q"), _heads(k, T, D, dtype, "k"), _heads(v, T, D, dtype, "v")
    if v.shape[1] != Hkv:
        raise ValueError(f"k and v must have the same heads, got {Hkv} and {v.shape[1]}")
    if slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of shape {(T,)}")
    kp, vp = _pool(k_pool, Hkv, D, dtype, "k_pool"), _pool(v_pool, Hkv, D, dtype, "v_pool")
    n_pages, page_size = k_pool.shape[0], k_pool.shape[2]
    if page_size & (page_size - 1) or page_size < 1 or v_pool.shape != k_pool.shape:
        raise ValueError("k_pool and v_pool must have one shape and a page size that is a power of two")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dtype, device=dev)
    elif out.shape != q.shape or out.dtype != dtype or (D > 1 and out.stride(2) != 1):
        raise ValueError("out must match q's shape and dtype, with contiguous channels")
    d = _lib.RopeDesc(_lib.dtype_code(dtype), T, Hq, Hkv, D, rot, axes, *sec, interleaved, 0, round_tables, p64, ps,
                      positions.data_ptr(), inv_freq.data_ptr(), q.data_ptr(), q.stride(0), q.stride(1),
                      out.data_ptr(), out.stride(0), out.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                      v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(), page_size, n_pages, *kp, *vp)
    st = _lib.bind(dev)
    _lib.check(_lib.load().fade_rope_axes(ctypes.byref(d), st), "rope_append")
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
_WS: dict = {}


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

    Returns [T, Hq, D] (zeros where no key is visible; tokens past cu_q[R] are
    not written); with ``return_lse`` a dict of that as "out" and the float32
    [T, Hq] log of the sum of exponentials as "lse" (-inf where no key is
    visible).  Head_dim 64 or 128, page
    size 16 to 128, Hq / Hkv up to 128.  What the pool holds past a request's
    kv_len is never used.  Workspace is cached per (device, stream); calls on
    one stream run in order, so sharing it is safe."""
    dev = _lib.require_cuda(q, k_pool, v_pool, block_table, cu_q, kv_lens, out)
    if q.dim() != 3 or k_pool.dim() != 4:
        raise ValueError(f"q must be [tokens, heads, head_dim] and k_pool [pages, heads, page size, head_dim], got "
                         f"{tuple(q.shape)} and {tuple(k_pool.shape)}")
    T, Hq, D = q.shape
    n_pages, Hkv, page_size = k_pool.shape[:3]
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported dtype {dtype}; expected float16 or bfloat16")
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page size must be one of {PAGE_SIZES}, got {page_size}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > 128:
        raise ValueError(f"Hq={Hq} must be a multiple of Hkv={Hkv}, at most 128 times it")
    kp, vp = _pool(k_pool, Hkv, D, dtype, "k_pool"), _pool(v_pool, Hkv, D, dtype, "v_pool")
    if v_pool.shape != k_pool.shape:
        raise ValueError(f"k_pool and v_pool must have one shape, got {tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    R = kv_lens.numel()
    bt, width, stride = _table(block_table, R)
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"sm_scale must be positive, got {sm_scale}")
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.contiguous()              # rows must be 16-byte aligned for the kernel's loads
        if q.data_ptr() % 16:
            q = q.clone()
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dtype, device=dev)
    elif out.shape != (T, Hq, D) or out.dtype != dtype or out.stride(2) != 1:
        raise ValueError("out must match q's shape and dtype, with contiguous channels")
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    d = _lib.ChunkDesc(
        _lib.dtype_code(dtype), R, T, Hq, Hkv, D, page_size, n_pages, width, stride, causal, window or 0, scale,
        q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
        None if lse is None else lse.data_ptr(), *kp, *vp, bt, _int32(cu_q, (R + 1,), "cu_q"),
        _int32(kv_lens, (R,), "kv_lens"))
    lib = _lib.load()
    st = _lib.bind(dev)
    ref = ctypes.byref(d)
    need = lib.fade_chunk_attn_workspace_size(ref)
    if need == 0:
        raise ValueError(f"unsupported chunk attention sizes (R={R}, T={T}, n_pages={n_pages}, table width {width})")
    key = (dev, st)
    ws = _WS.get(key)
    if ws is None or ws.numel() < need:
        ws = _WS[key] = torch.zeros(need, dtype=torch.uint8, device=dev)
    _lib.check(lib.fade_chunk_attn(ref, ws.data_ptr(), ws.numel(), st), "chunk_attention")
    return {"out": out, "lse": lse} if return_lse else out


def check_device_errors(device: torch.device | str = "cuda") -> None:
    """Raise if a bounded device wait of an earlier ``chunk_attention`` call on
    the current stream gave up (synchronises)."""
    dev = torch.device(device)
    if dev.index is None:
        dev = torch.device(dev.type, torch.cuda.current_device())
    st = _lib.bind(dev)
    ws = _WS.get((dev, st))
    if ws is not None:
        status = _lib.load().fade_workspace_check(ws.data_ptr(), ws.numel(), st)
        if status != _lib.FADE_OK:
            del _WS[(dev, st)]          # its counters may have stopped half way
        _lib.check(status, "chunk_attention")


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
        self._release_status = torch.zeros(1, dtype=torch.int32, device=dev)

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
        """Drop the requests of the bool [max_requests] mask `rows`."""
        release_rows(rows, self.kv_lens, self.block_table, self.page_size, self.free_pages, self.n_free,
                     self._release_status)

    def check(self) -> None:
        """Raise if a release failed or a device wait gave up (synchronises)."""
        code = int(self._release_status.item())
        if code:
            raise RuntimeError(f"release: {_PLAN_ERRORS.get(code, f'status {code}')}")
        check_device_errors(self._state.device)

    def gather(self, layer: int, rows, length: int) -> tuple[Tensor, Tensor]:
        """K, V [len(rows), n_kv_heads, length, head_dim] of the first `length`
        tokens of the given rows, contiguous: what the tier quantisers and
        ``TieredDecoder.load_prompt`` take."""
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
