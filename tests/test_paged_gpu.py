"""Paged serving step (``fade_b200.paged``) against plain 64-bit implementations:
page planning, rotary positions with several axes, chunk attention, the cache."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# half the spacing at 1: significands of 8, 11 and 24 bits
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


# ---------------------------------------------------------------------------
# plan_step / release_rows
# ---------------------------------------------------------------------------
def _plan_ref(new, kv, table, free, n_free, page, total):
    """Plain Python restatement; None where the step does not fit."""
    R, W = table.shape
    if min(new, default=0) < 0 or min(kv, default=0) < 0 or not 0 <= n_free <= len(free) or sum(new) > total:
        return None
    if any(-(-(c + n) // page) > W for c, n in zip(kv, new)):
        return None
    table = table.copy()
    cu, positions, slots, left = [0], [], [], n_free
    for r in range(R):
        for j in range(-(-kv[r] // page), -(-(kv[r] + new[r]) // page)):
            left -= 1
            if left < 0:
                return None
            table[r, j] = free[left]
        for pos in range(kv[r], kv[r] + new[r]):
            positions.append(pos)
            slots.append(int(table[r, pos // page]) * page + pos % page)
        cu.append(cu[-1] + new[r])
    pad = total - len(slots)
    return dict(cu_q=cu, kv_lens=[c + n for c, n in zip(kv, new)], positions=positions + [0] * pad,
                slots=slots + [-1] * pad, n_free=[left], table=table)


def _plan_inputs(new, kv, page, width, spare, seed, stride=None):
    rng = np.random.default_rng(seed)
    held = [-(-c // page) for c in kv]
    pages = rng.permutation(sum(held) + spare).astype(np.int32)
    R = len(new)
    table = rng.integers(-5, 5, (R, width)).astype(np.int32)      # stale entries past the held pages
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = pages[at:at + n]
        at += n
    return table, pages[at:].copy()


def _run_plan(new, kv, table, free, n_free, page, total, dev, width_stride=0):
    from fade_b200.paged import plan_step

    R, W = table.shape
    wide = torch.full((R, W + width_stride), -9, dtype=torch.int32, device=dev)
    bt = wide[:, :W]
    bt.copy_(torch.from_numpy(table))

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    plan = plan_step(i32(new), i32(kv), bt, torch.from_numpy(free).to(dev), i32([n_free]), page, total)
    assert (wide[:, W:] == -9).all()
    return plan, bt


@pytest.mark.parametrize("R,page,total_pad,high,seed", [
    (1, 16, 0, 1, 0),            # one decode
    (1, 128, 5, 700, 1),         # one prompt, padded
    (3, 1, 0, 9, 2),             # one-token pages
    (33, 16, 3, 40, 3),
    (257, 32, 0, 2, 4),
    (1025, 64, 77, 130, 5),      # more requests than threads
    (5, 16, 0, 9000, 6),         # many tokens, few requests
    (2500, 16, 1, 3, 7),
])
def test_plan_matches_plain(cuda_device, R, page, total_pad, high, seed):
    rng = random.Random(seed)
    new = [rng.choice((0, 1, rng.randint(0, high))) for _ in range(R)]
    kv = [rng.choice((0, page, rng.randint(0, 5 * page))) for _ in range(R)]
    width = max(-(-(c + n) // page) for c, n in zip(kv, new)) + rng.randint(0, 3)
    need = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(kv, new))
    table, free = _plan_inputs(new, kv, page, max(width, 1), need + 4, seed)
    for n_free in (need + 4, need):                                # some left, none left
        ref = _plan_ref(new, kv, table, free, n_free, page, sum(new) + total_pad)
        plan, bt = _run_plan(new, kv, table, free, n_free, page, sum(new) + total_pad, cuda_device, width_stride=seed % 3)
        plan.check()
        for name in ("cu_q", "kv_lens", "positions", "slots", "n_free"):
            assert getattr(plan, name).tolist() == ref[name], name
        assert np.array_equal(bt.cpu().numpy(), ref["table"])


def test_plan_no_requests_and_no_tokens(cuda_device):
    plan, _ = _run_plan([], [], np.zeros((0, 4), np.int32), np.arange(3, dtype=np.int32), 3, 16, 5, cuda_device)
    plan.check()
    assert plan.cu_q.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and plan.n_free.item() == 3
    plan, bt = _run_plan([0, 0], [17, 0], np.array([[4, 5], [7, 7]], np.int32), np.arange(3, dtype=np.int32), 2, 16, 0,
                         cuda_device)
    plan.check()
    assert plan.kv_lens.tolist() == [17, 0] and bt.tolist() == [[4, 5], [7, 7]] and plan.n_free.item() == 2


@pytest.mark.parametrize("what,code", [("pages", 1), ("row", 2), ("tokens", 3), ("negative", 4), ("free", 4), ("huge", 2)])
def test_plan_all_or_nothing(cuda_device, what, code):
    """A step that does not fit hands out nothing and says why."""
    page, new, kv, width, total, n_free = 16, [3, 40, 1], [16, 5, 0], 6, 44, 9
    if what == "pages":
        n_free = 3                                                 # the step needs 1 + 2 + 1
    elif what == "row":
        width = 2
    elif what == "tokens":
        total = 43
    elif what == "negative":
        kv[1] = -1
    elif what == "free":
        n_free = 50
    table, free = _plan_inputs([0] * 3, [max(c, 0) for c in kv], page, width, 9, 3)
    if what == "huge":
        from fade_b200.paged import plan_step

        def i32(x):
            return torch.tensor(x, dtype=torch.int32, device=cuda_device)

        bt = torch.from_numpy(table).to(cuda_device)
        plan = plan_step(i32([2 ** 31 - 1, 0, 0]), i32([16, 5, 0]), bt, torch.from_numpy(free).to(cuda_device), i32([9]),
                         page, 44)
        assert plan.status.item() in (2, 3)
    else:
        plan, bt = _run_plan(new, kv, table, free, n_free, page, total, cuda_device)
        assert plan.status.item() == code
    with pytest.raises(RuntimeError, match="plan_step"):
        plan.check()
    assert plan.cu_q.tolist() == [0] * 4 and (plan.slots == -1).all() and (plan.positions == 0).all()
    assert plan.n_free.item() == n_free and plan.kv_lens.tolist() == kv
    assert np.array_equal(bt.cpu().numpy(), table)


def test_plan_reuses_buffers_and_other_stream(cuda_device):
    from fade_b200.paged import StepPlan, plan_step

    R, page = 7, 16
    new, kv = [1, 20, 0, 3, 16, 2, 1], [0, 3, 9, 16, 15, 31, 100]
    table, free = _plan_inputs(new, kv, page, 9, 30, 11)
    ref = _plan_ref(new, kv, table, free, 30, page, 43)
    buf = StepPlan.empty(R, 43, cuda_device)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        def i32(x):
            return torch.tensor(x, dtype=torch.int32, device=cuda_device)

        bt = torch.from_numpy(table).to(cuda_device)
        args = (i32(new), i32(kv), bt, torch.from_numpy(free).to(cuda_device), i32([30]), page, 43)
        for _ in range(2):                                        # the same step twice: the same plan
            assert plan_step(*args, out=buf) is buf
    s.synchronize()
    assert buf.slots.tolist() == ref["slots"] and buf.cu_q.tolist() == ref["cu_q"]
    assert np.array_equal(bt.cpu().numpy(), ref["table"])


def test_plan_refusals(cuda_device):
    from fade_b200.paged import StepPlan, plan_step, release_rows

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=cuda_device)

    good = dict(new_lens=i32([1]), kv_lens=i32([0]), block_table=i32([[0, 0]]), free_pages=i32([0, 1]),
                n_free=i32([2]), page_size=16, total=1)
    plan_step(**good).check()
    for change in (dict(page_size=24), dict(page_size=0), dict(total=-1), dict(new_lens=i32([1, 2])),
                   dict(new_lens=torch.ones(1, device=cuda_device)), dict(block_table=i32([0, 0])),
                   dict(block_table=i32([[0, 0, 0, 0]])[:, ::2]), dict(n_free=i32([1, 1])),
                   dict(kv_lens=i32([[0]])), dict(out=StepPlan.empty(1, 2, cuda_device)),
                   dict(new_lens=torch.zeros(16385, dtype=torch.int32, device=cuda_device))):
        with pytest.raises(ValueError):
            plan_step(**{**good, **change})
    out = StepPlan.empty(1, 1, cuda_device)
    out.kv_lens = good["kv_lens"]
    with pytest.raises(ValueError, match="share"):
        plan_step(**good, out=out)
    with pytest.raises(RuntimeError, match="CUDA"):
        plan_step(**{**good, "new_lens": torch.ones(1, dtype=torch.int32)})
    with pytest.raises(ValueError):
        release_rows(i32([1]), good["kv_lens"], good["block_table"], 16, good["free_pages"], good["n_free"])


@pytest.mark.parametrize("R,page,seed", [(1, 16, 0), (40, 32, 1), (1500, 16, 2)])
def test_release_rows(cuda_device, R, page, seed):
    from fade_b200.paged import release_rows

    rng = np.random.default_rng(seed)
    kv = rng.integers(0, 6 * page, R).astype(np.int32)
    table, free = _plan_inputs([0] * R, kv.tolist(), page, 7, 5, seed)
    rows = rng.random(R) < 0.5
    if R == 1:
        rows[:] = True
    stack = free.tolist()
    for r in range(R):
        if rows[r]:
            stack += table[r, :-(-int(kv[r]) // page)].tolist()
    cap = np.full(len(stack) + 2, -1, np.int32)
    cap[:len(free)] = free
    d = dict(kv=torch.from_numpy(kv).to(cuda_device), bt=torch.from_numpy(table).to(cuda_device),
             free=torch.from_numpy(cap).to(cuda_device),
             n=torch.tensor([len(free)], dtype=torch.int32, device=cuda_device))
    status = release_rows(torch.from_numpy(rows).to(cuda_device), d["kv"], d["bt"], page, d["free"], d["n"])
    assert status.item() == 0
    assert d["n"].item() == len(stack) and d["free"].tolist() == stack + [-1, -1]
    assert d["kv"].tolist() == np.where(rows, 0, kv).tolist()
    # a stack without room: nothing changes
    small = d["free"][:len(stack)].clone()
    kv2 = torch.full((R,), page, dtype=torch.int32, device=cuda_device)
    n2 = d["n"].clone()
    status = release_rows(torch.ones(R, dtype=torch.uint8, device=cuda_device), kv2, d["bt"], page, small, n2)
    assert status.item() == 1 and n2.item() == len(stack) and (kv2 == page).all()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _rope_ref(x, positions, inv_freq, axes, inverse, round_dtype=None):
    """(value, error bound before the last rounding) in 64 bits; the angle is the fp32 product."""
    half = inv_freq.numel()
    rows = positions[torch.tensor(axes, device=positions.device)].float() if half else positions[:0].float()
    angle = (rows * inv_freq[:, None]).double().t()[:, None]
    c, s = angle.cos(), angle.sin()
    table_err = 2.0 ** -22                       # cos and sin in fp32: 2 ulp of values up to 1
    if round_dtype is not None:
        c, s = c.to(round_dtype).double(), s.to(round_dtype).double()
        table_err = 2 * HALF_ULP[round_dtype]    # a value next to a rounding boundary may go the other way
    if inverse:
        s = -s
    x = x.double()
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    err = (a.abs() + b.abs()) * (table_err + 3 * 2.0 ** -24)
    return (torch.cat([a * c - b * s, b * c + a * s, rest], -1), torch.cat([err, err, torch.zeros_like(rest)], -1))


def _assert_rounded(out, ref, err):
    lim = err + HALF_ULP[out.dtype] * (ref.abs() + err) + 2.0 ** -25 * (out.dtype == torch.float16)
    bad = (out.double() - ref).abs() - lim
    assert float(bad.max()) <= 0 if bad.numel() else True, float(bad.max())


def _inv_freq(half, dev, theta=500000.0):
    return (theta ** -(torch.arange(half, dtype=torch.float64) / max(half, 1))).float().to(dev)


@pytest.mark.parametrize("T,H,D,sections,inter,dt,inverse,rounded", [
    (1, 1, 64, (32,), False, torch.bfloat16, False, False),
    (5, 7, 128, (16, 24, 24), False, torch.bfloat16, False, False),
    (33, 4, 128, (24, 20, 20), True, torch.float16, False, False),
    (17, 16, 80, (20, 20), False, torch.float16, True, False),
    (9, 3, 72, (12, 12, 12), True, torch.float32, False, False),
    (64, 2, 128, (32,), False, torch.bfloat16, False, False),          # half of the head turns
    (3, 5, 66, (5, 4, 4, 3), True, torch.float32, True, False),        # four axes, odd halves
    (7, 2, 10, (1, 0, 2), False, torch.bfloat16, False, False),        # an empty axis
    (11, 3, 7, (0,), False, torch.float16, False, False),              # nothing turns: a copy
    (300, 8, 64, (8, 12, 12), False, torch.bfloat16, False, True),
    (130, 8, 64, (8, 12, 12), True, torch.float16, True, True),
])
def test_rope_axes(cuda_device, T, H, D, sections, inter, dt, inverse, rounded):
    from fade_b200.paged import rope_axes, section_axes

    g = torch.Generator(device="cuda").manual_seed(T + D)
    x = torch.randn(T, H, D, generator=g, device=cuda_device).to(dt)
    pos = torch.randint(0, 40000, (len(sections), T), generator=g, device=cuda_device, dtype=torch.int32)
    inv = _inv_freq(sum(sections), cuda_device)
    ref, err = _rope_ref(x, pos, inv, section_axes(sections, inter), inverse, dt if rounded else None)
    kw = dict(interleaved=inter, inverse=inverse, round_tables=rounded)
    out = rope_axes(x, pos, inv, sections, **kw)
    _assert_rounded(out, ref, err)
    assert torch.equal(rope_axes(x, pos.long(), inv, sections, **kw), out)          # 64-bit positions
    wide = torch.zeros(T, 2 * H + 1, D + 3, dtype=dt, device=cuda_device)           # odd strides and offset
    view = wide[:, 1::2, 1:D + 1]
    view.copy_(x)
    assert torch.equal(rope_axes(view, pos, inv, sections, **kw), out)
    assert torch.equal(rope_axes(view, pos, inv, sections, out=view, **kw), out)    # in place, in the view
    assert torch.equal(view, out) and (wide[:, ::2] == 0).all() and (wide[:, :, 0] == 0).all()
    assert (wide[:, :, D + 1:] == 0).all()
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)                         # heads outermost
    assert torch.equal(rope_axes(turned, pos, inv, sections, **kw), out)


def test_rope_inverse_is_the_transpose(cuda_device):
    """rope(x) . y = x . rope^-1(y), and the derivative along a difference."""
    from fade_b200.paged import rope_axes

    g = torch.Generator(device="cuda").manual_seed(3)
    x, y, dx = (torch.randn(19, 4, 64, generator=g, device=cuda_device) for _ in range(3))
    pos = torch.randint(0, 3000, (3, 19), generator=g, device=cuda_device)
    inv = _inv_freq(32, cuda_device)
    a = (rope_axes(x, pos, inv, (8, 12, 12)).double() * y.double()).sum()
    b = (x.double() * rope_axes(y, pos, inv, (8, 12, 12), inverse=True).double()).sum()
    scale = float(x.double().norm() * y.double().norm())
    assert abs(float(a - b)) <= scale * 2.0 ** -20                 # rounding of 2 x 4864 terms in fp32
    plus, minus = (rope_axes(x + e * dx, pos, inv, (8, 12, 12)).double() for e in (0.5, -0.5))
    along = ((plus - minus) * y.double()).sum()
    grad = (dx.double() * rope_axes(y, pos, inv, (8, 12, 12), inverse=True).double()).sum()
    assert abs(float(along - grad)) <= scale * 2.0 ** -18


def test_rope_matches_the_schemes_tables(cuda_device):
    """round_tables gives what MRope's tables give, text and several axes."""
    from fade_b200.paged import rope_axes
    from fade_b200.rope import MRope
    from gpu_util import t_vals
    from oracle.rope import apply_rope

    g = torch.Generator(device="cuda").manual_seed(4)
    for dt, name, inter in ((torch.bfloat16, "bf16", False), (torch.float16, "f16", True)):
        scheme = MRope(theta=1e6, head_dim=128, mrope_section=[16, 24, 24], interleaved=inter)
        x = torch.randn(50, 6, 128, generator=g, device=cuda_device).to(dt)
        pos = torch.randint(0, 9000, (3, 50), generator=g, device=cuda_device)
        cos, sin = scheme.compute_cos_sin(pos, cuda_device, model_dtype=dt)
        want = apply_rope(t_vals(x.transpose(0, 1)), t_vals(cos)[0], t_vals(sin)[0], name)
        got = t_vals(rope_axes(x, pos, scheme.inv_freq(cuda_device), (16, 24, 24), interleaved=inter, round_tables=True))
        got = got.transpose(1, 0, 2)
        # equal but where one of the two sincos lands across a rounding boundary of the table
        near = np.abs(got - want) <= 4 * HALF_ULP[dt] * (np.abs(want) + np.abs(t_vals(x.transpose(0, 1))).max())
        assert near.all() and np.mean(got == want) > 0.99


def _pools(n_pages, hkv, page, D, dt, dev, layout, fill):
    if layout == "heads":                       # [pages, heads, tokens, D]
        return tuple(torch.full((n_pages, hkv, page, D), fill, dtype=dt, device=dev) for _ in range(2))
    return tuple(torch.full((n_pages, page, hkv, D), fill, dtype=dt, device=dev).transpose(1, 2) for _ in range(2))


@pytest.mark.parametrize("T,hq,hkv,D,page,sections,dt,layout", [
    (1, 14, 2, 64, 16, (32,), torch.float16, "heads"),
    (37, 4, 4, 128, 32, (16, 24, 24), torch.bfloat16, "tokens"),
    (200, 28, 4, 128, 64, (64,), torch.bfloat16, "heads"),
    (75, 6, 3, 66, 1, (11, 11, 11), torch.float32, "tokens"),
])
def test_rope_append(cuda_device, T, hq, hkv, D, page, sections, dt, layout):
    from fade_b200.paged import rope_append, section_axes

    g = torch.Generator(device="cuda").manual_seed(T)
    fused = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device=cuda_device).to(dt)
    q, k, v = (x.unflatten(-1, (-1, D)) for x in fused.split([hq * D, hkv * D, hkv * D], -1))
    n_pages = -(-T // page) + 4
    kp, vp = _pools(n_pages, hkv, page, D, dt, cuda_device, layout, 7.0)
    slots = torch.randperm(n_pages * page, generator=g, device=cuda_device)[:T]
    slots[T // 2] = -1                                             # padding
    if T > 4:
        slots[3] = n_pages * page                                  # past the pool: dropped, too
    pos = torch.randint(0, 5000, (len(sections), T), generator=g, device=cuda_device, dtype=torch.int32)
    inv = _inv_freq(sum(sections), cuda_device)
    out = rope_append(q, k, v, pos, inv, sections, slots, kp, vp)
    axes = section_axes(sections)
    _assert_rounded(out, *_rope_ref(q, pos, inv, axes, False))
    k_ref, k_err = _rope_ref(k, pos, inv, axes, False)
    live = (slots >= 0) & (slots < n_pages * page)
    at = slots[live]
    got_k, got_v = kp[at // page, :, at % page], vp[at // page, :, at % page]
    _assert_rounded(got_k, k_ref[live], k_err[live])
    assert torch.equal(got_v, v[live])
    untouched = torch.ones(n_pages, page, dtype=torch.bool, device=cuda_device)
    untouched[at // page, at % page] = False
    assert (kp.transpose(1, 2)[untouched] == 7).all() and (vp.transpose(1, 2)[untouched] == 7).all()
    assert torch.equal(rope_append(q, k, v, pos, inv, sections, slots, kp, vp, out=q), out)     # in place


def test_rope_non_finite_and_large_positions(cuda_device):
    """NaN and infinities stay in their pair; angles far beyond 2 pi keep their accuracy."""
    from fade_b200.paged import rope_axes

    x = torch.ones(2, 1, 8, device=cuda_device)
    x[0, 0, 1], x[1, 0, 6] = math.nan, math.inf
    pos = torch.tensor([3, 2 ** 24], device=cuda_device)
    inv = _inv_freq(4, cuda_device)
    out = rope_axes(x, pos, inv)
    assert out[0, 0].isnan().tolist() == [False, True, False, False, False, True, False, False]
    assert out[1, 0].isfinite().tolist() == [True, True, False, True, True, True, False, True]
    one = torch.ones(3, 2, 8, device=cuda_device)
    p = torch.tensor([[10 ** 6, 2 ** 24, 123456789]], device=cuda_device)
    _assert_rounded(rope_axes(one, p, inv), *_rope_ref(one, p, inv, [0] * 4, False))


def test_rope_refusals(cuda_device):
    from fade_b200.paged import rope_append, rope_axes

    x = torch.zeros(3, 2, 8, device=cuda_device)
    pos, inv = torch.zeros(2, 3, dtype=torch.int32, device=cuda_device), _inv_freq(4, cuda_device)
    rope_axes(x, pos, inv, (2, 2))
    for args in ((x[0], pos, inv, (2, 2)), (x, pos[:, :2], inv, (2, 2)), (x, pos.float(), inv, (2, 2)),
                 (x, pos, inv, (2, 1)), (x, pos, inv, (4,)), (x, pos, inv.double(), (2, 2)), (x.double(), pos, inv, (2, 2)),
                 (x, pos, _inv_freq(5, cuda_device), (3, 2)), (x, pos, inv, (5, -1)), (x, pos, inv, (1, 1, 1, 1, 0))):
        with pytest.raises(ValueError):
            rope_axes(*args)
    with pytest.raises(ValueError, match="out"):
        rope_axes(x, pos, inv, (2, 2), out=x[:2])
    with pytest.raises(RuntimeError, match="CUDA"):
        rope_axes(x.cpu(), pos, inv, (2, 2))
    k, pool, slots = x[:, :1], torch.zeros(2, 1, 4, 8, device=cuda_device), torch.arange(3, device=cuda_device)
    rope_append(x, k, k, pos, inv, (2, 2), slots, pool, pool.clone())
    for change in (dict(k=k[:2]), dict(v=x), dict(v=k.half()), dict(slots=slots.int()), dict(slots=slots[:2]),
                   dict(k_pool=pool[0]), dict(k_pool=pool[:, :, :3]), dict(v_pool=pool.half()),
                   dict(v_pool=pool[:1]), dict(k_pool=pool.expand(2, 2, 4, 8))):
        good = dict(q=x, k=k, v=k, positions=pos, inv_freq=inv, sections=(2, 2), slots=slots, k_pool=pool, v_pool=pool)
        with pytest.raises(ValueError):
            rope_append(**{**good, **change})


# ---------------------------------------------------------------------------
# chunk attention
# ---------------------------------------------------------------------------
def _attn_inputs(new, kv, hq, hkv, D, page, dt, dev, seed, layout="heads", poison=True, scale=1.0):
    """Paged caches whose unused places hold NaN (and infinities), a table with garbage past the pages in use."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    R = len(kv)
    held = [-(-c // page) for c in kv]
    n_pages = sum(held) + 3
    kp, vp = _pools(n_pages, hkv, page, D, dt, dev, layout, math.nan if poison else 0.0)
    if poison:
        kp[-1], vp[-1] = math.inf, -math.inf
    order = torch.randperm(n_pages, generator=g, device=dev)
    width = max(held + [1]) + 2
    table = torch.tensor([-1, n_pages, 2 ** 31 - 1, 0], device=dev)[
        torch.randint(0, 4, (R, width), generator=g, device=dev)].to(torch.int32)
    at = 0
    for r in range(R):
        pages = order[at:at + held[r]]
        table[r, :held[r]] = pages.to(torch.int32)
        at += held[r]
        if kv[r] > 0:
            j = torch.arange(kv[r], device=dev)
            chan = torch.ones(D, device=dev)
            chan[:3] = 6.0                                         # outlier channels, as keys have them
            kp[pages[j // page], :, j % page] = (scale * torch.randn(kv[r], hkv, D, generator=g, device=dev) * chan).to(dt)
            vp[pages[j // page], :, j % page] = torch.randn(kv[r], hkv, D, generator=g, device=dev).to(dt)
    T = sum(new)
    q = torch.randn(T, hq, D, generator=g, device=dev).to(dt)
    cu = torch.tensor([sum(new[:r]) for r in range(R + 1)], dtype=torch.int32, device=dev)
    return q, kp, vp, table, cu, torch.tensor(kv, dtype=torch.int32, device=dev)


def _attn_ref(q, kp, vp, table, new, kv, causal, window, sm):
    """out, lse, and the error bounds of both, in 64 bits."""
    T, hq, D = q.shape
    hkv, page = kp.shape[1:3]
    dev, u = q.device, HALF_ULP[q.dtype]
    out = torch.zeros(T, hq, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=dev)
    lim, lim_lse = torch.zeros_like(out), torch.zeros_like(lse)
    t0 = 0
    for r, (n, c) in enumerate(zip(new, kv)):
        if n and c:
            j = torch.arange(c, device=dev)
            pg = table[r].long()[j // page]
            k = kp[pg, :, j % page].double().repeat_interleave(hq // hkv, 1)       # [c, hq, D]
            v = vp[pg, :, j % page].double().repeat_interleave(hq // hkv, 1)
            x = q[t0:t0 + n].double()
            s = torch.einsum("thd,chd->htc", x, k) * sm
            # scores: D products summed in fp32 by the tensor core, then scaled
            ds = torch.einsum("thd,chd->htc", x.abs(), k.abs()).amax(-1) * sm * 2.0 ** -18
            p = (c - n + torch.arange(n, device=dev))[:, None]
            seen = torch.ones(n, c, dtype=torch.bool, device=dev)
            if causal:
                seen &= j <= p
            if window:
                seen &= j > p - window
            s = s.masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(s, -1)
            w = torch.exp(s - norm.clamp(min=-1e300)[..., None])
            o = torch.einsum("htc,chd->thd", w, v)
            mass = torch.einsum("htc,chd->thd", w, v.abs())        # sum of weights times |v|
            out[t0:t0 + n], lse[t0:t0 + n] = o, norm.t()
            # weights rounded to 16 bits, scores off by ds, fp32 sums; one rounding of the result
            lim[t0:t0 + n] = mass * (u + 2 * ds.t()[..., None] + 2.0 ** -13) + u * o.abs() + 2.0 ** -24
            lim_lse[t0:t0 + n] = ds.t() + 2.0 ** -20 * (norm.t().abs().nan_to_num(posinf=0.0) + 1)
        t0 += n
    return out, lse, lim, lim_lse


def _check_attn(new, kv, hq, hkv, D, page, dt, dev, seed=0, causal=True, window=None, layout="heads", sm=None,
                scale=1.0, **kw):
    from fade_b200.paged import check_device_errors, chunk_attention

    args = _attn_inputs(new, kv, hq, hkv, D, page, dt, dev, seed, layout, scale=scale)
    q, kp, vp, table = args[:4]
    out, lse = chunk_attention(*args, causal=causal, window=window, sm_scale=sm, return_lse=True, **kw).values()
    check_device_errors(dev)
    ref, ref_lse, lim, lim_lse = _attn_ref(q, kp, vp, table, new, kv, causal, window, sm or 1 / math.sqrt(D))
    assert out.isfinite().all()
    err = (out.double() - ref).abs()
    worst = float((err / lim.clamp(min=1e-30)).max()) if err.numel() else 0.0
    print(f"[chunk attn] worst err/limit {worst:.3f}")
    assert (err <= lim).all(), worst
    empty = ref_lse.isinf()
    assert torch.equal(lse.isinf(), empty) and (out[empty] == 0).all()
    assert ((lse.double() - ref_lse).abs()[~empty] <= lim_lse[~empty]).all()
    return args, out, lse


BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("new,kv,hq,hkv,D,page,dt", [
    ([1], [1], 1, 1, 64, 16, HF),                                    # one token over itself
    ([1], [2048], 14, 2, 64, 64, HF),
    ([1], [127], 28, 4, 128, 16, BF),
    ([1], [128], 28, 4, 128, 128, BF),
    ([1], [129], 28, 4, 128, 32, BF),
    ([1] * 16, [5 + 517 * r for r in range(16)], 32, 8, 128, 128, BF),
    ([2], [1], 8, 8, 64, 16, BF),                                    # more queries than keys: an empty row
    ([5, 0, 3], [5, 77, 0], 8, 2, 128, 16, HF),                      # idle row, request without a cache
    ([300], [300], 4, 4, 64, 32, HF),                                # plain causal prompt
    ([257], [700], 32, 8, 128, 64, BF),
    ([64], [5000], 64, 8, 128, 128, BF),                             # few rows, long cache
    ([31, 1, 200, 0, 65], [31, 900, 333, 40, 1065], 28, 4, 128, 16, BF),
    ([3], [1000], 7, 1, 64, 16, HF),                                 # all heads on one
    ([2], [400], 128, 1, 128, 32, BF),                               # 128 heads on one
    ([9], [400], 100, 1, 64, 32, HF),                                # one token per tile
    ([1], [40000], 8, 1, 128, 128, BF),                              # one row over a long cache
])
def test_chunk_attention(cuda_device, new, kv, hq, hkv, D, page, dt):
    _check_attn(new, kv, hq, hkv, D, page, dt, cuda_device, seed=len(new) + kv[0])


@pytest.mark.parametrize("new,kv,window", [
    ([1], [1000], 1),
    ([1, 1], [1000, 60], 129),
    ([200], [1200], 64),
    ([513], [513], 100),
    ([70, 1, 5], [3000, 2000, 5], 1000),
    ([130], [100], 50),                                              # empty rows and a window
])
@pytest.mark.parametrize("causal", [True, False])
def test_chunk_attention_window(cuda_device, new, kv, window, causal):
    _check_attn(new, kv, 16, 4, 128, 16, BF, cuda_device, seed=window, causal=causal, window=window)
    _check_attn(new, kv, 6, 2, 64, 128, HF, cuda_device, seed=window, causal=causal, window=window)


def test_chunk_attention_not_causal(cuda_device):
    """All of a cache of another length (an encoder's states), empty caches among them."""
    _check_attn([300, 4, 7, 1], [150, 0, 1025, 3000], 12, 4, 64, 32, HF, cuda_device, causal=False)
    _check_attn([33, 150], [1, 400], 8, 8, 128, 64, BF, cuda_device, causal=False)


def test_chunk_attention_many_requests(cuda_device):
    rng = random.Random(5)
    new = [rng.choice((1, 1, 1, 0, 2, rng.randint(3, 40))) for _ in range(700)]
    kv = [n + rng.randint(0, 300) for n in new]
    _check_attn(new, kv, 8, 2, 64, 16, BF, cuda_device, seed=6)


def test_chunk_attention_random_batches(cuda_device):
    rng = random.Random(7)
    for i in range(20):
        R = rng.randint(1, 9)
        new = [rng.choice((0, 1, 1, rng.randint(2, 9), rng.randint(10, 400))) for _ in range(R)]
        kv = [max(0, n + rng.choice((0, -1, rng.randint(0, 200), rng.randint(0, 3000)))) for n in new]
        hq, hkv, D = rng.choice(((14, 2, 64), (32, 8, 128), (28, 4, 128), (8, 8, 64), (5, 1, 128)))
        _check_attn(new, kv, hq, hkv, D, rng.choice((16, 32, 64, 128)), rng.choice((BF, HF)), cuda_device, seed=i,
                    causal=rng.random() < 0.8, window=rng.choice((None, None, rng.randint(1, 500))),
                    layout=rng.choice(("heads", "tokens")))


def test_chunk_attention_large_scores(cuda_device):
    """Scores of hundreds: the running maximum moves late and far."""
    _check_attn([40, 1], [900, 2500], 8, 2, 128, 32, HF, cuda_device, seed=8, scale=12.0)
    _check_attn([300], [900], 8, 2, 64, 32, BF, cuda_device, seed=9, scale=12.0, sm=0.5)
    from fade_b200.paged import chunk_attention

    # keys in rising order: every block brings a new maximum
    q, kp, vp, table, cu, kl = _attn_inputs([3], [1500], 4, 1, 64, 16, BF, cuda_device, 10)
    j = torch.arange(1500, device=cuda_device)
    pg = table[0].long()[j // 16]
    q.fill_(1.0)
    kp[pg, :, j % 16] = (j.float() / 40)[:, None, None].expand(-1, 1, 64).to(BF)
    out, lse = chunk_attention(q, kp, vp, table, cu, kl, return_lse=True).values()
    ref, ref_lse, lim, lim_lse = _attn_ref(q, kp, vp, table, [3], [1500], True, None, 0.125)
    assert ((out.double() - ref).abs() <= lim).all() and ((lse.double() - ref_lse).abs() <= lim_lse).all()


def test_chunk_attention_repeats_bit_for_bit(cuda_device):
    from fade_b200.paged import chunk_attention

    args, out, lse = _check_attn([100, 1, 40], [3000, 9000, 40], 32, 8, 128, 64, BF, cuda_device, seed=11)
    other = _attn_inputs([1] * 30, [700] * 30, 8, 2, 64, 16, HF, cuda_device, 12)
    for _ in range(3):
        chunk_attention(*other)                                     # the same workspace in between
        again, lse2 = chunk_attention(*args, return_lse=True).values()
        assert torch.equal(again, out) and torch.equal(lse2, lse)


def test_chunk_attention_strides_streams_and_padding(cuda_device):
    from fade_b200.paged import chunk_attention

    new, kv = [20, 1, 3], [200, 333, 3]
    args, out, lse = _check_attn(new, kv, 28, 4, 128, 32, BF, cuda_device, seed=13)
    q, kp, vp, table, cu, kl = args
    # q inside a fused projection, an odd offset (copied), token rows past the last request
    fused = torch.full((40, 36, 128), math.nan, dtype=BF, device=cuda_device)
    fused[:24, :28] = q
    dest = torch.full((40, 30, 128), 3.0, dtype=BF, device=cuda_device)
    got = chunk_attention(fused[:, :28], kp, vp, table, cu, kl, out=dest[:, 1:29])
    assert got.data_ptr() == dest[:, 1:].data_ptr()
    assert torch.equal(got[:24], out) and (dest[24:] == 3).all() and (dest[:, 0] == 3).all() and (dest[:, 29] == 3).all()
    odd = torch.zeros(24 * 28 * 128 + 1, dtype=BF, device=cuda_device)[1:].view(24, 28, 128)
    odd.copy_(q)
    assert torch.equal(chunk_attention(odd, kp, vp, table, cu, kl), out)
    wide = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :table.shape[1]] = table
    assert torch.equal(chunk_attention(q, kp, vp, wide[:, :table.shape[1]], cu, kl), out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other, lse2 = chunk_attention(*args, return_lse=True).values()
    s.synchronize()
    assert torch.equal(other, out) and torch.equal(lse2, lse)


def test_chunk_attention_in_a_graph(cuda_device):
    """Lengths on the device: one captured call serves steps of other lengths."""
    from fade_b200.paged import chunk_attention

    kv = [500, 90, 1300]
    q, kp, vp, table, cu, kl = _attn_inputs([4, 4, 4], kv, 8, 2, 128, 64, BF, cuda_device, 14)
    out = torch.zeros_like(q)
    chunk_attention(q, kp, vp, table, cu, kl, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chunk_attention(q, kp, vp, table, cu, kl, out=out)           # this stream's workspace, before the capture
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            chunk_attention(q, kp, vp, table, cu, kl, out=out)
    torch.cuda.current_stream().wait_stream(s)
    for new, lens in (([4, 4, 4], kv), ([10, 0, 2], [400, 90, 1299]), ([1, 1, 1], [1, 2, 3])):
        cu.copy_(torch.tensor([sum(new[:r]) for r in range(4)], dtype=torch.int32))
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        g.replay()
        ref, _, lim, _ = _attn_ref(q[:sum(new)], kp, vp, table, new, lens, True, None, 128 ** -0.5)
        assert ((out[:sum(new)].double() - ref).abs() <= lim).all()


def test_chunk_attention_offsets_past_32_bits(cuda_device):
    """Pages beyond 2^32 bytes and 2^31 elements of the pool."""
    from fade_b200.paged import chunk_attention, rope_append

    n_pages, hkv, page, D = 140000, 2, 128, 64                       # 4.6 GB per pool
    kp = torch.empty(n_pages, hkv, page, D, dtype=BF, device=cuda_device)
    vp = torch.empty_like(kp)
    kv, g = [300, 129], torch.Generator(device="cuda").manual_seed(15)
    table = torch.tensor([[n_pages - 1, n_pages - 2, n_pages - 3], [n_pages - 70000, 5, 0]], dtype=torch.int32,
                         device=cuda_device)
    for r, c in enumerate(kv):
        k, v = (torch.randn(c, hkv, D, generator=g, device=cuda_device).to(BF) for _ in range(2))
        j = torch.arange(c, device=cuda_device)
        slots = table[r].long()[j // page] * page + j % page
        q = torch.zeros(c, 1, D, dtype=BF, device=cuda_device)
        rope_append(q, k, v, j, _inv_freq(0, cuda_device), (0,), slots, kp, vp)    # no rotation: a write
        assert torch.equal(kp[table[r].long()[j // page], :, j % page], k)
        assert torch.equal(vp[table[r].long()[j // page], :, j % page], v)
    new = [3, 1]
    q = torch.randn(4, 4, D, generator=g, device=cuda_device).to(BF)
    cu = torch.tensor([0, 3, 4], dtype=torch.int32, device=cuda_device)
    out = chunk_attention(q, kp, vp, table, cu, torch.tensor(kv, dtype=torch.int32, device=cuda_device))
    ref, _, lim, _ = _attn_ref(q, kp, vp, table, new, kv, True, None, 0.125)
    assert ((out.double() - ref).abs() <= lim).all()


def test_chunk_attention_nothing_to_do(cuda_device):
    from fade_b200.paged import chunk_attention

    q, kp, vp, table, cu, kl = _attn_inputs([0, 0], [5, 0], 4, 2, 64, 16, BF, cuda_device, 16)
    assert chunk_attention(q, kp, vp, table, cu, kl).shape == (0, 4, 64)
    empty = torch.zeros(0, 3, dtype=torch.int32, device=cuda_device)
    cu0 = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert chunk_attention(q, kp, vp, empty, cu0, kl[:0]).shape == (0, 4, 64)


def test_chunk_attention_refusals(cuda_device):
    from fade_b200.paged import chunk_attention

    q, kp, vp, table, cu, kl = _attn_inputs([3, 2], [30, 20], 4, 2, 64, 16, BF, cuda_device, 17)
    good = dict(q=q, k_pool=kp, v_pool=vp, block_table=table, cu_q=cu, kv_lens=kl)
    chunk_attention(**good)
    big = torch.zeros(4, 2, 16, 96, dtype=BF, device=cuda_device)
    for change in (dict(q=q[0]), dict(q=q.half()), dict(q=q.float(), k_pool=kp.float(), v_pool=vp.float()),
                   dict(q=q[:, :3]), dict(k_pool=kp[:, :, :8], v_pool=vp[:, :, :8]), dict(v_pool=vp[:2]),
                   dict(k_pool=kp[..., :32]), dict(q=torch.zeros(5, 4, 96, dtype=BF, device=cuda_device), k_pool=big, v_pool=big),
                   dict(block_table=table[:1]), dict(block_table=table.long()), dict(cu_q=cu[:2]), dict(cu_q=cu.long()),
                   dict(kv_lens=kl.float()), dict(window=0), dict(sm_scale=0.0), dict(sm_scale=-1.0),
                   dict(sm_scale=math.nan), dict(out=q[:2])):
        with pytest.raises(ValueError):
            chunk_attention(**{**good, **change})
    with pytest.raises(RuntimeError, match="CUDA"):
        chunk_attention(**{**good, "kv_lens": kl.cpu()})
    odd = torch.zeros(kp.numel() + 1, dtype=BF, device=cuda_device)[1:].view(kp.shape)
    with pytest.raises(RuntimeError, match="16-byte"):
        chunk_attention(**{**good, "k_pool": odd})


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def test_cache_steps_and_release(cuda_device):
    """Prompts in chunks, decodes and a release through PagedKVCache against one dense attention per request."""
    from fade_b200.paged import PagedKVCache, rope_axes

    L, hq, hkv, D, page, R = 2, 8, 2, 64, 16, 4
    cache = PagedKVCache(L, hkv, D, n_pages=40, max_requests=R, max_tokens=256, page_size=page, dtype=BF,
                         device=cuda_device)
    g = torch.Generator(device="cuda").manual_seed(18)
    inv = _inv_freq(D // 2, cuda_device)
    hist = [[([], []) for _ in range(R)] for _ in range(L)]
    lens = [0] * R
    for step, new in enumerate(([40, 7, 0, 1], [40, 1, 16, 1], [13, 1, 1, 1], "drop", [1, 1, 30, 20], [1, 1, 1, 1])):
        if new == "drop":
            rows = torch.tensor([False, True, False, True], device=cuda_device)
            cache.release(rows)
            for r in (1, 3):
                lens[r] = 0
                for lay in hist:
                    lay[r] = ([], [])
            continue
        total = sum(new) + 3
        plan = cache.plan(torch.tensor(new, dtype=torch.int32, device=cuda_device), total)
        plan.check()
        for layer in range(L):
            q, k, v = (torch.randn(total, h, D, generator=g, device=cuda_device).to(BF) for h in (hq, hkv, hkv))
            qr = cache.append(layer, plan, q, k, v, inv)
            out = cache.attend(layer, plan, qr)
            t0 = 0
            for r in range(R):
                pos = torch.arange(lens[r], lens[r] + new[r], device=cuda_device)
                hist[layer][r][0].append(rope_axes(k[t0:t0 + new[r]], pos, inv))
                hist[layer][r][1].append(v[t0:t0 + new[r]])
                if new[r]:
                    kk, vv = (torch.cat(x) for x in hist[layer][r])
                    c = kk.shape[0]
                    tab = torch.arange(c, device=cuda_device, dtype=torch.int32)[None]
                    ref, _, lim, _ = _attn_ref(qr[t0:t0 + new[r]], kk[:, :, None], vv[:, :, None], tab, [new[r]], [c],
                                               True, None, D ** -0.5)
                    assert ((out[t0:t0 + new[r]].double() - ref).abs() <= lim).all()
                    gk, gv = cache.gather(layer, [r], c)
                    assert torch.equal(gk[0].transpose(0, 1), kk) and torch.equal(gv[0].transpose(0, 1), vv)
                t0 += new[r]
        lens = [a + b for a, b in zip(lens, new)]
        assert cache.kv_lens.tolist() == lens
        assert cache.n_free.item() == 40 - sum(-(-n // page) for n in lens)
    cache.check()
    held = [cache.block_table[r, :-(-lens[r] // page)].tolist() for r in range(R)]
    pages = sum(held, []) + cache.free_pages[:cache.n_free.item()].tolist()
    assert sorted(pages) == list(range(40))                        # every page in one place


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,kv,hq,hkv,D,page,dt,causal,window,where", [
    ([5], [3000], 8, 1, 128, 64, BF, True, None, {0: [2999, 2997]}),          # later drafts, a tile over many SMs
    ([5] * 16, [900 + 37 * r for r in range(16)], 32, 8, 128, 32, HF, True, None, {3: [1010], 9: [1231, 1232]}),
    ([300], [700], 8, 2, 64, 16, HF, True, None, {0: [450, 640, 699]}),       # inside the chunk
    ([129], [129], 4, 4, 64, 32, BF, True, None, {0: [0, 128]}),              # the first key reaches every row
    ([200, 1], [1200, 700], 16, 4, 128, 16, BF, True, 64, {0: [990, 1100], 1: [630, 636]}),
    ([1, 1, 1], [1000, 60, 5], 14, 2, 64, 64, HF, True, 129, {0: [800, 870]}),      # before every row's window
    ([130], [100], 8, 2, 64, 16, HF, True, None, {0: [99, 40]}),              # rows without keys beside it
    ([40], [500], 8, 2, 128, 128, BF, False, 300, {0: [170, 210]}),
    ([1021], [4000], 8, 2, 128, 128, HF, True, 1024, {0: [2100, 3500]}),
])
def test_chunk_attention_masked_values(cuda_device, new, kv, hq, hkv, D, page, dt, causal, window, where, bad):
    """A NaN or an infinity in V reaches the rows that see its key, in its channel, and nothing else."""
    from fade_b200.paged import check_device_errors, chunk_attention

    q, kp, vp, table, cu, kl = _attn_inputs(new, kv, hq, hkv, D, page, dt, cuda_device, 21)
    clean = vp.clone()
    ref, ref_lse, lim, lim_lse = _attn_ref(q, kp, clean, table, new, kv, causal, window, D ** -0.5)
    hit = torch.zeros_like(ref, dtype=torch.bool)
    t0 = 0
    for r, n in enumerate(new):
        for j in where.get(r, ()):
            chan = (7 * j) % D
            vp[int(table[r, j // page]), :, j % page, chan] = bad
            p = kv[r] - n + torch.arange(n, device=cuda_device)
            sees = ((p >= j) if causal else p >= -n) & ((p - window < j) if window else p >= -n)
            hit[t0:t0 + n, :, chan] |= sees[:, None]
        t0 += n
    out, lse = chunk_attention(q, kp, vp, table, cu, kl, causal=causal, window=window, return_lse=True).values()
    check_device_errors(cuda_device)
    assert not out[hit].isfinite().any()
    assert out[~hit].isfinite().all()
    assert ((out.double() - ref).abs() <= lim)[~hit].all()
    some = ~ref_lse.isinf()
    assert torch.equal(~lse.isinf(), some) and ((lse.double() - ref_lse).abs() <= lim_lse)[some].all()
    again = chunk_attention(q, kp, clean, table, cu, kl, causal=causal, window=window)   # nothing stays behind
    assert again.isfinite().all() and ((again.double() - ref).abs() <= lim).all()


def test_chunk_attention_refuses_to_overwrite_q(cuda_device):
    from fade_b200.paged import chunk_attention

    args = _attn_inputs([3, 2], [30, 20], 4, 2, 64, 16, BF, cuda_device, 17)
    with pytest.raises(ValueError):
        chunk_attention(*args, out=args[0])
