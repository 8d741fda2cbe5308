"""The operators of a serving step over a paged cache: cases, plain forms and exact values.

One step of a continuous batch goes through three operators of ``fade_b200.paged``:
``plan_step`` (block tables, slot map and positions from the requests' lengths),
``rope_append`` / ``rope_axes`` (rotary positions with several axes, K and V written to
their page slots) and ``chunk_attention`` (the step's new tokens over the paged cache).
With ``own`` false ``run`` computes them from elementary torch operations in 32 bits.
"""

import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# (query heads, kv heads, head_dim) of the benchmark configurations, and one without shared heads
HEADS = ((14, 2, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (8, 8, 64))


def listed():
    return [
        # --- plan_step ---
        # a decode step of a small batch: one new token each
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "mode": "decode", "ctx": 8192, "page": 128,
         "pad": 0, "lens": 1},
        # a mixed step: decodes, idle rows and prompt chunks, padded to a fixed token count
        {"name": "plan_mixed_509", "op": "plan", "requests": 509, "mode": "mixed", "ctx": 4096, "page": 16,
         "pad": 77, "lens": 2},
        # admission of a large queue of prompts in one step
        {"name": "plan_prefill_2048", "op": "plan", "requests": 2048, "mode": "prefill", "ctx": 1024, "page": 16,
         "pad": 0, "lens": 3},
        # --- rope ---
        # a decode step: 16 tokens, text positions, appended to the cache
        {"name": "rope_decode_16", "op": "rope", "tokens": 16, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "axes": 1,
         "interleaved": False, "dtype": "bf16", "append": True, "page": 128},
        # patches of images in a vision tower: two axes (height, width), no cache
        {"name": "rope_image_6399", "op": "rope", "tokens": 6399, "hq": 16, "hkv": 0, "dim": 64, "rot": 64, "axes": 2,
         "interleaved": False, "dtype": "f16", "append": False, "page": 16},
        # a prompt chunk of text and video: three axes, interleaved, appended
        {"name": "rope_video_16384", "op": "rope", "tokens": 16384, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "axes": 3, "interleaved": True, "dtype": "bf16", "append": True, "page": 64},
        # --- chunk_attention ---
        # a single token of a single request (the smallest model shape)
        {"name": "attn_one_token", "op": "attn", "requests": 1, "mode": "decode", "new": 1, "ctx": 2048, "hq": 14,
         "hkv": 2, "dim": 64, "dtype": "f16", "page": 64, "window": 0, "lse": False, "lens": 4},
        # a decode step of a ragged batch of 16, up to 8192 tokens each
        {"name": "attn_decode_16", "op": "attn", "requests": 16, "mode": "decode", "new": 1, "ctx": 8192, "hq": 32,
         "hkv": 8, "dim": 128, "dtype": "bf16", "page": 128, "window": 0, "lse": False, "lens": 5},
        # drafts checked: 5 tokens for each of 16 long requests
        {"name": "attn_verify_16x5", "op": "attn", "requests": 16, "mode": "even", "new": 5, "ctx": 32768, "hq": 64,
         "hkv": 8, "dim": 128, "dtype": "bf16", "page": 64, "window": 0, "lse": True, "lens": 6},
        # a mixed step: a chunk of 509 tokens beside decodes and an idle row, small pages
        {"name": "attn_mixed_509", "op": "attn", "requests": 9, "mode": "mixed", "new": 509, "ctx": 4096, "hq": 28,
         "hkv": 4, "dim": 128, "dtype": "bf16", "page": 16, "window": 0, "lse": False, "lens": 7},
        # a chunk under a sliding window
        {"name": "attn_window_1021", "op": "attn", "requests": 4, "mode": "even", "new": 1021, "ctx": 8192, "hq": 32,
         "hkv": 8, "dim": 128, "dtype": "f16", "page": 128, "window": 1024, "lse": True, "lens": 8},
        # prompt chunks of 2048 tokens over long prefixes
        {"name": "attn_chunk_4x2048", "op": "attn", "requests": 4, "mode": "even", "new": 2048, "ctx": 8192, "hq": 32,
         "hkv": 8, "dim": 128, "dtype": "bf16", "page": 128, "window": 0, "lse": False, "lens": 9},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "rope", "attn", "attn"))
    if op == "plan":
        mode = rng.choice(("decode", "mixed", "prefill"))
        return {"op": "plan", "requests": _log(rng, 1, 2048), "mode": mode,
                "ctx": _log(rng, 64, 1024 if mode == "prefill" else 8192), "page": rng.choice((16, 32, 64, 128)),
                "pad": rng.choice((0, 0, rng.randrange(1, 300))), "lens": rng.randrange(1 << 30)}
    if op == "rope":
        append = rng.random() < 0.6
        hq, hkv, dim = rng.choice(HEADS)
        if not append:
            hq, hkv, dim = rng.choice((4, 7, 16, 32)), 0, rng.choice((64, 72, 80, 128))
        rot = rng.choice((dim, dim, dim // 2))
        dtype = rng.choice(("bf16", "f16")) if append else rng.choice(("bf16", "f16", "f32"))
        axes = rng.choice((1, 2, 3))
        most = 16384 * 48 * 128 // ((hq + 2 * hkv) * dim * (2 if dtype == "f32" else 1))
        return {"op": "rope", "tokens": _log(rng, 1, min(16384, most)), "hq": hq, "hkv": hkv, "dim": dim, "rot": rot,
                "axes": axes, "interleaved": axes > 1 and rng.random() < 0.5, "dtype": dtype, "append": append,
                "page": rng.choice((16, 32, 64, 128))}
    most = work(listed()[-1])["flops"]
    while True:
        hq, hkv, dim = rng.choice(HEADS)
        mode = rng.choice(("decode", "even", "mixed"))
        case = {"op": "attn", "requests": _log(rng, 2 if mode == "mixed" else 1, 32), "mode": mode,
                "new": 1 if mode == "decode" else _log(rng, 2, 2048), "ctx": _log(rng, 16, 32768), "hq": hq,
                "hkv": hkv, "dim": dim, "dtype": rng.choice(("bf16", "f16")), "page": rng.choice((16, 32, 64, 128)),
                "window": rng.choice((0, 0, 0, _log(rng, 16, 4096))), "lse": rng.random() < 0.5,
                "lens": rng.randrange(1 << 30)}
        scores = case["requests"] * hq * case["new"] * (case["ctx"] + case["new"])
        cache = case["requests"] * (case["ctx"] + case["new"]) * hkv * dim
        if scores < 3 << 30 and cache < 1 << 29 and work(case)["flops"] <= most:
            return case


def _lengths(case):
    """(cached, new) tokens of each request, from the case alone."""
    rng = random.Random(case["lens"])
    R, ctx, mode = case["requests"], case["ctx"], case["mode"]
    cached, new = [], []
    for r in range(R):
        c = rng.randint(ctx // 2, ctx)
        if mode == "decode":
            n = 1
        elif mode == "even":            # attention: the same number of new tokens each
            n = case["new"]
        elif mode == "prefill":         # plan: prompts of their own length, nothing cached yet
            c, n = 0, rng.randint(1, max(1, ctx // 8))
        elif case["op"] == "plan":      # mixed: mostly decodes, some idle rows, some prompt chunks
            n = rng.choice((1, 1, 1, 1, 1, 1, 0, rng.randint(2, 256)))
        else:                           # mixed: one chunk, one idle row where there is room, else decodes
            n = case["new"] if r == 0 else 0 if r == 1 and R > 2 else 1
        cached.append(c)
        new.append(n)
    return cached, new


def _sections(case):
    """Frequencies per axis (time, height, width): the first axis takes what does not divide."""
    half, A = case["rot"] // 2, case["axes"]
    if A == 1:
        return (half,)
    if A == 3 and half == 64:
        return (16, 24, 24)
    rest = half // A
    return (half - rest * (A - 1),) + (rest,) * (A - 1)


def _axis_of(case):
    """The axis of each frequency: sections one after the other, or interleaved."""
    sec, A = _sections(case), case["axes"]
    half = case["rot"] // 2
    if case["interleaved"]:
        return [j % A if j % A and j < A * sec[j % A] else 0 for j in range(half)]
    return [a for a in range(A) for _ in range(sec[a])]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        P, T = case["page"], sum(new) + case["pad"]
        need = sum(_pages(c + n, P) - _pages(c, P) for c, n in zip(cached, new))
        return {"bytes": 17 * len(new) + 8 * need + 12 * T, "flops": 0}
    if case["op"] == "rope":
        T, eb = case["tokens"], 4 if case["dtype"] == "f32" else 2
        elems = T * (case["hq"] + 2 * case["hkv"]) * case["dim"]
        pairs = T * (case["hq"] + case["hkv"]) * case["rot"] // 2
        return {"bytes": 2 * elems * eb + 4 * case["axes"] * T + 2 * case["rot"] + (8 * T if case["append"] else 0),
                "flops": 6 * pairs}
    cached, new = _lengths(case)
    W, D = case["window"], case["dim"]
    keys = pairs = 0
    for c, n in zip(cached, new):
        first = c + 1                    # keys that the first new token sees without a window
        if W:
            keys += n and min(c + n, n - 1 + W)
            short = max(0, min(n, W - first))        # tokens that see fewer than W keys
            pairs += short * first + short * (short - 1) // 2 + (n - short) * min(W, c + n) if n else 0
        else:
            keys += (c + n) if n else 0
            pairs += n * first + n * (n - 1) // 2
    T = sum(new)
    return {"bytes": 2 * 2 * keys * case["hkv"] * D + 2 * 2 * T * case["hq"] * D
            + (4 * T * case["hq"] if case["lse"] else 0) + 4 * sum(_pages(c + n, case["page"]) for c, n in zip(cached, new))
            + 8 * len(new), "flops": 4 * D * case["hq"] * pairs}


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _outliers(g, shape, dtype):
    """N(0, 1) with a few channels eight times as large, as keys have them."""
    x = torch.randn(shape, generator=g, device="cuda")
    scale = torch.ones(shape[-1], device="cuda")
    scale[torch.randperm(shape[-1], generator=g, device="cuda")[:4]] = 8.0
    return (x * scale).to(dtype)


def _tables(g, tokens, page, spare):
    """Block table rows for `tokens` per request out of shuffled pages; `spare` pages are left over."""
    pages = [_pages(t, page) for t in tokens]
    n_pages = sum(pages) + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    width = max(pages) if pages else 1
    counts = _int32(pages).long()
    column = torch.arange(width, device="cuda")
    live = column < counts[:, None]
    index = (counts.cumsum(0) - counts)[:, None] + column
    table = torch.where(live, order[index.clamp(max=n_pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    return table.contiguous(), order[sum(pages):].contiguous(), n_pages


def prepare(case, seed):
    g = _generator(seed)
    s = SimpleNamespace(case=case)
    if case["op"] == "plan":
        cached, new = _lengths(case)
        P = case["page"]
        need = sum(_pages(c + n, P) - _pages(c, P) for c, n in zip(cached, new))
        s.total = sum(new) + case["pad"]
        table, s.free_pages, _ = _tables(g, cached, P, need + 64)
        wide = max(_pages(c + n, P) for c, n in zip(cached, new)) + 8
        s.block_table = torch.zeros(len(new), wide, dtype=torch.int32, device="cuda")
        s.block_table[:, :table.shape[1]] = table
        s.n_free = _int32([need + 64])
        s.kv_lens, s.new_lens = _int32(cached), _int32(new)
        if own:
            from fade_b200.paged import StepPlan

            s.plan = StepPlan.empty(len(new), s.total, device="cuda")     # buffers that a server keeps
        return s
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rope":
        T, hq, hkv, D = case["tokens"], case["hq"], case["hkv"], case["dim"]
        fused = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device="cuda").to(dtype)
        s.q, s.k, s.v = (x.unflatten(-1, (-1, D)) for x in fused.split([hq * D, hkv * D, hkv * D], -1))
        half = case["rot"] // 2
        s.inv_freq = (500000.0 ** -(torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
        top = 32768 if case["append"] else 1024
        s.positions = torch.randint(0, top, (case["axes"], T), generator=g, device="cuda", dtype=torch.int32)
        if case["append"]:
            P = case["page"]
            n_pages = _pages(T, P) + 3
            s.k_pool = torch.randn(n_pages, hkv, P, D, generator=g, device="cuda").to(dtype)
            s.v_pool = torch.randn(n_pages, hkv, P, D, generator=g, device="cuda").to(dtype)
            at = torch.arange(T, device="cuda") + P // 2          # consecutive tokens over shuffled pages
            s.slots = torch.randperm(n_pages, generator=g, device="cuda")[at // P] * P + at % P
        return s
    cached, new = _lengths(case)
    hkv, D, P = case["hkv"], case["dim"], case["page"]
    kv = [c + n for c, n in zip(cached, new)]
    s.block_table, _, n_pages = _tables(g, kv, P, 5)
    s.k_pool = _outliers(g, (n_pages, hkv, P, D), dtype)
    s.v_pool = torch.randn(n_pages, hkv, P, D, generator=g, device="cuda").to(dtype)
    s.q = torch.randn(sum(new), case["hq"], D, generator=g, device="cuda").to(dtype)
    s.cu_q = _int32([sum(new[:r]) for r in range(len(new) + 1)])
    s.kv_lens = _int32(kv)
    s.most_new = max(new)
    return s


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(s):
    c = s.case
    if c["op"] == "plan":
        return _plan_own(s) if own else _plan_plain(s)
    if c["op"] == "rope":
        return _rope_own(s) if own else _rope_plain(s)
    return _attn_own(s) if own else _attn_plain(s)


def _plan_own(s):
    from fade_b200.paged import plan_step

    p = plan_step(s.new_lens, s.kv_lens, s.block_table, s.free_pages, s.n_free, s.case["page"], s.total, out=s.plan)
    return {"cu_q": p.cu_q, "kv_lens": p.kv_lens, "positions": p.positions, "slots": p.slots, "n_free": p.n_free,
            "block_table": s.block_table}


def _plan_plain(s):
    P, T = s.case["page"], s.total
    new, kv = s.new_lens.long(), s.kv_lens.long()
    have = (kv + P - 1) // P
    need = (kv + new + P - 1) // P - have
    base = need.cumsum(0) - need
    ends = new.cumsum(0)
    starts = ends - new
    column = torch.arange(s.block_table.shape[1], device="cuda")[None] - have[:, None]
    fresh = (column >= 0) & (column < need[:, None])
    index = s.n_free.long() - 1 - base[:, None] - column
    table = torch.where(fresh, s.free_pages[index.clamp(0, s.free_pages.shape[0] - 1)], s.block_table)
    t = torch.arange(T, device="cuda")
    row = torch.searchsorted(ends, t, right=True)
    live = row < new.shape[0]
    row = row.clamp(max=new.shape[0] - 1)
    pos = torch.where(live, kv[row] + t - starts[row], 0)
    slot = torch.where(live, table[row, pos // P].long() * P + pos % P, -1)
    cu_q = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), ends])
    return {"cu_q": cu_q.int(), "kv_lens": (kv + new).int(), "positions": pos.int(), "slots": slot,
            "n_free": (s.n_free.long() - need.sum()).int(), "block_table": table}


def _rope_own(s):
    from fade_b200.paged import rope_append, rope_axes

    c = s.case
    if not c["append"]:
        return rope_axes(s.q, s.positions, s.inv_freq, _sections(c), interleaved=c["interleaved"])
    q = rope_append(s.q, s.k, s.v, s.positions, s.inv_freq, _sections(c), s.slots, s.k_pool, s.v_pool,
                    interleaved=c["interleaved"])
    return {"q": q, "k_pool": s.k_pool, "v_pool": s.v_pool}


def _rotate(x, cos, sin, rot):
    a, b, rest = x.float().split([rot // 2, rot // 2, x.shape[-1] - rot], -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(x.dtype)


def _rope_plain(s):
    c = s.case
    axis = torch.tensor(_axis_of(c), device="cuda")
    angle = s.positions[axis].float().t() * s.inv_freq
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    q = _rotate(s.q, cos, sin, c["rot"])
    if not c["append"]:
        return q
    P = c["page"]
    s.k_pool[s.slots // P, :, s.slots % P] = _rotate(s.k, cos, sin, c["rot"])
    s.v_pool[s.slots // P, :, s.slots % P] = s.v
    return {"q": q, "k_pool": s.k_pool, "v_pool": s.v_pool}


def _attn_own(s):
    from fade_b200.paged import chunk_attention

    c = s.case
    return chunk_attention(s.q, s.k_pool, s.v_pool, s.block_table, s.cu_q, s.kv_lens, window=c["window"] or None,
                           return_lse=c["lse"])


def _attn_plain(s):
    c = s.case
    hkv, D, P = c["hkv"], c["dim"], c["page"]
    g = c["hq"] // hkv
    R, N = s.kv_lens.shape[0], s.most_new
    keys = s.k_pool[s.block_table.long()].transpose(1, 2).flatten(2, 3).float()       # [R, hkv, S, D]
    values = s.v_pool[s.block_table.long()].transpose(1, 2).flatten(2, 3).float()
    S = keys.shape[2]
    starts, ends = s.cu_q[:-1].long(), s.cu_q[1:].long()
    token = starts[:, None] + torch.arange(N, device="cuda")
    q = s.q.float()[token.clamp(max=s.q.shape[0] - 1)]                                # [R, N, hq, D]
    q = q.unflatten(2, (hkv, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)                 # [R, hkv, g N, D]
    scores = (q @ keys.transpose(2, 3)).unflatten(2, (g, N)).mul_(1.0 / math.sqrt(D))
    j = torch.arange(S, device="cuda")
    p = (s.kv_lens.long() - (ends - starts))[:, None, None] + torch.arange(N, device="cuda")[:, None]
    seen = (j <= p) & (j < s.kv_lens[:, None, None])
    if c["window"]:
        seen &= j > p - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ values).unflatten(2, (g, N)) / total.clamp(min=1e-30)
    t = torch.arange(s.q.shape[0], device="cuda")
    row = torch.searchsorted(ends, t, right=True)
    at = t - starts[row]
    out = out.permute(0, 3, 1, 2, 4)[row, at].flatten(1, 2).to(s.q.dtype)             # [T, hq, D]
    if not c["lse"]:
        return out
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2)[row, at].flatten(1, 2)
    return {"out": out, "lse": lse}


# ----------------------------------------------------------------------------------------------
# 64-bit values, request by request
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":
        return None                       # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "rope":
        theta = torch.stack([s.positions[a].double() * f for a, f in zip(_axis_of(case), s.inv_freq.double())], -1)
        turn = torch.polar(torch.ones_like(theta), theta)[:, None]
        half = case["rot"] // 2

        def rotated(x):
            x = x.double()
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        if not case["append"]:
            return rotated(s.q)
        k_pool, v_pool = s.k_pool.double(), s.v_pool.double()
        k_pool.transpose(1, 2)[s.slots // case["page"], s.slots % case["page"]] = rotated(s.k)
        v_pool.transpose(1, 2)[s.slots // case["page"], s.slots % case["page"]] = s.v.double()
        return {"q": rotated(s.q), "k_pool": k_pool, "v_pool": v_pool}
    P, hq, hkv, D = case["page"], case["hq"], case["hkv"], case["dim"]
    cached, new = _lengths(case)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        slots = torch.arange(c + n, device="cuda")
        pages = s.block_table[r].long()[slots // P]
        for h in range(hq if n else 0):
            k = s.k_pool[pages, h * hkv // hq, slots % P].double()
            v = s.v_pool[pages, h * hkv // hq, slots % P].double()
            for a in range(0, n, 512):
                b = min(n, a + 512)
                x = torch.einsum("td,sd->ts", s.q[first + a:first + b, h].double(), k) / math.sqrt(D)
                ahead = slots[None] - (c + torch.arange(a, b, device="cuda"))[:, None]
                x[ahead > 0] = -math.inf
                if case["window"]:
                    x[ahead <= -case["window"]] = -math.inf
                norm = torch.logsumexp(x, -1)
                out[first + a:first + b, h] = torch.exp(x - norm[:, None]) @ v
                lse[first + a:first + b, h] = norm
        first += n
    return {"out": out, "lse": lse} if case["lse"] else out
