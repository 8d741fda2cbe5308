"""The paged serving step where things go wrong: waits that run out, threads,
captured steps, strides that are never stepped, values at the types' limits."""

from __future__ import annotations

import math
import threading

import pytest
import torch

from test_paged_gpu import BF, HF, _attn_inputs, _attn_ref

pytestmark = pytest.mark.gpu


# (new, kv, hq, hkv, D, page, dtype): decodes over split tiles, chunks of two half tiles, both in one batch
GIVE_UP = [
    ([1, 1, 5], [3000, 700, 900], 8, 2, 128, 32, BF),
    ([300], [2000], 8, 2, 64, 64, HF),
    ([260, 1, 0, 3], [1500, 4000, 9, 3], 28, 4, 128, 16, BF),
]


@pytest.mark.parametrize("polls", [0, 1, 3, 40, 1000])
@pytest.mark.parametrize("new,kv,hq,hkv,D,page,dt", GIVE_UP)
def test_waits_that_run_out_are_reported(cuda_device, polls, new, kv, hq, hkv, D, page, dt):
    """A call whose device waits give up ends, says so, and leaves nothing behind for the next one."""
    from fade_b200 import _lib
    from fade_b200.paged import check_device_errors, chunk_attention

    lib = _lib.load()
    args = _attn_inputs(new, kv, hq, hkv, D, page, dt, cuda_device, 31)
    clean = chunk_attention(*args)
    check_device_errors(cuda_device)
    ref, _, lim, _ = _attn_ref(*args[:4], new, kv, True, None, D ** -0.5)
    for _ in range(5):
        try:
            assert lib.fade_set_wait_polls(polls) == _lib.FADE_OK
            out = chunk_attention(*args)
        finally:
            assert lib.fade_set_wait_polls(-1) == _lib.FADE_OK
        try:
            check_device_errors(cuda_device)
            assert polls > 0 and ((out.double() - ref).abs() <= lim).all()
        except RuntimeError as e:
            assert "timed out" in str(e)
        check_device_errors(cuda_device)                          # reported once
        assert torch.equal(chunk_attention(*args), clean)
        check_device_errors(cuda_device)


def _in_new_thread(work):
    """work() in a thread that has not used the GPU."""
    got = []

    def loop():
        try:
            got.append(work())
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=loop)
    t.start()
    t.join(timeout=60)
    torch.cuda.synchronize()
    assert got and not isinstance(got[0], Exception), got
    return got[0]


def test_first_call_of_a_thread(cuda_device):
    """The tensor maps are made in a thread that has no context yet."""
    from fade_b200.attention import Int4Tier, tiered_decode_attention
    from fade_b200.paged import chunk_attention
    from fade_b200.quant import quant_k_int4, quant_v_int4

    args = _attn_inputs([3, 1], [900, 40], 8, 2, 64, 16, HF, cuda_device, 32)
    want = chunk_attention(*args)
    out = torch.zeros_like(want)                                  # (torch's own launches would make the context current)
    assert torch.equal(_in_new_thread(lambda: chunk_attention(*args, out=out)), want)
    g = torch.Generator(device="cuda").manual_seed(33)
    k, v = (torch.randn(1, 2, 256, 128, generator=g, device=cuda_device).to(BF) for _ in range(2))
    tier = Int4Tier(*quant_k_int4(k), *quant_v_int4(v))
    q = torch.randn(1, 8, 1, 128, generator=g, device=cuda_device).to(BF)
    want = tiered_decode_attention(q, [tier])
    assert torch.equal(_in_new_thread(lambda: tiered_decode_attention(q, [tier])), want)


def _in_threads(works, rounds, stream):
    """Each work over and over in a thread of its own, all on one stream; their results in order."""
    results, errors = [[] for _ in works], []
    start = threading.Barrier(len(works))

    def loop(i):
        try:
            with torch.cuda.stream(stream):
                start.wait(timeout=30)
                for _ in range(rounds):
                    results[i].append(works[i]())
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(len(works))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=120)
    torch.cuda.synchronize()
    assert not errors and not any(t.is_alive() for t in threads), errors
    return results


@pytest.mark.parametrize("own_stream", [False, True])
def test_chunk_attention_from_threads_on_one_stream(cuda_device, own_stream):
    """Batches of other sizes from other threads on the same stream: each gets its own result, bit for bit."""
    from fade_b200.paged import check_device_errors, chunk_attention

    batches = [_attn_inputs(new, kv, 8, 2, 128, 32, BF, cuda_device, 40 + i) for i, (new, kv) in enumerate(
        (([1, 1, 1], [5000, 900, 2000]), ([300], [2500]), ([40, 1, 70], [1000, 7000, 70]), ([1], [9000])))]
    alone = [chunk_attention(*b, return_lse=True) for b in batches]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
    results = _in_threads([lambda b=b: chunk_attention(*b, return_lse=True) for b in batches], 60, stream)
    with torch.cuda.stream(stream):
        check_device_errors(cuda_device)
    for want, got in zip(alone, results):
        assert len(got) == 60
        for g in got:
            assert torch.equal(g["out"], want["out"]) and torch.equal(g["lse"], want["lse"])


def test_tiered_decode_attention_from_threads_on_one_stream(cuda_device):
    """As above for the decode over tiers, whose kernels hand partials on through a workspace, too."""
    from fade_b200.attention import FPTier, Int4Tier, tiered_decode_attention
    from fade_b200.quant import quant_k_int4, quant_v_int4

    g = torch.Generator(device="cuda").manual_seed(50)

    def batch(B, n):
        k, v, rk, rv = (torch.randn(B, 2, m, 128, generator=g, device=cuda_device).to(BF) for m in (n, n, 64, 64))
        q = torch.randn(B, 8, 1, 128, generator=g, device=cuda_device).to(BF)
        return q, [Int4Tier(*quant_k_int4(k), *quant_v_int4(v)), FPTier(rk, rv)]

    batches = [batch(1, 8192), batch(6, 1024), batch(3, 3000 // 8 * 8)]
    alone = [tiered_decode_attention(*b) for b in batches]
    torch.cuda.synchronize()
    results = _in_threads([lambda b=b: tiered_decode_attention(*b) for b in batches], 60, torch.cuda.default_stream())
    for want, got in zip(alone, results):
        assert len(got) == 60 and all(torch.equal(g, want) for g in got)


def test_captured_calls_report_their_errors(cuda_device):
    """A wait that gives up in a replayed graph is found from any stream, without the stream of the capture."""
    from fade_b200 import _lib
    from fade_b200.paged import check_device_errors, chunk_attention

    args = _attn_inputs([3, 1], [900, 40], 8, 2, 64, 16, HF, cuda_device, 34)
    want = chunk_attention(*args)
    graph, broken = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    try:
        assert _lib.load().fade_set_wait_polls(0) == _lib.FADE_OK
        with torch.cuda.graph(broken):
            chunk_attention(*args)
    finally:
        assert _lib.load().fade_set_wait_polls(-1) == _lib.FADE_OK
    with torch.cuda.graph(graph):
        out = chunk_attention(*args)
    graph.replay()
    check_device_errors(cuda_device)
    assert torch.equal(out, want)
    broken.replay()
    with pytest.raises(RuntimeError, match="timed out"):
        check_device_errors(cuda_device)
    graph.replay()
    check_device_errors(cuda_device)
    assert torch.equal(out, want)


def test_graphs_replayed_at_the_same_time(cuda_device):
    """Graphs captured on one stream and replayed on several, beside direct calls: each has its own workspace."""
    from fade_b200.paged import check_device_errors, chunk_attention

    batches = [_attn_inputs(new, kv, 8, 2, 128, 32, BF, cuda_device, 60 + i) for i, (new, kv) in enumerate(
        (([1, 1, 1], [5000, 900, 2000]), ([200], [2500]), ([40, 1, 70], [1000, 7000, 70])))]
    alone = [chunk_attention(*b) for b in batches]
    graphs = []
    for b in batches:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chunk_attention(*b)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(40):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        direct = [chunk_attention(*b) for b in batches]
    torch.cuda.synchronize()
    check_device_errors(cuda_device)
    for want, (_, out), also in zip(alone, graphs, direct):
        assert torch.equal(out, want) and torch.equal(also, want)


def test_captured_cache_step(cuda_device):
    """A whole decode step of PagedKVCache in a graph: replays advance the cache as direct steps do."""
    from fade_b200.paged import PagedKVCache

    L, hq, hkv, D, R = 2, 8, 2, 64, 3
    g = torch.Generator(device="cuda").manual_seed(70)
    inv = (10000.0 ** -(torch.arange(D // 2, device=cuda_device) / (D // 2))).float()
    prompt = torch.tensor([20, 33, 7], dtype=torch.int32, device=cuda_device)
    one = torch.ones(R, dtype=torch.int32, device=cuda_device)
    first = [torch.randn(L, 60, h, D, generator=g, device=cuda_device).to(BF) for h in (hq, hkv, hkv)]
    steps = [[torch.randn(L, R, h, D, generator=g, device=cuda_device).to(BF) for h in (hq, hkv, hkv)] for _ in range(20)]

    def step(cache, qkv, lens, total):
        plan = cache.plan(lens, total)
        return torch.stack([cache.attend(i, plan, cache.append(i, plan, qkv[0][i], qkv[1][i], qkv[2][i], inv))
                            for i in range(L)])

    caches = [PagedKVCache(L, hkv, D, n_pages=20, max_requests=R, max_tokens=64, page_size=16, dtype=BF,
                           device=cuda_device) for _ in range(2)]
    for c in caches:
        step(c, first, prompt, 60)
    static = [x.clone() for x in steps[0]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(caches[1], static, one, R)
    for qkv in steps:
        want = step(caches[0], qkv, one, R)
        for s, x in zip(static, qkv):
            s.copy_(x)
        graph.replay()
        assert torch.equal(out, want)
    for c in caches:
        c.check()
        assert c.kv_lens.tolist() == [40, 53, 27]
    assert torch.equal(caches[0].n_free, caches[1].n_free) and torch.equal(caches[0].k, caches[1].k)


def test_strides_that_are_never_stepped(cuda_device):
    """A dimension of one may have any stride: a token out of a wider row, a pool of one page or one head."""
    from fade_b200.paged import chunk_attention

    dev = cuda_device
    q, kp, vp, table, cu, kl = _attn_inputs([1], [40], 2, 1, 64, 64, HF, dev, 35)
    want = chunk_attention(q, kp, vp, table, cu, kl)
    rows = torch.zeros(5, 132, dtype=HF, device=dev)
    rows[2, :128] = q.view(-1)
    one = rows[:, :128].unflatten(1, (2, 64))[2:3]
    assert one.stride() == (132, 64, 1)
    assert torch.equal(chunk_attention(one, kp, vp, table, cu, kl), want)
    wide = torch.full((3, 2 * 64 + 5), 3.0, dtype=HF, device=dev)
    dest = wide[:, :128].unflatten(1, (2, 64))[:1]
    assert dest.stride()[0] % 8 and chunk_attention(q, kp, vp, table, cu, kl, out=dest) is dest
    assert torch.equal(dest, want) and (wide[1:] == 3).all() and (wide[:, 128:] == 3).all()
    # a token at an odd address is copied, from its odd stride too
    flat = torch.zeros(129, dtype=HF, device=dev)
    flat[1:] = q.view(-1)
    odd = flat.as_strided((1, 2, 64), (131, 64, 1), 1)
    assert torch.equal(chunk_attention(odd, kp, vp, table, cu, kl), want)
    # one head of its own: [T, 1, D] and pools [pages, 1, page, D]
    page = int(table[0, 0])
    zero = torch.zeros_like(table)
    single = [torch.zeros(64 * 64 + 12, dtype=HF, device=dev) for _ in range(2)]
    for s, p in zip(single, (kp, vp)):
        s[:64 * 64] = p[page, 0].reshape(-1)
    k1, v1 = (s.as_strided((1, 1, 64, 64), (4099, 4097, 64, 1)) for s in single)
    assert torch.equal(chunk_attention(q, k1, v1, zero, cu, kl), want)
    thin = q[:, :1].clone().as_strided((1, 1, 64), (77, 33, 1))
    assert torch.equal(chunk_attention(thin, kp, vp, table, cu, kl), chunk_attention(q[:, :1].clone(), kp, vp, table, cu, kl))
    # broadcast tokens and heads
    for b in (q[:, :1].expand(1, 2, 64), q.expand(3, 2, 64)):
        n = torch.tensor([0, b.shape[0]], dtype=torch.int32, device=dev)
        assert torch.equal(chunk_attention(b, kp, vp, table, n, kl), chunk_attention(b.clone(), kp, vp, table, n, kl))


def test_a_failed_release_is_remembered(cuda_device):
    """The status of a release outlives the releases after it, until it was looked at."""
    from fade_b200.paged import PagedKVCache, release_rows

    cache = PagedKVCache(1, 2, 64, n_pages=8, max_requests=2, max_tokens=64, page_size=16, dtype=BF, device=cuda_device)
    cache.plan(torch.tensor([20, 30], dtype=torch.int32, device=cuda_device), 50).check()
    first, second = (torch.tensor(m, device=cuda_device) for m in ([True, False], [False, True]))
    for lens, text in ((65, "row"), (-1, "negative")):          # a page more than a row of the table holds; no length
        cache.kv_lens[0] = lens
        cache.release(first)                                     # fails: nothing changes
        assert cache.kv_lens.tolist() == [lens, 30] and cache.n_free.item() == 4
        cache.kv_lens[0] = 20
        cache.release(torch.zeros_like(first))                   # succeeds
        with pytest.raises(RuntimeError, match=text):
            cache.check()
        cache.check()
    cache.release(first)
    cache.release(second)
    cache.check()
    assert cache.kv_lens.tolist() == [0, 0] and cache.n_free.item() == 8
    assert sorted(cache.free_pages.tolist()) == list(range(8))
    # the operator's own status: a negative length of a row that stays counts, too
    kv = torch.tensor([16, -3], dtype=torch.int32, device=cuda_device)
    assert release_rows(first, kv, cache.block_table, 16, cache.free_pages, cache.n_free).item() == 4
    assert kv.tolist() == [16, -3] and cache.n_free.item() == 8


def test_rope_axes_of_every_scheme(cuda_device):
    """rope_axes with a scheme's step frequencies against its tables, in the tier cache's pairing (j, j + D/2)."""
    from fade_b200 import rope
    from fade_b200.paged import rope_axes

    g = torch.Generator(device="cuda").manual_seed(80)
    D, x = 64, torch.randn(40, 3, 64, generator=g, device=cuda_device)
    pos = torch.randint(0, 30000, (40,), generator=g, device=cuda_device)
    for scheme in (rope.Vanilla(head_dim=D), rope.LinearScaled(head_dim=D, factor=3.0), rope.Llama3(head_dim=D, factor=8.0),
                   rope.NtkAware(head_dim=D, factor=2.0), rope.Yarn(head_dim=D, factor=4.0),
                   rope.Proportional(head_dim=D, partial_rotary_factor=0.5),
                   rope.MRope(head_dim=D, mrope_section=[32]), rope.NoRope(head_dim=D)):
        f = scheme.axes_inv_freq(cuda_device)
        cos, sin = (t[0, 0].double()[:, None] for t in scheme.compute_cos_sin(pos, cuda_device, model_dtype=torch.float32))
        a, b = x.double().split(D // 2, -1)
        want = torch.cat([a * cos[..., :D // 2] - b * sin[..., :D // 2], b * cos[..., D // 2:] + a * sin[..., D // 2:]], -1)
        angle = torch.zeros(40, 1, D // 2, device=cuda_device)
        angle[:, 0, :f.numel()] = pos.float()[:, None] * f
        lim = (a.abs() + b.abs()) * (4 * 2.0 ** -24 * angle + 2.0 ** -21)
        assert ((rope_axes(x, pos, f).double() - want).abs() <= torch.cat([lim, lim], -1)).all(), type(scheme).__name__


def test_hand_over_to_the_tier_cache_at_text_positions(cuda_device):
    """Pages gathered into TieredKVCache go through an eviction (un-rotated and rotated again) as the model's own keys do."""
    from fade_b200.cache import TieredKVCache
    from fade_b200.paged import PagedKVCache
    from fade_b200.policy import _assign_one_layer
    from fade_b200.rope import LinearScaled

    g = torch.Generator(device="cuda").manual_seed(90)
    hq, hkv, D, n = 4, 2, 64, 150
    scheme = LinearScaled(theta=10000.0, head_dim=D, factor=2.0)
    q, k, v = (torch.randn(n, h, D, generator=g, device=cuda_device).half() for h in (hq, hkv, hkv))
    pages = PagedKVCache(1, hkv, D, n_pages=16, max_requests=2, max_tokens=256, page_size=16, dtype=HF, device=cuda_device)
    plan = pages.plan(torch.tensor([0, n], dtype=torch.int32, device=cuda_device), n)
    # sin and cos rounded to fp16 as the scheme's tables are; half of an integer position is exact, so the angles agree
    pages.append(0, plan, q, k, v, scheme.axes_inv_freq(cuda_device), round_tables=True)
    plan.check()
    cos, sin = (t[0, 0][:, None] for t in scheme.compute_cos_sin(torch.arange(n, device=cuda_device), cuda_device, torch.float16))
    turned = torch.cat([-k[..., D // 2:], k[..., :D // 2]], -1).float()
    direct = (k.float() * cos + turned * sin).half().transpose(0, 1)[None]
    caches = []
    for keys, values in ((direct, v.transpose(0, 1)[None]), pages.gather(0, [1], n)):
        cache = TieredKVCache(n_sink=4, recent_window=16, int4_budget=40, dtype=HF, rope_theta=10000.0, head_dim=D,
                              rope_scheme=scheme)
        cache.update(keys.contiguous(), values.contiguous(), 0)
        scores = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(91), device=cuda_device)
        cache.apply_tier_assignment(0, _assign_one_layer(n, scores, 4, 16, 40, 0))
        caches.append(cache)
    a, b = (c._materialize(0) for c in caches)
    assert a[0].shape == b[0].shape and a[0].shape[2] == 60
    assert torch.equal(a[1], b[1])
    # K: one fp16 rounding of the rotation apart, then 4-bit codes of the middle: a step of the scale
    step = float(a[0].abs().max()) / 7 + 4 * 2.0 ** -11 * float(a[0].abs().max())
    assert float((a[0] - b[0]).abs().max()) <= step
    sinks = slice(0, 4)
    assert float((a[0][:, :, sinks] - b[0][:, :, sinks]).abs().max()) <= 8 * 2.0 ** -11 * float(direct.abs().max())


def test_overlapping_outputs_are_refused(cuda_device):
    """An output that shares elements with the input is refused, one that only lies between them is not."""
    from fade_b200.paged import chunk_attention, rope_axes

    _, kp, vp, table, cu, kl = _attn_inputs([6, 5], [30, 20], 4, 2, 64, 16, BF, cuda_device, 36)
    g = torch.Generator(device="cuda").manual_seed(37)
    pos = torch.arange(11, device=cuda_device)
    inv = torch.rand(32, generator=g, device=cuda_device)

    def attend(x, out=None):
        return chunk_attention(x, kp, vp, table, cu, kl, out=out)

    def rotate(x, out=None):
        return rope_axes(x, pos, inv, out=out)

    for call in (attend, rotate):
        rows = torch.randn(12, 4, 64, generator=g, device=cuda_device).to(BF)
        heads = torch.randn(11, 9, 64, generator=g, device=cuda_device).to(BF)
        turned = torch.randn(4, 11, 64, generator=g, device=cuda_device).to(BF)
        flat = torch.randn(11 * 4 * 64 + 8, generator=g, device=cuda_device).to(BF)
        for x, out in ((rows[:-1], rows[1:]), (heads[:, :4], heads[:, 3:7]), (heads[:, :8:2], heads[:, 2:9:2]),
                       (flat[:-8].view(11, 4, 64), flat[8:].view(11, 4, 64)),
                       (turned.transpose(0, 1), turned.view(11, 4, 64))):
            with pytest.raises(ValueError):
                call(x, out)
        # the other heads of the same tensor, side by side and alternating
        for x, out in ((heads[:, :4], heads[:, 4:8]), (heads[:, :8:2], heads[:, 1:8:2]), (heads[:, 1:8:2], heads[:, 2:9:2])):
            want = call(x.clone())
            assert torch.equal(call(x, out), want)
    x = torch.randn(11, 4, 64, generator=g, device=cuda_device).to(BF)
    want = rotate(x)
    assert rotate(x, x) is x and torch.equal(x, want)              # in place


@pytest.mark.parametrize("R,new,D", [(40, 1, 64), (20, 40, 128)])      # one half tile (decodes), two half tiles
def test_averages_of_the_largest_fp16_values_stay_finite(cuda_device, R, new, D):
    """Weights are rounded to fp16 for their product with V, their sum is not: 65504 averaged must not become an infinity."""
    from fade_b200.paged import chunk_attention

    n = 1400
    q, kp, vp, table, cu, kl = _attn_inputs([new] * R, [n] * R, 32, 8, D, 16, HF, cuda_device, 38, poison=False)
    # 256 keys of score 0, then equal keys whose weight 1 + 1.01 * 2^-11 against them rounds up to 1 + 2^-10
    q.zero_(), kp.zero_()
    q[..., 0] = 1.0
    j = torch.arange(256, n, device=cuda_device)
    for r in range(R):
        kp[table[r].long()[j // 16], :, j % 16, 0] = 1.0
    vp[..., ::2], vp[..., 1::2] = 65504.0, -65504.0
    sm = math.log(1 + 1.01 * 2.0 ** -11)
    want = torch.full((D,), 65504.0, device=cuda_device)
    want[1::2] = -65504.0
    out = chunk_attention(q, kp, vp, table, cu, kl, sm_scale=sm)
    assert out.isfinite().all()
    # weights rounded: 2^-11 of the value, and the result's own rounding
    assert ((out.float() - want).abs() <= 65504 * 2.0 ** -10).all()
    # a visible infinity is one, also beside hidden ones of the other sign that make other rows look again
    last = table[:, (n - 1) // 16].long()
    vp[last, :, (n - 1) % 16, 2] = float("inf")
    out = chunk_attention(q, kp, vp, table, cu, kl, sm_scale=sm).unflatten(0, (R, new))
    assert (out[:, -1, :, 2] == float("inf")).all()
    assert out[:, :-1].isfinite().all() and ((out[:, :-1].float() - want).abs() <= 65504 * 2.0 ** -10).all()
    assert ((out[:, -1].float() - want).abs()[..., 3:] <= 65504 * 2.0 ** -10).all()


def test_smallest_scale(cuda_device):
    """Scores far below any difference: the plain average of the visible values, and no NaN from hidden ones."""
    from fade_b200.paged import chunk_attention

    q, kp, vp, table, cu, kl = _attn_inputs([30], [200], 4, 2, 64, 16, HF, cuda_device, 39)
    for sm in (1e-45, 1e-40, 1e-30):
        out = chunk_attention(q, kp, vp, table, cu, kl, sm_scale=sm)
        ref, _, lim, _ = _attn_ref(q, kp, vp, table, [30], [200], True, None, sm)
        assert ((out.double() - ref).abs() <= lim).all()
    with pytest.raises(ValueError, match="sm_scale"):
        chunk_attention(q, kp, vp, table, cu, kl, sm_scale=1e-46)


@pytest.mark.parametrize("new,kv,T,hq,hkv,D,dt", [
    ([3, 0, 2], [40, 9, 700], 5, 8, 2, 64, HF),          # no padding
    ([3, 0, 2], [40, 9, 700], 37, 8, 2, 128, BF),
    ([300], [2000], 1024, 14, 2, 64, HF),
    ([0, 0], [5, 6], 9, 4, 4, 128, BF),                  # a step without tokens (or one that could not be planned)
])
def test_tokens_past_the_last_request_are_zeros(cuda_device, new, kv, T, hq, hkv, D, dt):
    """Fresh outputs hold 0 and -inf for padding tokens, whatever their memory held; a given one keeps its rows."""
    from fade_b200.paged import check_device_errors, chunk_attention

    q, kp, vp, table, cu, kl = _attn_inputs(new, kv, hq, hkv, D, 16, dt, cuda_device, 41)
    n = sum(new)
    ref, ref_lse, lim, lim_lse = _attn_ref(q, kp, vp, table, new, kv, True, None, D ** -0.5)
    padded = torch.full((T, hq, D), math.nan, dtype=dt, device=cuda_device)
    padded[:n] = q
    junk = [torch.full((T, hq, D), math.nan, dtype=dt, device=cuda_device),
            torch.full((T, hq), math.nan, device=cuda_device)]
    del junk                                             # the next outputs take this memory
    out, lse = chunk_attention(padded, kp, vp, table, cu, kl, return_lse=True).values()
    check_device_errors(cuda_device)
    assert ((out[:n].double() - ref).abs() <= lim).all() and ((lse[:n].double() - ref_lse).abs() <= lim_lse).all()
    assert (out[n:] == 0).all() and (lse[n:] == -math.inf).all()
    mine = torch.full((T, hq + 1, D), 3.0, dtype=dt, device=cuda_device)
    lse = chunk_attention(padded, kp, vp, table, cu, kl, out=mine[:, 1:], return_lse=True)["lse"]
    assert torch.equal(mine[:n, 1:], out[:n]) and (mine[n:] == 3).all() and (mine[:, 0] == 3).all()
    assert (lse[n:] == -math.inf).all()
    none = torch.zeros(0, table.shape[1], dtype=torch.int32, device=cuda_device)
    out, lse = chunk_attention(padded, kp, vp, none, cu[:1], kl[:0], return_lse=True).values()
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("new,kv,D", [([300], [900], 128), ([1, 5], [3000, 700], 64)])
def test_channels_beside_an_infinity_are_what_they_were(cuda_device, new, kv, D):
    """A visible infinity in one channel changes no bit of the others."""
    from fade_b200.paged import chunk_attention

    for dt in (HF, BF):
        q, kp, vp, table, cu, kl = _attn_inputs(new, kv, 8, 2, D, 16, dt, cuda_device, 42)
        want = chunk_attention(q, kp, vp, table, cu, kl)
        vp[table[:, 0].long(), :, 0, 5] = float("inf")                # the first token of each request: every row sees it
        out = chunk_attention(q, kp, vp, table, cu, kl)
        others = torch.arange(D, device=cuda_device) != 5
        assert torch.equal(out[..., others], want[..., others]) and not out[..., 5].isfinite().any()
