"""Host side of the paged serving step at its edges (no GPU)."""

from __future__ import annotations

import pytest
import torch

from fade_b200 import _lib


def test_wait_polls_are_bounded():
    lib = _lib.load()
    try:
        assert lib.fade_set_wait_polls((1 << 22) + 1) == _lib.FADE_ERR_INVALID_ARG
        assert lib.fade_set_wait_polls(0) == lib.fade_set_wait_polls(1 << 22) == _lib.FADE_OK
    finally:
        assert lib.fade_set_wait_polls(-1) == _lib.FADE_OK


class _Devices:
    """Two devices: torch's calls and a library that records what is current when it is called."""

    def __init__(self, monkeypatch):
        self.now, self.seen = 0, []
        monkeypatch.setattr(_lib, "_lib", self)
        monkeypatch.setattr(_lib, "_current", lambda: self.now, raising=False)
        monkeypatch.setattr(_lib, "_stream", lambda idx: 0)           # the default stream has the same handle on both
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.now)
        monkeypatch.setattr(torch.cuda, "set_device", self._set)
        monkeypatch.setattr(_lib, "_capturing", lambda: False, raising=False)
        monkeypatch.setattr(_lib, "same_device", lambda *t: 1)
        monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cuda", 1))

    def _set(self, idx):
        self.now = torch.device("cuda", idx).index

    def fade_set_device(self, idx):
        self.now = idx
        return _lib.FADE_OK

    def fade_status_string(self, status):
        return b"status"

    def fade_chunk_attn_workspace_size(self, d):
        self.seen.append(self.now)
        return 256

    def __getattr__(self, name):
        def call(*args):
            self.seen.append(self.now)
            return _lib.FADE_OK

        if not name.startswith("fade_"):
            raise AttributeError(name)
        return call


def test_bind_follows_the_current_device(monkeypatch):
    """torch changes the current device between two calls for the same one."""
    lib = _Devices(monkeypatch)
    _lib.bind(torch.device("cuda", 1))
    assert lib.now == 1
    torch.cuda.set_device(0)                      # the end of a `with torch.cuda.device(1)`, say
    _lib.bind(torch.device("cuda", 1))
    assert lib.now == 1


@pytest.mark.parametrize("op", ["plan_step", "release_rows", "rope_axes", "rope_append", "chunk_attention", "quant_k_int4"])
def test_calls_run_on_their_tensors_device(monkeypatch, op):
    """... and leave the caller's device current, whatever was current in between."""
    from fade_b200 import paged, quant

    lib = _Devices(monkeypatch)
    monkeypatch.setattr(paged, "_WS", {})
    monkeypatch.setattr(quant, "_contig_out", lambda shape, dtype, dev: torch.empty(shape, dtype=dtype))
    i = torch.zeros(1, dtype=torch.int32)
    x, pool = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(1, 1, 16, 64, dtype=torch.float16)
    call = {
        "plan_step": lambda: paged.plan_step(i, i, i[None], i, i, 16, 1,
                                             out=paged.StepPlan.empty(1, 1, "cpu")),
        "release_rows": lambda: paged.release_rows(i.bool(), i, i[None], 16, i, i, i.clone()),
        "rope_axes": lambda: paged.rope_axes(x, i, torch.zeros(32)),
        "rope_append": lambda: paged.rope_append(x, x, x, i, torch.zeros(32), None, i.long(), pool, pool),
        "chunk_attention": lambda: paged.chunk_attention(x, pool, pool, i[None], torch.zeros(2, dtype=torch.int32), i),
        "quant_k_int4": lambda: quant.quant_k_int4(x[None]),
    }[op]
    for _ in range(2):
        lib.seen.clear()
        call()
        assert lib.seen and set(lib.seen) == {1}
        assert lib.now == 0


def _schemes():
    from fade_b200 import rope

    return [rope.Vanilla(head_dim=16), rope.LinearScaled(head_dim=16, factor=4.0), rope.LinearScaled(head_dim=16, factor=3.0),
            rope.Llama3(head_dim=16, factor=8.0), rope.NtkAware(head_dim=16, factor=2.0), rope.Yarn(head_dim=16, factor=4.0),
            rope.Proportional(head_dim=16, partial_rotary_factor=0.5), rope.MRope(head_dim=16, mrope_section=[2, 3, 3]),
            rope.NoRope(head_dim=16)]


@pytest.mark.parametrize("scheme", _schemes(), ids=lambda s: type(s).__name__)
def test_step_frequencies_give_the_schemes_tables(scheme):
    """cos and sin of position * axes_inv_freq are what the scheme's own tables hold, for every scheme."""
    pos = torch.tensor([0, 1, 17, 1000, 30011])
    cos, sin = scheme.compute_cos_sin(pos, "cpu", model_dtype=torch.float32)
    f = scheme.axes_inv_freq("cpu")
    assert f.dtype == torch.float32 and f.numel() in (0, 8)
    angle = torch.zeros(5, 8)
    angle[:, :f.numel()] = pos.float()[:, None] * f
    # two roundings of the angle either way, and of cos and sin
    lim = 4 * 2.0 ** -24 * angle.abs() + 2.0 ** -22
    for half in (slice(0, 8), slice(8, 16)):
        assert ((angle.double().cos() - cos[0, 0, :, half]).abs() <= lim).all()
        assert ((angle.double().sin() - sin[0, 0, :, half]).abs() <= lim).all()


@pytest.mark.parametrize("sm_scale,ok", [(1e-46, False), (5e-324, False), (1e-45, True), (1e-40, True), (1e30, True), (1.1e30, False)])
def test_scales_that_fp32_cannot_hold_are_refused(sm_scale, ok):
    """A scale that is 0 in fp32 would make 0 x infinity of every hidden key's score."""
    import ctypes

    d = _lib.ChunkDesc(dtype=_lib.FADE_BF16, R=1, T=1, Hq=1, Hkv=1, D=64, page_size=16, n_pages=1, table_width=1,
                       table_stride=1, causal=1, sm_scale=sm_scale)
    assert (_lib.load().fade_chunk_attn_workspace_size(ctypes.byref(d)) > 0) == ok


def test_return_lse_is_a_truth_value(monkeypatch):
    from fade_b200 import paged

    _Devices(monkeypatch)
    monkeypatch.setattr(paged, "_WS", {})
    i = torch.zeros(1, dtype=torch.int32)
    x, pool = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(1, 1, 16, 64, dtype=torch.float16)
    for flag in (None, 0, 1, False, True):
        got = paged.chunk_attention(x, pool, pool, i[None], torch.zeros(2, dtype=torch.int32), i, return_lse=flag)
        assert isinstance(got, dict) == bool(flag)
