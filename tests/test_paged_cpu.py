"""Host side of the paged serving step (no GPU): argument checks of the C entry
points, axis sections and the M-RoPE tables of several axes."""

from __future__ import annotations

import ctypes

import pytest
import torch

from fade_b200 import _lib


def _plan(**kw):
    d = _lib.PlanDesc(R=1, total=1, page_size=16, table_width=2, table_stride=2, free_cap=4)
    for name in ("new_lens", "kv_lens", "block_table", "free_pages", "n_free", "cu_q", "kv_out", "positions", "slots",
                 "n_free_out", "status"):
        setattr(d, name, 16 * (1 + len(name)) + ord(name[0]) * 4096)     # distinct, never read
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.load().fade_plan_step(ctypes.byref(d), None)


@pytest.mark.parametrize("change,status", [
    (dict(R=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(total=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(page_size=0), _lib.FADE_ERR_INVALID_ARG),
    (dict(page_size=48), _lib.FADE_ERR_INVALID_ARG),
    (dict(status=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(slots=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(new_lens=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(free_pages=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(kv_lens=64, kv_out=64), _lib.FADE_ERR_INVALID_ARG),
    (dict(n_free=64, n_free_out=64), _lib.FADE_ERR_INVALID_ARG),
    (dict(R=_lib.PLAN_MAX_ROWS + 1), _lib.FADE_ERR_UNSUPPORTED),
    (dict(total=2 ** 31), _lib.FADE_ERR_UNSUPPORTED),
])
def test_plan_entry_point_refusals(change, status):
    assert _plan(**change) == status


def test_release_entry_point_refusals():
    f = _lib.load().fade_release_rows
    good = [64, 1, 64, 64, 2, 2, 16, 64, 4, 64, 64, None]
    for i, v in ((1, -1), (0, None), (2, None), (3, None), (4, -1), (6, 24), (7, None), (8, -1), (9, None), (10, None)):
        args = list(good)
        args[i] = v
        assert f(*args) == _lib.FADE_ERR_INVALID_ARG, i
    assert f(*good[:1], _lib.PLAN_MAX_ROWS + 1, *good[2:]) == _lib.FADE_ERR_UNSUPPORTED


def _rope(**kw):
    d = _lib.RopeDesc(dtype=_lib.FADE_BF16, T=3, Hq=2, Hkv=1, D=8, rot=8, axes=2, section0=2, section1=2, page_size=16,
                      n_pages=4)
    for name in ("positions", "inv_freq", "q", "q_out", "k", "v", "slots", "k_pool", "v_pool"):
        setattr(d, name, 4096)
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.load().fade_rope_axes(ctypes.byref(d), None)


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(D=0), _lib.FADE_ERR_INVALID_ARG),
    (dict(rot=7), _lib.FADE_ERR_ODD_DIM),
    (dict(rot=10, section0=3), _lib.FADE_ERR_INVALID_ARG),
    (dict(axes=0), _lib.FADE_ERR_INVALID_ARG),
    (dict(axes=5), _lib.FADE_ERR_INVALID_ARG),
    (dict(section1=3), _lib.FADE_ERR_INVALID_ARG),
    (dict(section0=5, section1=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(dtype=9), _lib.FADE_ERR_INVALID_ARG),
    (dict(positions=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(inv_freq=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(q_out=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(page_size=12), _lib.FADE_ERR_INVALID_ARG),
    (dict(v_pool=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(slots=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(D=5000), _lib.FADE_ERR_UNSUPPORTED),
    (dict(T=2 ** 31), _lib.FADE_ERR_UNSUPPORTED),
    (dict(T=0), _lib.FADE_OK),
    (dict(Hq=0, Hkv=0), _lib.FADE_OK),
])
def test_rope_entry_point_refusals(change, status):
    assert _rope(**change) == status


def _chunk(ws=4096, **kw):
    d = _lib.ChunkDesc(dtype=_lib.FADE_BF16, R=2, T=3, Hq=8, Hkv=2, D=64, page_size=16, n_pages=4, table_width=2,
                       table_stride=2, causal=1, window=0, sm_scale=0.125, q_st=512, q_sh=64, o_st=512, o_sh=64,
                       kp_sp=2048, kp_sh=1024, kp_st=64, vp_sp=2048, vp_sh=1024, vp_st=64)
    for name in ("q", "out", "k_pool", "v_pool", "block_table", "cu_q", "kv_lens"):
        setattr(d, name, 4096)
    for k, v in kw.items():
        setattr(d, k, v)
    lib = _lib.load()
    return lib.fade_chunk_attn(ctypes.byref(d), ws, 16, None), lib.fade_chunk_attn_workspace_size(ctypes.byref(d))


@pytest.mark.parametrize("change,status", [
    (dict(R=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(Hq=7), _lib.FADE_ERR_INVALID_ARG),
    (dict(Hkv=0), _lib.FADE_ERR_INVALID_ARG),
    (dict(window=-1), _lib.FADE_ERR_INVALID_ARG),
    (dict(sm_scale=0.0), _lib.FADE_ERR_INVALID_ARG),
    (dict(sm_scale=float("nan")), _lib.FADE_ERR_INVALID_ARG),
    (dict(sm_scale=float("inf")), _lib.FADE_ERR_INVALID_ARG),
    (dict(dtype=_lib.FADE_F32), _lib.FADE_ERR_UNSUPPORTED),
    (dict(D=96), _lib.FADE_ERR_UNSUPPORTED),
    (dict(page_size=8), _lib.FADE_ERR_UNSUPPORTED),
    (dict(page_size=256), _lib.FADE_ERR_UNSUPPORTED),
    (dict(Hq=258), _lib.FADE_ERR_UNSUPPORTED),
])
def test_chunk_entry_point_unsupported(change, status):
    assert _chunk(**change) == (status, 0)


@pytest.mark.parametrize("change,status", [
    (dict(q=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(cu_q=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(block_table=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(v_pool=None), _lib.FADE_ERR_INVALID_ARG),
    (dict(q=4098), _lib.FADE_ERR_ALIGN),
    (dict(vp_st=68), _lib.FADE_ERR_ALIGN),
    (dict(o_sh=4), _lib.FADE_ERR_ALIGN),
    (dict(ws=None), _lib.FADE_ERR_WORKSPACE),
    (dict(), _lib.FADE_ERR_WORKSPACE),          # 16 bytes are too few
    (dict(T=0), _lib.FADE_OK),
    (dict(R=0), _lib.FADE_OK),
])
def test_chunk_entry_point_refusals(change, status):
    got, need = _chunk(**change)
    assert got == status and need > 16


def test_cpu_tensors_are_refused():
    from fade_b200.paged import chunk_attention, plan_step, release_rows, rope_append, rope_axes

    i = torch.zeros(1, dtype=torch.int32)
    x, pool = torch.zeros(1, 1, 64, dtype=torch.float16), torch.zeros(1, 1, 16, 64, dtype=torch.float16)
    for call in (lambda: plan_step(i, i, i[None], i, i, 16, 1), lambda: release_rows(i.bool(), i, i[None], 16, i, i),
                 lambda: rope_axes(x, i, torch.zeros(32)),
                 lambda: rope_append(x, x, x, i, torch.zeros(32), None, i.long(), pool, pool),
                 lambda: chunk_attention(x, pool, pool, i[None], torch.zeros(2, dtype=torch.int32), i)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_section_axes():
    from fade_b200.paged import section_axes

    assert section_axes((2, 3, 1)) == [0, 0, 1, 1, 1, 2]
    assert section_axes((2, 2, 2), interleaved=True) == [0, 1, 2, 0, 1, 2]
    assert section_axes((4, 1, 1), interleaved=True) == [0, 1, 2, 0, 0, 0]
    assert section_axes((5,)) == [0] * 5 and section_axes(()) == []


def test_mrope_tables_of_several_axes():
    """One axis after the other or interleaved; equal axes give the text tables."""
    from types import SimpleNamespace

    from fade_b200.rope import MRope, extract_rope_scheme

    pos = torch.tensor([[0, 5, 9], [1, 2, 3], [7, 7, 8]])
    scheme = MRope(theta=1e4, head_dim=16, mrope_section=[2, 3, 3])
    cos, sin = scheme.compute_cos_sin(pos, "cpu", model_dtype=torch.float32)
    inv = scheme.inv_freq("cpu")
    for j, a in enumerate([0, 0, 1, 1, 1, 2, 2, 2]):
        angle = pos[a].float() * inv[j]
        for c in (j, j + 8):
            assert torch.equal(cos[0, 0, :, c], angle.cos()) and torch.equal(sin[0, 0, :, c], angle.sin())
    text = scheme.compute_cos_sin(pos[0], "cpu")
    same = scheme.compute_cos_sin(pos[:1].expand(3, 3), "cpu")
    assert torch.equal(text[0], same[0]) and torch.equal(text[1], same[1])
    inter = MRope(theta=1e4, head_dim=16, mrope_section=[2, 3, 3], interleaved=True)
    got = inter.compute_cos_sin(pos, "cpu", model_dtype=torch.float32)[0][0, 0, :, :8]
    for j, a in enumerate([0, 1, 2, 0, 1, 2, 0, 1]):
        assert torch.equal(got[:, j], (pos[a].float() * inv[j]).cos())
    with pytest.raises(ValueError, match="mrope_section"):
        scheme.compute_cos_sin(pos[:2], "cpu")
    cfg = SimpleNamespace(head_dim=16, rope_parameters={"rope_theta": 1e4, "mrope_section": [2, 3, 3],
                                                        "mrope_interleaved": True})
    assert extract_rope_scheme(cfg).interleaved and not MRope().interleaved


def test_packed_descriptors_have_the_structures_layout():
    for pack, desc in ((_lib.PACK_PLAN, _lib.PlanDesc), (_lib.PACK_ROPE, _lib.RopeDesc), (_lib.PACK_CHUNK, _lib.ChunkDesc)):
        assert pack.size == ctypes.sizeof(desc)
        values = [float(i) if kind is ctypes.c_double else i for i, (_, kind) in enumerate(desc._fields_, 1)]
        d = desc.from_buffer_copy(pack.pack(*values))
        assert [getattr(d, name) for name, _ in desc._fields_] == values
