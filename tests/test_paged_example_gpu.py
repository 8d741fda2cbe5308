"""The serving example: chunked prompts, decodes, release and the hand-over to INT4 tiers."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("paged_serving", ROOT / "examples" / "paged_serving.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_chunk_size_does_not_change_the_result(cuda_device):
    ex = _example()
    model = ex.TinyDecoder(n_layers=3)
    g = torch.Generator().manual_seed(2)
    prompts = []
    for shape in ((3, (5, 7), 9), (30, (2, 2), 1), (1, (1, 1), 60)):
        pos = ex.image_prompt_positions(*shape)
        prompts.append((torch.randint(0, 1000, (pos.shape[1],), generator=g), pos))
    cache, last, _ = ex.serve(model, prompts, 1000, 1)
    cache.check()
    assert cache.kv_lens.tolist() == [len(t) for t, _ in prompts]
    for chunk in (1, 13, 16):
        other, hidden, _ = ex.serve(model, prompts, chunk, 1)
        other.check()
        for a, b in zip(last, hidden):
            # the weights of a row are summed in other blocks: bf16 steps of a 3-layer residual stream
            assert float((a - b).abs().max()) <= 8 * 2.0 ** -8 * float(a.abs().max())
        for layer in range(model.L):
            for r, (t, _) in enumerate(prompts):
                n = len(t)
                k, v = cache.gather(layer, [r], n)
                k2, v2 = other.gather(layer, [r], n)
                assert float((k - k2).abs().max()) <= 8 * 2.0 ** -8 * float(k.abs().max())
                assert float((v - v2).abs().max()) <= 8 * 2.0 ** -8 * float(v.abs().max())


def test_example_runs(cuda_device, capsys):
    _example().main()
    text = capsys.readouterr().out
    assert "after releasing request 1" in text
    errs = [float(line.rsplit(" ", 1)[1]) for line in text.splitlines() if line.startswith("layer")]
    assert len(errs) == 2 and all(e < 0.2 for e in errs)          # 4-bit K and V
