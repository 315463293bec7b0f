"""LoomDecoder.beam_search beyond one search: captured steps of many eos and pad ids,
and histories that a defect would confuse."""
import json
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

GOLD = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _cfg(name, **kw):
    from loom_amd.config import ModelConfig
    with open(os.path.join(GOLD, "configs.json")) as f:
        d = json.load(f)[name]
    d.update(kw)
    return ModelConfig.from_dict(d)


def _tiny():
    z = np.load(os.path.join(GOLD, "tiny_decode.npz"))
    state = {k[3:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("w::")}
    return _cfg("tiny"), state, torch.from_numpy(z["prompt"])


def test_captured_steps_of_many_eos_and_pad_ids_are_bounded():
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny()
    eng = LoomDecoder(cfg, state, batch=9, dtype=torch.float32)
    ids = [(e, p) for p in (0, 1) for e in (None, 2, 3, 4)]
    first = {}
    for eos, pad in ids + ids[::-1] + ids[:3]:
        got = eng.beam_search(prompt, 6, 3, eos_id=eos, pad_id=pad, page_size=16)
        assert len(eng._beams._graphs) <= 4
        if (eos, pad) in first:
            assert all(torch.equal(a, b) for a, b in zip(got, first[eos, pad]))
        else:
            eager = eng.beam_search(prompt, 6, 3, eos_id=eos, pad_id=pad, page_size=16, use_graph=False)
            assert all(torch.equal(a, b) for a, b in zip(got, eager))
            first[eos, pad] = got
    kept = list(eng._beams._graphs)
    eng.beam_search(prompt, 6, 3, eos_id=kept[0][0] if kept[0][0] >= 0 else None, pad_id=kept[0][1], page_size=16)
    assert sorted(eng._beams._graphs) == sorted(kept) and list(eng._beams._graphs)[-1] == kept[0]
