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


@pytest.mark.parametrize("dt,chunked,page", [(torch.bfloat16, False, 16), (torch.bfloat16, True, 64), (torch.float32, False, 16)])
def test_hypotheses_run_alone_give_the_same_bits(dt, chunked, page):
    """The checkpoint's shape, over a fire of the document state: every hypothesis run
    by itself, in a row that never forks and holds pages of its own, gives the search's
    last logits to the bit (a row's sums do not depend on the rows beside it), and its
    log-probabilities sum up to the score.  A page or a state of another hypothesis
    anywhere would show."""
    from loom_amd.engine import LoomDecoder, _BeamState
    from loom_amd.weights import init_state_dict
    cfg = _cfg("nano_chk", seq_len=512)
    state = init_state_dict(cfg, 2)
    S, W, P, n = 2, 4, 125, 12
    prompt = torch.randint(0, cfg.V, (S, P), generator=torch.Generator().manual_seed(5))
    eng = LoomDecoder(cfg, state, batch=S * W, dtype=dt)
    ids, scores = eng.beam_search(prompt, n, W, chunked_prefill=chunked, page_size=page)
    logits, parent = eng.logits.clone(), eng._beams.parent.long()
    moved = eng._beams.cache.refs.max()
    assert int(moved) == W                                    # the prompt's pages are still shared

    rows = prompt.repeat_interleave(W, 0)
    hyp = ids.view(S * W, n)
    if chunked:
        eng.prefill(rows)
    else:
        eng.start(rows)
        eng.replay_steps(P - 1)
    bs = _BeamState(eng, W, page, None)
    kc = bs.cache
    kc.reset()
    kc.start(torch.ones(S * W, dtype=torch.bool, device=eng.dev))
    kc.update(n_new=P)
    full = torch.full((S * W,), P, dtype=torch.int32, device=eng.dev)
    kc.load(eng.k_cache, eng.v_cache, torch.zeros_like(full), full)
    kc.lens.copy_(full - 1)
    total = torch.zeros(S * W, dtype=torch.float64, device=eng.dev)
    for t in range(n):
        total += torch.log_softmax(eng.logits.double(), 1).gather(1, hyp[:, t:t + 1])[:, 0]
        if t == n - 1:
            break
        eng.ids.copy_(hyp[:, t])
        kc.update(n_new=1, advance=1)
        eng._launch_step(first=False, prompt_len=0, paged=bs)
    assert int(kc.refs.max()) == 1
    assert torch.equal(eng.logits, logits[parent])
    # a choice's error in its score (the value's rounding, 40 units of the sum's, and the
    # exponentials' arguments of up to 8), n times
    tol = n * (2.0 ** -24 * float(scores.abs().max()) + 40 * 2.0 ** -24 + 2.0 ** -22 * 8)
    assert float((scores.view(-1).double() - total).abs().max()) <= tol
    # and another hypothesis' history would: the rows are not alike
    for s in range(S):
        own = logits[parent][s * W:(s + 1) * W]
        hist = [tuple(h) for h in hyp[s * W:(s + 1) * W, :-1].tolist()]
        assert len(set(hist)) > 1
        for a in range(W):
            for b in range(a):
                assert torch.equal(own[a], own[b]) == (hist[a] == hist[b])
