"""LoomDecoder.beam_search against a beam search that recomputes every hypothesis from
its first token with the dense engine (fp32), and its own invariants."""
import json
import math
import os

import numpy as np
import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu

# How far two candidates must lie apart for the two searches to choose alike.  They
# differ in the order of the attention's fp32 sums alone: over at most 32 positions
# that is 32 * 2^-24 = 2e-6 of values of size one per block, three blocks with a
# LayerNorm after each, and the same again in the other direction.
APART = 2e-5

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


def _tiny(variants=False):
    z = np.load(os.path.join(GOLD, "variants_decode.npz" if variants else "tiny_decode.npz"))
    state = {k[3:]: torch.from_numpy(z[k]) for k in z.files if k.startswith("w::")}
    return _cfg("tiny_variants" if variants else "tiny"), state, torch.from_numpy(z["prompt"])


def _recomputed(cfg, state, prompt, n_new, W, eos=-1, pad=0, carry=None):
    """Every step runs all hypotheses from scratch, token by token, and chooses with
    the plain selection."""
    from loom_amd.engine import LoomDecoder
    S, P = prompt.shape
    eng = LoomDecoder(cfg, state, batch=S * W, dtype=torch.float32, carry_token_id=carry)
    seqs = prompt.repeat_interleave(W, 0)
    scores = torch.full((S, W), -math.inf)
    scores[:, 0] = 0
    fin = torch.zeros(S * W, dtype=torch.bool)
    gap = math.inf
    for _ in range(n_new):
        for pos in range(seqs.shape[1]):
            logits = eng.step(seqs[:, pos], pos)
        more, _, _, _ = ref.beam_select(logits, scores, W + 1, fin, eos, pad)
        d = (more[:, :-1] - more[:, 1:])
        gap = min(gap, float(d[torch.isfinite(d)].min()))
        sc, par, tok, fin = ref.beam_select(logits, scores, W, fin, eos, pad)
        scores, fin = sc.float(), fin.view(-1)
        seqs = torch.cat([seqs[par.view(-1).long()], tok.view(-1, 1)], 1)
    return seqs[:, P:].view(S, W, n_new), scores, gap


@pytest.mark.parametrize("W,page,chunked,carry,variants", [(1, 16, False, None, False), (3, 16, False, None, False),
                                                           (4, 32, True, None, False), (3, 16, True, 5, False),
                                                           (2, 64, False, 5, False), (3, 16, False, None, True)])
def test_beams_equal_recomputed_hypotheses(W, page, chunked, carry, variants):
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny(variants)
    n_new = 9
    want, want_scores, gap = _recomputed(cfg, state, prompt, n_new, W, carry=carry)
    assert gap > APART, f"the case decides nothing: candidates {gap} apart"
    eng = LoomDecoder(cfg, state, batch=3 * W, dtype=torch.float32, carry_token_id=carry)
    ids, scores = eng.beam_search(prompt, n_new, W, chunked_prefill=chunked, page_size=page)
    assert torch.equal(ids.cpu(), want)
    assert ((scores.cpu() - want_scores).abs() <= n_new * APART).all()       # a log-probability per token


def test_beams_that_end():
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny()
    eng = LoomDecoder(cfg, state, batch=9, dtype=torch.float32)
    free, _ = eng.beam_search(prompt, 8, 3, page_size=16)
    eos = int(free[0, 0, 2])                                  # a token that the first prompt's best beam chooses
    want, want_scores, gap = _recomputed(cfg, state, prompt, 8, 3, eos=eos, pad=1)
    assert gap > APART
    ids, scores = eng.beam_search(prompt, 8, 3, eos_id=eos, pad_id=1, page_size=16)
    assert torch.equal(ids.cpu(), want)
    assert ((scores.cpu() - want_scores).abs() <= 8 * APART).all()
    ended = [(s, w) for s in range(3) for w in range(3) if eos in ids[s, w, :-1].tolist()]
    assert ended
    for s, w in ended:
        at = ids[s, w].tolist().index(eos)
        assert all(t == 1 for t in ids[s, w, at + 1:].tolist())


def test_one_beam_is_greedy_and_searches_repeat():
    """beams = 1 equals generate; a search after another one, other prompts and
    a greedy generation in between gives the same answer; eager equals captured."""
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny()
    eng = LoomDecoder(cfg, state, batch=3, dtype=torch.float32)
    greedy = eng.generate(prompt, 12)
    ids, _ = eng.beam_search(prompt, 12, 1, page_size=16)
    assert torch.equal(ids[:, 0], greedy)
    a = eng.beam_search(prompt[:1], 12, 3, page_size=16)
    eng.beam_search(prompt[1:2], 5, 3, page_size=16)
    assert torch.equal(eng.generate(prompt, 12), greedy)
    for kw in ({}, {"use_graph": False}, {"n_pages": 7}):
        b = eng.beam_search(prompt[:1], 12, 3, page_size=16, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), kw
    eng.free_beam_buffers()
    b = eng.beam_search(prompt[:1], 12, 3, page_size=16)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with pytest.raises(ValueError, match="exceeded"):
        eng.step(ids[:, 0, -1], eng.pos)                      # nothing to continue from


def test_nano_bf16_graph_equals_eager_and_scores_are_the_sums():
    """The checkpoint's shape in bf16: captured and eager searches agree to the bit, and
    a beam's score is the sum of the log-probabilities that the dense engine gives its
    tokens, within the bf16 logits' distance of two orders of rounding."""
    from loom_amd.engine import LoomDecoder
    from loom_amd.weights import init_state_dict
    cfg = _cfg("nano_chk", seq_len=512)
    state = init_state_dict(cfg, 2)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, cfg.V, (2, 125), generator=g)   # the continuation passes the fire at 128
    eng = LoomDecoder(cfg, state, batch=8, dtype=torch.bfloat16)
    ids, scores = eng.beam_search(prompt, 10, 4, page_size=16)
    ids2, scores2 = eng.beam_search(prompt, 10, 4, page_size=16, use_graph=False)
    assert torch.equal(ids, ids2) and torch.equal(scores, scores2)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    assert len({tuple(r) for r in ids.view(8, 10).tolist()}) == 8
    seq = torch.cat([prompt.repeat_interleave(4, 0), ids.view(8, 10).cpu()], 1)
    total = torch.zeros(8, dtype=torch.float64)
    for pos in range(seq.shape[1] - 1):
        logits = eng.step(seq[:, pos], pos)
        if pos >= 124:
            total += torch.log_softmax(logits.double().cpu(), 1).gather(1, seq[:, pos + 1:pos + 2])[:, 0]
    # the two attentions differ in their rounding of 10 tokens' logits: bf16 steps of logits of up to 4 in size
    assert ((scores.view(-1).cpu().double() - total).abs() <= 10 * 4 * 2.0 ** -7).all()


def test_beam_search_refuses():
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny()
    eng = LoomDecoder(cfg, state, batch=6, dtype=torch.float32)
    for args, kw, msg in [((prompt, 4, 3), {}, "engine batch"), ((prompt, 4, 0), {}, "engine batch"),
                          ((prompt[:2], 0, 3), {}, "at least one token"), ((prompt[:2, :0], 4, 3), {}, "at least one token"),
                          ((prompt[:2], 4, 3), dict(eos_id=cfg.V), "eos_id"), ((prompt[:2], 4, 3), dict(pad_id=-1), "pad_id"),
                          ((prompt[:2], 10 ** 6, 3), {}, "exceeded"), ((prompt[:2], 4, 3), dict(page_size=24), "power of two"),
                          ((prompt[:2], 4, 3), dict(n_pages=0), "n_pages"), ((prompt[:2] + cfg.V, 4, 3), {}, "token ids")]:
        with pytest.raises(ValueError, match=msg):
            eng.beam_search(*args, **kw)
    with pytest.raises(RuntimeError, match="pages could not be had"):
        eng.beam_search(prompt[:2], 4, 3, page_size=16, n_pages=3)
    ids, _ = eng.beam_search(prompt[:2], 4, 3, page_size=16)  # and works again
    assert ids.shape == (2, 3, 4)
