"""Beam search whose attention reads the beams' common pages once, against hypotheses
recomputed with the dense engine, and its own invariants."""
import pytest
import torch

from test_gpu_beam_search import APART, _cfg, _recomputed, _tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.mark.parametrize("W,page,variants", [(4, 16, False), (3, 32, True)])
def test_beams_equal_recomputed_hypotheses(W, page, variants):
    """A prompt of more than the positions from which reading once pays."""
    from loom_amd.engine import LoomDecoder
    _, state, _ = _tiny(variants)
    cfg = _cfg("tiny_variants" if variants else "tiny", seq_len=256)
    g = torch.Generator().manual_seed(3)
    prompt, n_new = torch.randint(0, cfg.V, (2, 101), generator=g), 6
    want, want_scores, gap = _recomputed(cfg, state, prompt, n_new, W)
    # (as there, over up to 107 positions instead of 32)
    apart = APART * 107 / 32
    assert gap > apart, f"the case decides nothing: candidates {gap} apart"
    eng = LoomDecoder(cfg, state, batch=2 * W, dtype=torch.float32)
    ids, scores = eng.beam_search(prompt, n_new, W, page_size=page, shared_reads=True)
    assert eng._beams.shared.tolist() == [101 // page * page] * (2 * W)
    assert torch.equal(ids.cpu(), want)
    assert ((scores.cpu() - want_scores).abs() <= n_new * apart).all()


def test_nano_bf16_graph_equals_eager_and_searches_of_both_kinds_alternate():
    from loom_amd.engine import LoomDecoder
    from loom_amd.weights import init_state_dict
    cfg = _cfg("nano_chk", seq_len=512)
    state = init_state_dict(cfg, 2)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, cfg.V, (2, 125), generator=g)
    eng = LoomDecoder(cfg, state, batch=8, dtype=torch.bfloat16)
    ids, scores = eng.beam_search(prompt, 10, 4, page_size=16, shared_reads=True)
    plain, plain_scores = eng.beam_search(prompt, 10, 4, page_size=16)
    for kw in ({}, {"use_graph": False}):
        ids2, scores2 = eng.beam_search(prompt, 10, 4, page_size=16, shared_reads=True, **kw)
        assert torch.equal(ids, ids2) and torch.equal(scores, scores2)
    again, again_scores = eng.beam_search(prompt, 10, 4, page_size=16)
    assert torch.equal(plain, again) and torch.equal(plain_scores, again_scores)
    assert len({tuple(r) for r in ids.view(8, 10).tolist()}) == 8
    # the two attentions differ in their rounding of 10 tokens' logits: bf16 steps of logits of up to 4 in size
    assert ((scores[:, 0] - plain_scores[:, 0]).abs() <= 10 * 4 * 2.0 ** -7).all()


def test_pages_that_run_out_raise():
    from loom_amd.engine import LoomDecoder
    cfg, state, prompt = _tiny()
    eng = LoomDecoder(cfg, state, batch=6, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="pages could not be had"):
        eng.beam_search(prompt[:2], 4, 3, page_size=16, n_pages=3, shared_reads=True)
    ids, _ = eng.beam_search(prompt[:2], 4, 3, page_size=16, shared_reads=True)   # and works again
    assert ids.shape == (2, 3, 4)
