"""Beam search on a paged key-value cache, as measurable cases.

Kinds (``case["kind"]``):
  step     one layer's attention of one new token per row over a paged cache: RoPE of the
           projection row [q | k | v], append of (k, v) to the row's page, both readouts
           C = A V and Kctx = A K over the row's own length
  update   the cache side of a beam step: every row takes its parent's pages, the pages that
           nobody holds any more become free, and the next token is made writable (a partly
           filled page that rows share is copied, a missing page is taken from the free ones),
           over the pools of all layers
  compact  the pages in use move to the lowest ids of the pool, and the tables follow
  select   the best continuations over beams and vocabulary
  reorder  the rows of the decoder's per-sequence states follow the selected parents

Heads and widths are those of the nano configurations (8 q heads of 96 over 2 kv heads, width 768,
hidden 4 times that, 10 layers, vocabularies of 4096 and 8192) and generic ones.  Plain forms are
elementary torch operations; with ``own`` set, ``run`` calls ``loom_amd.ops``.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _ops():
    """The framework's operators (only where ``own`` is true)."""
    pkg = os.path.join(os.getcwd(), "loomformer-paraplex_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from loom_amd import ops
    return ops


def listed():
    return [
        # one conversation, a few hundred tokens in: launches and latency
        dict(name="step_bf16_1x300", kind="step", dtype="bf16", B=1, T=300, ragged=False, idle=0, QH=8, KVH=2,
             HD=96, PS=16),
        # the decode workload at the middle of its generation: 32 sequences of one length
        dict(name="step_bf16_32x2176", kind="step", dtype="bf16", B=32, T=2176, ragged=False, idle=0, QH=8, KVH=2,
             HD=96, PS=64),
        # the fp32 reference configuration, a handful of rows of which one is idle, odd lengths
        dict(name="step_fp32_5x1001", kind="step", dtype="fp32", B=5, T=1001, ragged=True, idle=1, QH=8, KVH=2,
             HD=96, PS=16),
        # a serving batch of very different lengths, wide heads
        dict(name="step_bf16_64x16384", kind="step", dtype="bf16", B=64, T=16384, ragged=True, idle=2, QH=32,
             KVH=8, HD=128, PS=64),
        # one prompt searched with four beams: latency of the cache's bookkeeping
        dict(name="update_bf16_1x4x333", kind="update", dtype="bf16", S=1, W=4, T=333, L=10, KVH=2, HD=96, PS=16),
        # a serving batch: 32 prompts of eight beams each
        dict(name="update_bf16_32x8x4100", kind="update", dtype="bf16", S=32, W=8, T=4100, L=10, KVH=2, HD=96,
             PS=64),
        # a small fp32 pool in pieces
        dict(name="compact_fp32_151", kind="compact", dtype="fp32", NP=151, L=10, KVH=2, HD=96, PS=16, R=5),
        # a pool a third of whose pages are in use, after the rows of a large batch ended
        dict(name="compact_bf16_6000", kind="compact", dtype="bf16", NP=6000, L=10, KVH=2, HD=96, PS=64, R=32),
        # one prompt of the fp32 reference configuration, four beams of which one is at its end, eight continuations
        dict(name="select_fp32_1x4x8192", kind="select", dtype="fp32", S=1, W=4, V=8192, K=8, fin=1),
        # a large batch over a large vocabulary of an odd size
        dict(name="select_bf16_64x8x65537", kind="select", dtype="bf16", S=64, W=8, V=65537, K=8, fin=0),
        # the decoder's states of one prompt with four beams
        dict(name="reorder_bf16_4x512", kind="reorder", dtype="bf16", S=1, W=4, T=512, L=10, N=768),
        # and of 32 prompts with eight beams each
        dict(name="reorder_bf16_256x2304", kind="reorder", dtype="bf16", S=32, W=8, T=2304, L=10, N=768),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "update", "update", "compact", "select", "select", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "step":
        QH, KVH = rng.choice([(8, 2), (8, 2), (32, 8), (8, 8), (6, 2), (16, 2), (5, 1), (16, 1)])
        HD = rng.choice([96, 96, 64, 128])
        B = _log(rng, 1, 64)
        T = _log(rng, 1, min(16384, (3 << 26) // (B * KVH * HD * ESIZE[dtype])))       # K of a full batch: 192 MB
        return dict(kind=kind, dtype=dtype, B=B, T=T, ragged=rng.random() < 0.6, idle=min(B - 1, rng.choice([0, 0, 1, 3])),
                    QH=QH, KVH=KVH, HD=HD, PS=rng.choice([16, 32, 64, 128]))
    if kind == "update":
        W = rng.randint(2, 8)
        S = _log(rng, 1, 32)
        return dict(kind=kind, dtype=dtype, S=S, W=W, T=_log(rng, 1, 4100), L=rng.choice([1, 4, 10]), KVH=2,
                    HD=rng.choice([96, 64]), PS=rng.choice([16, 32, 64]))
    if kind == "compact":
        return dict(kind=kind, dtype=dtype, NP=_log(rng, 33, 3000), L=rng.choice([1, 4, 10]), KVH=2,
                    HD=rng.choice([96, 64]), PS=rng.choice([16, 32, 64]), R=rng.randint(1, 64))
    if kind == "select":
        W = rng.randint(1, 8)
        return dict(kind=kind, dtype=dtype, S=_log(rng, 1, 64), W=W, V=_log(rng, 100, 65537),
                    K=rng.choice([W, W, 2 * W]), fin=rng.choice([0, 0, 2]))
    return dict(kind=kind, dtype=dtype, S=_log(rng, 1, 32), W=rng.randint(2, 8), T=_log(rng, 128, 2304),
                L=rng.randint(1, 10), N=rng.choice([256, 512, 768]))


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(case):
    """Tokens each row holds before the new one (-1: an idle row), from the case alone."""
    B, top = case["B"], case["T"] - 1
    if case["ragged"] and B > 1:                     # spread over the logarithm of 1..T, mixed
        lens = [int(round((top + 1) ** (((7 * i) % B) / (B - 1)))) - 1 for i in range(B)]
    else:
        lens = [top] * B
    for i in range(case["idle"]):                    # idle rows between the others and at the end
        lens[B - 1 - 2 * i if B - 1 - 2 * i > 0 else 0] = -1
    return lens


def _prepare_step(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    B, QH, KVH, HD, PS = case["B"], case["QH"], case["KVH"], case["HD"], case["PS"]
    lens = _lengths(case)
    pages = [(n + PS) // PS if n >= 0 else 0 for n in lens]          # of len + 1 tokens
    MP = -(-case["T"] // PS)
    NP = sum(pages) + 3
    order = torch.randperm(NP, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, MP), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
    inv = 10000.0 ** (-torch.arange(0, HD, 2, device=DEV, dtype=torch.float64) / HD)
    ang = torch.arange(case["T"], device=DEV, dtype=torch.float64)[:, None] * torch.cat([inv, inv])[None]
    return dict(qkv=torch.randn(B, (QH + 2 * KVH) * HD, generator=g, device=DEV).to(dt),
                k_pages=torch.randn(NP, KVH, PS, HD, generator=g, device=DEV, dtype=dt),
                v_pages=torch.randn(NP, KVH, PS, HD, generator=g, device=DEV, dtype=dt),
                table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                cos=ang.cos().float(), sin=ang.sin().float())


def _prepare_update(case, seed):
    """Beams of S prompts: the first nine tenths of a prompt's pages are shared by its W rows, the
    rest are each row's own; half of the beams die at this step."""
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    S, W, T, PS, L = case["S"], case["W"], case["T"], case["PS"], case["L"]
    n = -(-T // PS)
    shared = (9 * n) // 10
    MP, R = n + 2, S * W
    used = S * shared + R * (n - shared)
    NP = used + R + 5
    order = torch.randperm(NP, generator=g, device=DEV)[:used].to(torch.int32)
    table = torch.full((S, W, MP), -1, dtype=torch.int32, device=DEV)
    table[:, :, :shared] = order[:S * shared].view(S, 1, shared)
    table[:, :, shared:n] = order[S * shared:].view(S, W, n - shared)
    table = table.view(R, MP).contiguous()
    refs = torch.zeros(NP, dtype=torch.int32, device=DEV)
    refs.scatter_add_(0, table[table >= 0].long(), torch.ones((), dtype=torch.int32, device=DEV).expand(int((table >= 0).sum())))
    pools = [torch.randn(L, NP, case["KVH"], PS, case["HD"], generator=g, device=DEV, dtype=dt) for _ in range(2)]
    return dict(k_pages=pools[0], v_pages=pools[1], table=table, refs=refs,
                lens=torch.full((R,), T, dtype=torch.int32, device=DEV),
                status=torch.zeros(1, dtype=torch.int32, device=DEV), parent=_parents(S, W, g))


def _parents(S, W, g):
    """Parent of each of S * W rows: W - W // 2 beams of each group live on (an odd one in three of
    the groups moves to another place), the others take the place of dead ones."""
    order = torch.rand(S, W, generator=g, device=DEV).argsort(1)
    live = W - W // 2
    par = torch.empty(S, W, dtype=torch.int64, device=DEV)
    par.scatter_(1, order[:, :live], order[:, :live])
    if W > 1:
        pick = torch.randint(0, live, (S, W // 2), generator=g, device=DEV)
        par.scatter_(1, order[:, live:], order.gather(1, pick))
    return (par + W * torch.arange(S, device=DEV)[:, None]).view(-1).to(torch.int32)


def _prepare_compact(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    NP, R, PS, L = case["NP"], case["R"], case["PS"], case["L"]
    used = NP // 3
    order = torch.randperm(NP, generator=g, device=DEV)[:used].to(torch.int32)
    MP = -(-used // R)
    table = torch.full((R * MP,), -1, dtype=torch.int32, device=DEV)
    table[:used] = order
    refs = torch.zeros(NP, dtype=torch.int32, device=DEV)
    refs[order.long()] = 1
    pools = [torch.randn(L, NP, case["KVH"], PS, case["HD"], generator=g, device=DEV, dtype=dt) for _ in range(2)]
    table = table.view(R, MP)
    return dict(k_pages=pools[0], v_pages=pools[1], table=table.clone(), refs=refs.clone(), table0=table, refs0=refs,
                used=torch.zeros(1, dtype=torch.int32, device=DEV))


def _prepare_select(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    S, W, V = case["S"], case["W"], case["V"]
    finished = torch.zeros(S * W, dtype=torch.bool, device=DEV)
    if W > 1:
        finished[torch.arange(case["fin"], device=DEV) * 3 % (S * W)] = True
    return dict(logits=(torch.randn(S * W, V, generator=g, device=DEV) * 3).to(dt),
                scores=-20 - 5 * torch.rand(S, W, generator=g, device=DEV), finished=finished)


def _prepare_reorder(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    S, W, N, L, T = case["S"], case["W"], case["N"], case["L"], case["T"]
    R, H, keys = S * W, 4 * case["N"], T // 128 + 1
    r = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=dt)  # noqa: E731
    return dict(tensors=[r(L, R, H), r(R, H, 3, 3), r(R, keys, N), r(R, keys, N),
                         torch.randint(0, 2, (R, keys), generator=g, device=DEV, dtype=torch.uint8),
                         torch.randint(0, 4096, (R, T), generator=g, device=DEV, dtype=torch.int64)],
                dims=[1, 0, 0, 0, 0, 0], parent=_parents(S, W, g))


def prepare(case, seed):
    make = dict(step=_prepare_step, update=_prepare_update, compact=_prepare_compact, select=_prepare_select,
                reorder=_prepare_reorder)[case["kind"]]
    return dict(case, **make(case, seed))


# ------------------------------------------------------------------ plain forms

def _rotate(x):
    a, b = x.chunk(2, -1)
    return torch.cat([-b, a], -1)


def _step_plain(s):
    B, QH, KVH, HD, PS = s["B"], s["QH"], s["KVH"], s["HD"], s["PS"]
    dt, G = s["qkv"].dtype, s["QH"] // s["KVH"]
    live = s["lens"] >= 0
    pos = s["lens"].clamp(min=0).long()
    x = s["qkv"].float().view(B, QH + 2 * KVH, HD)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = x[:, :QH + KVH] * cos + _rotate(x[:, :QH + KVH]) * sin
    qk = torch.where(live[:, None, None], qk, 0.0).to(dt)
    q, k, v = qk[:, :QH], qk[:, QH:], x[:, QH + KVH:].to(dt)
    rows = live.nonzero().view(-1)
    page = s["table"][rows, pos[rows] // PS].long()
    s["k_pages"][page, :, pos[rows] % PS] = k[rows]
    s["v_pages"][page, :, pos[rows] % PS] = v[rows]
    at = s["table"].clamp(min=0).long()
    kk = s["k_pages"][at].transpose(1, 2).reshape(B, KVH, -1, HD).float()
    vv = s["v_pages"][at].transpose(1, 2).reshape(B, KVH, -1, HD).float()
    sc = torch.matmul(q.float().view(B, KVH, G, HD), kk.transpose(2, 3)) / math.sqrt(HD)
    seen = (torch.arange(kk.shape[2], device=DEV)[None] <= pos[:, None]) & live[:, None]
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    w = torch.where(seen[:, None, None], torch.exp(sc - sc.amax(-1, keepdim=True)), 0.0)
    w = w / torch.where(live[:, None, None, None], w.sum(-1, keepdim=True), 1.0)
    c, kctx = torch.matmul(w, vv), torch.matmul(w, kk)
    return dict(c=c.view(B, QH, HD).to(dt), kctx=kctx.view(B, QH, HD).to(dt), q=q, k_pages=s["k_pages"],
                v_pages=s["v_pages"])


def _update_plain(s):
    table, refs, lens, par = s["table"], s["refs"], s["lens"], s["parent"].long()
    R, MP = table.shape
    PS, NP = s["PS"], refs.numel()
    rows = torch.arange(R, device=DEV)
    plen = lens[par]
    keep = torch.arange(MP, device=DEV)[None] < ((plen + PS - 1) // PS)[:, None]
    new = torch.where((par == rows)[:, None], table, torch.where(keep, table[par], -1))
    count = torch.bincount(new.view(-1).long() + 1, minlength=NP + 1)[1:]
    slot = (plen // PS).long()
    page = new.gather(1, slot[:, None]).view(-1).long()
    tail = plen % PS > 0
    same = (page[:, None] == page[None]) & tail[:, None] & tail[None]
    before = torch.tril(same, -1).sum(1)
    copy = tail & (count[page.clamp(min=0)] - before > 1)
    want = copy | (~tail & (page < 0))
    free = torch.argsort((count != 0).to(torch.uint8), stable=True)
    got = torch.where(want, free[(want.cumsum(0) - 1).clamp(min=0)], page)
    new.scatter_(1, slot[:, None], got[:, None].to(new.dtype))
    src, dst = page[copy], got[copy]
    held = (torch.arange(PS, device=DEV)[None] < (plen % PS)[copy][:, None])[None, :, None, :, None]
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, dst] = torch.where(held, pool[:, src], pool[:, dst])
    table.copy_(new)
    lens.copy_(plen)
    refs.copy_(torch.bincount(new.view(-1).long() + 1, minlength=NP + 1)[1:])
    return dict(table=table, lens=lens, refs=refs, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _compact_plain(s):
    table, refs = s["table"], s["refs"]
    NP = refs.numel()
    ids = torch.arange(NP, device=DEV)
    inuse = refs > 0
    U = inuse.sum()
    moves, holes = inuse & (ids >= U), ~inuse & (ids < U)
    src = torch.argsort((~moves).to(torch.uint8), stable=True)      # the pages that move, in order, first
    dst = torch.argsort((~holes).to(torch.uint8), stable=True)      # and the free places below U
    count = int(moves.sum())
    src, dst = src[:count], dst[:count]
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, dst] = pool[:, src]
    where = ids.clone()
    where[src] = dst
    table.copy_(torch.where(table >= 0, where[table.clamp(min=0).long()].to(table.dtype), table))
    held = refs[src]
    refs[src] = 0
    refs[dst] = held
    s["used"].copy_(U)
    return dict(table=table, refs=refs, used=s["used"], k_pages=s["k_pages"], v_pages=s["v_pages"])


EOS, PAD = 2, 1


def _select_plain(s):
    S, W, V, K = s["S"], s["W"], s["V"], s["K"]
    x = s["logits"].double()                       # candidates of two beams may be close together
    m = x.amax(1, keepdim=True)
    value = x - (m + torch.exp(x - m).sum(1, keepdim=True).log()) + s["scores"].view(-1, 1).double()
    only = torch.full_like(value, -math.inf)
    only[:, PAD] = s["scores"].view(-1).double()
    value = torch.where(s["finished"][:, None], only, value)
    best, at = torch.sort(value.view(S, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    none = torch.isinf(best)
    first = W * torch.arange(S, device=DEV)[:, None]
    parent = torch.where(none, first, first + at // V)
    token = torch.where(none, PAD, at % V)
    return dict(scores=best.float(), parent=parent.to(torch.int32), token=token,
                finished=~none & (s["finished"][parent] | (token == EOS)))


def _reorder_plain(s):
    at = s["parent"].long()
    return [t.copy_(t.index_select(d, at)) for t, d in zip(s["tensors"], s["dims"])]


def run(state):
    s, kind = state, state["kind"]
    if kind == "step":
        if own:
            c, kctx, q = _ops().paged_decode_step(s["qkv"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cos"], s["sin"])
            return dict(c=c, kctx=kctx, q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
        return _step_plain(s)
    if kind == "update":
        if own:
            _ops().paged_update(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["refs"], s["status"], parent=s["parent"], n_new=1)
            return dict(table=s["table"], lens=s["lens"], refs=s["refs"], k_pages=s["k_pages"], v_pages=s["v_pages"])
        return _update_plain(s)
    if kind == "compact":
        # the fragmented state again, so that every pass has the same pages to move
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        if own:
            _ops().paged_compact(s["k_pages"], s["v_pages"], s["table"], s["refs"], s["used"])
            return dict(table=s["table"], refs=s["refs"], used=s["used"], k_pages=s["k_pages"], v_pages=s["v_pages"])
        return _compact_plain(s)
    if kind == "select":
        if own:
            scores, parent, token, finished = _ops().beam_select(s["logits"], s["scores"], s["K"], finished=s["finished"], eos_id=EOS, pad_id=PAD)
            return dict(scores=scores, parent=parent, token=token, finished=finished)
        return _select_plain(s)
    if own:
        _ops().reorder_rows(s["tensors"], s["parent"], s["dims"])
        return list(s["tensors"])
    return _reorder_plain(s)


# ------------------------------------------------------------------ work and exact values

def work(case):
    kind, e = case["kind"], ESIZE[case["dtype"]]
    if kind == "step":
        B, QH, KVH, HD = case["B"], case["QH"], case["KVH"], case["HD"]
        lens = [n for n in _lengths(case) if n >= 0]
        row = 2 * KVH * HD * e                                   # K and V of one token
        pages = sum((n + case["PS"]) // case["PS"] for n in lens)
        rows = len(lens) * ((QH + 2 * KVH) * HD * e + row + 2 * HD * 4) + 3 * B * QH * HD * e
        return dict(bytes=sum(lens) * row + rows + 4 * (pages + B), flops=sum(6 * QH * HD * (n + 1) for n in lens))
    if kind == "update":
        S, W, T, PS = case["S"], case["W"], case["T"], case["PS"]
        dead, n = S * (W // 2), -(-T // PS)
        new = S * W if T % PS == 0 else dead
        copied = 0 if T % PS == 0 else dead * (T % PS) * case["L"] * 2 * case["KVH"] * case["HD"] * e
        return dict(bytes=2 * copied + dead * (2 * n * 4 + 16) + 12 * new + 12 * S * W, flops=0)
    if kind == "compact":
        NP, used = case["NP"], case["NP"] // 3
        moved = used * (NP - used) // NP                         # of a random third of the pages
        return dict(bytes=2 * moved * case["L"] * 2 * case["KVH"] * case["PS"] * case["HD"] * e + 4 * NP + 8 * used, flops=0)
    if kind == "select":
        rows, V = case["S"] * case["W"], case["V"]
        return dict(bytes=(rows - (case["fin"] if case["W"] > 1 else 0)) * V * e + rows * 5 + case["S"] * case["K"] * 17, flops=3 * rows * V)
    R, N, keys = case["S"] * case["W"], case["N"], case["T"] // 128 + 1
    row = (case["L"] * 4 * N + 36 * N + 2 * keys * N) * e + keys + 8 * case["T"]
    return dict(bytes=2 * row * case["S"] * (case["W"] // 2) + 4 * R, flops=0)


def _exact_step(s):
    B, QH, KVH, HD, PS = s["B"], s["QH"], s["KVH"], s["HD"], s["PS"]
    dt, half = s["qkv"].dtype, s["HD"] // 2
    G = QH // KVH
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    c, kctx, qo = (torch.zeros(B, QH, HD, dtype=torch.float64, device=DEV) for _ in range(3))
    for b, n in enumerate(_lengths(s)):
        if n < 0:
            continue
        x = s["qkv"][b].double().view(QH + 2 * KVH, HD)
        co, si = s["cos"][n].double(), s["sin"][n].double()
        turned = torch.empty_like(x)
        turned[:, :half] = x[:, :half] * co[:half] - x[:, half:] * si[:half]
        turned[:, half:] = x[:, half:] * co[half:] + x[:, :half] * si[half:]
        turned = turned.to(dt).double()
        qo[b] = turned[:QH]
        last = int(s["table"][b, n // PS])
        kp[last, :, n % PS] = turned[QH:QH + KVH]
        vp[last, :, n % PS] = x[QH + KVH:]
        ids = s["table"][b, :n // PS + 1].long()
        for j in range(KVH):
            k, v = kp[ids, j].reshape(-1, HD)[:n + 1], vp[ids, j].reshape(-1, HD)[:n + 1]
            a = torch.softmax(qo[b, j * G:(j + 1) * G] @ k.t() * HD ** -0.5, 1)
            c[b, j * G:(j + 1) * G], kctx[b, j * G:(j + 1) * G] = a @ v, a @ k
    return dict(c=c, kctx=kctx, q=qo, k_pages=kp, v_pages=vp)


def _exact_update(s):
    PS, T = s["PS"], s["T"]
    old, parent = s["table"].tolist(), s["parent"].tolist()
    have = -(-T // PS)
    rows = [list(old[p][:have]) + [-1] * (len(old[r]) - have) if p != r else list(old[r]) for r, p in enumerate(parent)]
    refs = [0] * s["refs"].numel()
    for row in rows:
        for p in row:
            if p >= 0:
                refs[p] += 1
    free = [p for p, n in enumerate(refs) if n == 0]
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    for row in rows:
        p = row[T // PS]
        if T % PS and refs[p] > 1:
            q = free.pop(0)
            for pool in pools:
                pool[:, q, :, :T % PS] = pool[:, p, :, :T % PS]
            refs[p] -= 1
        elif T % PS == 0 and p < 0:
            q = free.pop(0)
        else:
            continue
        refs[q] = 1
        row[T // PS] = q
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(table=i32(rows), lens=i32([T] * len(rows)), refs=i32(refs), k_pages=pools[0], v_pages=pools[1])


def _exact_compact(s):
    refs = s["refs0"].tolist()
    U = sum(n > 0 for n in refs)
    holes = [p for p in range(U) if refs[p] == 0]
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    went = {}
    for p in range(U, len(refs)):
        if refs[p]:
            went[p] = holes.pop(0)
            refs[went[p]], refs[p] = refs[p], 0
    if went:
        a, b = torch.tensor(list(went), device=DEV), torch.tensor(list(went.values()), device=DEV)
        for pool in pools:
            pool[:, b] = pool[:, a]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(table=i32([[went.get(p, p) for p in row] for row in s["table0"].tolist()]), refs=i32(refs), used=i32([U]),
                k_pages=pools[0], v_pages=pools[1])


def _exact_select(s):
    S, W, V, K = s["S"], s["W"], s["V"], s["K"]
    x = s["logits"].double()
    logp = torch.log_softmax(x, 1)
    out = dict(scores=[], parent=[], token=[], finished=[])
    for i in range(S):
        found = []
        for r in range(i * W, (i + 1) * W):
            base = float(s["scores"].view(-1)[r])
            if bool(s["finished"][r]):
                found.append((-base, r, PAD))
                continue
            least = torch.topk(x[r], min(K, V)).values[-1]          # with every tie of the last one
            at = (x[r] >= least).nonzero().view(-1)
            found += [(-(base + p), r, t) for p, t in zip(logp[r, at].tolist(), at.tolist())]
        found = sorted(found)[:K]
        found += [(math.inf, i * W, PAD)] * (K - len(found))
        out["scores"].append([-v for v, _, _ in found])
        out["parent"].append([r for _, r, _ in found])
        out["token"].append([t for _, _, t in found])
        out["finished"].append([v < math.inf and (bool(s["finished"][r]) or t == EOS) for v, r, t in found])
    return dict(scores=torch.tensor(out["scores"], dtype=torch.float64, device=DEV),
                parent=torch.tensor(out["parent"], dtype=torch.int32, device=DEV),
                token=torch.tensor(out["token"], device=DEV), finished=torch.tensor(out["finished"], device=DEV))


def _exact_reorder(s):
    outs = []
    for t, d in zip(s["tensors"], s["dims"]):
        o = t.double() if t.is_floating_point() else t.clone()
        for r, p in enumerate(s["parent"].tolist()):
            o.select(d, r).copy_(t.select(d, p))
        outs.append(o)
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    return dict(step=_exact_step, update=_exact_update, compact=_exact_compact, select=_exact_select,
                reorder=_exact_reorder)[case["kind"]](s)
