"""A serving step over a paged key-value cache whose rows share prefixes, as measurable cases.

A batch has a request per row: lens[r] tokens of it are in the cache, new[r] more come in this
step (1: a token that was just chosen, more: a prompt or a piece of one, 0: none).  The new tokens
of all rows lie one behind the other in one flat batch of n_tokens, whose end may be padding.

Kinds (``case["kind"]``):
  plan    block tables and slot maps from the requests' lengths: pages for every row's new tokens
          (missing pages are taken from the free ones, a partly filled page that others hold is
          copied for its writer), then of every flat token its row, its position and its slot in
          the pools
  attend  the attention of a step's new tokens in L layers: the plan of the step once, then per
          layer RoPE of the projection rows [q | k | v], (k, v) into their slots, and both readouts
          C = A V and Kctx = A K of every token over its row up to the token itself.  The pages
          that rows of a batch have in common are read once for all of them

Heads and widths are those of the nano configurations (8 q heads of 96 over 2 kv heads, 10 layers)
and generic ones.  Plain forms are elementary torch operations; with ``own`` set, ``run`` calls
``loom_amd.ops``.
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


# A case has S groups of W rows.  The rows of a group have their first P tokens in common; each holds
# up to `held` further ones (spread over the logarithm where `ragged`), and brings tokens by `tokens`:
#   "one"     one each: a decode step
#   "prompt"  up to `new` each (spread over the logarithm where `ragged`): prompts, or pieces of them
#   "mixed"   one each, but every eighth row up to `new`: prompts that join a running batch
# `idle` rows hold no sequence; `pad` flat tokens behind the last are padding.

def listed():
    nano = dict(QH=8, KVH=2, HD=96)
    wide = dict(QH=32, KVH=8, HD=128)
    return [
        # four continuations of one prompt, a few tokens in: launches and latency
        dict(name="attend_bf16_1x4x333", kind="attend", dtype="bf16", S=1, W=4, P=333, held=20, new=1, tokens="one",
             ragged=True, idle=0, pad=0, PS=16, L=1, **nano),
        # eight prompts of 2048 tokens with four continuations each, two layers
        dict(name="attend_bf16_8x4x2048", kind="attend", dtype="bf16", S=8, W=4, P=2048, held=128, new=1, tokens="one",
             ragged=False, idle=0, pad=0, PS=64, L=2, **nano),
        # a serving batch behind one long instruction, answers of very different lengths, wide heads
        dict(name="attend_bf16_1x64x16384", kind="attend", dtype="bf16", S=1, W=64, P=16384, held=1024, new=1, tokens="one",
             ragged=True, idle=2, pad=0, PS=64, L=1, **wide),
        # the fp32 reference configuration, a handful of rows of which one is idle, odd lengths
        dict(name="attend_fp32_1x5x1001", kind="attend", dtype="fp32", S=1, W=5, P=1001, held=300, new=1, tokens="one",
             ragged=True, idle=1, pad=3, PS=16, L=1, **nano),
        # the chunked prefill's chunk: 32 rows of 128 tokens behind 1920 of their own
        dict(name="attend_bf16_32x128", kind="attend", dtype="bf16", S=32, W=1, P=0, held=1920, new=128, tokens="prompt",
             ragged=False, idle=0, pad=0, PS=64, L=1, **nano),
        # questions of different lengths behind one instruction, wide heads
        dict(name="attend_bf16_1x16x2048", kind="attend", dtype="bf16", S=1, W=16, P=1024, held=0, new=2048, tokens="prompt",
             ragged=True, idle=0, pad=37, PS=64, L=1, **wide),
        # three fp32 prompts of odd lengths into an empty cache
        dict(name="attend_fp32_3x257", kind="attend", dtype="fp32", S=3, W=1, P=0, held=0, new=257, tokens="prompt",
             ragged=True, idle=0, pad=1, PS=16, L=1, **nano),
        # a running batch of four instructions that prompts join, half, two layers
        dict(name="attend_fp16_4x12x1500", kind="attend", dtype="fp16", S=4, W=12, P=1500, held=200, new=300, tokens="mixed",
             ragged=True, idle=1, pad=16, QH=16, KVH=2, HD=64, PS=32, L=2),
        # four continuations begin from one prompt whose last page is partly filled
        dict(name="plan_bf16_1x4x333", kind="plan", dtype="bf16", S=1, W=4, P=333, held=0, new=1, tokens="one",
             ragged=False, idle=0, pad=0, PS=16, L=2, **nano),
        # 64 prompts of different lengths are admitted to an empty cache
        dict(name="plan_bf16_64x2048", kind="plan", dtype="bf16", S=64, W=1, P=0, held=0, new=2048, tokens="prompt",
             ragged=True, idle=3, pad=100, PS=16, L=2, **nano),
        # a large running batch that long prompts join
        dict(name="plan_bf16_32x8x4100", kind="plan", dtype="bf16", S=32, W=8, P=4100, held=500, new=2048, tokens="mixed",
             ragged=True, idle=5, pad=64, PS=64, L=2, **nano),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        kind = rng.choice(["attend", "attend", "attend", "plan"])
        QH, KVH = rng.choice([(8, 2), (8, 2), (32, 8), (8, 8), (6, 2), (16, 2), (5, 1), (16, 1)])
        tokens = rng.choice(["one", "one", "prompt", "mixed"])
        W = _log(rng, 1, 64)
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"]), S=_log(rng, 1, 64 // W), W=W,
                    P=rng.choice([0, 1, 1, 1]) * _log(rng, 1, 16384), held=rng.choice([0, 1, 1]) * _log(rng, 1, 2048),
                    new=1 if tokens == "one" else _log(rng, 1, 2048), tokens=tokens, ragged=rng.random() < 0.7,
                    idle=rng.choice([0, 0, 1, 3]), pad=rng.choice([0, 0, 1, 50]), QH=QH, KVH=KVH,
                    HD=rng.choice([96, 96, 64, 128]), PS=rng.choice([16, 32, 64, 128]), L=rng.choice([1, 1, 2]))
        case["idle"] = min(case["idle"], case["S"] * W - 1)
        w = work(case)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return case


# ------------------------------------------------------------------ inputs

def _spread(i, n, top):
    """The i-th of n whole numbers over the logarithm of 1..top, mixed."""
    return int(round(top ** (((7 * i) % n) / (n - 1)))) if n > 1 else top


def _requests(case):
    """(lens, new) of the rows, from the case alone (-1, 0: an idle row)."""
    R, lens, new = case["S"] * case["W"], [], []
    for i in range(R):
        lens.append(case["P"] + (_spread(i, R, case["held"] + 1) - 1 if case["ragged"] else case["held"]))
        n = 1
        if case["tokens"] == "prompt" or (case["tokens"] == "mixed" and i % 8 == 3):
            n = _spread(i + 1, R, case["new"]) if case["ragged"] else case["new"]
        new.append(n)
    for i in range(case["idle"]):                    # idle rows between the others and at the end
        at = R - 1 - 2 * i if R - 1 - 2 * i > 0 else 0
        lens[at], new[at] = -1, 0
    return lens, new


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    W, P, PS, L, KVH, HD = (case[k] for k in ("W", "P", "PS", "L", "KVH", "HD"))
    lens, new = _requests(case)
    R = len(lens)
    ready = case["kind"] == "attend"                 # pages for the new tokens are there already
    MP = max(1, -(-max(n + m for n, m in zip(lens, new)) // PS))
    rows, used, spare = [], 0, 5
    for r, n in enumerate(lens):
        if r % W == 0:
            common = {}                              # the group's pages
        row = [-1] * MP
        if n >= 0:
            # rows that hold no more than the common tokens share a partly filled last page too
            shared = -(-P // PS) if n == P and not ready else P // PS
            for s in range(-(-(n + (new[r] if ready else 0)) // PS)):
                if s < shared and s in common:
                    row[s] = common[s]
                else:
                    row[s] = used
                    used += 1
                    if s < shared:
                        common[s] = row[s]
            spare += 0 if ready else -(-(n + new[r]) // PS) - n // PS
        rows.append(row)
    NP = used + spare
    order = torch.randperm(NP, generator=g, device=DEV).to(torch.int32)
    at = _i32(rows)
    table = torch.where(at >= 0, order[at.clamp(min=0).long()], -1).to(torch.int32)
    pools = [torch.randn(L, NP, KVH, PS, HD, generator=g, device=DEV, dtype=dt) for _ in range(2)]
    s = dict(case, k_pages=pools[0], v_pages=pools[1], table=table, lens=_i32(lens), news=_i32(new),
             n_tokens=sum(new) + case["pad"])
    if not ready:
        refs = torch.bincount(table.view(-1).long() + 1, minlength=NP + 1)[1:].to(torch.int32)
        return dict(s, table=table.clone(), refs=refs.clone(), table0=table, refs0=refs,
                    status=torch.zeros(1, dtype=torch.int32, device=DEV))
    inv = 10000.0 ** (-torch.arange(0, HD, 2, device=DEV, dtype=torch.float64) / HD)
    ang = torch.arange(MP * PS, device=DEV, dtype=torch.float64)[:, None] * torch.cat([inv, inv])[None]
    width = (case["QH"] + 2 * KVH) * HD
    return dict(s, qkv=[torch.randn(s["n_tokens"], width, generator=g, device=DEV).to(dt) for _ in range(L)],
                cos=ang.cos().float(), sin=ang.sin().float())


# ------------------------------------------------------------------ plain forms

def _maps_plain(s, table):
    """starts, rows, positions and slots of the flat tokens."""
    lens, new, PS = s["lens"], s["news"], s["PS"]
    count = torch.where(lens >= 0, new, 0).long()
    starts = torch.cat([count.new_zeros(1), count.cumsum(0)])
    t = torch.arange(s["n_tokens"], device=DEV)
    row = (t[:, None] >= starts[None, 1:]).sum(1)
    there = row < lens.numel()
    at = row.clamp(max=lens.numel() - 1)
    pos = lens[at].long() + t - starts[at]
    page = table[at, torch.where(there, pos, 0) // PS].long()
    slots = torch.where(there, page * PS + pos % PS, -1)
    i32 = lambda v: torch.where(there, v, -1).to(torch.int32)  # noqa: E731
    return dict(starts=starts.to(torch.int32), rows=i32(row), positions=i32(pos), slots=slots)


def _plan_plain(s):
    table, refs, lens, PS = s["table"], s["refs"], s["lens"], s["PS"]
    new = torch.where(lens >= 0, s["news"], 0)
    R, MP = table.shape
    tail = (new > 0) & (lens % PS > 0)
    slot = (lens.clamp(min=0) // PS).long()
    page = table.gather(1, slot.clamp(max=MP - 1)[:, None]).view(-1).long()
    same = (page[:, None] == page[None]) & tail[:, None] & tail[None]
    before = torch.tril(same, -1).sum(1)
    copy = tail & (refs[page.clamp(min=0)] - before > 1)
    col = torch.arange(MP, device=DEV)[None]
    miss = (col >= ((lens + PS - 1) // PS)[:, None]) & (col < ((lens + new + PS - 1) // PS)[:, None]) & (new > 0)[:, None]
    want = miss | (copy[:, None] & (col == slot[:, None]))
    free = torch.argsort((refs != 0).to(torch.uint8), stable=True)
    rank = (want.view(-1).long().cumsum(0) - 1).clamp(min=0).view(R, MP)
    table.copy_(torch.where(want, free[rank].to(torch.int32), table))
    got = table.gather(1, slot.clamp(max=MP - 1)[:, None]).view(-1).long()
    src, dst = page[copy], got[copy]
    held = (torch.arange(PS, device=DEV)[None] < (lens % PS)[copy][:, None])[None, :, None, :, None]
    for pool in (s["k_pages"], s["v_pages"]):
        pool[:, dst] = torch.where(held, pool[:, src], pool[:, dst])
    refs.copy_(torch.bincount(table.view(-1).long() + 1, minlength=refs.numel() + 1)[1:])
    return dict(_maps_plain(s, table), table=table, refs=refs, k_pages=s["k_pages"], v_pages=s["v_pages"])


def _rotate(x):
    a, b = x.chunk(2, -1)
    return torch.cat([-b, a], -1)


def _attend_plain(s):
    QH, KVH, HD, PS = s["QH"], s["KVH"], s["HD"], s["PS"]
    dt, G, N = s["qkv"][0].dtype, s["QH"] // s["KVH"], s["n_tokens"]
    m = _maps_plain(s, s["table"])
    total = int(m["starts"][-1])
    pos, slots = m["positions"][:total].long(), m["slots"][:total]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lens, starts = s["lens"].tolist(), m["starts"].tolist()
    outs = dict(c=[], kctx=[], q=[])
    for layer, qkv in enumerate(s["qkv"]):
        kp, vp = s["k_pages"][layer], s["v_pages"][layer]
        x = qkv[:total].float().view(total, QH + 2 * KVH, HD)
        qk = (x[:, :QH + KVH] * cos + _rotate(x[:, :QH + KVH]) * sin).to(dt)
        kp[slots // PS, :, slots % PS] = qk[:, QH:]
        vp[slots // PS, :, slots % PS] = x[:, QH + KVH:].to(dt)
        c, kctx, q = (torch.zeros(N, QH, HD, dtype=dt, device=DEV) for _ in range(3))
        q[:total] = qk[:, :QH]
        for r, n in enumerate(lens):
            a, e = starts[r], starts[r + 1]
            if a == e:
                continue
            T = n + e - a
            ids = s["table"][r, :-(-T // PS)].long()
            kk = kp[ids].transpose(0, 1).reshape(KVH, -1, HD)[:, :T].float()
            vv = vp[ids].transpose(0, 1).reshape(KVH, -1, HD)[:, :T].float()
            qr = q[a:e].float().view(e - a, KVH, G, HD).permute(1, 2, 0, 3).reshape(KVH, G * (e - a), HD)
            sc = torch.matmul(qr, kk.transpose(1, 2).contiguous()) / math.sqrt(HD)
            unseen = torch.arange(T, device=DEV)[None] > torch.arange(n, T, device=DEV)[:, None]
            sc = sc.view(KVH, G, e - a, T).masked_fill(unseen, -math.inf)
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            w = (w / w.sum(-1, keepdim=True)).view(KVH, G * (e - a), T)
            for out, rows in ((c, vv), (kctx, kk)):
                o = torch.matmul(w, rows).view(KVH, G, e - a, HD).permute(2, 0, 1, 3)
                out[a:e] = o.reshape(e - a, QH, HD).to(dt)
        outs["c"].append(c)
        outs["kctx"].append(kctx)
        outs["q"].append(q)
    return dict(outs, k_pages=s["k_pages"], v_pages=s["v_pages"])


def run(state):
    s = state
    if s["kind"] == "plan":
        # the tables of before the step again, so that every pass has the same pages to find
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
        if not own:
            return _plan_plain(s)
        ops = _ops()
        ops.paged_reserve(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["refs"], s["status"], s["news"])
        p = ops.paged_plan(s["k_pages"], s["table"], s["lens"], s["news"], s["n_tokens"], s["QH"])
        return dict(starts=p.starts, rows=p.rows, positions=p.positions, slots=p.slots, table=s["table"], refs=s["refs"],
                    k_pages=s["k_pages"], v_pages=s["v_pages"])
    if not own:
        return _attend_plain(s)
    ops = _ops()
    p = ops.paged_plan(s["k_pages"], s["table"], s["lens"], s["news"], s["n_tokens"], s["QH"])
    outs = dict(c=[], kctx=[], q=[])
    for layer, qkv in enumerate(s["qkv"]):
        c, kctx, q = ops.paged_batch_step(p, qkv, s["k_pages"][layer], s["v_pages"][layer], s["table"], s["cos"], s["sin"])
        outs["c"].append(c)
        outs["kctx"].append(kctx)
        outs["q"].append(q)
    return dict(outs, k_pages=s["k_pages"], v_pages=s["v_pages"])


# ------------------------------------------------------------------ work and exact values

def work(case):
    e, W, P, PS, L, KVH, HD, QH = (ESIZE[case["dtype"]],) + tuple(case[k] for k in ("W", "P", "PS", "L", "KVH", "HD", "QH"))
    lens, new = _requests(case)
    total, N, R = sum(new), sum(new) + case["pad"], len(lens)
    live = [(r, n, m) for r, (n, m) in enumerate(zip(lens, new)) if n >= 0]
    row = 2 * KVH * HD * e                                       # K and V of one token in one layer
    maps = 4 * (R + 1) + 16 * N
    if case["kind"] == "plan":
        pages = sum(-(-(n + m) // PS) - -(-n // PS) for _, n, m in live)
        forks = [r for r, n, _ in live if n == P and P % PS]
        copies = len(forks) - len({r // W for r in forks})       # the last of a group's rows keeps the page
        # lens and new, the counts of all pages, the table's entries for the new tokens, the maps, the copies
        return dict(bytes=8 * R + 4 * pages + 12 * (pages + copies) + maps + copies * (8 + 2 * (P % PS) * row * L), flops=0)
    groups = {}
    for r, n, m in live:
        groups.setdefault(r // W, []).append(n - P // PS * PS)   # its own tokens (the common whole pages once)
    seen = sum(P // PS * PS + sum(v) for v in groups.values())
    entries = sum(-(-(n + m) // PS) for _, n, m in live)
    step = seen * row + total * ((QH + 2 * KVH) * HD * e + row) + 3 * N * QH * HD * e + 8 * HD * max(n + m for _, n, m in live if m)
    keys = sum(m * n + m * (m + 1) // 2 for _, n, m in live)
    return dict(bytes=L * step + 4 * entries + 8 * R + maps, flops=L * 6 * QH * HD * keys)


def _exact_plan(s):
    PS, L = s["PS"], s["L"]
    lens, new = _requests(s)
    table, refs = s["table0"].tolist(), s["refs0"].tolist()
    free = [p for p, n in enumerate(refs) if n == 0]
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    starts, rows, positions, slots = [0], [], [], []
    for r, (n, m) in enumerate(zip(lens, new)):
        if m and n % PS and refs[table[r][n // PS]] > 1:
            p, q = table[r][n // PS], free.pop(0)
            for pool in pools:
                pool[:, q, :, :n % PS] = pool[:, p, :, :n % PS]
            refs[p] -= 1
            refs[q] = 1
            table[r][n // PS] = q
        for t in range(n, n + m):
            if table[r][t // PS] < 0:
                table[r][t // PS] = free.pop(0)
                refs[table[r][t // PS]] = 1
            rows.append(r)
            positions.append(t)
            slots.append(table[r][t // PS] * PS + t % PS)
        starts.append(len(rows))
    pad = [-1] * s["pad"]
    return dict(starts=_i32(starts), rows=_i32(rows + pad), positions=_i32(positions + pad),
                slots=torch.tensor(slots + pad, dtype=torch.int64, device=DEV), table=_i32(table), refs=_i32(refs),
                k_pages=pools[0], v_pages=pools[1])


def _exact_attend(s):
    QH, KVH, HD, PS, N = s["QH"], s["KVH"], s["HD"], s["PS"], s["n_tokens"]
    lens, new = _requests(s)
    half, G, dt = HD // 2, QH // KVH, s["qkv"][0].dtype
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    outs = dict(c=[], kctx=[], q=[])
    for layer in range(s["L"]):
        c, kctx, q = (torch.zeros(N, QH, HD, dtype=torch.float64, device=DEV) for _ in range(3))
        a = 0
        for r, (n, m) in enumerate(zip(lens, new)):
            if m == 0:
                continue
            x = s["qkv"][layer][a:a + m].double().view(m, QH + 2 * KVH, HD)
            co, si = s["cos"][n:n + m].double()[:, None], s["sin"][n:n + m].double()[:, None]
            turned = torch.empty_like(x)
            turned[..., :half] = x[..., :half] * co[..., :half] - x[..., half:] * si[..., :half]
            turned[..., half:] = x[..., half:] * co[..., half:] + x[..., :half] * si[..., half:]
            turned = turned.to(dt).double()
            q[a:a + m] = turned[:, :QH]
            for i in range(m):
                if i == 0 or (n + i) % PS == 0:      # page by page
                    page, e = int(s["table"][r, (n + i) // PS]), min(m, i + PS - (n + i) % PS)
                    at = slice((n + i) % PS, (n + i) % PS + e - i)
                    kp[layer, page, :, at] = turned[i:e, QH:QH + KVH].transpose(0, 1)
                    vp[layer, page, :, at] = x[i:e, QH + KVH:].transpose(0, 1)
            ids = s["table"][r, :-(-(n + m) // PS)].long()
            ok = torch.ones(m, n + m, dtype=torch.bool, device=DEV).tril(n)
            for h in range(QH):
                k = kp[layer, ids, h // G].reshape(-1, HD)[:n + m]
                v = vp[layer, ids, h // G].reshape(-1, HD)[:n + m]
                w = torch.softmax((q[a:a + m, h] @ k.t() * HD ** -0.5).masked_fill(~ok, -math.inf), 1)
                c[a:a + m, h], kctx[a:a + m, h] = w @ v, w @ k
            a += m
        outs["c"].append(c)
        outs["kctx"].append(kctx)
        outs["q"].append(q)
    return dict(outs, k_pages=kp, v_pages=vp)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_plan(s) if case["kind"] == "plan" else _exact_attend(s)
