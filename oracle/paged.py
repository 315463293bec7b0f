"""Plain restatements (64 bits, loops over rows) of the paged cache's operators,
the beam selection and the row reordering.  Floating inputs of any type on any
device; results in float64 on the CPU unless they are whole numbers or copies."""
from __future__ import annotations

import math

import torch


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x cos + rotate_half(x) sin over the last dimension, in 64 bits."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    a, b = x.chunk(2, -1)
    return x * cos + torch.cat([-b, a], -1) * sin


def rows_of(pages: torch.Tensor, table_row, n: int) -> torch.Tensor:
    """The first n tokens of a row: [kv_heads, n, head_dim] in 64 bits."""
    PS = pages.shape[2]
    ids = [int(p) for p in table_row[:-(-n // PS)]]
    return pages[ids].double().transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def attention(q, k_pages, v_pages, table, counts):
    """C = A V, Kctx = A K of each row over its first counts[r] tokens (none:
    zeros), and what the bounds of a computed result go by: the same sums of
    absolute values, and the largest score and sum of |q k| of each head."""
    q = q.cpu().double()
    kp, vp = k_pages.cpu(), v_pages.cpu()
    B, QH, HD = q.shape
    KVH = kp.shape[1]
    G = QH // KVH
    out = {n: torch.zeros(B, QH, HD, dtype=torch.float64) for n in ("c", "kctx", "c_abs", "kctx_abs")}
    out.update(s_max=torch.zeros(B, QH, dtype=torch.float64), qk_abs=torch.zeros(B, QH, dtype=torch.float64))
    for b in range(B):
        n = int(counts[b])
        if n <= 0:
            continue
        k, v = rows_of(kp, table[b], n), rows_of(vp, table[b], n)
        for h in range(QH):
            kk, vv = k[h // G], v[h // G]
            s = kk @ q[b, h] / math.sqrt(HD)
            w = torch.exp(s - s.max())
            w = w / w.sum()
            out["c"][b, h], out["kctx"][b, h] = w @ vv, w @ kk
            out["c_abs"][b, h], out["kctx_abs"][b, h] = w @ vv.abs(), w @ kk.abs()
            out["s_max"][b, h] = s.abs().max()
            out["qk_abs"][b, h] = (kk.abs() @ q[b, h].abs()).max() / math.sqrt(HD)
    return out


def update(k_pages, v_pages, table, lens, refs, parent=None, n_new=0, advance=0):
    """paged_update on copies: (k_pages, v_pages, table, lens, refs, status).  Pools
    [layers, pages, kv_heads, page_size, head_dim]."""
    kp, vp = k_pages.clone(), v_pages.clone()
    NP, PS = kp.shape[1], kp.shape[3]
    old, l0 = table.tolist(), lens.tolist()
    rf = refs.tolist()
    R, MP = len(old), len(old[0])
    rows, ln, status = [list(r) for r in old], list(l0), 0
    valid = lambda p: 0 <= p < NP  # noqa: E731
    if parent is not None:
        for r, p in enumerate(parent.tolist()):
            if p == r:
                continue
            held = -(-(l0[p] + advance) // PS) if 0 <= p < R and l0[p] >= 0 else 0
            rows[r] = [old[p][s] if s < held else -1 for s in range(MP)]
            ln[r] = l0[p] if 0 <= p < R else -1
        for r in range(R):
            for a, b in zip(old[r], rows[r]):
                if a != b:
                    if valid(a):
                        rf[a] -= 1
                    if valid(b):
                        rf[b] += 1
    ln = [n + advance if n >= 0 else -1 for n in ln]
    held, gone = list(rf), []
    for r in range(R):                                # pages behind the tokens that are not the row's alone
        n = min(n_new, MP * PS - ln[r]) if ln[r] >= 0 else 0
        kept = True
        for s in range(-(-ln[r] // PS), (ln[r] + n - 1) // PS + 1) if n > 0 else ():
            kept = kept and valid(rows[r][s]) and held[rows[r][s]] <= 1
            if not kept and valid(rows[r][s]):
                gone.append(rows[r][s])
                rows[r][s] = -1
    for p in gone:
        rf[p] -= 1
    free = [p for p in range(NP) if rf[p] <= 0]
    for r in range(R):
        if ln[r] < 0 or n_new == 0:
            continue
        n = min(n_new, MP * PS - ln[r])
        if n < n_new:
            status += 1
        if n <= 0:
            continue
        tail, slot = ln[r] % PS, ln[r] // PS
        if tail and valid(rows[r][slot]) and rf[rows[r][slot]] > 1:
            src = rows[r][slot]
            rf[src] -= 1
            if free:
                dst = free.pop(0)
                for pool in (kp, vp):
                    pool[:, dst, :, :tail] = pool[:, src, :, :tail]
                rf[dst] = 1
                rows[r][slot] = dst
            else:
                rows[r][slot] = -1
                status += 1
        s = -(-ln[r] // PS)
        last = (ln[r] + n - 1) // PS
        while s <= last and valid(rows[r][s]):
            s += 1
        for s in range(s, last + 1):
            if free:
                rows[r][s] = free.pop(0)
                rf[rows[r][s]] = 1
            else:
                status += 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return kp, vp, i32(rows).view(R, MP), i32(ln), i32(rf), status


def compact(k_pages, v_pages, table, refs):
    """paged_compact on copies: (k_pages, v_pages, table, refs, used)."""
    kp, vp = k_pages.clone(), v_pages.clone()
    rf = refs.tolist()
    used = sum(n > 0 for n in rf)
    movers = [p for p in range(used, len(rf)) if rf[p] > 0]
    holes = [p for p in range(used) if rf[p] <= 0]
    for a, b in zip(movers, holes):
        kp[:, b], vp[:, b] = kp[:, a], vp[:, a]
        rf[b], rf[a] = rf[a], 0
    went = dict(zip(movers, holes))
    rows = [[went.get(p, p) for p in row] for row in table.tolist()]
    return kp, vp, torch.tensor(rows, dtype=torch.int32).view(table.shape), torch.tensor(rf, dtype=torch.int32), used


def beam_select(logits, scores, n_out, finished=None, eos_id=-1, pad_id=0):
    """beam_select: (scores in 64 bits, parent, token, finished)."""
    x, sc = logits.cpu().double(), scores.cpu().double()
    S, W = sc.shape
    fin = [False] * (S * W) if finished is None else [bool(f) for f in finished.cpu().view(-1)]
    out = [[], [], [], []]
    for g in range(S):
        found = []
        for w in range(W):
            r, base = g * W + w, float(sc[g, w])
            if fin[r]:
                found.append((base, w, pad_id))
                continue
            m = x[r].max()
            lse = float(m + torch.log(torch.exp(x[r] - m).sum()))
            found += [(v - lse + base, w, t) for t, v in enumerate(x[r].tolist())]
        found = sorted((-v, w, t) for v, w, t in found if math.isfinite(v))[:n_out]
        rows = [(-v, g * W + w, t, fin[g * W + w] or t == eos_id) for v, w, t in found]
        rows += [(-math.inf, g * W, pad_id, False)] * (n_out - len(rows))
        for o, col in zip(out, zip(*rows)):
            o.append(list(col))
    return (torch.tensor(out[0], dtype=torch.float64), torch.tensor(out[1], dtype=torch.int32),
            torch.tensor(out[2], dtype=torch.int64), torch.tensor(out[3], dtype=torch.bool))


def reorder_rows(t: torch.Tensor, parent, dim: int = 0) -> torch.Tensor:
    """A copy of t with row r = the former row parent[r] (outside: unchanged)."""
    R = t.shape[dim]
    at = [p if 0 <= p < R else r for r, p in enumerate(parent.tolist())]
    return t.index_select(dim, torch.tensor(at, device=t.device))
