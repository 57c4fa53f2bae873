"""Plain references of the operators that verify drafted tokens (omniserver_b200/ops/speculative.py), from their definitions, in
64 bits, with loops over requests, nodes and heads."""

from __future__ import annotations

import math

import torch


def sees_list(mask_row, n):
    """The nodes below n whose bit is set in a row of mask words."""
    return [j for j in range(n) if j // 32 < len(mask_row) and (int(mask_row[j // 32]) >> (j % 32)) & 1]


def tree_attention(qkv, k_cache, v_cache, block_table, cu_q, seq_lens, mask, nh, nkv, hd, scale, window=None, depth=None):
    """(out, spread, weight) [T, nh*hd] in 64 bits: the attention; sum of p |v| (what the rounding of weights can move); and the
    largest sum |q k| scale of a row (what the rounding of scores can move). Rows of no request are NaN."""
    T, ps, grp = qkv.shape[0], k_cache.shape[2], nh // nkv
    q = qkv[:, :nh * hd].double().cpu().view(T, nh, hd)
    K, V = k_cache.double().cpu(), v_cache.double().cpu()
    bt, cu, lens = block_table.cpu().tolist(), cu_q.cpu().tolist(), seq_lens.cpu().tolist()
    mask = mask.cpu().tolist()
    out = torch.full((T, nh, hd), math.nan, dtype=torch.float64)
    spread, weight = torch.zeros_like(out), 0.0
    for s in range(len(lens)):
        n = cu[s + 1] - cu[s]
        base = lens[s] - n
        for i in range(n):
            t = cu[s] + i
            at = base + (int(depth[t]) if depth is not None else 0)
            places = [p for p in range(base) if not window or p > at - window]
            for j in sees_list(mask[t], n):
                if not window or base + int(depth[cu[s] + j]) > at - window:
                    places.append(base + j)
            if not places:
                out[t] = 0.0
                continue
            pages = torch.tensor([bt[s][p // ps] for p in places])
            offs = torch.tensor([p % ps for p in places])
            k, v = K[pages, :, offs], V[pages, :, offs]          # [keys, nkv, hd]
            for h in range(nh):
                sc = (k[:, h // grp] @ q[t, h]) * scale
                if sc.isfinite().all():
                    weight = max(weight, float((k[:, h // grp].abs() @ q[t, h].abs()).max()) * abs(scale))
                if bool((sc == -math.inf).all()):
                    out[t, h] = 0.0
                    continue
                p = torch.exp(sc - sc.max())
                p = p / p.sum()
                out[t, h] = p @ v[:, h // grp]
                spread[t, h] = p @ v[:, h // grp].abs()
    return out.view(T, nh * hd), spread.view(T, nh * hd), weight


def verify(logits, tokens, parents, cu_q, uniform, max_depth, temperature=None, draft_probs=None):
    """Lists (tokens, path, count) per request."""
    V = logits.shape[1]
    cu, tok, par, u = cu_q.tolist(), tokens.tolist(), parents.tolist(), uniform.double().tolist()
    got = []
    for s in range(len(cu) - 1):
        t0, n = cu[s], cu[s + 1] - cu[s]
        if n == 0:
            got.append(([-1] * (max_depth + 1), [-1] * (max_depth + 1), 0))
            continue
        temp = float(temperature[s]) if temperature is not None else 0.0

        def target(i):
            x = logits[t0 + i].double()
            x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
            top = x.max()
            if top == -math.inf:
                return None, 0
            first = int((x == top).nonzero()[0])
            if temp <= 0:
                r = torch.zeros_like(x)
                r[first] = 1.0
            else:
                r = torch.where(x == top, torch.ones_like(x), torch.exp((x - (top if top < math.inf else 0.0)) / temp))
                if top == math.inf:
                    r = (x == top).double()
                r = r / r.sum()
            return r, first

        path, node = [0], 0
        r, first = target(0)
        while True:
            nxt = None
            for c in range(node + 1, n):
                if par[t0 + c] != node or len(path) > max_depth or r is None or not 0 <= tok[t0 + c] < V:
                    continue
                x = tok[t0 + c]
                if temp <= 0:
                    if x == first:
                        nxt = c
                        break
                    continue
                if draft_probs is None:
                    if u[t0 + c] < float(r[x]):
                        nxt = c
                        break
                    left = r.clone()
                    left[x] = 0.0
                else:
                    q = draft_probs[t0 + node].double()
                    q = torch.where(q > 0, q, torch.zeros_like(q))
                    if u[t0 + c] * float(q[x]) < float(r[x]):
                        nxt = c
                        break
                    left = (r - q).clamp(min=0.0)
                if float(left.sum()) > 0:
                    r = left / left.sum()
            if nxt is None:
                break
            node = nxt
            path.append(node)
            r, first = target(node)
        if r is None or temp <= 0:
            word = first
        else:
            run = torch.cumsum(r, 0)
            over = (run > u[t0] * float(run[-1])).nonzero()
            word = int(over[0]) if len(over) else int((r > 0).nonzero()[-1])
        pad = [-1] * (max_depth + 1 - len(path))
        got.append(([tok[t0 + c] for c in path[1:]] + [word] + pad, path + pad, len(path)))
    return got


def compact(cache, block_table, cu_q, seq_lens, path, count):
    """The cache after the move (a copy)."""
    out, ps = cache.clone(), cache.shape[4]
    bt, cu = block_table.tolist(), cu_q.tolist()
    for s in range(len(count)):
        base = int(seq_lens[s]) - (cu[s + 1] - cu[s])
        for i in range(int(count[s])):
            a, b = base + int(path[s, i]), base + i
            out[:, :, bt[s][b // ps], :, b % ps] = cache[:, :, bt[s][a // ps], :, a % ps]
    return out
