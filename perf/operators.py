"""The operators of a step that verifies drafted tokens, in their plain form and through the framework.

A request brings a tree of drafted tokens. Its keys and values go into the paged cache behind the request's committed
tokens; attention lets a node see the committed tokens and its ancestors; the verification walks the tree with the
target's logits and given random numbers; the tokens of the accepted path move together in the cache. Forked requests
copy pages.

``listed()`` and ``draw(rng)`` give cases, ``prepare`` a case's inputs, ``run`` makes one pass: with ``own`` through
``omniserver_b200.ops.kernels()``, otherwise in elementary torch operations. ``exact`` computes the same from the
definitions in 64 bits, ``work`` says what a pass cannot do without.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
# (query heads, kv heads) of the framework's benchmark sizes
HEADS = ((12, 2), (28, 4), (64, 8))


# ------------------------------------------------------------------ cases
def listed():
    tree = dict(op="tree", hd=128, page=32, window=0, dtype="bf16")
    verify = dict(op="verify", greedy=0)
    cache = dict(hd=128, page=32, layers=28, dtype="bf16")
    return [
        # one user, a small tree, the benchmark's context: the smallest call, latency counts
        dict(tree, name="tree one request", reqs=1, nodes=16, ctx=2048, nh=12, nkv=2),
        # a small batch of ragged trees and contexts
        dict(tree, name="tree ragged batch", reqs=8, nodes=32, ctx=4096, nh=28, nkv=4),
        # a busy server: many requests with a few drafted tokens each (some with one)
        dict(tree, name="tree many requests", reqs=64, nodes=8, ctx=2100, nh=28, nkv=4),
        # one long context with a wide tree: the most arithmetic
        dict(tree, name="tree long context", reqs=1, nodes=64, ctx=32768, nh=64, nkv=8),
        # the 32-bit path
        dict(tree, name="tree 32 bits", reqs=4, nodes=24, ctx=1000, nh=12, nkv=2, dtype="f32"),
        # one user, a chain of five drafted tokens found without a draft model (a point mass each)
        dict(verify, name="verify one chain", reqs=1, nodes=6, branch=1, vocab=151936, dense=False),
        # a small batch of trees of a draft head's best guesses; every fourth request is greedy
        dict(verify, name="verify trees", reqs=8, nodes=32, branch=3, vocab=152064, dense=False, greedy=4),
        # a busy server with a draft model: chains drawn from its probabilities
        dict(verify, name="verify drawn chains", reqs=32, nodes=7, branch=1, vocab=152064, dense=True),
        # accepted paths of one request, and of a full batch, over all layers
        dict(cache, name="compact one", op="compact", reqs=1, nodes=16, ctx=300, nkv=2),
        dict(cache, name="compact batch", op="compact", reqs=64, nodes=12, ctx=90, nkv=4),
        # a fork copies the parent's last page; a batch of prompts is forked with whole pages
        dict(cache, name="copy one page", op="copy", pages=1, nkv=2),
        dict(cache, name="copy many pages", op="copy", pages=64, nkv=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tree", "tree", "verify", "verify", "compact", "copy"))
    if op == "tree":
        nh, nkv = rng.choice(HEADS)
        reqs, nodes, dtype = _log(rng, 1, 64), _log(rng, 1, 64), rng.choice(("bf16", "bf16", "bf16", "f32"))
        # keys of all requests: at most what the largest listed cases read; in 32 bits less
        most = 130000 * 8 // nkv // reqs if dtype == "bf16" else 4000 // reqs
        if reqs * nodes > 512:
            nodes = max(1, 512 // reqs)
        if dtype == "f32":
            nodes = min(nodes, 24)
        ctx = _log(rng, 40, max(60, min(32768, most)))
        return dict(op="tree", reqs=reqs, nodes=nodes, ctx=ctx, nh=nh, nkv=nkv, hd=rng.choice((64, 128)),
                    page=rng.choice((16, 32, 64)), window=rng.choice((0, 0, 0, 1 + ctx // 3)), dtype=dtype)
    if op == "verify":
        dense = rng.random() < 0.5
        branch = 1 if dense and rng.random() < 0.6 else rng.choice((1, 2, 3))
        reqs = _log(rng, 1, 32)
        nodes = max(2, min(_log(rng, 2, 40), 224 // reqs))
        return dict(op="verify", reqs=reqs, nodes=nodes, branch=branch, vocab=rng.choice((_log(rng, 900, 152064), 151936, 152064)),
                    dense=dense, greedy=rng.choice((0, 0, 3)))
    layers, nkv, page = rng.choice((4, 28, 40)), rng.choice((2, 4, 8)), rng.choice((16, 32, 64))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "compact":
        ctx, nodes = _log(rng, 20, 200), _log(rng, 3, 40)
        token = layers * 2 * nkv * 128 * SIZE[dtype]
        reqs = min(_log(rng, 1, 64), max(1, 400_000_000 // ((ctx + nodes + page) * token)))
        return dict(op="compact", reqs=reqs, nodes=nodes, ctx=ctx, nkv=nkv, hd=128, page=page, layers=layers, dtype=dtype)
    one = layers * 2 * nkv * page * 128 * SIZE[dtype]
    pages = max(1, min(_log(rng, 1, 64), 117_000_000 // one))
    return dict(op="copy", pages=pages, nkv=nkv, hd=128, page=page, layers=layers, dtype=dtype)


# ------------------------------------------------------------------ sizes of a case (from the case alone)
def _q_lens(c):
    r = random.Random(7 * c["reqs"] + c["nodes"])
    return np.array([c["nodes"] if i == 0 else r.randint(max(1, c["nodes"] // 4), c["nodes"]) for i in range(c["reqs"])])


def _bases(c):
    """Committed tokens in front of each request's tree."""
    r = random.Random(11 * c["reqs"] + c["ctx"])
    return np.array([c["ctx"] if i == 0 else r.randint(max(0, c["ctx"] // 2), c["ctx"]) for i in range(c["reqs"])])


def _depth_of(nodes, branch):
    """Depth of the last node of the tree in which node j's parent is (j - 1) // branch."""
    d, j = 0, nodes - 1
    while j > 0:
        j, d = (j - 1) // branch, d + 1
    return d


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed % 1000003) + salt)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _tables(kv_lens, page, rng):
    """Pages in random order: (block table, pages in all)."""
    need = -(-kv_lens // page)
    total = int(need.sum())
    ids = rng.permutation(total + 3)[:total]
    bt = np.full((len(kv_lens), int(need.max())), -1, dtype=np.int32)
    o = 0
    for s, n in enumerate(need):
        bt[s, :n] = ids[o:o + n]
        o += n
    return bt, total + 3


def _parents(n, rng):
    """A random tree in which parents come before their children."""
    p = [-1] + [int(rng.integers((j - 1) // 3, j)) for j in range(1, n)]
    return p


def _ancestors(parents):
    """For each node the list of the nodes from the root to itself."""
    out = []
    for j, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [j])
    return out


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    return {"tree": _prepare_tree, "verify": _prepare_verify, "compact": _prepare_compact, "copy": _prepare_copy}[case["op"]](case, seed)


def _prepare_tree(c, seed):
    rng, g, dt = np.random.default_rng(seed), _gen(seed, 1), DTYPES[c["dtype"]]
    q_lens, base = _q_lens(c), _bases(c)
    kv_lens = base + q_lens
    bt, pages = _tables(kv_lens, c["page"], rng)
    T, width = int(q_lens.sum()), (c["nh"] + 2 * c["nkv"]) * c["hd"]
    trees = [_parents(int(n), rng) for n in q_lens]
    words = -(-int(q_lens.max()) // 32)
    mask, depth = np.zeros((T, words), dtype=np.uint32), np.zeros(T, dtype=np.int32)
    t = 0
    for parents in trees:
        for line in _ancestors(parents):
            for j in line:
                mask[t, j // 32] |= np.uint32(1 << (j % 32))
            depth[t] = len(line) - 1
            t += 1
    cache = torch.randn((2, pages, c["nkv"], c["page"], c["hd"]), generator=g, device=DEV, dtype=torch.float32).to(dt)
    return dict(case=c, trees=trees, q_lens=q_lens, kv_lens=kv_lens, k=cache[0], v=cache[1],
                qkv=torch.randn((T, width), generator=g, device=DEV, dtype=torch.float32).to(dt), bt=_dev(bt), cu=_dev(_cu(q_lens)),
                lens=_dev(kv_lens.astype(np.int32)), mask=_dev(mask.view(np.int32)), depth=_dev(depth),
                n_max=int(q_lens.max()), kv_max=int(kv_lens.max()))


def _prepare_verify(c, seed):
    g, V, n = _gen(seed, 2), c["vocab"], c["nodes"]
    S, T = c["reqs"], c["reqs"] * c["nodes"]
    parents = np.array([-1] + [(j - 1) // c["branch"] for j in range(1, n)], dtype=np.int32)
    # logits as peaked as a language model's: a handful of words share most of the probability
    logits = torch.randn((T, V), generator=g, device=DEV).mul_(math.sqrt(2 * math.log(V)))
    temp = torch.full((S,), 0.9, device=DEV)
    if c["greedy"]:
        temp[torch.arange(S, device=DEV) % c["greedy"] == 0] = 0.0
    par = torch.from_numpy(parents).to(DEV).long()
    row = torch.arange(S, device=DEV)[:, None] * n
    parent_row = (row + par.clamp(min=0)).reshape(-1)
    tokens = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    q = None
    if c["dense"]:
        # the draft model's probabilities are near the target's; its tokens are drawn from them
        q = torch.softmax(logits / 0.9 + torch.randn((T, V), generator=g, device=DEV).mul_(0.7), dim=-1)
        for j in range(1, n):
            pr = parent_row.view(S, n)[:, j]
            tokens.view(S, n)[:, j] = torch.multinomial(q[pr], 1, generator=g).to(torch.int32)[:, 0]
    else:
        # a draft head's best guesses: sibling k is its parent's k-th best word, at times a worse one
        best = torch.topk(logits, c["branch"] + 2, dim=-1).indices
        for j in range(1, n):
            k = (j - 1) % c["branch"] + torch.randint(0, 2, (S,), generator=g, device=DEV)
            tokens.view(S, n)[:, j] = best[parent_row.view(S, n)[:, j], k].to(torch.int32)
    uniform = torch.randint(0, 1 << 24, (T,), generator=g, device=DEV).float() / float(1 << 24)
    return dict(case=c, logits=logits, q=q, tokens=tokens, parents=torch.from_numpy(np.tile(parents, S)).to(DEV), temp=temp,
                uniform=uniform, cu=_dev(_cu(np.full(S, n))), depth_max=_depth_of(n, c["branch"]), par=par)


def _cache(c, pages, g):
    shape = (c["layers"], 2, pages, c["nkv"], c["page"], c["hd"])
    return torch.randn(shape, generator=g, device=DEV, dtype=DTYPES[c["dtype"]])


def _path_width(c):
    return min(8, (c["nodes"] + 1) // 2)


def _prepare_compact(c, seed):
    rng, g = np.random.default_rng(seed), _gen(seed, 3)
    q_lens, base = _q_lens(c), _bases(c)
    bt, pages = _tables(base + q_lens, c["page"], rng)
    S, W = c["reqs"], _path_width(c)
    path, counts = np.full((S, W), -1, dtype=np.int32), np.zeros(S, dtype=np.int32)
    for s, n in enumerate(q_lens):
        k = int(rng.integers(1, min(W, (n + 1) // 2) + 1))
        # the root, then nodes behind the places that the path ends up in: a second pass finds the same tokens there
        path[s, :k] = [0] + sorted(rng.choice(np.arange(k, n), k - 1, replace=False).tolist()) if k > 1 else [0]
        counts[s] = k
    return dict(case=c, cache=_cache(c, pages, g), bt=_dev(bt), cu=_dev(_cu(q_lens)), lens=_dev((base + q_lens).astype(np.int32)),
                path=_dev(path), counts=_dev(counts), host=(bt, base, path, counts))


def _prepare_copy(c, seed):
    rng, n = np.random.default_rng(seed), c["pages"]
    ids = rng.permutation(2 * n + 2).astype(np.int32)
    src, dst = ids[:n].copy(), ids[n:2 * n].copy()
    return dict(case=c, cache=_cache(c, 2 * n + 2, _gen(seed, 4)), src=src, dst=dst, src_dev=_dev(src).long(), dst_dev=_dev(dst).long())


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"tree": _own_tree, "verify": _own_verify, "compact": _own_compact, "copy": _own_copy}[op](s)
    return {"tree": _plain_tree, "verify": _plain_verify, "compact": _plain_compact, "copy": _plain_copy}[op](s)


def _own_tree(s):
    from omniserver_b200 import ops
    c = s["case"]
    return ops.kernels().tree_attention(s["qkv"], s["k"], s["v"], s["bt"], s["cu"], s["lens"], s["mask"], c["nh"], c["nkv"], c["hd"],
                                        c["hd"] ** -0.5, c["window"] or None, s["n_max"], s["kv_max"], DTYPES[c["dtype"]],
                                        depth=s["depth"])


def _own_verify(s):
    from omniserver_b200 import ops
    return ops.kernels().verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["uniform"], s["case"]["nodes"],
                                       s["depth_max"], temperature=s["temp"], draft_probs=s["q"])


def _own_compact(s):
    from omniserver_b200 import ops
    ops.kernels().compact_cache(s["cache"], s["bt"], s["cu"], s["lens"], s["path"], s["counts"])
    return s["cache"]


def _own_copy(s):
    from omniserver_b200 import ops
    ops.kernels().copy_pages(s["cache"], s["src"], s["dst"])
    return s["cache"]


def _plain_tree(s):
    c, N, L = s["case"], s["n_max"], s["kv_max"]
    nh, nkv, hd, page = c["nh"], c["nkv"], c["hd"], c["page"]
    S, grp = c["reqs"], nh // nkv
    cu, lens = s["cu"].long(), s["lens"].long()
    n = cu[1:] - cu[:-1]
    base = lens - n
    pos, node = torch.arange(L, device=DEV), torch.arange(N, device=DEV)
    there = node[None, :] < n[:, None]                                            # [S, N]
    row = (cu[:-1, None] + node[None, :]).clamp(max=s["qkv"].shape[0] - 1)
    pages = s["bt"].long()[:, pos // page].clamp(min=0)                           # [S, L]
    k = s["k"][pages, :, pos % page].float()                                      # [S, L, nkv, hd]
    v = s["v"][pages, :, pos % page].float()
    q = s["qkv"][row][..., :nh * hd].float().view(S, N, nkv, grp, hd)
    # node i sees the committed tokens and the nodes whose bit is set, of these the last `window` positions
    j = pos[None, :] - base[:, None]                                              # [S, L] index among the drafted tokens
    jc = j.clamp(0, N - 1)
    words = s["mask"][row].gather(2, (jc >> 5)[:, None, :].expand(S, N, L))       # [S, N, L]
    drafted = (words >> (jc & 31)[:, None, :]) & 1
    sees = (j < 0)[:, None, :] | ((drafted != 0) & (j < n[:, None])[:, None, :])
    if c["window"]:
        depth = s["depth"].long()[row]                                            # [S, N]
        at = torch.where(j < 0, pos[None, :], base[:, None] + depth.gather(1, jc))
        sees &= at[:, None, :] > (base[:, None] + depth - c["window"])[:, :, None]
    sees &= there[:, :, None]
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(S, nkv, N * grp, hd), k.permute(0, 2, 3, 1)) * hd ** -0.5
    score = score.view(S, nkv, N, grp, L).masked_fill(~sees[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, nkv, N * grp, L), v.permute(0, 2, 1, 3)).view(S, nkv, N, grp, hd)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(S * N, nh * hd).to(DTYPES[c["dtype"]])
    # back to one row per token of the step
    tok = torch.arange(s["qkv"].shape[0], device=DEV)
    req = (tok[:, None] >= cu[None, 1:]).sum(1)
    return o[req * N + tok - cu[req]]


def _plain_verify(s):
    c = s["case"]
    S, n, V, D = c["reqs"], c["nodes"], c["vocab"], s["depth_max"]
    logits, u, tokens = s["logits"].view(S, n, V), s["uniform"].view(S, n).double(), s["tokens"].view(S, n).long()
    q = s["q"].view(S, n, V) if s["q"] is not None else None
    greedy, ids = s["temp"] <= 0, torch.arange(S, device=DEV)

    def distribution(at):
        """The target's probabilities behind node at[s]; a greedy request's is one word. In 64 bits: the running sums of 150,000
        words decide which one is drawn."""
        x = logits[ids, at].double()
        top = x.amax(-1, keepdim=True)
        e = torch.exp((x - top) / torch.where(greedy, 1.0, s["temp"].double())[:, None])
        one = torch.zeros_like(e).scatter_(1, x.argmax(-1, keepdim=True), 1.0)
        return torch.where(greedy[:, None], one, e / e.sum(-1, keepdim=True))

    cur = torch.zeros(S, dtype=torch.long, device=DEV)
    count = torch.ones(S, dtype=torch.long, device=DEV)
    path = torch.full((S, D + 1), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    r = distribution(cur)
    for j in range(1, n):   # parents come before their children: one pass over the nodes meets every node of the walk
        tested = (s["par"][j] == cur) & (count <= D)
        x = tokens[:, j]
        px = r.gather(1, x[:, None])[:, 0]
        if q is None:
            qx, left = torch.ones_like(px), r.scatter(1, x[:, None], 0.0)
        else:
            dq = q[ids, cur].double()
            qx = torch.where(greedy, 1.0, dq.gather(1, x[:, None])[:, 0])
            left = torch.where(greedy[:, None], r, (r - dq).clamp(min=0))
        yes = tested & torch.where(greedy, px > 0, u[:, j] * qx < px)
        total = left.sum(-1, keepdim=True)
        left = torch.where(greedy[:, None] | (total <= 0), r, left / total)
        cur = torch.where(yes, j, cur)
        path.scatter_(1, count.clamp(max=D)[:, None], torch.where(yes, j, path.gather(1, count.clamp(max=D)[:, None])[:, 0])[:, None].to(torch.int32))
        count = count + yes
        r = torch.where(yes[:, None], distribution(cur), torch.where(tested[:, None], left, r))
    # the next word: the first whose running sum passes the root's random number
    run_ = r.cumsum(-1)
    nxt = (run_ <= (u[:, :1] * run_[:, -1:])).sum(-1).clamp(max=V - 1)
    out = torch.where(path >= 0, tokens.gather(1, path.clamp(min=0).long()), -1)
    out = torch.cat([out[:, 1:], torch.full((S, 1), -1, device=DEV)], dim=1)
    out.scatter_(1, (count - 1)[:, None], nxt[:, None])
    return out.to(torch.int32), path, count.to(torch.int32)


def _plain_compact(s):
    c, page = s["case"], s["case"]["page"]
    cu, path, counts = s["cu"].long(), s["path"].long(), s["counts"].long()
    base = s["lens"].long() - (cu[1:] - cu[:-1])
    i = torch.arange(path.shape[1], device=DEV)
    frm = base[:, None] + torch.where(i[None, :] < counts[:, None], path, 0)      # places without a token move the root onto itself
    to = base[:, None] + torch.where(i[None, :] < counts[:, None], i[None, :], 0)
    bt = s["bt"].long()
    a, b = bt.gather(1, frm // page).reshape(-1), bt.gather(1, to // page).reshape(-1)
    moved = s["cache"][:, :, a, :, (frm % page).reshape(-1)]
    s["cache"][:, :, b, :, (to % page).reshape(-1)] = moved
    return s["cache"]


def _plain_copy(s):
    s["cache"][:, :, s["dst_dev"]] = s["cache"][:, :, s["src_dev"]]
    return s["cache"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(c):
    if c["op"] == "tree":
        e, n, b = SIZE[c["dtype"]], _q_lens(c).astype(float), _bases(c).astype(float)
        if c["window"]:
            b = np.minimum(b, c["window"])
        # every visible key and value once, queries and outputs once; a node sees the committed tokens and itself at least
        return {"bytes": float(2 * (b + n).sum() * c["nkv"] * c["hd"] * e + 2 * n.sum() * c["nh"] * c["hd"] * e),
                "flops": float(4 * c["nh"] * c["hd"] * (n * (b + 1)).sum())}
    if c["op"] == "verify":
        # every row of logits once; of the draft's probabilities the row of the node at which a request's walk ends
        rows = c["reqs"] * c["nodes"] + (c["reqs"] if c["dense"] else 0)
        return {"bytes": float(4 * rows * c["vocab"]), "flops": float(6 * rows * c["vocab"])}
    token = c["layers"] * 2 * c["nkv"] * c["hd"] * SIZE[c["dtype"]]
    if c["op"] == "compact":
        # tokens that move are read and written: of a path of k tokens all but the root, k from 1 to its most, evenly
        most = np.minimum(_path_width(c), (_q_lens(c) + 1) // 2)
        return {"bytes": float(2 * token * ((most - 1) / 2).sum() + 4 * c["reqs"]), "flops": 0.0}
    return {"bytes": float(2 * token * c["page"] * c["pages"]), "flops": 0.0}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "verify": _exact_verify, "compact": _exact_compact, "copy": _exact_copy}[case["op"]](s)


def _exact_tree(s):
    c = s["case"]
    nh, nkv, hd, page, win = c["nh"], c["nkv"], c["hd"], c["page"], c["window"]
    if int((s["kv_lens"] * s["q_lens"]).sum()) * nh * hd > 2e11:
        return None
    bt, out, t = s["bt"].cpu().numpy(), [], 0
    for r, parents in enumerate(s["trees"]):
        n, kv = len(parents), int(s["kv_lens"][r])
        base, lines = kv - n, _ancestors(parents)
        where = torch.from_numpy(np.array([bt[r, p // page] * page + p % page for p in range(kv)])).to(DEV)
        keys = s["k"].transpose(1, 2).reshape(-1, nkv, hd)[where].double()
        vals = s["v"].transpose(1, 2).reshape(-1, nkv, hd)[where].double()
        sees = np.zeros((n, kv), dtype=bool)
        for i, line in enumerate(lines):
            sees[i, :base] = True
            sees[i, [base + a for a in line]] = True
            if win:
                at = base + len(line) - 1
                sees[i, :max(0, at - win + 1)] = False
                for a in line:
                    if base + len(lines[a]) - 1 <= at - win:
                        sees[i, base + a] = False
        hidden = torch.from_numpy(~sees).to(DEV)
        q = s["qkv"][t:t + n, :nh * hd].double().view(n, nh, hd)
        heads = []
        for h in range(nh):
            a = q[:, h] @ keys[:, h // (nh // nkv)].T / math.sqrt(hd)
            heads.append(torch.softmax(a.masked_fill(hidden, -math.inf), dim=-1) @ vals[:, h // (nh // nkv)])
        out.append(torch.stack(heads, dim=1).reshape(n, nh * hd))
        t += n
    return torch.cat(out)


def _exact_verify(s):
    c, D = s["case"], s["depth_max"]
    S, n = c["reqs"], c["nodes"]
    temp, u, tok = s["temp"].tolist(), s["uniform"].tolist(), s["tokens"].tolist()
    parents = s["parents"].tolist()[:n]
    words, paths, counts = [], [], []
    for r in range(S):
        node, path = 0, [0]
        while True:
            x = s["logits"][r * n + node].double()
            if temp[r] <= 0:
                p = torch.zeros_like(x)
                p[int(torch.nonzero(x == x.max())[0])] = 1.0
            else:
                p = torch.softmax(x / temp[r], dim=-1)
            kids = [j for j in range(n) if parents[j] == node] if len(path) <= D else []
            found = None
            for j in kids:
                w, px = tok[r * n + j], float(p[tok[r * n + j]])
                if temp[r] <= 0:
                    if px == 1.0:
                        found = j
                        break
                    continue
                if s["q"] is None:
                    if u[r * n + j] < px:
                        found = j
                        break
                    p[w] = 0.0
                else:
                    q = s["q"][r * n + node].double()
                    if u[r * n + j] * float(q[w]) < px:
                        found = j
                        break
                    p = torch.clamp(p - q, min=0.0)
                p = p / p.sum()
            if found is None:
                break
            node = found
            path.append(node)
        total = torch.cumsum(p, 0)
        nxt = int(torch.nonzero(total > u[r * n] * total[-1])[0])
        words.append([tok[r * n + j] for j in path[1:]] + [nxt] + [-1] * (D + 1 - len(path)))
        paths.append(path + [-1] * (D + 1 - len(path)))
        counts.append(len(path))
    return tuple(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (words, paths, counts))


def _exact_compact(s):
    page, (bt, base, path, counts) = s["case"]["page"], s["host"]
    out = s["cache"].clone()
    for r in range(len(base)):
        for i in range(int(counts[r])):
            a, b = int(base[r]) + int(path[r, i]), int(base[r]) + i
            out[:, :, int(bt[r, b // page]), :, b % page] = s["cache"][:, :, int(bt[r, a // page]), :, a % page]
    return out.double()


def _exact_copy(s):
    out = s["cache"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        out[:, :, b] = s["cache"][:, :, a]
    return out.double()
