"""The operators that verify drafted tokens against plain references in 64 bits (tests/plain/speculative.py)."""

import math

import numpy as np
import pytest
import torch

from plain import speculative as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from omniserver_b200 import ops
    return ops.kernels()


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def random_tree(n, rng):
    return [-1] + [int(rng.integers(max(0, (j - 1) // 3), j)) for j in range(1, n)] if n else []


class Step:
    """A batch of trees over a paged cache: everything on the CPU, pages in random order, what no request holds is NaN."""

    def __init__(self, q_lens, bases, nh, nkv, hd, page, dtype, cache_dtype=None, seed=0, extra_cols=0, spare_pages=3, extra_rows=0):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.q_lens, self.bases, self.nh, self.nkv, self.hd, self.page = q_lens, bases, nh, nkv, hd, page
        kv = [b + n for b, n in zip(bases, q_lens)]
        need = [-(-k // page) for k in kv]
        pages = sum(need) + spare_pages
        ids = rng.permutation(pages)
        width = max(need + [1])
        self.bt = torch.full((len(q_lens), width), -1, dtype=torch.int32)
        o = 0
        self.k = torch.full((pages, nkv, page, hd), math.nan)
        self.v = torch.full((pages, nkv, page, hd), math.nan)
        for s, n in enumerate(need):
            self.bt[s, :n] = torch.from_numpy(ids[o:o + n].astype(np.int32))
            o += n
            for p in range(kv[s]):
                at = int(self.bt[s, p // page])
                self.k[at, :, p % page] = torch.randn(nkv, hd, generator=g)
                self.v[at, :, p % page] = torch.randn(nkv, hd, generator=g)
        cache_dtype = cache_dtype or dtype
        self.k, self.v = self.k.to(cache_dtype), self.v.to(cache_dtype)
        T = sum(q_lens) + extra_rows
        self.qkv = torch.randn(T, (nh + 2 * nkv) * hd + extra_cols, generator=g).to(dtype)
        self.cu, self.lens = i32([0] + np.cumsum(q_lens).tolist()), i32(kv)
        self.parents = sum([random_tree(n, rng) for n in q_lens], [])
        from omniserver_b200.ops import CudaKernels
        mask, depth = CudaKernels.tree_plan(self.parents, q_lens)
        self.mask = torch.cat([torch.from_numpy(mask), torch.full((extra_rows, mask.shape[1]), -1, dtype=torch.int32)])
        self.depth = torch.cat([torch.from_numpy(depth), torch.zeros(extra_rows, dtype=torch.int32)])

    def want(self, window=None, scale=None):
        return plain.tree_attention(self.qkv, self.k, self.v, self.bt, self.cu, self.lens, self.mask, self.nh, self.nkv, self.hd,
                                    self.hd ** -0.5 if scale is None else scale, window, self.depth)

    def got(self, window=None, out_dtype=None, scale=None, dev=DEV, **kw):
        return K().tree_attention(self.qkv.to(dev), self.k.to(dev), self.v.to(dev), self.bt.to(dev), self.cu.to(dev), self.lens.to(dev),
                                  self.mask.to(dev), self.nh, self.nkv, self.hd, self.hd ** -0.5 if scale is None else scale, window,
                                  max(self.q_lens), max(int(x) for x in self.lens), out_dtype or self.qkv.dtype,
                                  depth=self.depth.to(dev) if window else None, **kw)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(step, got, want, spread, weight, tensor_cores):
    """|error| against what the roundings can do, A = sum of p |v|:
    * the output is rounded once: half a step of its type, relative to the value;
    * a score is a sum of hd products in 32 bits, scaled: off by at most (hd + 2) 2^-24 times sum |q k| scale, which moves its
      weight by that much relatively, and the sum of weights by no more: twice that times A. The tensor cores' sums are taken to
      round like that too, or to truncate (twice as much);
    * the exponential is right to 2 units in the last place (32 bits) or 2^-22 plus its argument's rounding, at most 2^-24 times
      the largest argument, which is at most twice `weight` (tensor cores);
    * sums over the keys in 32 bits: at most one rounding per key, for A and for the total;
    * the tensor-core kernel rounds a weight to bf16 before the product with V: half a step of bf16 times A."""
    kv = max(int(x) for x in step.lens)
    u = 2.0 ** -24
    rel = 2 * (step.hd + 2) * u * weight * (2 if tensor_cores else 1) + 2 * (4 + 4 * weight) * u + 2 * (kv + 40) * u
    if tensor_cores:
        rel += half_step(BF16)
    rows = sum(step.q_lens)
    err = (got.double().cpu() - want)[:rows].abs()
    bound = half_step(got.dtype) * want[:rows].abs() + rel * (1 + half_step(got.dtype)) * spread[:rows] + 1e-30
    assert got[:rows].isfinite().all()
    worst = (err / bound).max()
    assert worst <= 1, f"error {float(worst):.3g} times what the roundings can do"
    K().check_device_errors()


def runs_on_tensor_cores(step, exact=False):
    return (not exact and step.qkv.dtype == BF16 and step.k.dtype == BF16 and step.hd in (64, 128) and step.page >= 8
            and step.page & (step.page - 1) == 0)


BATCHES = [
    ([1], [0]), ([1], [1]), ([3], [0]), ([1], [700]), ([16], [1000]), ([5, 1, 0, 9], [37, 128, 50, 0]), ([33], [256]), ([64, 2], [127, 129]),
    ([20, 7, 1], [255, 600, 64]), ([130], [300]),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,hd", [(12, 2, 128), (4, 4, 64), (7, 1, 128), (6, 2, 20), (2, 1, 256), (3, 1, 80)])
@pytest.mark.parametrize("q_lens,bases", BATCHES)
def test_tree_attention(q_lens, bases, nh, nkv, hd, dtype):
    step = Step(q_lens, bases, nh, nkv, hd, 16, dtype, seed=len(q_lens) + hd)
    before = K().counts["attn_tree_tc"]
    got = step.got()
    assert K().counts["attn_tree_tc"] - before == (1 if runs_on_tensor_cores(step) else 0)
    check(step, got, *step.want(), runs_on_tensor_cores(step))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 5, 8, 32, 64, 128, 256])
def test_tree_attention_page_sizes(page, dtype):
    step = Step([9, 17, 1], [130, 63, 300], 4, 2, 64, page, dtype, seed=page)
    check(step, step.got(), *step.want(), runs_on_tensor_cores(step))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 2, 5, 16, 100, 129, 5000])
def test_tree_attention_windows(window, dtype):
    step = Step([12, 1, 30], [200, 77, 0], 4, 2, 64, 16, dtype, seed=window)
    # pages that every row's window has passed were given back
    for s, b in enumerate(step.bases):
        for pi in range(max(0, b - window + 1) // 16):
            step.bt[s, pi] = -1
    check(step, step.got(window), *step.want(window), runs_on_tensor_cores(step))


@pytest.mark.parametrize("qd,cd,od", [(F32, BF16, F32), (BF16, F32, BF16), (BF16, BF16, F32), (F32, F32, BF16)])
def test_tree_attention_mixed_types(qd, cd, od):
    step = Step([12, 3], [90, 5], 6, 2, 64, 16, qd, cd, seed=3)
    check(step, step.got(out_dtype=od), *step.want(), False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("grp", [1, 2, 3, 5, 8, 11, 16, 29, 64, 127, 128, 130])
def test_tree_attention_group_sizes(grp, dtype):
    step = Step([5, 2], [40, 150], grp, 1, 64, 16, dtype, seed=grp)
    check(step, step.got(), *step.want(), runs_on_tensor_cores(step) and grp <= 128)


def test_tree_attention_long_requests_beside_shorter_ones():
    """The 32-bit kernel cuts 8,000 keys into more ranges than 8,200."""
    step = Step([3, 2, 1], [8197, 7998, 10], 2, 1, 64, 64, F32, seed=1)
    check(step, step.got(), *step.want(), False)
    one = Step([3, 2, 1], [8197, 7998, 10], 2, 1, 64, 64, BF16, seed=1)
    check(one, one.got(), *one.want(), True)
    check(one, one.got(exact=True), *one.want(), False)


def test_tree_attention_32_bits_does_not_depend_on_the_batch():
    step = Step([6, 9, 1], [700, 20, 300], 4, 2, 64, 16, F32, seed=5)
    whole = step.got()
    for s in range(3):
        one = Step([6, 9, 1], [700, 20, 300], 4, 2, 64, 16, F32, seed=5)
        a, b = int(step.cu[s]), int(step.cu[s + 1])
        one.qkv, one.mask, one.depth, one.bt = step.qkv[a:b], step.mask[a:b], step.depth[a:b], step.bt[s:s + 1]
        one.cu, one.lens, one.q_lens = i32([0, b - a]), step.lens[s:s + 1], [b - a]
        assert torch.equal(one.got(), whole[a:b])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_repeats_its_bits(dtype):
    step = Step([16, 40, 3], [900, 20, 300], 12, 2, 128, 32, dtype, seed=8)
    first = step.got()
    for _ in range(3):
        assert torch.equal(step.got(), first)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_rows_that_see_nothing_are_zero(dtype):
    step = Step([5, 3], [0, 0], 4, 2, 64, 16, dtype, seed=2)
    step.mask[1] = 0
    step.mask[6] = 1 << 3          # a bit beyond its request's nodes
    got, (want, spread, weight) = step.got(), step.want()
    assert not got[1].any() and not got[6].any() and got[0].any()
    check(step, got, want, spread, weight, runs_on_tensor_cores(step))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_any_mask(dtype):
    """Not only ancestors: any set of nodes, later ones too, and bits beyond the request's nodes, which do not count."""
    step = Step([40, 1, 7], [100, 128, 3], 6, 2, 128, 16, dtype, seed=4)
    g = torch.Generator().manual_seed(9)
    step.mask = torch.randint(-2**31, 2**31 - 1, step.mask.shape, generator=g).to(torch.int32)
    check(step, step.got(), *step.want(), runs_on_tensor_cores(step))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_tree_attention_does_not_look_at_hidden_places(dtype, what, where):
    """What a branch's siblings hold does not reach it, whatever it is; the rows that see it go by the formula."""
    step = Step([24, 5], [120, 250], 6, 2, 128, 16, dtype, seed=6)
    leaf = [j for j in range(1, 24) if j not in step.parents[:24]][0]
    clean, spread, weight = step.want()
    place = 120 + leaf
    getattr(step, where)[int(step.bt[0, place // 16]), :, place % 16, ::3] = what
    got = step.got()
    rows = [t for t in range(29) if t != leaf]
    ref = Step([24, 5], [120, 250], 6, 2, 128, 16, dtype, seed=6)
    ref_got = ref.got()
    assert torch.equal(got[rows], ref_got[rows])
    mine, plain_row = got[leaf].double().cpu(), step.want()[0][leaf]
    if where == "v":
        assert torch.equal(mine.isfinite(), plain_row.isfinite())
        assert torch.equal(mine.isnan(), plain_row.isnan())
        assert torch.equal(mine[~mine.isfinite() & ~mine.isnan()], plain_row[~mine.isfinite() & ~mine.isnan()])
        ok = mine.isfinite()
        assert torch.allclose(mine[ok], clean[leaf][ok], rtol=2 ** -6, atol=float(2 ** -6 * spread[leaf].max()))
    K().check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [7, 40])
def test_tree_attention_does_not_look_behind_a_window(dtype, window):
    step = Step([12], [200], 4, 2, 64, 16, dtype, seed=7)
    ref = step.got(window)
    seen = [p for p in range(200) if p > 200 - window]
    for p in range(200):
        if p not in seen:
            step.k[int(step.bt[0, p // 16]), :, p % 16] = math.nan
            step.v[int(step.bt[0, p // 16]), :, p % 16] = math.inf
    # places that only the shallow nodes see
    deep = int(step.depth.max())
    assert deep >= 2
    step.v[int(step.bt[0, (200 - window + 1) // 16]), :, (200 - window + 1) % 16] = math.nan
    got = step.got(window)
    for t in range(12):
        if int(step.depth[t]) == 0:
            assert got[t].isnan().all()
        else:
            assert torch.equal(got[t], ref[t])
    K().check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_leaves_other_rows_alone(dtype):
    step = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=1, extra_rows=6, extra_cols=8)
    out = torch.full((20, 4 * 64), 7.0, dtype=dtype, device=DEV)
    got = step.got(out=out)
    assert got is out and (got[14:] == 7.0).all()
    check(step, got, *step.want(), runs_on_tensor_cores(step))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [1, 3, 8])
def test_tree_attention_row_strides(dtype, cols):
    step = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=cols, extra_cols=cols)
    check(step, step.got(), *step.want(), runs_on_tensor_cores(step) and cols % 8 == 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.5, 0.0, -0.2])
def test_tree_attention_scales(dtype, scale):
    step = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=2)
    check(step, step.got(scale=scale), *step.want(scale=scale), runs_on_tensor_cores(step) and scale > 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [-1, 99])
def test_tree_attention_reports_a_page_outside_the_pool(dtype, bad):
    from omniserver_b200.ops import KernelError
    step = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=2)
    ref = step.got()
    step.bt[0, 0] = bad
    got = step.got()
    with pytest.raises(KernelError, match="outside the page pool"):
        K().check_device_errors()
    assert torch.equal(got[5:14], ref[5:14])       # the other request
    K().check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_reports_bounds_that_are_too_small(dtype):
    from omniserver_b200.ops import KernelError
    s = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=2)
    d = [t.to(DEV) for t in (s.qkv, s.k, s.v, s.bt, s.cu, s.lens, s.mask)]
    for most_q, most_kv in ((8, 149), (9, 148)):
        out = K().tree_attention(*d, 4, 2, 64, 0.125, None, most_q, most_kv, dtype)
        with pytest.raises(KernelError, match="more nodes or keys"):
            K().check_device_errors()
        ref = s.got()
        assert torch.equal(out[:5], ref[:5]) or dtype == BF16
    bt = d[3][:, :9].contiguous()
    K().tree_attention(*d[:3], bt, *d[4:], 4, 2, 64, 0.125, None, 9, 149, dtype)
    with pytest.raises(KernelError, match="more nodes or keys"):
        K().check_device_errors()


def test_tree_attention_refuses():
    from omniserver_b200.ops import KernelError
    s = Step([5, 9], [30, 140], 4, 2, 64, 16, F32, seed=2)
    good = dict(qkv=s.qkv, k_cache=s.k, v_cache=s.v, block_table=s.bt, cu_q=s.cu, seq_lens=s.lens, tree_mask=s.mask)
    good = {n: t.to(DEV) for n, t in good.items()}
    args = dict(nh=4, nkv=2, hd=64, scale=0.125, window=None, max_q_len=9, max_kv_len=149, out_dtype=F32)
    K().tree_attention(**good, **args)
    for over, match in [
        (dict(qkv=s.qkv), "CUDA tensor"), (dict(qkv=good["qkv"].t().contiguous().t()), "contiguous"),
        (dict(seq_lens=good["seq_lens"].long()), "int32"), (dict(nh=3), "multiple"), (dict(nh=64), "columns"), (dict(hd=32), "caches"),
        (dict(v_cache=good["v_cache"].bfloat16()), "caches"), (dict(block_table=good["block_table"][:1]), "block_table"),
        (dict(cu_q=good["cu_q"][:2]), "cu_q"), (dict(tree_mask=good["tree_mask"][:3]), "tree_mask"), (dict(max_q_len=33), "tree_mask"),
        (dict(window=3), "depth"), (dict(window=-3), "window"), (dict(window=3, depth=good["seq_lens"]), "depth"),
        (dict(qkv=good["qkv"].half()), "float32 or bfloat16"), (dict(out=torch.empty(3, 3, device=DEV)), "out"),
    ]:
        with pytest.raises(KernelError, match=match):
            K().tree_attention(**{**good, **args, **over})
    empty = K().tree_attention(**{**good, **args, "max_q_len": 0})
    assert empty.shape == (14, 256)


# ------------------------------------------------------------------ verification
def drafts(q_lens, V, seed, branch=2, peak=4.0, dense=False, repeat=False):
    """Logits, tokens, parents, uniforms and (dense) draft probabilities; children often carry their parent's best words."""
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    T = sum(q_lens)
    logits = torch.randn(T, V, generator=g) * peak
    parents, tokens = [], torch.randint(0, V, (T,), generator=g).to(torch.int32)
    t0 = 0
    for n in q_lens:
        par = [-1] + [int(rng.integers((j - 1) // branch, j)) for j in range(1, n)] if n else []
        parents += par
        seen = {}
        for j in range(1, n):
            k = seen.get(par[j], 0)
            seen[par[j]] = 0 if repeat else k + 1
            best = torch.topk(logits[t0 + par[j]], min(V, 4)).indices
            tokens[t0 + j] = best[min(k, len(best) - 1)]
        t0 += n
    q = torch.softmax(logits + torch.randn(T, V, generator=g), dim=-1) if dense else None
    if dense:
        t0 = 0
        for n in q_lens:
            for j in range(1, n):
                tokens[t0 + j] = int(torch.multinomial(q[t0 + parents[t0 + j]], 1, generator=g))
            t0 += n
    u = torch.randint(0, 1 << 24, (T,), generator=g).float() / (1 << 24)
    return dict(logits=logits, tokens=tokens, parents=i32(parents).view(T), cu_q=i32([0] + np.cumsum(q_lens).tolist()), uniform=u), q


def verify_both(args, most, depth, temperature=None, q=None):
    dev = {n: t.to(DEV) for n, t in args.items()}
    got = K().verify_drafts(**dev, max_q_len=most, max_depth=depth, temperature=None if temperature is None else temperature.to(DEV),
                            draft_probs=None if q is None else q.to(DEV))
    want = plain.verify(args["logits"], args["tokens"], args["parents"], args["cu_q"], args["uniform"], depth, temperature, q)
    return [list(x) for x in zip(got[0].tolist(), got[1].tolist(), got[2].tolist())], [list(w) for w in want]


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("V", [1, 2, 50, 1001, 4096, 4097, 20000, 151936])
@pytest.mark.parametrize("q_lens", [[1], [6], [4, 0, 17, 1, 2], [40, 3]])
def test_verify(q_lens, V, dense):
    if V > 100000 and sum(q_lens) > 24:
        q_lens = [12, 3]
    args, q = drafts(q_lens, V, seed=V + len(q_lens) + 2 * dense, dense=dense)
    for t, name in ((None, "greedy"), (0.9, "sampled"), (0.0, "mixed")):
        temp = None if t is None else torch.tensor([1.3 if (name == "mixed" and s % 2) else t for s in range(len(q_lens))])
        got, want = verify_both(args, max(q_lens), 5, temp, q)
        assert got == want, name
    K().check_device_errors()


@pytest.mark.parametrize("dense", [False, True])
def test_verify_many_random_walks(dense):
    accepted = 0
    for seed in range(12):
        q_lens = [7, 12, 3, 20]
        args, q = drafts(q_lens, 3000, seed=100 + seed, branch=3, peak=3.0, dense=dense, repeat=seed % 3 == 0)
        got, want = verify_both(args, 20, 6, torch.tensor([0.7, 1.0, 1.5, 0.3]), q)
        assert got == want, seed
        accepted += sum(x[2] - 1 for x in got)
    assert accepted > 20


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("depth", [0, 1, 3])
def test_verify_stops_at_max_depth(depth, dense):
    args, q = drafts([8], 500, seed=1, branch=1, peak=30.0, dense=dense)
    got, want = verify_both(args, 8, depth, torch.tensor([1.0]), q)
    assert got == want and len(got[0][0]) == depth + 1


@pytest.mark.parametrize("dense", [False, True])
def test_verify_random_numbers_at_their_ends(dense):
    for u in (0.0, 1.0 - 2.0 ** -24):
        args, q = drafts([9, 4], 5000, seed=3, dense=dense)
        args["uniform"] = torch.full_like(args["uniform"], u)
        got, want = verify_both(args, 9, 4, torch.tensor([1.0, 0.5]), q)
        assert got == want


def test_verify_random_number_passes_the_last_word():
    """u times the total, rounded, can be the total: the last word with weight is taken, not one behind it."""
    logits = torch.full((1, 6000), -math.inf)
    logits[0, [5, 77, 4500]] = 0.0
    args = dict(logits=logits, tokens=i32([0]), parents=i32([-1]), cu_q=i32([0, 1]), uniform=torch.tensor([1.0]))
    got, _ = verify_both(args, 1, 0, torch.tensor([1.0]))
    assert got == [[[4500], [0], 1]]


@pytest.mark.parametrize("dense", [False, True])
def test_verify_infinite_and_missing_logits(dense):
    V = 9000
    args, q = drafts([3, 3, 3, 3], V, seed=5, branch=1, dense=dense)
    lg = args["logits"]
    lg[0] = -math.inf                                   # nothing to accept, nothing to draw: word 0
    lg[3, ::2] = math.nan
    lg[6, [8, 5000]] = math.inf                         # two words share everything
    args["tokens"][7] = 5000
    lg[9, 10:] = -math.inf
    for temp in (None, torch.tensor([1.0, 0.8, 0.7, 1.2])):
        got, want = verify_both(args, 3, 2, temp, q)
        assert got == want
    assert got[0] == [[0, -1, -1], [0, -1, -1], 1]
    lg.fill_(math.nan)
    got, want = verify_both(args, 3, 2, torch.ones(4), q)
    assert got == want and all(x[0][0] == 0 and x[2] == 1 for x in got)


@pytest.mark.parametrize("gaps", [(0.0, 1e-3), (0.0, 1e-7), (0.0, 0.1, 1e-4), (0.0, 1e-5, 1e-9), (0.0, 1e-12)])
@pytest.mark.parametrize("together", [True, False])
def test_verify_what_is_left_of_dominant_words(gaps, together):
    """A few words hold nearly everything and are all rejected: what is left, down to 10^-12 of the row, keeps its digits."""
    V, S = 30000, 24
    g = torch.Generator().manual_seed(11)
    words = [5000 + 3 * i if together else 700 + 5000 * i for i in range(len(gaps))]
    rows = torch.randn(S, V, generator=g) * 2.0
    rest = torch.logsumexp(rows.double(), -1)
    for i, gap in enumerate(gaps):
        nxt = gaps[i + 1] if i + 1 < len(gaps) else None
        # word i outweighs everything behind it by 1 / (what is left next)
        rows[:, words[i]] = (rest + sum(-math.log(x) for x in gaps[i + 1:]) if nxt else rest - 60).float()
    n = len(gaps)
    logits = torch.zeros(S * n, V)
    logits[::n] = rows
    tokens = i32(([0] + words[:n - 1]) * S)
    u = torch.rand(S * n, generator=g)
    u = (torch.floor(u * 2 ** 24) / 2 ** 24).float()
    for k in range(1, n):
        u[k::n] = 1.0 - 2.0 ** -24            # rejected wherever it can be
    args = dict(logits=logits, tokens=tokens, parents=i32(([-1] + [0] * (n - 1)) * S), cu_q=i32(list(range(0, S * n + 1, n))), uniform=u)
    got, want = verify_both(args, n, 1, torch.ones(S))
    assert got == want


def test_verify_equal_distributions_accept_everything():
    args, q = drafts([9], 4000, seed=6, branch=1, dense=True)
    q = torch.softmax(args["logits"].double(), -1)
    # a word's probability rounded down, so that no rejection is possible: u q < q <= r
    q32 = q.float()
    q32 = torch.where(q32.double() > q * (1 - 1e-6), q32 * (1 - 2.0 ** -18), q32)
    got, want = verify_both(args, 9, 8, torch.tensor([1.0]), q32)
    assert got == want and got[0][2] == 9


def test_verify_bad_draft_entries_count_as_zero():
    args, q = drafts([6, 4], 700, seed=8, branch=2, dense=True)
    q[:, ::5] = math.nan
    q[:, 1::7] = -0.5
    got, want = verify_both(args, 6, 3, torch.tensor([1.0, 0.9]), q)
    assert got == want


def test_verify_ties_go_to_the_lowest_index():
    logits = torch.zeros(2, 10000)
    logits[0, [4095, 4096, 9000]] = 3.0
    args = dict(logits=logits, tokens=i32([0, 4095]), parents=i32([-1, 0]), cu_q=i32([0, 2]), uniform=torch.tensor([0.5, 0.5]))
    got, want = verify_both(args, 2, 1)
    assert got == want == [[[4095, 0], [0, 1], 2]]


def test_verify_reports_a_token_outside_the_vocabulary():
    from omniserver_b200.ops import KernelError
    for dense in (False, True):
        args, q = drafts([4, 4], 9000, seed=9, branch=3, dense=dense)
        args["tokens"][1], args["tokens"][6] = 9000, -2
        args["tokens"][4] = -7            # a root's token is not looked at
        got, want = verify_both(args, 4, 3, torch.tensor([1.0, 1.0]), q)
        with pytest.raises(KernelError, match="outside the vocabulary reached the verification"):
            K().check_device_errors()
        assert got == want
    K().check_device_errors()


def test_verify_parents_that_are_none():
    """Parents that are not smaller than their child, or negative, belong to no walk."""
    args, _ = drafts([6], 300, seed=10, branch=1, peak=30.0)
    args["parents"] = i32([-1, 0, 2, 5, -1, 99])
    got, want = verify_both(args, 6, 5, torch.tensor([1.0]))
    assert got == want
    K().check_device_errors()


@pytest.mark.parametrize("n", [300, 1024])
def test_verify_large_trees(n):
    args, _ = drafts([n, 5], 64, seed=n, branch=1, peak=200.0)
    got, want = verify_both(args, n, n - 1, torch.tensor([1.0, 1.0]))
    assert got == want and got[0][2] > 100
    got, want = verify_both(args, n, 700, None)
    assert got == want


def test_verify_follows_the_targets_distribution():
    """Whatever the draft is, the first emitted token is distributed like the target: 20,000 walks over 8 words, each with its own
    random numbers. A count's standard deviation is at most sqrt(N / 4): 6 of them."""
    N, V = 20000, 8
    g = torch.Generator().manual_seed(1)
    target, draft = torch.randn(V, generator=g), torch.softmax(torch.randn(V, generator=g), 0)
    for dense in (False, True):
        logits = target.expand(2 * N, V).contiguous()
        tokens = torch.zeros(2 * N, dtype=torch.int32)
        tokens[1::2] = torch.multinomial(draft, N, replacement=True, generator=g).to(torch.int32)
        u = torch.randint(0, 1 << 24, (2 * N,), generator=g).float() / (1 << 24)
        new, _, count = K().verify_drafts(logits.to(DEV), tokens.to(DEV), i32([-1, 0] * N).to(DEV), torch.arange(0, 2 * N + 1, 2, dtype=torch.int32).to(DEV),
                                          u.to(DEV), 2, 1, torch.ones(N, device=DEV), draft.expand(2 * N, V).contiguous().to(DEV) if dense else None)
        p = torch.softmax(target.double(), 0)
        first = torch.bincount(new[:, 0].cpu(), minlength=V).double()
        assert ((first - N * p).abs() <= 6 * math.sqrt(N / 4)).all()
        assert 0 < int((count == 2).sum()) < N


def test_verify_refuses():
    from omniserver_b200.ops import KernelError
    args, q = drafts([4, 4], 100, seed=1, dense=True)
    good = {n: t.to(DEV) for n, t in args.items()}
    rest = dict(max_q_len=4, max_depth=3, temperature=torch.ones(2, device=DEV), draft_probs=q.to(DEV))
    K().verify_drafts(**good, **rest)
    for over, match in [
        (dict(logits=args["logits"]), "CUDA tensor"), (dict(logits=good["logits"].bfloat16()), "float32"),
        (dict(tokens=good["tokens"].long()), "int32"), (dict(tokens=good["tokens"][:3]), "tokens"), (dict(uniform=good["uniform"][:3]), "uniform"),
        (dict(parents=good["parents"][:3]), "parents"), (dict(max_q_len=1025), "nodes"), (dict(max_q_len=-1), "nodes"),
        (dict(max_depth=-1), "max_depth"), (dict(temperature=torch.ones(3, device=DEV)), "temperature"),
        (dict(draft_probs=q[:, :50].contiguous().to(DEV)), "draft_probs"), (dict(logits=good["logits"][:, :0]), "vocabulary"),
    ]:
        with pytest.raises(KernelError, match=match):
            K().verify_drafts(**{**good, **rest, **over})
    new, path, count = K().verify_drafts(good["logits"][:0], good["tokens"][:0], good["parents"][:0], i32([0, 0]).to(DEV),
                                         good["uniform"][:0], 0, 1)
    assert new.tolist() == [[-1, -1]] and path.tolist() == [[-1, -1]] and count.tolist() == [0]


# ------------------------------------------------------------------ cache
def paged(kv_lens, layers, nkv, page, hd, dtype, seed=0):
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    need = [-(-k // page) for k in kv_lens]
    ids = rng.permutation(sum(need) + 2)
    bt = torch.full((len(kv_lens), max(need)), -1, dtype=torch.int32)
    o = 0
    for s, n in enumerate(need):
        bt[s, :n] = torch.from_numpy(ids[o:o + n].astype(np.int32))
        o += n
    return torch.randn(layers, 2, sum(need) + 2, nkv, page, hd, generator=g).to(dtype), bt


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layers,nkv,page,hd", [(3, 2, 16, 128), (1, 1, 1, 20), (2, 3, 5, 7), (28, 4, 32, 64), (2, 1, 64, 33)])
def test_compact_cache(layers, nkv, page, hd, dtype):
    q_lens, bases = [9, 1, 30, 12, 0, 300], [37, 5, 0, 63, 10, 3]
    kv = [a + b for a, b in zip(q_lens, bases)]
    cache, bt = paged(kv, layers, nkv, page, hd, dtype, seed=hd)
    paths = [[0, 2, 3, 8], [0], list(range(0, 30, 2)), [0, 1, 2], [], [i for i in range(300) if i % 7 != 3]]
    path = torch.full((6, 300), -9, dtype=torch.int32)
    for s, p in enumerate(paths):
        path[s, :len(p)] = i32(p)
    count, cu, lens = i32([len(p) for p in paths]), i32([0] + np.cumsum(q_lens).tolist()), i32(kv)
    want = plain.compact(cache, bt, cu, lens, path, count)
    dev = cache.to(DEV)
    K().compact_cache(dev, bt.to(DEV), cu.to(DEV), lens.to(DEV), path.to(DEV), count.to(DEV))
    assert torch.equal(dev.cpu(), want)
    K().check_device_errors()


@pytest.mark.parametrize("bad", [[0, 2, 2], [0, 3, 1], [-1, 2, 3], [0, 2, 9], [3, 2, 1]])
def test_compact_cache_reports_bad_paths_and_moves_nothing(bad):
    from omniserver_b200.ops import KernelError
    cache, bt = paged([20, 20], 2, 2, 8, 16, F32)
    path, cu, lens = i32([bad, [0, 2, 4]]), i32([0, 9, 18]), i32([20, 20])
    dev = cache.to(DEV)
    K().compact_cache(dev, bt.to(DEV), cu.to(DEV), lens.to(DEV), path.to(DEV), i32([3, 3]).to(DEV))
    with pytest.raises(KernelError, match="does not ascend"):
        K().check_device_errors()
    assert torch.equal(dev.cpu(), plain.compact(cache, bt, cu, lens, path, i32([0, 3])))
    for counts, starts in (([4, 0], [20, 20]), ([-3, 0], [20, 20]), ([3, 0], [5, 20])):
        dev = cache.to(DEV)
        K().compact_cache(dev, bt.to(DEV), cu.to(DEV), i32(starts).to(DEV), i32([[0, 2, 4], [0, 2, 4]]).to(DEV), i32(counts).to(DEV))
        if counts[0] < 0:
            K().check_device_errors()          # no tokens: nothing to move
        else:
            with pytest.raises(KernelError, match="does not ascend"):
                K().check_device_errors()
        assert torch.equal(dev.cpu(), cache)


@pytest.mark.parametrize("bad", [-1, 77])
def test_compact_cache_reports_pages_outside_the_pool(bad):
    from omniserver_b200.ops import KernelError
    cache, bt = paged([20, 20], 2, 2, 8, 16, F32)
    cu, lens, path = i32([0, 9, 18]), i32([20, 20]), i32([[0, 2, 8], [0, 2, 4]])
    broken = bt.clone()
    broken[0, 2] = bad                        # holds places 16 to 19: node 8 of request 0 lies at 11 + 8
    dev = cache.to(DEV)
    K().compact_cache(dev, broken.to(DEV), cu.to(DEV), lens.to(DEV), path.to(DEV), i32([3, 3]).to(DEV))
    with pytest.raises(KernelError, match="outside the page pool"):
        K().check_device_errors()
    assert torch.equal(dev.cpu(), plain.compact(cache, bt, cu, lens, path, i32([2, 3])))


def test_compact_cache_refuses():
    from omniserver_b200.ops import KernelError
    cache, bt = paged([20, 20], 2, 2, 8, 16, F32)
    good = dict(cache=cache, block_table=bt, cu_q=i32([0, 9, 18]), seq_lens=i32([20, 20]), path=i32([[0, 1], [0, 1]]), count=i32([2, 2]))
    good = {n: t.to(DEV) for n, t in good.items()}
    K().compact_cache(**good)
    for over, match in [(dict(cache=cache), "CUDA tensor"), (dict(cache=good["cache"][0]), "cache"), (dict(cache=good["cache"].half()), "float32"),
                        (dict(path=good["path"][0]), "path"), (dict(count=good["count"][:1]), "count"), (dict(cu_q=good["cu_q"][:2]), "cu_q"),
                        (dict(block_table=good["block_table"][:1]), "block_table"), (dict(path=good["path"].long()), "int32")]:
        with pytest.raises(KernelError, match=match):
            K().compact_cache(**{**good, **over})


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layers,nkv,page,hd,n", [(3, 2, 16, 128, 5), (1, 1, 1, 3, 2), (2, 3, 5, 7, 4), (28, 4, 32, 128, 1), (1, 1, 2, 4, 300)])
def test_copy_pages(layers, nkv, page, hd, n, dtype):
    cache, _ = paged([page * (2 * n + 1)], layers, nkv, page, hd, dtype, seed=n)
    ids = np.random.default_rng(n).permutation(2 * n + 2)
    src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
    if n > 3:
        src[1] = src[0]           # one source may go to several places
    dev = cache.to(DEV)
    K().copy_pages(dev, src, dst)
    want = cache.clone()
    want[:, :, dst] = cache[:, :, src]
    assert torch.equal(dev.cpu(), want)
    K().copy_pages(dev, np.array(dst), tuple(src) if len(set(src)) == n else torch.tensor(ids[:n]))
    K().copy_pages(dev, [], [])


def test_copy_pages_refuses():
    from omniserver_b200.ops import KernelError
    cache = paged([40], 2, 2, 8, 16, F32)[0].to(DEV)
    before = cache.clone()
    for src, dst, match in [([0], [7], "outside the pool"), ([-1], [1], "outside the pool"), ([0.5], [1], "whole"), ([0, 1], [2, 2], "every destination once"),
                            ([0, 1], [1, 2], "none of them a source"), ([0], [0], "none of them a source"), ([0, 1], [2], "as many"),
                            ([[0]], [[1]], "whole"), (torch.tensor([0], device=DEV), [1], "whole")]:
        with pytest.raises(KernelError, match=match):
            K().copy_pages(cache, src, dst)
    with pytest.raises(KernelError, match="CUDA tensor"):
        K().copy_pages(cache.cpu(), [0], [1])
    assert torch.equal(cache, before)
