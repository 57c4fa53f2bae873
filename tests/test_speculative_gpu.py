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


@pytest.mark.parametrize("dense", [False, True])
def test_verify_reports_a_request_with_more_nodes_than_the_call_allowed(dense):
    from omniserver_b200.ops import KernelError
    args, q = drafts([4, 9], 300, seed=9, branch=1, dense=dense)
    temp = torch.ones(2)
    _, whole = verify_both(args, 9, 8, temp, q)
    dev = {n: t.to(DEV) for n, t in args.items()}
    got = K().verify_drafts(**dev, max_q_len=8, max_depth=8, temperature=temp.to(DEV), draft_probs=None if q is None else q.to(DEV))
    with pytest.raises(KernelError, match="more nodes or keys"):
        K().check_device_errors()
    assert got[0][0].tolist() == whole[0][0] and got[1][0].tolist() == whole[0][1]
    K().check_device_errors()


@pytest.mark.parametrize("temp", [1e-38, 1e-12, 1e-8, 1e-7, 1e-6, 1e-5, 1e5, 1e30, math.inf])
def test_verify_extreme_temperatures(temp):
    """Logits with ties at the top. (The oracle takes 1e38 for infinity: behind that a difference of ordinary logits is nothing either way.)"""
    args, _ = drafts([6, 5], 3001, seed=3)
    args["logits"].clamp_(-12, 12)
    got = K().verify_drafts(**{n: t.to(DEV) for n, t in args.items()}, max_q_len=6, max_depth=5, temperature=torch.full((2,), temp, device=DEV))
    want = plain.verify(args["logits"], args["tokens"], args["parents"], args["cu_q"], args["uniform"], 5, torch.full((2,), min(temp, 1e38)))
    assert [list(x) for x in zip(got[0].tolist(), got[1].tolist(), got[2].tolist())] == [list(w) for w in want]
    K().check_device_errors()


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("top", [3e6, 5e6])
def test_verify_slices_of_very_different_size(top, dense):
    """Logits a little apart around `top`, where m c rounds by halves, beside slices of small ones and of ones just below: with c = log2(e),
    the maxima lie on both sides of 2^22."""
    g = torch.Generator().manual_seed(6)
    V = 4 * 1024
    args, q = drafts([5, 4], V, seed=8, dense=dense)
    x = torch.randn(9, V, generator=g)
    x[:, :1024] = top + torch.randint(-3, 4, (9, 1024), generator=g) * 0.5
    x[:, 2 * 1024:][:, :1024] = top * 0.9999995 + torch.randint(-3, 4, (9, 1024), generator=g) * 0.5
    args["logits"] = x
    for j in range(1, 9):
        args["tokens"][j] = int(torch.randint(0, 1024, (1,), generator=g))
    got, want = verify_both(args, 5, 4, torch.ones(2), q)
    assert got == want
    K().check_device_errors()


# ------------------------------------------------------------------ streams, graphs, devices, and a step as a whole
def device_step(step):
    d = {n: getattr(step, n).to(DEV) for n in ("qkv", "k", "v", "bt", "cu", "lens", "mask", "depth")}

    def call(out=None):
        return K().tree_attention(d["qkv"], d["k"], d["v"], d["bt"], d["cu"], d["lens"], d["mask"], step.nh, step.nkv, step.hd,
                                  step.hd ** -0.5, None, max(step.q_lens), max(int(x) for x in step.lens), step.qkv.dtype, out=out)
    return d, call


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_on_two_streams_at_once(dtype):
    """Calls on two streams, interleaved, share nothing: each gives what it gives alone."""
    big = device_step(Step([40, 9, 17], [2500, 700, 30], 12, 2, 128, 32, dtype, seed=1))[1]
    small = device_step(Step([5, 1], [300, 900], 12, 2, 128, 32, dtype, seed=2))[1]
    want = big(), small()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, f in enumerate((big, small)):
            with torch.cuda.stream(streams[i]):
                got[i].append(f())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    K().check_device_errors()


def test_verify_on_two_streams_at_once():
    calls, want = [], []
    for seed, q_lens in ((1, [9, 4, 30]), (2, [6])):
        args, q = drafts(q_lens, 30000, seed=seed, dense=True)
        dev = {n: t.to(DEV) for n, t in args.items()}
        temp, qd = torch.full((len(q_lens),), 0.9, device=DEV), q.to(DEV)
        calls.append(lambda dev=dev, temp=temp, qd=qd, n=max(q_lens): K().verify_drafts(**dev, max_q_len=n, max_depth=5, temperature=temp, draft_probs=qd))
        want.append([t.clone() for t in calls[-1]()])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(calls[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))
    K().check_device_errors()


def test_captured_calls_replay_with_new_data():
    """Two graphs of the calls, captured one after the other, replayed in turn with other lengths, masks, logits and paths in the
    same buffers."""
    steps = [Step([20, 7, 3], b, 12, 2, 128, 32, BF16, seed=5) for b in ([900, 40, 333], [10, 500, 800], [0, 1000, 64])]
    # one pool of pages and one width of table for all of them
    pages, width = max(s.k.shape[0] for s in steps), max(s.bt.shape[1] for s in steps)
    k, v = torch.zeros(pages, 2, 32, 128, dtype=BF16, device=DEV), torch.zeros(pages, 2, 32, 128, dtype=BF16, device=DEV)
    bt = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    qkv, mask, lens, cu = steps[0].qkv.to(DEV), steps[0].mask.to(DEV), steps[0].lens.to(DEV), steps[0].cu.to(DEV)
    args, _ = drafts([20, 7, 3], 5000, seed=1)
    dev = {n: t.to(DEV) for n, t in args.items()}
    temp = torch.ones(3, device=DEV)
    cache = torch.zeros(2, 2, pages, 2, 32, 128, dtype=BF16, device=DEV)

    def whole():
        o = K().tree_attention(qkv, k, v, bt, cu, lens, mask, 12, 2, 128, 0.09, None, 20, 1100, BF16)
        new, path, count = K().verify_drafts(**dev, max_q_len=20, max_depth=6, temperature=temp)
        K().compact_cache(cache, bt, cu, lens, path, count)
        return o, new, path, count

    def load(i):
        s = steps[i]
        for dst, src in ((qkv, s.qkv), (mask, s.mask), (lens, s.lens)):
            dst.copy_(src)
        k.zero_()[:s.k.shape[0]].copy_(s.k)
        v.zero_()[:s.v.shape[0]].copy_(s.v)
        bt.fill_(-1)[:, :s.bt.shape[1]].copy_(s.bt)
        other, _ = drafts([20, 7, 3], 5000, seed=10 + i)
        for n, t in other.items():
            dev[n].copy_(t)
        cache.copy_(torch.randn(cache.shape, generator=torch.Generator().manual_seed(i)))

    load(0)
    whole()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(whole())
        graphs.append(g)
    for i in (1, 0, 2, 1):
        for g, o in zip(graphs, outs):
            load(i)
            g.replay()
            got = [t.clone() for t in o] + [cache.clone()]
            load(i)
            want = list(whole()) + [cache]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    K().check_device_errors()


def test_tensors_have_to_be_on_the_current_device(monkeypatch):
    """(Shown with a device number that is not this one's: the tests run on one GPU.)"""
    from omniserver_b200.ops import KernelError
    s = Step([5], [30], 4, 2, 64, 16, F32)
    d, call = device_step(s)
    call()
    cache = torch.zeros(1, 2, 4, 2, 8, 16, device=DEV)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    with pytest.raises(KernelError, match="not the current device"):
        call()
    with pytest.raises(KernelError, match="not the current device"):
        K().copy_pages(cache, [0], [1])
    with pytest.raises(KernelError, match="not the current device"):
        K().verify_drafts(torch.zeros(1, 4, device=DEV), d["cu"][:1], d["cu"][:1], d["cu"], torch.zeros(1, device=DEV), 1, 1)


def test_empty_batches():
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    k = torch.zeros(3, 2, 16, 64, dtype=BF16, device=DEV)
    out = K().tree_attention(torch.zeros(0, 512, dtype=BF16, device=DEV), k, k, z.view(0, 4), one, z, z.view(0, 1), 4, 2, 64, 1.0, None, 0, 0, BF16)
    assert out.shape == (0, 256)
    new, path, count = K().verify_drafts(torch.zeros(0, 7, device=DEV), z, z, one, torch.zeros(0, device=DEV), 0, 2)
    assert new.shape == (0, 3) and path.shape == (0, 3) and count.shape == (0,)
    K().compact_cache(torch.zeros(1, 2, 3, 2, 16, 64, device=DEV), z.view(0, 4), one, z, z.view(0, 3), z)
    K().check_device_errors()


def test_many_requests_in_one_step():
    """More requests than a CTA has threads: the line of tiles is laid out in several rounds."""
    rng = np.random.default_rng(3)
    q_lens, bases = rng.integers(0, 4, 900).tolist(), rng.integers(0, 40, 900).tolist()
    for dtype in (BF16, F32):
        step = Step(q_lens, bases, 2, 1, 64, 16, dtype, seed=3)
        check(step, step.got(), *step.want(), runs_on_tensor_cores(step))


def test_fork_then_both_go_on():
    """A forked request's cache is its parent's until they go on; then neither sees the other."""
    from omniserver_b200.cache import CacheManager
    from omniserver_b200.models.decoder import EntryNeeds
    from omniserver_b200.parts.base import KVCacheNeed
    m = CacheManager([EntryNeeds(KVCacheNeed(2, 64, None), [], None)] * 3, [], 16, 12, 4, BF16, DEV)
    st = m.groups[0].storage
    m.begin("a")
    m.reserve("a", 37)
    slots = torch.from_numpy(m.slot_map(0, ["a"], [37])).long()
    m.commit("a", 37)
    st[:, :, slots // 16, :, slots % 16] = torch.randn(37, 3, 2, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)

    def tokens(r):
        t = torch.tensor(list(m.requests[r].tables[0]))
        p = torch.arange(m.requests[r].cursor)
        return st[:, :, t[p // 16], :, p % 16].clone()

    was = tokens("a")
    m.fork("a", "b")
    assert torch.equal(tokens("b"), was)
    m.reserve("b", 5)
    new = torch.from_numpy(m.slot_map(0, ["b"], [5])).long()
    m.accept("b", 4)
    st[:, :, new // 16, :, new % 16] = 9.0
    assert torch.equal(tokens("a"), was) and torch.equal(tokens("b")[:37], was) and (tokens("b")[37:] == 9.0).all()
    m.finish("a")
    assert torch.equal(tokens("b")[:37], was)
    m.check_invariants()


class TreeDecoder:
    """A small decoder out of the framework's kernels, a step of drafted trees: two layers of attention over a paged cache, with
    rotary positions, and a head. Weights in 32 bits; ``dtype`` is that of the cache and the activations."""

    V, H, NH, NKV, HD, LAYERS, PAGE = 97, 64, 4, 2, 64, 2, 16

    def __init__(self, dtype, manager, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.m = dtype, manager
        n = (self.NH + 2 * self.NKV) * self.HD

        def w(*s, scale):
            return (torch.randn(*s, generator=g) * scale).to(dtype).to(DEV)

        self.embed = w(self.V, self.H, scale=1.0)
        self.qkv = [w(n, self.H, scale=self.H ** -0.5) for _ in range(self.LAYERS)]
        self.out = [w(self.H, self.NH * self.HD, scale=(self.NH * self.HD) ** -0.5) for _ in range(self.LAYERS)]
        self.norm = torch.ones(self.H, device=DEV, dtype=dtype)
        self.head = w(self.V, self.H, scale=2.0 * self.H ** -0.5)
        self.inv_freq = (10000.0 ** (-torch.arange(0, self.HD, 2).float() / self.HD)).to(DEV)

    def step(self, requests, tokens, parents):
        """Logits [T, V] for each node of each request's tree, whose keys and values are then in the cache; and the batch."""
        k = K()
        q_lens = [len(t) for t in tokens]
        flat = sum(tokens, [])
        mask, depth = k.tree_plan(sum(parents, []), q_lens)
        for r, n in zip(requests, q_lens):
            self.m.reserve(r, n)
        base = np.repeat([self.m.requests[r].cursor for r in requests], q_lens)
        pos = torch.from_numpy(np.stack([base + depth] * 3).astype(np.int32)).to(DEV)
        tok_seq = torch.from_numpy(np.repeat(np.arange(len(requests)), q_lens).astype(np.int32)).to(DEV)
        cu = i32([0] + np.cumsum(q_lens).tolist()).to(DEV)
        kv = [self.m.requests[r].cursor + n for r, n in zip(requests, q_lens)]
        lens, bt = i32(kv).to(DEV), torch.from_numpy(self.m.block_table(0, requests)).to(DEV)
        slots = torch.from_numpy(self.m.slot_map(0, requests, q_lens)).to(DEV)
        zero = torch.zeros(len(requests), dtype=torch.int32, device=DEV)
        cos, sin = k.rope_tables(pos, zero, tok_seq, cu, zero, torch.zeros(1, 2, dtype=torch.int32, device=DEV), self.inv_freq,
                                 torch.zeros(self.HD // 2, dtype=torch.int32, device=DEV))
        x, res = k.embed_lookup(self.embed, i32(flat).to(DEV), self.dtype), None
        mask_d = torch.from_numpy(mask).to(DEV)
        for l in range(self.LAYERS):
            h, res = k.add_rmsnorm(x, res, self.norm, 1e-6, self.dtype)
            y = k.linear(h, self.qkv[l], None, self.dtype)
            st = self.m.groups[0].storage
            k.rope_kv_write(y, cos, sin, st[l, 0], st[l, 1], slots, self.NH, self.NKV, self.HD, self.HD)
            a = k.tree_attention(y, st[l, 0], st[l, 1], bt, cu, lens, mask_d, self.NH, self.NKV, self.HD, self.HD ** -0.5, None,
                                 max(q_lens), max(kv), self.dtype)
            x = k.linear(a, self.out[l], None, self.dtype)
        h, _ = k.add_rmsnorm(x, res, self.norm, 1e-6, self.dtype)
        return k.linear(h, self.head, None, F32), dict(cu_q=cu, seq_lens=lens, block_table=bt)


def new_manager(dtype):
    from omniserver_b200.cache import CacheManager
    from omniserver_b200.models.decoder import EntryNeeds
    from omniserver_b200.parts.base import KVCacheNeed
    t = TreeDecoder
    return CacheManager([EntryNeeds(KVCacheNeed(t.NKV, t.HD, None), [], None)] * t.LAYERS, [], t.PAGE, 60, 8, dtype, DEV, poison_freed=True)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_step_as_a_whole_emits_what_single_tokens_do(temperature):
    """Prompts as chains, then steps of random trees: attention, verification, compaction, acceptance, forks in between. Greedy: the
    tokens are those of decoding one by one. Sampled without draft probabilities, the root's children being all 97 words in an order
    of chance, of which one is therefore accepted: the logits where the walk ended are those of a fresh request of the same tokens."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 97, n).tolist() for n in (5, 23, 40)]

    def chain(n):
        return list(range(-1, n - 1))

    # one by one
    m1 = new_manager(F32)
    d1 = TreeDecoder(F32, m1)
    ids = [f"r{i}" for i in range(3)]
    for r in ids:
        m1.begin(r)
    logits, _ = d1.step(ids, prompts, [chain(len(p)) for p in prompts])
    ends = np.cumsum([len(p) for p in prompts]) - 1
    for r, p in zip(ids, prompts):
        m1.commit(r, len(p))
    last = logits[torch.from_numpy(ends).to(DEV)].argmax(-1).tolist()
    plain_tokens = [[t] for t in last]
    for _ in range(24):
        logits, _ = d1.step(ids, [[t[-1]] for t in plain_tokens], [[-1]] * 3)
        for r in ids:
            m1.commit(r, 1)
        for t, w in zip(plain_tokens, logits.argmax(-1).tolist()):
            t.append(w)
    # by trees: the drafts are the right words at times
    m2 = new_manager(F32)
    d2 = TreeDecoder(F32, m2)
    for r in ids:
        m2.begin(r)
    d2.step(ids, prompts, [chain(len(p)) for p in prompts])
    for r, p in zip(ids, prompts):
        m2.commit(r, len(p))
    got = [[t] for t in last]
    g = torch.Generator().manual_seed(5)
    accepted = 0
    for _ in range(12):
        trees, parents = [], []
        for i in range(3):
            n = int(rng.integers(1, 14))
            par = random_tree(n, rng)
            depth = [0] * n
            for j in range(1, n):
                depth[j] = depth[par[j]] + 1
            ahead = plain_tokens[i][len(got[i]):]
            toks = [got[i][-1]] + [ahead[depth[j] - 1] if depth[j] <= len(ahead) and rng.random() < 0.7 else int(rng.integers(0, 97)) for j in range(1, n)]
            if temperature > 0:   # every word below the root, then some nodes anywhere
                par = [-1] + [0] * 97 + [int(rng.integers(0, 98)) for _ in range(n)]
                toks = toks[:1] + rng.permutation(97).tolist() + rng.integers(0, 97, n).tolist()
            trees.append(toks)
            parents.append(par)
        logits, batch = d2.step(ids, trees, parents)
        T = sum(len(t) for t in trees)
        u = (torch.randint(0, 1 << 24, (T,), generator=g).float() / (1 << 24)).to(DEV)
        flat_t, flat_p = i32(sum(trees, [])).to(DEV), i32(sum(parents, [])).to(DEV)
        new, path, count = K().verify_drafts(logits, flat_t, flat_p, batch["cu_q"], u, 128, 13, temperature=torch.full((3,), temperature, device=DEV))
        want = plain.verify(logits.cpu(), flat_t.cpu(), flat_p.cpu(), batch["cu_q"].cpu(), u.cpu(), 13, torch.full((3,), temperature))
        assert [list(x) for x in zip(new.tolist(), path.tolist(), count.tolist())] == [list(w) for w in want]
        K().compact_cache(m2.groups[0].storage, batch["block_table"], batch["cu_q"], batch["seq_lens"], path, count)
        if temperature > 0:
            # a fresh request of the same tokens sees the same logits where the walk ended
            t0 = 0
            for i in range(3):
                seq = prompts[i] + got[i][:-1] + [trees[i][j] for j in path[i, :int(count[i])].tolist()]
                m2.begin("fresh")
                ref, _ = d2.step(["fresh"], [seq], [chain(len(seq))])
                m2.rollback("fresh")
                m2.finish("fresh")
                node = int(path[i, int(count[i]) - 1])
                assert torch.allclose(logits[t0 + node], ref[-1], rtol=1e-3, atol=1e-3)
                t0 += len(trees[i])
        for i, r in enumerate(ids):
            c = int(count[i])
            accepted += c - 1
            m2.accept(r, c)
            got[i] += new[i, :c].tolist()
            if temperature == 0.0:
                assert got[i][:25] == plain_tokens[i][:len(got[i])][:25]
        m2.check_invariants()
        # a fork goes on from here like its parent would
        m2.fork("r1", "child")
        fl, _ = d2.step(["child"], [[got[1][-1]]], [[-1]])
        pl, _ = d2.step(["r1"], [[got[1][-1]]], [[-1]])
        assert torch.equal(fl, pl)
        m2.rollback("r1")
        m2.finish("child")
        if temperature > 0 and min(len(x) for x in got) > 24:
            break
    assert accepted > 5
    K().check_device_errors()


# ------------------------------------------------------------------ caches that 32-bit offsets do not reach
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_in_a_cache_of_more_than_2_to_the_32_elements(dtype):
    """The same pages, once in a small pool and once spread up to the end of one of 2^32 elements and more: the same bits."""
    s = Step([9, 3], [200, 75], 4, 2, 128, 32, dtype, seed=4)
    used = s.k.shape[0]
    pages = (1 << 32) // (2 * 32 * 128) + 7
    move = torch.arange(used, dtype=torch.long) * ((pages - 1) // (used - 1))
    move[-1] = pages - 1
    k = torch.empty(pages, 2, 32, 128, dtype=dtype, device=DEV)
    v = torch.empty(pages, 2, 32, 128, dtype=dtype, device=DEV)
    k[move.to(DEV)], v[move.to(DEV)] = s.k.to(DEV), s.v.to(DEV)
    bt = torch.where(s.bt >= 0, move[s.bt.clamp(min=0).long()].to(torch.int32), -1)
    want = s.got()
    d = [t.to(DEV) for t in (s.qkv, bt, s.cu, s.lens, s.mask)]
    got = K().tree_attention(d[0], k, v, *d[1:], 4, 2, 128, 128 ** -0.5, None, 9, 209, dtype)
    assert torch.equal(got, want)
    del k, v
    torch.cuda.empty_cache()
    K().check_device_errors()


def test_cache_operators_in_a_cache_of_more_than_2_to_the_32_bytes():
    layers, nkv, page, hd = 3, 2, 16, 64
    pages = (1 << 32) // (2 * layers * nkv * page * hd) + 5
    cache = torch.empty(layers, 2, pages, nkv, page, hd, dtype=BF16, device=DEV)
    ids = [pages - 1, 3, pages - 2]
    rows = torch.randn(layers, 2, 3, nkv, page, hd, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    at = torch.tensor(ids, device=DEV)
    cache[:, :, at] = rows
    K().copy_pages(cache, [pages - 1, 3], [pages - 4, 0])
    assert torch.equal(cache[:, :, pages - 4], rows[:, :, 0]) and torch.equal(cache[:, :, 0], rows[:, :, 1])
    dev = [i32(x).to(DEV) for x in ([ids], [0, 20], [45], [[0, 4, 18, -1]], [3])]
    K().compact_cache(cache, *dev)
    want = rows.clone()
    for i, n in ((1, 4), (2, 18)):
        a, b = 25 + n, 25 + i
        want[:, :, b // page, :, b % page] = rows[:, :, a // page, :, a % page]
    assert torch.equal(cache[:, :, at], want)
    K().check_device_errors()


@pytest.mark.parametrize("hd", [64, 128])
def test_tree_attention_over_and_over(hd):
    """Batches whose requests are cut at many places, or fit in whole, in many calls: the same bits every time, no wait given up."""
    rng = np.random.default_rng(8)
    for bases in (rng.integers(1500, 2200, 64).tolist(), rng.integers(0, 300, 200).tolist(), [20000, 5, 700, 64, 3000]):
        call = device_step(Step([int(x) for x in rng.integers(1, 9, len(bases))], bases, 28, 4, hd, 64, BF16, seed=8))[1]
        want = call()
        for _ in range(60):
            outs = [call() for _ in range(5)]
            assert all(torch.equal(o, want) for o in outs)
    K().check_device_errors()


def test_tree_attention_values_that_are_not_finite_in_neighbouring_stretches():
    """Infinities in places that some rows see and others do not, in every request of a batch cut at many places: they reach the rows that
    see them, in every one, and no others."""
    step = Step([9] * 40, [100 + 37 * i for i in range(40)], 12, 2, 128, 32, BF16, seed=2)
    for s in range(40):
        at = step.bases[s] + 4                        # node 4: seen by itself and its descendants
        step.v[int(step.bt[s, at // 32]), :, at % 32, :] = math.inf
    got = step.got()
    cu = step.cu.tolist()
    words = step.mask[:, 0].tolist()
    for s in range(40):
        for t in range(cu[s], cu[s + 1]):
            sees = (words[t] >> 4) & 1
            assert bool((got[t] == math.inf).all()) if sees else bool(got[t].isfinite().all()), (s, t)
    K().check_device_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cu", [[0, 5, 15], [-1, 5, 14], [0, 16, 14], [0, 5, 2]])
def test_tree_attention_reports_tokens_that_are_not_there(dtype, cu):
    """Offsets outside the rows of qkv, or falling: reported; rows outside are not written, and what is right is computed."""
    from omniserver_b200.ops import KernelError
    s = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=2)
    d = [t.to(DEV) for t in (s.qkv, s.k, s.v, s.bt, i32(cu), s.lens, s.mask)]
    buf = torch.full((20, 256), 7.0, dtype=dtype, device=DEV)
    K().tree_attention(*d, 4, 2, 64, 0.125, None, 9, 149, dtype, out=buf[3:17])
    with pytest.raises(KernelError, match="tokens outside"):
        K().check_device_errors()
    assert (buf[:3] == 7.0).all() and (buf[17:] == 7.0).all()
    if cu[:2] == [0, 5]:
        assert torch.equal(buf[3:8], s.got(scale=0.125)[:5]) or dtype == BF16


@pytest.mark.parametrize("dense", [False, True])
def test_verify_reports_tokens_that_are_not_there(dense):
    from omniserver_b200.ops import KernelError
    args, q = drafts([4, 9], 300, seed=9, branch=1, dense=dense)
    temp = torch.ones(2)
    want = verify_both(args, 9, 8, temp, q)[1]
    for cu in ([0, 4, 14], [-2, 4, 13], [0, 4, 2]):
        dev = {n: t.to(DEV) for n, t in args.items()}
        dev["cu_q"] = i32(cu).to(DEV)
        new, path, count = K().verify_drafts(**dev, max_q_len=9, max_depth=8, temperature=temp.to(DEV), draft_probs=None if q is None else q.to(DEV))
        with pytest.raises(KernelError, match="tokens outside"):
            K().check_device_errors()
        bad = 0 if cu[0] < 0 else 1
        assert int(count[bad]) == 0 and (new[bad] == -1).all() and (path[bad] == -1).all()
        if cu == [0, 4, 14]:
            assert new[0].tolist() == want[0][0] and path[0].tolist() == want[0][1]
