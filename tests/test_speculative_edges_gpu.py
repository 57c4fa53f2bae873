"""Where the operators that verify drafted tokens went wrong once, or are easily got wrong, against the plain references in 64 bits."""

import math

import numpy as np
import pytest
import torch

from test_speculative_gpu import BF16, DEV, F32, K, Step, check, drafts, i32, runs_on_tensor_cores, verify_both

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ verification
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("what", [-math.inf, math.nan])
def test_verify_accepts_nothing_on_a_row_without_logits(what, dense):
    """A row of which no logit is above -inf says nothing, not that word 0 is the best: a drafted word 0 behind it is not accepted, by a
    greedy request either. (Rows 1 and 4 are behind the root; row 6 is a root's.)"""
    args, q = drafts([3, 3, 2], 3000, seed=2, branch=1, dense=dense)
    for row in (1, 4, 6):
        args["logits"][row] = what
    for node in (1, 4):
        args["tokens"][node] = int(args["logits"][node - 1].argmax())
    for node in (2, 5, 7):
        args["tokens"][node] = 0
    for temp in (None, torch.zeros(3), torch.tensor([0.0, 0.9, 0.0]), torch.tensor([0.9, 0.0, 0.9])):
        got, want = verify_both(args, 3, 2, temp, q)
        assert got == want
        assert got[2] == [[0, -1, -1], [0, -1, -1], 1]
        for s in range(2):
            if temp is None or temp[s] == 0:
                assert got[s][2] == 2 and got[s][0][1] == 0
    K().check_device_errors()


def uniforms(n, g):
    return torch.randint(0, 1 << 24, (n,), generator=g).float() / (1 << 24)


@pytest.mark.parametrize("temp,others", [(1.0, -math.inf), (0.05, -50.0)])
def test_verify_slices_of_which_only_rejected_words_had_weight(temp, others):
    """Two siblings hold all the weight of the first 1,024 words, and the next token's random number is 0: it is the first word with
    weight behind them. (Their weights are 2^30 and more apart, so that 64 bits do not hold the sum of both.)"""
    S, V = 64, 5000
    g = torch.Generator().manual_seed(3)
    logits = torch.zeros(3 * S, V)
    rows = torch.full((S, V), others)
    rows[:, 10] = 0.0
    rows[:, 500] = (-22.0 - torch.rand(S, generator=g)) * temp
    rows[:, [3100, 4100]] = (torch.rand(S, 2, generator=g) + 0.1) * temp
    logits[::3] = rows
    u = torch.full((3 * S,), 0.99)
    u[::3] = 0.0
    for order in ((10, 500), (500, 10)):
        args = dict(logits=logits, tokens=i32([0, *order] * S), parents=i32([-1, 0, 0] * S), cu_q=i32(list(range(0, 3 * S + 1, 3))), uniform=u)
        got, want = verify_both(args, 3, 1, torch.full((S,), temp))
        assert got == want
        assert all(x == [[3100, -1], [0, -1], 1] for x in got)
    K().check_device_errors()


@pytest.mark.parametrize("apart", [3, 1100])
@pytest.mark.parametrize("n", [1, 2, 3, 4])
def test_verify_little_is_left_behind_rejected_words(n, apart):
    """n siblings, each of which holds all but 2^-22 of what those before it leave, are rejected one after the other (u = 1 - 2^-24): what
    is left, 2^-88 of the row at the end, is drawn from like any other distribution. The words lie in one slice or in n of them."""
    S, V = 64, 6000
    g = torch.Generator().manual_seed(n)
    words = [700 + apart * i for i in range(n)]
    rows = torch.randn(S, V, generator=g) * 2.0
    rows[:, words] = -math.inf
    rest = torch.logsumexp(rows.double(), -1)
    for w in reversed(words):
        rows[:, w] = (rest + 22 * math.log(2.0)).float()
        rest = torch.logaddexp(rest, rows[:, w].double())
    logits = torch.zeros(S * (n + 1), V)
    logits[::n + 1] = rows
    u = torch.full((S * (n + 1),), 1.0 - 2.0 ** -24)
    u[::n + 1] = uniforms(S, g)
    args = dict(logits=logits, tokens=i32(([0] + words) * S), parents=i32(([-1] + [0] * n) * S),
                cu_q=i32(list(range(0, S * (n + 1) + 1, n + 1))), uniform=u)
    got, want = verify_both(args, n + 1, 1, torch.ones(S))
    assert all(x[2] == 1 and x[0][0] not in words for x in want)
    assert got == want
    K().check_device_errors()


@pytest.mark.parametrize("slices", [(7, 9), (7, 1500)])
def test_verify_draws_words_down_to_the_end_of_32_bits(slices):
    """A random number of 0 draws the first word that has weight: one of 2^-120 of the largest has, one of 2^-160 may have (a slice's own
    largest word counts for it), one of -inf has not. Before a rejection and behind one (the first of two words of a half each goes), with and
    without draft probabilities."""
    V = 4000
    light, heavy = slices
    row = torch.full((V,), -math.inf)
    row[5], row[light], row[[heavy, 3000]] = -160 * math.log(2.0), -120 * math.log(2.0), 0.0
    logits = torch.stack([row] * 3)
    q = torch.zeros(3, V)
    q[:, heavy] = 1.0
    args = dict(logits=logits, tokens=i32([0, 0, heavy]), parents=i32([-1, -1, 0]), cu_q=i32([0, 1, 3]), uniform=torch.tensor([0.0, 0.0, 0.9]))
    for dense in (False, True):
        got, _ = verify_both(args, 2, 1, torch.ones(2), q if dense else None)
        assert all(x[0][0] in (5, light) and x[1:] == [[0, -1], 1] for x in got)
    K().check_device_errors()


def test_verify_siblings_drawn_independently_leave_the_targets_distribution():
    """Three siblings and, below the first, another: drawn independently of one another from their parent's row of draft probabilities, or,
    without draft probabilities, the same different words every time. The first two emitted tokens are distributed like the target's:
    20,000 walks, a count's standard deviation is at most sqrt(N / 4): 6 of them."""
    N, V, n = 20000, 8, 5
    g = torch.Generator().manual_seed(4)
    target = torch.randn(V, V, generator=g)                  # by the word before: node c's row is that of its token
    draft = torch.softmax(torch.randn(V, V, generator=g), -1)
    p = torch.softmax(target.double(), -1)
    for dense in (False, True):
        tokens = torch.zeros(N, n, dtype=torch.long)         # the root's token is 0
        if dense:
            tokens[:, 1:4] = torch.multinomial(draft[0], 3 * N, replacement=True, generator=g).view(N, 3)
            tokens[:, 4] = torch.multinomial(draft[tokens[:, 1]], 1, generator=g)[:, 0]
        else:
            tokens[:, 1:] = torch.tensor([5, 2, 7, 1])
        u = uniforms(N * n, g)
        flat = tokens.view(-1)
        new, path, count = K().verify_drafts(target[flat].to(DEV), flat.to(torch.int32).to(DEV), i32([-1, 0, 0, 0, 1] * N).to(DEV),
                                             torch.arange(0, n * N + 1, n, dtype=torch.int32).to(DEV), u.to(DEV), n, 2, torch.ones(N, device=DEV),
                                             draft[flat].to(DEV) if dense else None)
        new, count = new.cpu().long(), count.cpu()
        first = torch.bincount(new[:, 0], minlength=V).double()
        assert ((first - N * p[0]).abs() <= 6 * math.sqrt(N / 4)).all()
        # where there is a second token in this step, it follows the first like the target says
        for w in range(V):
            second = torch.bincount(new[(new[:, 0] == w) & (count > 1), 1], minlength=V).double()
            m = float(second.sum())
            assert ((second - m * p[w]).abs() <= 6 * math.sqrt(m / 4) + 1e-9).all()
        assert len(count.unique()) == 3
    K().check_device_errors()


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("V", [170001, 330000])
def test_verify_rows_of_more_slices_than_a_lane_holds(V, dense):
    """Most of the weight, the drawn words and the drafted ones lie behind the first 160 slices of 1,024 words, or in the last ones."""
    for q_lens, tail in (([5], 3000), ([3, 4], 1000), ([4, 3, 3], V - 163840)):
        args, q = drafts(q_lens, V, seed=V + tail, branch=2, peak=3.0, dense=dense)
        args["logits"][:, -tail:] += 9.0
        if dense:
            q[:, -tail:] *= 1000.0
            q /= q.sum(-1, keepdim=True)
        for j in range(1, sum(q_lens)):
            if j not in args["cu_q"].tolist():
                s = sum(j >= x for x in args["cu_q"][1:].tolist())
                row = int(args["cu_q"][s]) + int(args["parents"][j])
                args["tokens"][j] = int(args["logits"][row, -tail:].topk(3).indices[j % 3]) + V - tail
        seen = 0
        for temp in (None, torch.full((len(q_lens),), 0.9)):
            got, want = verify_both(args, max(q_lens), 3, temp, q)
            assert got == want
            seen += sum(x[0][x[2] - 1] >= V - tail for x in got)
        assert seen > 0
    K().check_device_errors()


@pytest.mark.parametrize("reqs", [1, 9])
@pytest.mark.parametrize("V", [33000, 40001, 70000, 99999])
def test_verify_walks_by_two_and_four_ctas(V, reqs):
    accepted = 0
    for seed in range(3):
        args, q = drafts([4 + (i + seed) % 3 for i in range(reqs)], V, seed=seed + reqs, branch=3, peak=3.0, dense=True)
        got, want = verify_both(args, 6, 4, torch.full((reqs,), 0.8), q)
        assert got == want
        accepted += sum(x[2] - 1 for x in got)
    assert accepted > 0 or reqs == 1      # (three trees of one request may accept nothing)
    K().check_device_errors()


# ------------------------------------------------------------------ attention
def window_step(q_lens, bases, nh, nkv, hd, window, dtype, seed):
    step = Step(q_lens, bases, nh, nkv, hd, 16, dtype, seed=seed)
    for s, b in enumerate(bases):                 # pages that every row's window has passed were given back
        for pi in range(max(0, b - window + 1) // 16):
            step.bt[s, pi] = -1
    return step


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_lens,bases,nh,nkv,hd,window", [
    ([24], [3000], 12, 2, 128, 1500), ([70], [2049], 8, 2, 64, 640), ([40], [1000], 28, 4, 128, 5000),      # row tiles abreast
    ([8, 5, 12], [3000, 2000, 2500], 12, 2, 128, 1100), ([30, 1, 9], [4000, 700, 1300], 28, 4, 64, 2000),   # units cut, one row tile and two
    ([64, 33], [1700, 900], 7, 1, 128, 1001), ([6, 20], [2100, 2500], 2, 2, 64, 2047)])
def test_tree_attention_windows_of_units_that_are_cut(q_lens, bases, nh, nkv, hd, window, dtype):
    step = window_step(q_lens, bases, nh, nkv, hd, window, dtype, seed=window)
    check(step, step.got(window), *step.want(window), runs_on_tensor_cores(step))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tree_attention_batches_cut_at_many_places(hd, which):
    rng = np.random.default_rng(8)
    bases = (rng.integers(1500, 2200, 64).tolist(), rng.integers(0, 300, 200).tolist(), [20000, 5, 700, 64, 3000])[which]
    step = Step([int(x) for x in rng.integers(1, 9, len(bases))], bases, 28, 4, hd, 64, BF16, seed=8)
    check(step, step.got(), *step.want(), True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_lens,bases", [([3], [40]), ([5, 1, 9], [300, 20, 1100]), ([17, 2], [2000, 129])])
def test_tree_attention_with_bounds_above_what_is_there(q_lens, bases, dtype):
    """As a captured step passes them: the most nodes and keys that there may be."""
    step = Step(q_lens, bases, 12, 2, 128, 32, dtype, seed=5)
    wide = torch.full((len(q_lens), 300), -1, dtype=torch.int32)
    wide[:, :step.bt.shape[1]] = step.bt
    mask = torch.zeros(step.mask.shape[0], 4, dtype=torch.int32)
    mask[:, :step.mask.shape[1]] = step.mask
    for most_q, most_kv in ((32, 2100), (100, 9600), (128, 1 << 20)):
        out = K().tree_attention(step.qkv.to(DEV), step.k.to(DEV), step.v.to(DEV), wide.to(DEV), step.cu.to(DEV), step.lens.to(DEV), mask.to(DEV),
                                 12, 2, 128, 128 ** -0.5, None, most_q, most_kv, dtype)
        check(step, out, *step.want(), runs_on_tensor_cores(step))


class Rows:
    """Some requests of a step, for `check`."""

    def __init__(self, step, n):
        self.q_lens, self.lens, self.hd = step.q_lens[:n], step.lens[:n], step.hd


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_computes_the_requests_beside_a_reported_one(dtype):
    from omniserver_b200.ops import KernelError
    s = Step([5, 9], [30, 140], 4, 2, 64, 16, dtype, seed=2)
    want, spread, weight = s.want()
    d = [t.to(DEV) for t in (s.qkv, s.k, s.v, s.bt, s.cu, s.lens, s.mask)]
    cases = [(d, 8, 149), (d, 9, 148)]                                       # too many nodes, too many keys
    cases += [(d[:4] + [i32(cu).to(DEV)] + d[5:], 9, 149) for cu in ([0, 5, 15], [0, 5, 2])]   # tokens that are not there
    cases += [(d[:5] + [i32([35, 4]).to(DEV)] + d[6:], 9, 149)]              # fewer keys than nodes
    for args, most_q, most_kv in cases:
        got = K().tree_attention(*args, 4, 2, 64, 0.125, None, most_q, most_kv, dtype)
        with pytest.raises(KernelError, match="more nodes or keys"):
            K().check_device_errors()
        check(Rows(s, 1), got[:5], want[:5], spread[:5], weight, dtype == BF16)


# ------------------------------------------------------------------ bounds of a call
def test_bounds_that_32_bits_do_not_hold_are_refused():
    """(The kernels' C entries take these as 32-bit integers: what is beyond would arrive as something else.)"""
    from omniserver_b200.ops import KernelError
    z, one = torch.zeros(1, dtype=torch.int32, device=DEV), i32([0, 0]).to(DEV)
    logits, u = torch.zeros(1, 8, device=DEV), torch.zeros(1, device=DEV)
    for depth in (1 << 30, (1 << 31) - 1, (1 << 32) + 2):
        with pytest.raises(KernelError, match="max_depth"):
            K().verify_drafts(logits, z, z, one, u, 1, depth)
    k = torch.zeros(1, 1, 16, 64, device=DEV)
    mask = torch.zeros(1, (1 << 26) + 1, dtype=torch.int32, device=DEV)
    for most_q, most_kv in (((1 << 31) + 5, 16), (1, (1 << 32) + 16)):
        with pytest.raises(KernelError, match="2\\^30"):
            K().tree_attention(torch.zeros(1, 64, device=DEV), k, k, z.view(1, 1), one, z, mask, 1, 1, 64, 1.0, None, most_q, most_kv, torch.float32)
