"""The verification of drafted tokens without a GPU: the plan of a step's trees, forking and accepting in the cache manager, and
what the kernels' C entry points refuse before they launch anything."""

import ctypes

import numpy as np
import pytest
import torch

from omniserver_b200.cache import CacheManager, OutOfPages, OutOfSlots, PagePool
from omniserver_b200.models.decoder import EntryNeeds
from omniserver_b200.ops import CudaKernels, KernelError, library
from omniserver_b200.parts.base import KVCacheNeed, StateNeed
from plain import speculative as plain


def manager(num_pages=16, page_size=4, windows=(None, 6), max_requests=4, allocate=False):
    needs = [EntryNeeds(KVCacheNeed(2, 8, w), [], None) for w in windows]
    shared = [StateNeed("rope_cursor", (2,), torch.int32, shared=True)]
    return CacheManager(needs, shared, page_size, num_pages, max_requests, torch.float32, "cpu", allocate=allocate)


# ------------------------------------------------------------------ the plan
def test_tree_plan_lists_ancestors_and_depths():
    parents = [-1, 0, 0, 1, 2, 4, -1] + [-1]
    mask, depth = CudaKernels.tree_plan(parents, [7, 0, 1])
    assert mask.dtype == np.int32 and mask.shape == (8, 1) and depth.dtype == np.int32
    want = [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 4, 5], [6], [0]]
    assert [plain.sees_list(row, 7) for row in mask.tolist()] == want
    assert depth.tolist() == [0, 1, 1, 2, 2, 3, 0, 0]


def test_tree_plan_of_a_long_chain_fills_several_words():
    n = 70
    mask, depth = CudaKernels.tree_plan(list(range(-1, n - 1)), [n])
    assert mask.shape == (n, 3) and depth.tolist() == list(range(n))
    assert [plain.sees_list(row, n) for row in mask.tolist()] == [list(range(i + 1)) for i in range(n)]


@pytest.mark.parametrize("parents,q_lens", [([-1, 1], [2]), ([0], [1]), ([-1, -2], [2]), ([-1, 0], [3]), ([-1], [2, -1])])
def test_tree_plan_refuses(parents, q_lens):
    with pytest.raises(ValueError, match="tree_plan"):
        CudaKernels.tree_plan(parents, q_lens)


def test_tree_plan_of_nothing():
    mask, depth = CudaKernels.tree_plan([], [])
    assert mask.shape == (0, 1) and depth.shape == (0,)


# ------------------------------------------------------------------ the cache manager
def test_a_shared_page_is_free_when_its_last_holder_gives_it_back():
    p = PagePool(2)
    a = p.alloc()
    p.share(a)
    assert p.holders(a) == 2 and p.num_held == 1
    p.free(a)
    assert p.is_held(a) and p.num_free == 1
    p.free(a)
    assert not p.is_held(a) and p.num_free == 2
    with pytest.raises(ValueError, match="freed twice"):
        p.free(a)
    with pytest.raises(ValueError, match="not held"):
        p.share(a)


class Copies:
    """Stands where the kernels would be: notes the page copies."""

    def __init__(self):
        self.done = []

    def copy_pages(self, cache, src, dst):
        self.done.append((list(src), list(dst)))
        cache[:, :, list(dst)] = cache[:, :, list(src)]


@pytest.fixture
def copies(monkeypatch):
    from omniserver_b200 import ops
    c = Copies()
    monkeypatch.setattr(ops, "_KERNELS", c)
    return c


@pytest.mark.parametrize("tokens", [0, 1, 3, 4, 6, 8])
def test_fork_shares_full_pages_and_copies_the_partial_one(copies, tokens):
    m = manager(windows=(None,), allocate=True)
    m.begin("a")
    m.state.write("rope_cursor", m.requests["a"].slot, [5, 7])
    if tokens:
        m.reserve("a", tokens)
        m.commit("a", tokens)
        m.groups[0].storage.normal_(generator=torch.Generator().manual_seed(1))
    child = m.fork("a", "b")
    m.check_invariants()
    a, b = list(m.requests["a"].tables[0]), list(child.tables[0])
    full = tokens // 4
    assert child.cursor == tokens and len(b) == len(a) == -(-tokens // 4)
    assert b[:full] == a[:full] and (tokens % 4 == 0 or b[full] != a[full])
    assert copies.done == ([] if tokens % 4 == 0 else [([a[-1]], [b[-1]])])
    if b:
        st = m.groups[0].storage
        assert torch.equal(st[:, :, a], st[:, :, b])
    assert m.state.tensors["rope_cursor"][child.slot].tolist() == [5, 7]
    # both go on by themselves, in pages of their own
    m.reserve("a", 3)
    m.reserve("b", 3)
    ids = ["a", "b"]
    slots = m.slot_map(0, ids, [3, 3]).tolist()
    assert not set(slots[:3]) & set(slots[3:])
    m.commit("a", 3)
    m.commit("b", 3)
    m.check_invariants()
    m.finish("a")
    m.check_invariants()
    assert list(m.requests["b"].tables[0])[:full] == b[:full]
    m.finish("b")
    m.check_invariants()
    assert m.pages_in_use() == [0]


def test_fork_of_a_windowed_group_keeps_what_was_given_back(copies):
    m = manager(windows=(6, None), num_pages=16)
    m.begin("a")
    for _ in range(5):
        m.reserve("a", 3)
        m.commit("a", 3)
    m.fork("a", "b")
    m.check_invariants()
    m.fork("b", "c")
    m.check_invariants()
    assert list(m.requests["c"].tables[0])[:2] == [-1, -1]
    for rid in "abc":
        m.reserve(rid, 4)
        m.commit(rid, 4)
        m.check_invariants()
    m.reset("b")
    m.check_invariants()
    for rid in "abc":
        m.finish(rid)
    m.check_invariants()
    assert m.pages_in_use() == [0, 0]


def test_fork_refuses_and_leaves_everything_as_it_was(copies):
    m = manager(windows=(None,), num_pages=2, max_requests=2)
    m.begin("a")
    m.reserve("a", 6)
    with pytest.raises(ValueError, match="while a step"):
        m.fork("a", "b")
    m.commit("a", 6)
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    with pytest.raises(ValueError, match="already live"):
        m2 = manager()
        m2.begin("a")
        m2.fork("a", "a")
    assert not m.has("b") and m.state.num_free == 1
    m.check_invariants()
    m = manager(windows=(None,), max_requests=1)
    m.begin("a")
    with pytest.raises(OutOfSlots):
        m.fork("a", "b")
    with pytest.raises(KeyError):
        m.fork("x", "b")


def test_a_copy_that_fails_gives_the_child_back(monkeypatch):
    from omniserver_b200 import ops

    class Fails:
        def copy_pages(self, *a):
            raise KernelError("no")

    monkeypatch.setattr(ops, "_KERNELS", Fails())
    m = manager(windows=(None,), allocate=True)
    m.begin("a")
    m.reserve("a", 6)
    m.commit("a", 6)
    with pytest.raises(KernelError):
        m.fork("a", "b")
    assert not m.has("b")
    m.check_invariants()
    assert m.pages_in_use() == [2]


def test_freed_pages_are_poisoned_when_the_last_holder_leaves(copies):
    m = manager(windows=(None,), allocate=True)
    m.poison_freed = True
    m.begin("a")
    m.reserve("a", 4)
    m.commit("a", 4)
    page = m.requests["a"].tables[0][0]
    m.fork("a", "b")
    m.finish("a")
    assert not m.groups[0].storage[:, :, page].isnan().any()
    m.finish("b")
    assert m.groups[0].storage[:, :, page].isnan().all()


@pytest.mark.parametrize("kept", [1, 2, 5, 9])
def test_accept_keeps_the_first_tokens_and_gives_the_other_pages_back(kept):
    m = manager(windows=(None, 6))
    m.begin("a")
    m.reserve("a", 7)
    m.commit("a", 7)
    m.reserve("a", 9)
    m.accept("a", kept)
    m.check_invariants()
    rc = m.requests["a"]
    assert rc.cursor == 7 + kept and rc.reserved == 0 and len(rc.tables[0]) == -(-(7 + kept) // 4)
    with pytest.raises(ValueError):
        m.accept("a", 1)


# ------------------------------------------------------------------ refusals at the C entry points (nothing is launched)
BAD_SHAPE, UNSUPPORTED, TOO_LARGE = 10002, 10003, 10004
NULL = ctypes.c_void_p(0)


def tree_args(**over):
    a = dict(S=1, nh=4, nkv=2, hd=64, page=16, pages=4, window=0, max_q=4, max_kv=64, depth=NULL, part=NULL, dtypes=(0, 0, 0))
    a.update(over)
    o, q, c = a["dtypes"]
    return (NULL, o, NULL, q, 512, 64, NULL, NULL, c, NULL, 4, NULL, NULL, NULL, 1, a["depth"], a["S"], a["nh"], a["nkv"], a["hd"],
            a["page"], a["pages"], ctypes.c_float(1.0), a["window"], a["max_q"], a["max_kv"], a["part"], NULL, NULL)


@pytest.mark.parametrize("over,status", [
    (dict(hd=257), UNSUPPORTED), (dict(hd=0), BAD_SHAPE), (dict(nh=5), BAD_SHAPE), (dict(nkv=0), BAD_SHAPE), (dict(page=0), BAD_SHAPE),
    (dict(window=3), BAD_SHAPE), (dict(max_kv=2000), BAD_SHAPE), (dict(S=70000), TOO_LARGE), (dict(max_kv=(1 << 30) + 1), TOO_LARGE), (dict(dtypes=(2, 0, 0)), 10001),
    (dict(dtypes=(0, 7, 0)), 10001), (dict(dtypes=(0, 0, -1)), 10001), (dict(S=0), 0), (dict(max_q=0), 0)])
def test_tree_attention_entry_refuses(over, status):
    assert library.load().osb_attn_tree(*tree_args(**over)) == status


@pytest.mark.parametrize("over", [
    dict(hd=80), dict(hd=0), dict(nh=5), dict(nkv=0), dict(nh=129 * 2), dict(page=4), dict(page=24), dict(stride=516), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(max_q=(1 << 24) + 1), dict(max_kv=(1 << 30) + 1), dict(max_kv=0), dict(window=-1),
    dict(S=1 << 26, max_q=1024), dict(S=1 << 20, max_kv=1 << 20)])
def test_tensor_core_tree_attention_does_not_take(over):
    a = dict(S=1, nh=4, nkv=2, hd=64, page=16, stride=512, scale=1.0, window=0, max_q=4, max_kv=64)
    a.update(over)
    lib, scale = library.load(), ctypes.c_float(a["scale"])
    lib.osb_attn_tree_tc_scratch.restype = ctypes.c_longlong
    assert lib.osb_attn_tree_tc_scratch(a["S"], a["nh"], a["nkv"], a["hd"], a["page"], a["stride"], scale, a["window"], a["max_q"],
                                        a["max_kv"]) == 0
    assert lib.osb_attn_tree_tc(NULL, NULL, a["stride"], 4, NULL, NULL, NULL, 4, NULL, NULL, NULL, 1, NULL, a["S"], a["nh"], a["nkv"], a["hd"],
                                a["page"], 4, scale, a["window"], a["max_q"], a["max_kv"], NULL, NULL, NULL) == UNSUPPORTED


def test_tree_entries_refuse_too_few_mask_words():
    lib = library.load()
    args = list(tree_args(max_q=33))
    assert lib.osb_attn_tree(*args) == BAD_SHAPE
    assert lib.osb_attn_tree_tc(NULL, NULL, 512, 64, NULL, NULL, NULL, 4, NULL, NULL, NULL, 1, NULL, 1, 4, 2, 64, 16, 4, ctypes.c_float(1.0), 0, 33, 64, NULL, NULL,
                                NULL) == BAD_SHAPE


def test_scratch_of_the_32_bit_tree_attention_holds_every_smaller_request():
    """A request's rows x ranges never need more than what the largest request of its batch was given."""
    f = library.load().osb_attn_tree_scratch
    f.restype = ctypes.c_longlong
    assert f(1, 4, 2, 64, 8, 64) == 0 and f(0, 4, 2, 64, 8, 640) == 0

    def ranges(kv, rows):      # as the kernel cuts
        most = max(1, 128 // -(-rows // 32))
        per = -(-kv // most)
        return -(-kv // (-(-per // 64) * 64))

    for max_q, grp, max_kv in [(1, 1, 65), (3, 6, 700), (24, 6, 1000), (64, 8, 5000), (300, 8, 4097), (9, 4, 100000)]:
        cap = (f(1, grp, 1, 62, max_q, max_kv) - 1) // 64
        for q in sorted({1, 2, max_q // 3 + 1, max_q}):
            for kv in sorted({1, 64, 65, 128, max_kv // 2, 4096, 4100, max_kv - 1, max_kv}):
                if kv <= max_kv and q <= max_q and ranges(kv, q * grp) > 1:      # (one range goes straight to the output)
                    assert q * grp * ranges(kv, q * grp) <= cap, (max_q, grp, max_kv, q, kv)
                    assert ranges(kv, q * grp) <= ranges(min(max_kv, 8192), 1)


def verify_args(**over):
    a = dict(S=1, T=4, V=100, nodes=4, depth=3)
    a.update(over)
    return (NULL,) * 11 + (a["S"], a["T"], a["V"], a["nodes"], a["depth"], NULL, NULL)


@pytest.mark.parametrize("over,status", [
    (dict(V=0), BAD_SHAPE), (dict(T=-1), BAD_SHAPE), (dict(nodes=-1), BAD_SHAPE), (dict(depth=-1), BAD_SHAPE),
    (dict(nodes=1025), TOO_LARGE), (dict(V=17 << 20), TOO_LARGE), (dict(T=1 << 30, V=1 << 20), TOO_LARGE), (dict(S=0), 0)])
def test_verify_entry_refuses(over, status):
    assert library.load().osb_verify_drafts(*verify_args(**over)) == status


@pytest.mark.parametrize("over,status", [
    (dict(elem=1), BAD_SHAPE), (dict(elem=8), BAD_SHAPE), (dict(pages=0), BAD_SHAPE), (dict(hd=0), BAD_SHAPE),
    (dict(S=65536), TOO_LARGE), (dict(S=0), 0), (dict(planes=0), 0)])
def test_compact_entry_refuses(over, status):
    a = dict(elem=2, planes=2, pages=4, nkv=2, page=16, hd=8, S=1)
    a.update(over)
    assert library.load().osb_compact_cache(NULL, a["elem"], a["planes"], a["pages"], a["nkv"], a["page"], a["hd"], NULL, 4, NULL,
                                            NULL, NULL, 4, NULL, a["S"], NULL, NULL) == status


@pytest.mark.parametrize("src,dst,page_bytes,status", [
    ([0], [4], 64, BAD_SHAPE), ([-1], [1], 64, BAD_SHAPE), ([0], [1], 0, BAD_SHAPE), ([0], [1], 3, BAD_SHAPE), ([], [], 64, 0)])
def test_copy_entry_refuses(src, dst, page_bytes, status):
    a, b = np.array(src, dtype=np.int32), np.array(dst, dtype=np.int32)
    assert library.load().osb_copy_pages(NULL, ctypes.c_longlong(page_bytes), 2, 4, ctypes.c_void_p(a.ctypes.data),
                                         ctypes.c_void_p(b.ctypes.data), len(src), NULL) == status


@pytest.mark.parametrize("depth", [1 << 30, (1 << 31) - 1])
def test_verify_entry_refuses_more_columns_than_it_counts(depth):
    assert library.load().osb_verify_drafts(*verify_args(depth=depth)) == TOO_LARGE
