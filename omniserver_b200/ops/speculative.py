"""The operators of a step that verifies drafted tokens (``csrc/attn_tree*.cu``, ``csrc/verify.cu``, ``csrc/cache_ops.cu``).
A mixin of ``ops.CudaKernels``, which provides ``lib``, ``_stream()``, ``_ok()`` and ``err_flag()``.

Such a step, in order: a request brings a *tree* of tokens, node 0 the last token it has and the others drafted, parents
before children. ``tree_plan`` makes the mask and the depths on the host; the step's keys and values go into the cache behind the
committed tokens (``rope_kv_write``, a node's position being base + depth); ``tree_attention`` takes the place of
``paged_attention``; ``verify_drafts`` that of ``sample``; ``compact_cache`` moves the accepted path together, and
``CacheManager.accept`` keeps that many tokens of the reservation. Everything between is on the device; only the tokens go to
the host. ``copy_pages`` is what ``CacheManager.fork`` copies a partly filled page with.

The reference has none of these (it decodes one token per request and step, omniserve/runners/multimodal.py:227-304).
"""

from __future__ import annotations

import ctypes
import struct
from operator import index
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from ._common import KernelError, _check, _cuda_contig, _dt

_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16

# The arguments of the entry points: Q an address (0: none), q an integer, d a number.
_ENTRIES = {
    "attn_tree_scratch": "qqqqqq",
    "attn_tree": "QqQqqqQQqQqQQQqQqqqqqqdqqqQQQ",
    "attn_tree_tc_scratch": "qqqqqqdqqq",
    "attn_tree_tc": "QQqqQQQqQQQqQqqqqqqdqqqQQQ",
    "verify_drafts": "QQQQQQQQQQQqqqqqQQ",
    "compact_cache": "QqqqqqqQqQQQqQqQQ",
    "copy_pages": "QqqqQQqQ",
}


class Entries:
    """This file's entry points of the library, ``osb_attn_tree`` as ``attn_tree(...)`` and so on, with every call's arguments packed
    into one array: these calls are made where a step's launches take a few microseconds, and converting 26 arguments one by
    one takes four."""

    def __init__(self, lib: ctypes.CDLL):
        for name, args in _ENTRIES.items():
            setattr(self, name, self._entry(getattr(lib, f"osb_{name}_packed"), struct.Struct("=" + args).pack))

    @staticmethod
    def _entry(fn, pack):
        fn.argtypes, fn.restype = [ctypes.c_char_p], ctypes.c_longlong
        return lambda *args: fn(pack(*args))


def _on_device(ref: torch.Tensor) -> int:
    """The index of the tensor's device, which has to be the current one: a launch goes to a stream of that."""
    _check(ref.is_cuda, "the operands must be CUDA tensors (there is no CPU path)")
    dev = ref.get_device()
    if dev != torch.cuda.current_device():
        raise KernelError(f"the tensors are on cuda:{dev}, which is not the current device")
    return dev


def _operands(dev: int, dtype: Optional[torch.dtype], names: str, *tensors: torch.Tensor) -> None:
    """Contiguous tensors of this type on this device; ``names``: theirs, for the message."""
    for t in tensors:
        if t.get_device() != dev or (dtype is not None and t.dtype is not dtype) or not t.is_contiguous():
            name = names.split()[next(i for i, x in enumerate(tensors) if x is t)]
            _cuda_contig(name, t, dtype)
            raise KernelError(f"{name} must be on cuda:{dev}")


def _page_numbers(pages: Sequence[int]) -> List[int]:
    """The numbers as a list; anything but a row of whole numbers on the host is refused."""
    try:
        return [index(p) for p in (pages if isinstance(pages, (list, tuple)) else np.asarray(pages))]
    except TypeError as e:
        raise KernelError(f"copy_pages: page numbers are whole numbers on the host: {e}") from None


class SpeculativeOps:
    MAX_TREE_NODES = 1024      # of one request, in ``verify_drafts``
    VERIFY_SLICE = 1024        # words of a logits row that a warp of the verification takes at a time

    def _raw_stream(self, dev: int) -> int:
        """The current stream of device ``dev`` (the pinned one inside ``pinned_stream``) as an address. Looking up
        ``torch.cuda.current_stream()`` makes a Stream object, 3.4 us of the 14 that a small call takes on the host."""
        if self._pinned_stream is not None:
            return self._pinned_stream.value or 0
        return torch._C._cuda_getCurrentRawStream(dev)

    # ------------------------------------------------------------------ plan of a step (host)
    @staticmethod
    def tree_plan(parents: Sequence[int], q_lens: Sequence[int]) -> Tuple[np.ndarray, np.ndarray]:
        """(mask words [T, W] int32, depth [T] int32) of a step's trees. ``parents`` [T]: each node's parent, numbered within its
        request and smaller than the node's own number; -1 for a root. Bit j % 32 of word j / 32 of a node's row says that it
        sees node j of its request: itself and its ancestors. W holds the longest of ``q_lens``."""
        par, lens = [int(p) for p in parents], [int(n) for n in q_lens]
        if any(n < 0 for n in lens) or sum(lens) != len(par):
            raise ValueError(f"tree_plan: {len(par)} parents for trees of {sum(lens)} nodes")
        words = max(1, -(-max(lens, default=0) // 32))
        rows, depth, t0 = [], np.zeros(len(par), dtype=np.int32), 0
        for n in lens:
            for j in range(n):
                p = par[t0 + j]
                if not -1 <= p < j:
                    raise ValueError(f"tree_plan: node {j} of a request has parent {p}: parents come before their children")
                rows.append((rows[t0 + p] if p >= 0 else 0) | (1 << j))
                if p >= 0:
                    depth[t0 + j] = depth[t0 + p] + 1
            t0 += n
        raw = b"".join(r.to_bytes(4 * words, "little") for r in rows)
        return np.frombuffer(raw, dtype="<i4").reshape(len(par), words).astype(np.int32), depth

    # ------------------------------------------------------------------ attention
    def tree_attention(self, qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                       cu_q: torch.Tensor, seq_lens: torch.Tensor, tree_mask: torch.Tensor, nh: int, nkv: int, hd: int,
                       scale: float, window: Optional[int], max_q_len: int, max_kv_len: int, out_dtype: torch.dtype,
                       depth: Optional[torch.Tensor] = None, exact: bool = False, out: Optional[torch.Tensor] = None
                       ) -> torch.Tensor:
        """Attention of the step's trees over the paged cache (arguments as ``paged_attention``).

        Request s brings nodes ``cu_q[s] .. cu_q[s + 1] - 1``, whose keys and values lie in its last places
        ``base = seq_lens[s] - (cu_q[s + 1] - cu_q[s])`` onward. A node sees every committed key and the nodes of its request
        whose bits are set in its row of ``tree_mask`` [T, W] int32 (``tree_plan``; bits at or beyond its request's nodes do
        not count). With a ``window`` it sees the last ``window`` places up to its own, a node's place being base +
        ``depth`` [T] int32. A node that sees nothing gets zeros. What hidden places hold does not matter.

        ``max_q_len`` / ``max_kv_len``: at least the most nodes and keys of a request; a larger one, tokens outside qkv, and a
        page outside the pool among the visible ones, are reported by ``check_device_errors``, and that request's rows are
        then not defined. (With 0 for either nothing is done, and nothing reported.) Both also decide how the work is cut: bounds far above
        what is there, as a captured step has them, cost up to 5 us in bf16; in 32 bits 34 us became 50 to 56 where 32,768 keys were
        allowed for 4 requests of 1,000.
        Rows of ``out`` [T, nh*hd] (made here if not given) that belong to no request are not written. float32 operands,
        ``exact=True`` and shapes the tensor-core kernel does not take run in 32 bits throughout.
        """
        dev = _on_device(qkv)
        _operands(dev, None, "qkv k_cache v_cache", qkv, k_cache, v_cache)
        _operands(dev, _I32, "block_table cu_q seq_lens tree_mask", block_table, cu_q, seq_lens, tree_mask)
        win = min(int(window), 1 << 30) if window else 0      # (no request has more keys)
        _check(win >= 0, "tree_attention: a window is positive")
        _check(qkv.dim() == 2 and seq_lens.dim() == 1 and block_table.dim() == 2 and tree_mask.dim() == 2 and k_cache.dim() == 4,
               "tree_attention: qkv [T,*], seq_lens [S], block_table [S,*], tree_mask [T,W], caches [pages, nkv, page_size, hd]")
        T, width = qkv.shape
        S, = seq_lens.shape
        pages, heads, page_size, head_dim = shape = k_cache.shape
        rows, words = tree_mask.shape
        tables, bt_width = block_table.shape
        _check(nh > 0 and nkv > 0 and hd > 0 and nh % nkv == 0, "tree_attention: heads must be a multiple of kv heads")
        _check(width >= nh * hd, "tree_attention: q columns missing")
        _check(heads == nkv and head_dim == hd and v_cache.shape == shape and v_cache.dtype is k_cache.dtype,
               "tree_attention: caches [pages, nkv, page_size, hd]")
        _check(tables == S, "tree_attention: block_table [S,*]")
        _check(cu_q.shape == (S + 1,), "tree_attention: cu_q [S+1]")
        _check(rows == T and 32 * words >= max_q_len, "tree_attention: tree_mask [T, W] with 32 W >= max_q_len")
        _check(hd <= 256, "tree_attention: head sizes up to 256")
        _check(max_kv_len <= 1 << 30 and max_q_len <= 1 << 30, "tree_attention: up to 2^30 keys and nodes per request")
        if depth is not None:
            _operands(dev, _I32, "depth", depth)
            _check(depth.shape == (T,), "tree_attention: depth [T]")
        else:
            _check(win == 0, "tree_attention: a window needs the nodes' depth")
        if out is None:
            out = qkv.new_empty((T, nh * hd)) if out_dtype is qkv.dtype else qkv.new_empty((T, nh * hd), dtype=out_dtype)
        else:
            _operands(dev, out_dtype, "out", out)
            _check(out.shape == (T, nh * hd), "tree_attention: out [T, nh*hd]")
        if S == 0 or T == 0 or max_q_len <= 0 or max_kv_len <= 0 or pages == 0:
            return out
        qp, kp, vp, op = qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr()
        dp = depth.data_ptr() if depth is not None else 0
        err = self.err_flag(qkv.device).data_ptr()
        need = 0
        if (not exact and qkv.dtype is _BF16 and k_cache.dtype is _BF16 and out_dtype is _BF16 and (qp | kp | vp | op) % 16 == 0):
            need = self._entries.attn_tree_tc_scratch(S, nh, nkv, hd, page_size, width, scale, win, max_q_len, max_kv_len)
        if need > 0:
            scratch = qkv.new_empty(need, dtype=torch.uint8) if need > 1 else None
            rc = self._entries.attn_tree_tc(
                op, qp, width, T, kp, vp, block_table.data_ptr(), bt_width, cu_q.data_ptr(), seq_lens.data_ptr(),
                tree_mask.data_ptr(), words, dp, S, nh, nkv, hd, page_size, pages, scale, win, max_q_len, max_kv_len,
                0 if scratch is None else scratch.data_ptr(), err, self._raw_stream(dev))
            self._ok(rc, "attn_tree_tc")
            self.launches += 1 if need > 1 else 0      # the second kernel, which joins what was cut
        else:
            need = self._entries.attn_tree_scratch(S, nh, nkv, hd, max_q_len, max_kv_len)
            scratch = qkv.new_empty(need, dtype=_F32) if need > 0 else None
            rc = self._entries.attn_tree(
                op, _dt(out), qp, _dt(qkv), width, T, kp, vp, _dt(k_cache), block_table.data_ptr(), bt_width, cu_q.data_ptr(),
                seq_lens.data_ptr(), tree_mask.data_ptr(), words, dp, S, nh, nkv, hd, page_size, pages, scale, win, max_q_len,
                max_kv_len, scratch.data_ptr() if need > 0 else 0, err, self._raw_stream(dev))
            self._ok(rc, "attn_tree")
            self.launches += 1 if need > 0 else 0
        return out

    # ------------------------------------------------------------------ verification
    def verify_drafts(self, logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_q: torch.Tensor,
                      uniform: torch.Tensor, max_q_len: int, max_depth: int, temperature: Optional[torch.Tensor] = None,
                      draft_probs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Walks each request's tree with the target's logits: (tokens [S, max_depth + 1], path [S, max_depth + 1], count [S]).

        ``logits`` [T, V] fp32, ``tokens`` / ``parents`` [T] int32 (as for ``tree_plan``; node 0 is the token the request had),
        ``uniform`` [T] fp32 in [0, 1): node c > 0 is tested with its own, the last token drawn with the root's. ``temperature``
        [S] fp32 (<= 0, or None for all: greedy). A child with token x is accepted if u q(x) < r(x), r being the target's
        softmax(logits / temperature) behind its parent less what the siblings rejected before it took: max(r - q, 0)
        renormalised, or without ``draft_probs`` (drafts that are certain of their token) the word itself. ``draft_probs`` [T, V]
        fp32: row i is the distribution that node i's children were drawn from, each independently of the others (with replacement; the new
        tokens follow the target's distribution only then, without ``draft_probs`` always); negative and NaN entries count as 0. NaN logits
        count as -inf; where no logit of a row is above -inf nothing is accepted and the next token is 0. Words of 2^-126 of the likeliest
        one's probability and less may count as having none. ``max_q_len``: at least the
        most nodes of a request; what a larger one has beyond it is not looked at, nor a request whose tokens are outside
        ``logits`` (count 0), and ``check_device_errors`` reports them.

        Out: ``path`` the accepted nodes from 0 on, ``tokens`` the new tokens (the accepted nodes' and the next one), both -1
        behind the first ``count``: that many nodes stay in the cache, and that many tokens are new. At most ``max_depth``
        drafted tokens are accepted. A request without nodes has count 0. A token outside the vocabulary is never accepted, and
        reported by ``check_device_errors`` where a request brings it as a draft.
        """
        dev = _on_device(logits)
        _operands(dev, _F32, "logits uniform", logits, uniform)
        _operands(dev, _I32, "tokens parents cu_q", tokens, parents, cu_q)
        _check(logits.dim() == 2 and cu_q.dim() == 1 and cu_q.shape[0] >= 1, "verify_drafts: logits [T,V], cu_q [S+1]")
        T, V = logits.shape
        S = cu_q.shape[0] - 1
        _check(V > 0, "verify_drafts: an empty vocabulary")
        _check(tokens.shape == (T,) and parents.shape == (T,) and uniform.shape == (T,),
               "verify_drafts: tokens, parents and uniform [T]")
        _check(0 <= max_q_len <= self.MAX_TREE_NODES, "verify_drafts: up to 1024 nodes per request")
        _check(0 <= max_depth < 1 << 30, "verify_drafts: max_depth must not be negative, and below 2^30")
        tp = qp = 0
        if temperature is not None:
            _operands(dev, _F32, "temperature", temperature)
            _check(temperature.shape == (S,), "verify_drafts: temperature [S]")
            tp = temperature.data_ptr()
        if draft_probs is not None:
            _operands(dev, _F32, "draft_probs", draft_probs)
            _check(draft_probs.shape == (T, V), "verify_drafts: draft_probs [T,V]")
            qp = draft_probs.data_ptr()
        shape = (S, max_depth + 1)
        new, path, count = tokens.new_empty(shape), tokens.new_empty(shape), tokens.new_empty(S)
        if S == 0:
            return new, path, count
        stats = tokens.new_empty(4 * T * -(-V // self.VERIFY_SLICE))      # 16 bytes per slice of a row
        rc = self._entries.verify_drafts(new.data_ptr(), path.data_ptr(), count.data_ptr(), stats.data_ptr(), logits.data_ptr(),
                                         tokens.data_ptr(), parents.data_ptr(), cu_q.data_ptr(), uniform.data_ptr(), tp, qp, S, T, V,
                                         max_q_len, max_depth, self.err_flag(logits.device).data_ptr(), self._raw_stream(dev))
        self._ok(rc, "verify_drafts")
        self.launches += 1 if T > 0 else 0
        return new, path, count

    # ------------------------------------------------------------------ cache
    @staticmethod
    def _storage(cache: torch.Tensor) -> Tuple[int, Tuple[int, ...]]:
        """(device index, shape) of a page group's storage."""
        dev = _on_device(cache)
        _operands(dev, None, "cache", cache)
        _check(cache.dim() == 6 and cache.shape[1] == 2, "cache must be [layers, 2, pages, nkv, page_size, hd]")
        _dt(cache)
        return dev, cache.shape

    def compact_cache(self, cache: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
                      path: torch.Tensor, count: torch.Tensor) -> None:
        """Moves the accepted tokens of a verified step together, in every layer, keys and values, in place: what lies at place
        base + path[s, i] of request s goes to base + i for i < count[s], base = seq_lens[s] - (cu_q[s + 1] - cu_q[s]), as if
        all were read before any was written. ``cache`` is a page group's storage [layers, 2, pages, nkv, page_size, hd];
        ``path`` and ``count`` as ``verify_drafts`` returns them. A path that does not ascend, leaves its tree, or is longer than
        it moves nothing of its request, and a token in a page outside the pool stays; both are reported by
        ``check_device_errors``."""
        dev, (L, _, P, nkv, ps, hd) = self._storage(cache)
        _operands(dev, _I32, "block_table cu_q seq_lens path count", block_table, cu_q, seq_lens, path, count)
        S = seq_lens.shape[0]
        _check(seq_lens.dim() == 1 and cu_q.shape == (S + 1,) and count.shape == (S,),
               "compact_cache: seq_lens, count [S], cu_q [S+1]")
        _check(block_table.dim() == 2 and block_table.shape[0] == S, "compact_cache: block_table [S,*]")
        _check(path.dim() == 2 and path.shape[0] == S, "compact_cache: path [S,*]")
        if S == 0 or cache.numel() == 0:
            return
        rc = self._entries.compact_cache(cache.data_ptr(), cache.element_size(), 2 * L, P, nkv, ps, hd, block_table.data_ptr(),
                                         block_table.shape[1], cu_q.data_ptr(), seq_lens.data_ptr(), path.data_ptr(),
                                         path.shape[1], count.data_ptr(), S, self.err_flag(cache.device).data_ptr(),
                                         self._raw_stream(dev))
        self._ok(rc, "compact_cache")

    def copy_pages(self, cache: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copies page src[i] to page dst[i] in every layer, keys and values. ``cache`` as for ``compact_cache``; the page numbers
        are on the host (as the block tables are): every dst once, and none of them a src."""
        dev, (L, _, P, nkv, ps, hd) = self._storage(cache)
        a, b = _page_numbers(src), _page_numbers(dst)
        n = len(a)
        _check(n == len(b), "copy_pages: as many sources as destinations")
        if n == 0:
            return
        _check(min(a) >= 0 and max(a) < P and min(b) >= 0 and max(b) < P, "copy_pages: a page outside the pool")
        to = set(b)
        _check(len(to) == n and to.isdisjoint(a), "copy_pages: every destination once, and none of them a source")
        if cache.numel() == 0:
            return
        pages = (ctypes.c_int * (2 * n))(*a, *b)
        at = ctypes.addressof(pages)
        rc = self._entries.copy_pages(cache.data_ptr(), nkv * ps * hd * cache.element_size(), 2 * L, P, at, at + 4 * n, n,
                                      self._raw_stream(dev))
        self._ok(rc, "copy_pages")
