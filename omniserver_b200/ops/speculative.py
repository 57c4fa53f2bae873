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
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from ._common import _check, _cuda_contig, _dt, _p


def _on_device(ref: torch.Tensor, **tensors: Optional[torch.Tensor]) -> None:
    """Every tensor on the current device: a launch goes to a stream of that one."""
    dev = ref.device
    _check(dev.index == torch.cuda.current_device(), f"the tensors are on {dev}, which is not the current device")
    for name, t in tensors.items():
        _check(t is None or t.device == dev, f"{name} must be on {dev}")


class SpeculativeOps:
    MAX_TREE_NODES = 1024      # of one request, in ``verify_drafts``
    VERIFY_SLICE = 4096        # words of a logits row that one CTA of the verification takes

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

        ``max_q_len`` / ``max_kv_len``: at least the most nodes and keys of a request; a larger one, and a page outside the pool
        among the visible ones, is reported by ``check_device_errors``, and that request's rows are then not defined.
        Rows of ``out`` [T, nh*hd] (made here if not given) that belong to no request are not written. float32 operands,
        ``exact=True`` and shapes the tensor-core kernel does not take run in 32 bits throughout.
        """
        _cuda_contig("qkv", qkv)
        _cuda_contig("k_cache", k_cache)
        _cuda_contig("v_cache", v_cache)
        for n, t in (("block_table", block_table), ("cu_q", cu_q), ("seq_lens", seq_lens), ("tree_mask", tree_mask)):
            _cuda_contig(n, t, torch.int32)
        win = int(window) if window else 0
        _check(win >= 0, "tree_attention: a window is positive")
        _check(win == 0 or depth is not None, "tree_attention: a window needs the nodes' depth")
        if depth is not None:
            _cuda_contig("depth", depth, torch.int32)
        _on_device(qkv, k_cache=k_cache, v_cache=v_cache, block_table=block_table, cu_q=cu_q, seq_lens=seq_lens,
                   tree_mask=tree_mask, depth=depth, out=out)
        _check(qkv.dim() == 2 and seq_lens.dim() == 1, "tree_attention: qkv [T,*], seq_lens [S]")
        T, S = qkv.shape[0], seq_lens.shape[0]
        _check(nh > 0 and nkv > 0 and hd > 0 and nh % nkv == 0, "tree_attention: heads must be a multiple of kv heads")
        _check(qkv.shape[1] >= nh * hd, "tree_attention: q columns missing")
        _check(k_cache.dim() == 4 and k_cache.shape[1] == nkv and k_cache.shape[3] == hd and v_cache.shape == k_cache.shape
               and v_cache.dtype == k_cache.dtype, "tree_attention: caches [pages, nkv, page_size, hd]")
        _check(block_table.dim() == 2 and block_table.shape[0] == S, "tree_attention: block_table [S,*]")
        _check(cu_q.shape == (S + 1,), "tree_attention: cu_q [S+1]")
        _check(tree_mask.dim() == 2 and tree_mask.shape[0] == T and 32 * tree_mask.shape[1] >= max_q_len,
               "tree_attention: tree_mask [T, W] with 32 W >= max_q_len")
        _check(depth is None or depth.shape == (T,), "tree_attention: depth [T]")
        _check(hd <= 256, "tree_attention: head sizes up to 256")
        if out is None:
            out = torch.empty((T, nh * hd), dtype=out_dtype, device=qkv.device)
        else:
            _cuda_contig("out", out, out_dtype)
            _check(out.shape == (T, nh * hd), "tree_attention: out [T, nh*hd]")
        if S == 0 or T == 0 or max_q_len <= 0 or max_kv_len <= 0 or k_cache.shape[0] == 0:
            return out
        part_o = part_ml = None
        splits = 0
        if (not exact and qkv.dtype == k_cache.dtype == out_dtype == torch.bfloat16
                and (qkv.data_ptr() | k_cache.data_ptr() | v_cache.data_ptr() | out.data_ptr()) % 16 == 0):
            splits = self.lib.osb_attn_tree_tc_splits(S, nh, nkv, hd, k_cache.shape[2], qkv.shape[1], ctypes.c_float(scale), win,
                                                      max_q_len, max_kv_len)
        if splits > 0:
            if splits > 1:
                nodes = 128 // (nh // nkv)
                rows = S * nkv * -(-max_q_len // nodes) * splits * 128
                part_o = torch.empty(rows * hd, dtype=torch.float32, device=qkv.device)
                part_ml = torch.empty(rows * 2, dtype=torch.float32, device=qkv.device)
            rc = self.lib.osb_attn_tree_tc(
                _p(out), _p(qkv), qkv.shape[1], T, _p(k_cache), _p(v_cache), _p(block_table), block_table.shape[1], _p(cu_q),
                _p(seq_lens), _p(tree_mask), tree_mask.shape[1], _p(depth), S, nh, nkv, hd, k_cache.shape[2], k_cache.shape[0],
                ctypes.c_float(scale), win, max_q_len, max_kv_len, splits, _p(part_o), _p(part_ml),
                _p(self.err_flag(qkv.device)), self._stream())
            self._ok(rc, "attn_tree_tc")
            self.launches += 1 if splits > 1 else 0
            return out
        splits = self.lib.osb_attn_tree_splits(max_kv_len)
        if splits > 1:
            part_o = torch.empty(T * nh * splits * hd, dtype=torch.float32, device=qkv.device)
            part_ml = torch.empty(T * nh * splits * 2, dtype=torch.float32, device=qkv.device)
        rc = self.lib.osb_attn_tree(
            _p(out), _dt(out), _p(qkv), _dt(qkv), qkv.shape[1], _p(k_cache), _p(v_cache), _dt(k_cache), _p(block_table),
            block_table.shape[1], _p(cu_q), _p(seq_lens), _p(tree_mask), tree_mask.shape[1], _p(depth), S, nh, nkv, hd,
            k_cache.shape[2], k_cache.shape[0], ctypes.c_float(scale), win, max_q_len, max_kv_len, _p(part_o), _p(part_ml),
            _p(self.err_flag(qkv.device)), self._stream())
        self._ok(rc, "attn_tree")
        self.launches += 1 if splits > 1 else 0
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
        fp32: row i is the distribution that node i's children were drawn from; negative and NaN entries count as 0. NaN logits
        count as -inf; where no logit of a row is above -inf nothing is accepted and the next token is 0.

        Out: ``path`` the accepted nodes from 0 on, ``tokens`` the new tokens (the accepted nodes' and the next one), both -1
        behind the first ``count``: that many nodes stay in the cache, and that many tokens are new. At most ``max_depth``
        drafted tokens are accepted. A request without nodes has count 0. A token outside the vocabulary is never accepted, and
        reported by ``check_device_errors`` where a request brings it as a draft.
        """
        _cuda_contig("logits", logits, torch.float32)
        for n, t in (("tokens", tokens), ("parents", parents), ("cu_q", cu_q)):
            _cuda_contig(n, t, torch.int32)
        _cuda_contig("uniform", uniform, torch.float32)
        _check(logits.dim() == 2 and cu_q.dim() == 1 and cu_q.shape[0] >= 1, "verify_drafts: logits [T,V], cu_q [S+1]")
        T, V = logits.shape
        S = cu_q.shape[0] - 1
        _check(V > 0, "verify_drafts: an empty vocabulary")
        _check(tokens.shape == (T,) and parents.shape == (T,) and uniform.shape == (T,),
               "verify_drafts: tokens, parents and uniform [T]")
        _check(0 <= max_q_len <= self.MAX_TREE_NODES, f"verify_drafts: up to {self.MAX_TREE_NODES} nodes per request")
        _check(max_depth >= 0, "verify_drafts: max_depth must not be negative")
        if temperature is not None:
            _cuda_contig("temperature", temperature, torch.float32)
            _check(temperature.shape == (S,), "verify_drafts: temperature [S]")
        if draft_probs is not None:
            _cuda_contig("draft_probs", draft_probs, torch.float32)
            _check(draft_probs.shape == (T, V), "verify_drafts: draft_probs [T,V]")
        _on_device(logits, tokens=tokens, parents=parents, cu_q=cu_q, uniform=uniform, temperature=temperature,
                   draft_probs=draft_probs)
        out = torch.empty((2 * (max_depth + 1) + 1) * S, dtype=torch.int32, device=logits.device)
        n = S * (max_depth + 1)
        new, path, count = out[:n].view(S, max_depth + 1), out[n:2 * n].view(S, max_depth + 1), out[2 * n:]
        if S == 0:
            return new, path, count
        stats = torch.empty(max(1, T) * -(-V // self.VERIFY_SLICE) * 2, dtype=torch.float64, device=logits.device)
        rc = self.lib.osb_verify_drafts(_p(new), _p(path), _p(count), _p(stats), _p(logits), _p(tokens), _p(parents), _p(cu_q),
                                        _p(uniform), _p(temperature), _p(draft_probs), S, T, V, max_q_len, max_depth,
                                        _p(self.err_flag(logits.device)), self._stream())
        self._ok(rc, "verify_drafts")
        self.launches += 1 if T > 0 else 0
        return new, path, count

    # ------------------------------------------------------------------ cache
    @staticmethod
    def _check_storage(what: str, cache: torch.Tensor) -> None:
        _cuda_contig("cache", cache)
        _check(cache.dim() == 6 and cache.shape[1] == 2, f"{what}: cache [layers, 2, pages, nkv, page_size, hd]")
        _dt(cache)

    def compact_cache(self, cache: torch.Tensor, block_table: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor,
                      path: torch.Tensor, count: torch.Tensor) -> None:
        """Moves the accepted tokens of a verified step together, in every layer, keys and values, in place: what lies at place
        base + path[s, i] of request s goes to base + i for i < count[s], base = seq_lens[s] - (cu_q[s + 1] - cu_q[s]), as if
        all were read before any was written. ``cache`` is a page group's storage [layers, 2, pages, nkv, page_size, hd];
        ``path`` and ``count`` as ``verify_drafts`` returns them. A path that does not ascend, leaves its tree, or is longer than
        it moves nothing of its request, and a token in a page outside the pool stays; both are reported by
        ``check_device_errors``."""
        self._check_storage("compact_cache", cache)
        for n, t in (("block_table", block_table), ("cu_q", cu_q), ("seq_lens", seq_lens), ("path", path), ("count", count)):
            _cuda_contig(n, t, torch.int32)
        S = seq_lens.shape[0]
        _check(seq_lens.dim() == 1 and cu_q.shape == (S + 1,) and count.shape == (S,), "compact_cache: seq_lens, count [S], cu_q [S+1]")
        _check(block_table.dim() == 2 and block_table.shape[0] == S, "compact_cache: block_table [S,*]")
        _check(path.dim() == 2 and path.shape[0] == S, "compact_cache: path [S,*]")
        _on_device(cache, block_table=block_table, cu_q=cu_q, seq_lens=seq_lens, path=path, count=count)
        if S == 0 or cache.numel() == 0:
            return
        L, _, P, nkv, ps, hd = cache.shape
        rc = self.lib.osb_compact_cache(_p(cache), cache.element_size(), 2 * L, P, nkv, ps, hd, _p(block_table), block_table.shape[1],
                                        _p(cu_q), _p(seq_lens), _p(path), path.shape[1], _p(count), S,
                                        _p(self.err_flag(cache.device)), self._stream())
        self._ok(rc, "compact_cache")

    def copy_pages(self, cache: torch.Tensor, src: Sequence[int], dst: Sequence[int]) -> None:
        """Copies page src[i] to page dst[i] in every layer, keys and values. ``cache`` as for ``compact_cache``; the page numbers
        are on the host (as the block tables are): every dst once, and none of them a src."""
        self._check_storage("copy_pages", cache)
        _on_device(cache)
        a = np.ascontiguousarray(src, dtype=np.int32)
        b = np.ascontiguousarray(dst, dtype=np.int32)
        _check(a.ndim == 1 and a.shape == b.shape, "copy_pages: as many sources as destinations")
        n = a.shape[0]
        if n == 0:
            return
        la, lb = a.tolist(), b.tolist()
        L, _, P, nkv, ps, hd = cache.shape
        _check(min(la) >= 0 and max(la) < P and min(lb) >= 0 and max(lb) < P, f"copy_pages: pages 0 to {P - 1}")
        to = set(lb)
        _check(len(to) == n and to.isdisjoint(la), "copy_pages: every destination once, and none of them a source")
        if cache.numel() == 0:
            return
        rc = self.lib.osb_copy_pages(_p(cache), ctypes.c_longlong(nkv * ps * hd * cache.element_size()), 2 * L, P,
                                     ctypes.c_void_p(a.ctypes.data), ctypes.c_void_p(b.ctypes.data), n, self._stream())
        self._ok(rc, "copy_pages")
