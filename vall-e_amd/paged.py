"""A paged KV cache for serving loops, on libvalle_hip.so: memory follows the requests page by page, and a step may carry a tree of
drafted tokens per request.  One step of a loop, per layer where it says so:

    table.plan(len_old, len_new, parents)                       # pages, slots, positions, tree masks -- on the device, no sync
    q = rope_kv_paged(q, k, v, table.positions, rope, table.slots, k_cache[l], v_cache[l])               # per layer
    o = attn_tree(q, k_cache[l], v_cache[l], table.block_table, len_old, table.cu_rows, table.tree_mask)    # per layer
    len_old = kv_commit(k_cache, v_cache, table.block_table, len_old, path, n_accept, table.n_blocks, table.status)   # accepted nodes become context

Caches are ``[n_layers][n_pages][kv_heads][page_size][64]`` (``kv_cache``), head_dim 64, bf16 or fp32, q and k heads
pair-interleaved as the model's packed weights are (a rotation mixes elements 2i and 2i + 1).  The reference has no counterpart:
it recomputes the whole sequence every step (vall_e/models/base.py:521, ``use_cache=False``); the same products over one
contiguous slot per utterance are ``valle_rope_kv`` / ``valle_attn_decode``.

Every call is enqueued on the current stream of its tensors' device, reads nothing back and may be captured into a HIP graph.
Inference only: no autograd, no CPU fallback.  Arguments are checked in C++ (csrc/bind_serving.cpp): a wrong shape, layout or
device raises ValueError, a wrong type TypeError, a CPU tensor or a refusal of the C entry ValleHipError."""
from __future__ import annotations

import torch

from . import _lib as L

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_NODES = 64                 # drafted tokens per request: one 64-bit mask word
HEAD_DIM = 64


_S = L.serving()


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def kv_cache(n_layers, n_pages, page_size, kv_heads, dtype=torch.bfloat16, device="cuda"):
    """(k, v) page pools ``[n_layers][n_pages][kv_heads][page_size][64]``."""
    _need(page_size in PAGE_SIZES, f"page_size {page_size}: one of {PAGE_SIZES}")
    L.dtype_code(dtype)
    shape = (n_layers, n_pages, kv_heads, page_size, HEAD_DIM)
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


class PageTable:
    """The pages of a batch of up to ``max_requests`` requests over a pool of ``n_pages``, kept on the device.  One plan at a time: plans of
    one table on two streams must wait for each other.

    State: ``block_table [max_requests][max_blocks]`` int32 (entries behind a request's ``n_blocks`` mean nothing), ``n_blocks``
    [max_requests], ``free_list`` [n_pages] (a stack of the first ``free_count[0]`` entries).
    Written by every ``plan``: ``cu_rows`` [max_requests + 1] (row offsets of the step's packed rows), ``slots`` / ``positions``
    [max_rows] (slot = page * page_size + offset; -1: padding row, or a request without pages), ``tree_mask`` [max_rows] int64
    (plain rows: chains), ``status`` [max_requests]: 0 served, 1 no pages left (it keeps what it had), 2 lengths out of range,
    3 its rows lie behind ``max_rows``; what a step computes for rows of requests that were not served means nothing."""

    def __init__(self, max_requests, max_blocks, n_pages, page_size, max_rows, device="cuda"):
        _need(page_size in PAGE_SIZES, f"page_size {page_size}: one of {PAGE_SIZES}")
        _need(0 < max_requests <= 4096, f"max_requests {max_requests}: 1 .. 4096")
        _need(max_blocks > 0 and n_pages > 0 and max_rows > 0, "max_blocks, n_pages and max_rows must be positive")
        _need(n_pages * page_size < 2 ** 31 and max_blocks * max(page_size, max_requests) < 2 ** 31, "the pool or the tables pass 2^31 entries")
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device, self.page_size, self.max_rows = dev, page_size, max_rows
        self.max_requests, self.max_blocks, self.n_pages = max_requests, max_blocks, n_pages
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
        self.block_table, self.n_blocks, self.status = i32(max_requests, max_blocks), i32(max_requests), i32(max_requests)
        self.free_list = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=dev)          # page 0 on top
        self.free_count = torch.full((1,), n_pages, dtype=torch.int32, device=dev)
        self.next_n_blocks, self.next_free_count, self._ticket = i32(max_requests), i32(1), i32(1)
        self.cu_rows, self.slots, self.positions = i32(max_requests + 1), i32(max_rows), i32(max_rows)
        self.tree_mask = torch.zeros(max_rows, dtype=torch.int64, device=dev)

    def plan(self, len_old, len_new, parents=None, in_place=True):
        """Takes every request from ``len_old[b]`` to ``len_new[b]`` cached rows (int32 [max_requests] on the device; an idle
        request has 0 and 0): surplus pages go back to the pool (``len_new`` 0 gives back all), missing ones are taken in request
        order until the pool is empty, and the rows ``len_old .. len_new`` get their slots.  ``parents`` (int32 [max_rows]): row r
        is a drafted node whose parent is node ``parents[r]`` of the same request, an earlier one (anything else: a child of the
        context); positions are then ``len_old`` + depth and ``tree_mask`` holds every node's ancestors and itself; at most 64
        new rows per request.  Without them ``tree_mask`` holds what ``attn_tree`` takes for no mask: row i sees rows 0 .. i.  ``in_place=False`` leaves ``n_blocks`` and ``free_count`` and writes ``next_n_blocks`` /
        ``next_free_count`` (a plan that may be thrown away)."""
        if in_place:
            nb, fc = self.n_blocks, self.free_count
        else:
            nb, fc = self.next_n_blocks, self.next_free_count
        _S.page_plan(len_old, len_new, parents, self.block_table, self.n_blocks, nb, self.free_list, self.free_count, fc, self.status, self.cu_rows,
                     self.slots, self.positions, self.tree_mask, self._ticket, self.page_size)
        return self


def rope_kv_paged(q, k, v, positions, rope, slots, k_cache, v_cache, out=None):
    """RoPE on the rows' q and k (``[rows][heads][64]``, views of a fused projection work as they are), k and v written into the
    pages: row r goes to slot ``slots[r]`` of ``k_cache`` / ``v_cache`` ``[n_pages][kv_heads][page_size][64]`` (a slot outside the
    pool, -1 for instance: not written; a slot named twice: pieces of either row).  ``rope`` fp32 ``[positions][32][2]`` = (cos, sin);
    positions outside the table take its nearest row.  Returns the rotated q (``out``, which may be q itself)."""
    return _S.rope_kv_paged(q, k, v, positions, rope, slots, k_cache, v_cache, out)


def attn_tree(q, k_cache, v_cache, block_table, ctx_len, cu_rows, tree_mask=None, max_nodes=None, max_ctx=None, softmax_scale=None, out=None):
    """Attention of each request's new rows over its pages: request b asks with rows ``cu_rows[b] .. cu_rows[b+1]`` of q
    (``[rows][heads][64]``, heads a multiple of the cache's kv_heads; up to 64 rows per request), which see all of its
    ``ctx_len[b]`` cached rows and, of the new rows (cached behind them), those whose bit is set in ``tree_mask[row]`` (None: a
    chain, row i sees rows 0 .. i; one row: a plain decode step).  A row that sees nothing is zero.  Requests with a negative
    ``ctx_len`` and rows behind ``cu_rows[-1]`` are left as they were (``out=`` to say what that is; it may be q).  ``max_nodes``: the largest
    number of rows of a request (rows behind it are left); the default, min(64, all rows), is right for any batch but cuts the work for trees of that
    size: a plain decode step passes 1.  ``max_ctx``: the longest context, a hint for how to split the work (default: the table's width).  A prompt of
    more than 64 rows takes several calls, 64 rows a step; rows beyond are not computed."""
    return _S.attn_tree(q, k_cache, v_cache, block_table, ctx_len, cu_rows, tree_mask, max_nodes, max_ctx,
                        HEAD_DIM ** -0.5 if softmax_scale is None else softmax_scale, out)


def kv_commit(k_cache, v_cache, block_table, ctx_len, path, n_accept, n_blocks=None, status=None):
    """The accepted nodes of every request's tree become context, in all layers: cached row ``ctx_len[b] + path[b][j]`` moves to
    ``ctx_len[b] + j`` for ``j < n_accept[b]`` (``path`` int32 [requests][up to 64], node numbers 0 .. 63; others stay where they
    are).  Caches ``[n_layers][n_pages][kv_heads][page_size][64]``, changed in place.  Returns the new lengths, ``ctx_len + n_accept`` with
    ``n_accept`` held to 0 .. the path's width (a negative ``ctx_len`` stays).

    ``n_blocks`` and ``status`` (int32 [requests], the table's after ``plan``; ``next_n_blocks`` after a plan that was not in place): a request
    that was not served accepts nothing and keeps its length, whatever ``n_accept`` says; rows behind the pages a request holds are absent, and its
    length does not pass them (an ended request's becomes 0; for requests that are cut short pass the shorter of both lengths as ``ctx_len``).  Without them ``n_accept`` must not pass the rows that were planned, and has to be 0 where
    the plan refused the request: the table's entries behind ``n_blocks`` are left over and name pages of others."""
    return _S.kv_commit(k_cache, v_cache, block_table, ctx_len, path, n_accept, n_blocks, status)
