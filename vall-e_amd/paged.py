"""A paged KV cache for serving loops, on libvalle_hip.so: memory follows the requests page by page, and a step may carry a tree of
drafted tokens per request.  One step of a loop, per layer where it says so:

    table.plan(len_old, len_new, parents)                       # pages, slots, positions, tree masks -- on the device, no sync
    q = rope_kv_paged(q, k, v, table.positions, rope, table.slots, k_cache[l], v_cache[l])               # per layer
    o = attn_tree(q, k_cache[l], v_cache[l], table.block_table, len_old, table.cu_rows, table.tree_mask)    # per layer
    len_old = kv_commit(k_cache, v_cache, table.block_table, len_old, path, n_accept)     # the accepted nodes become context

Caches are ``[n_layers][n_pages][kv_heads][page_size][64]`` (``kv_cache``), head_dim 64, bf16 or fp32, q and k heads
pair-interleaved as the model's packed weights are (a rotation mixes elements 2i and 2i + 1).  The reference has no counterpart:
it recomputes the whole sequence every step (vall_e/models/base.py:521, ``use_cache=False``); the same products over one
contiguous slot per utterance are ``valle_rope_kv`` / ``valle_attn_decode``.

Every call is enqueued on the current stream of its tensors' device, reads nothing back and may be captured into a HIP graph.
Inference only: no autograd, no CPU fallback."""
from __future__ import annotations

import torch

from . import _lib as L

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_NODES = 64                 # drafted tokens per request: one 64-bit mask word
HEAD_DIM = 64


I32, I64, BF16, F32 = torch.int32, torch.int64, torch.bfloat16, torch.float32
_CODE = {BF16: L.BF16, F32: L.F32}


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _ints(name, t, dev, shape, dtype=I32):
    """Pointer of a contiguous whole-number tensor on GPU ``dev``."""
    if t.dtype is dtype and t.get_device() == dev and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name}: contiguous {dtype} tensor of shape {tuple(shape)} on GPU {dev} needed, got {t.dtype} {tuple(t.shape)} on {t.device}"
                     + ("" if t.is_contiguous() else " (not contiguous)"))


def _call(dev, fn, *args):
    """fn(*args, current stream of GPU dev) with that GPU current."""
    if torch.cuda.current_device() == dev:
        rc = fn(*args, L.raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, L.raw_stream(dev))
    if rc:
        L.check(rc)


def _gpu(t, what):
    dev = t.get_device()
    if dev < 0:
        raise L.ValleHipError(f"{what} needs GPU tensors; there is no CPU fallback")
    return dev


def kv_cache(n_layers, n_pages, page_size, kv_heads, dtype=torch.bfloat16, device="cuda"):
    """(k, v) page pools ``[n_layers][n_pages][kv_heads][page_size][64]``."""
    _need(page_size in PAGE_SIZES, f"page_size {page_size}: one of {PAGE_SIZES}")
    L.dtype_code(dtype)
    shape = (n_layers, n_pages, kv_heads, page_size, HEAD_DIM)
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


class PageTable:
    """The pages of a batch of up to ``max_requests`` requests over a pool of ``n_pages``, kept on the device.

    State: ``block_table [max_requests][max_blocks]`` int32 (entries behind a request's ``n_blocks`` mean nothing), ``n_blocks``
    [max_requests], ``free_list`` [n_pages] (a stack of the first ``free_count[0]`` entries).
    Written by every ``plan``: ``cu_rows`` [max_requests + 1] (row offsets of the step's packed rows), ``slots`` / ``positions``
    [max_rows] (slot = page * page_size + offset; -1: padding row, or a request without pages), ``tree_mask`` [max_rows] int64
    (with ``parents`` only), ``status`` [max_requests]: 0 served, 1 no pages left (it keeps what it had), 2 lengths out of range,
    3 its rows lie behind ``max_rows``."""

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
        self.next_n_blocks, self.next_free_count = i32(max_requests), i32(1)
        self.cu_rows, self.slots, self.positions = i32(max_requests + 1), i32(max_rows), i32(max_rows)
        self.tree_mask = torch.zeros(max_rows, dtype=torch.int64, device=dev)

    def plan(self, len_old, len_new, parents=None, in_place=True):
        """Takes every request from ``len_old[b]`` to ``len_new[b]`` cached rows (int32 [max_requests] on the device; an idle
        request has 0 and 0): surplus pages go back to the pool (``len_new`` 0 gives back all), missing ones are taken in request
        order until the pool is empty, and the rows ``len_old .. len_new`` get their slots.  ``parents`` (int32 [max_rows]): row r
        is a drafted node whose parent is node ``parents[r]`` of the same request, an earlier one (anything else: a child of the
        context); positions are then ``len_old`` + depth and ``tree_mask`` holds every node's ancestors and itself; at most 64
        new rows per request.  ``in_place=False`` leaves ``n_blocks`` and ``free_count`` and writes ``next_n_blocks`` /
        ``next_free_count`` (a plan that may be thrown away)."""
        dev = _gpu(self.block_table, "PageTable.plan")
        n = (self.max_requests,)
        lo, ln = _ints("len_old", len_old, dev, n), _ints("len_new", len_new, dev, n)
        par = mask = None
        if parents is not None:
            par, mask = _ints("parents", parents, dev, (self.max_rows,)), self.tree_mask.data_ptr()
        nb, fc = self.n_blocks.data_ptr(), self.free_count.data_ptr()
        nb2, fc2 = (nb, fc) if in_place else (self.next_n_blocks.data_ptr(), self.next_free_count.data_ptr())
        _call(dev, L.load().valle_page_plan, lo, ln, self.max_requests, self.page_size, self.block_table.data_ptr(), self.max_blocks, nb, nb2,
              self.free_list.data_ptr(), self.n_pages, fc, fc2, self.status.data_ptr(), self.cu_rows.data_ptr(), self.slots.data_ptr(),
              self.positions.data_ptr(), self.max_rows, par, mask)
        return self


def _heads(name, t, dev, dtype, rows=None):
    """(tensor, row stride) of [rows][heads][64] with the heads packed; any row stride that keeps rows 16-byte aligned, a copy otherwise."""
    shape, st = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != HEAD_DIM or (rows is not None and shape[0] != rows):
        raise ValueError(f"{name}: shape (rows{'' if rows is None else f' = {rows}'}, heads, {HEAD_DIM}) needed, got {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, {dtype} needed")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, GPU {dev} needed")
    if st[2] == 1 and (st[1] == HEAD_DIM or shape[1] == 1) and st[0] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, st[0]
    return t.clone(memory_format=torch.contiguous_format), shape[1] * HEAD_DIM


def _out(out, q, dev):
    """(tensor, row stride) of the result: a new one, or the caller's."""
    if out is None:
        out = torch.empty_like(q)
        return out, out.stride(0)
    if out.shape == q.shape and out.dtype is q.dtype:
        o, stride = _heads("out", out, dev, q.dtype)
        if o is out:
            return out, stride
    raise ValueError(f"out: like q {tuple(q.shape)} {q.dtype}, heads packed, rows 16-byte aligned")


def _pools(kc, vc, dev, dtype, layers=False):
    """Shape of the two page pools, checked."""
    shape = kc.shape
    if (kc.dtype is dtype and vc.dtype is dtype and vc.shape == shape and len(shape) == 4 and shape[3] == HEAD_DIM and shape[2] in PAGE_SIZES
            and kc.is_contiguous() and vc.is_contiguous() and kc.get_device() == dev and vc.get_device() == dev and not layers):
        return shape
    if kc.dtype is not dtype or vc.dtype is not dtype:
        raise TypeError(f"caches are {kc.dtype} / {vc.dtype}, {dtype} needed")
    if vc.shape != shape or len(shape) != (5 if layers else 4) or shape[-1] != HEAD_DIM or shape[-2] not in PAGE_SIZES or shape[0] == 0:
        raise ValueError(f"caches: two pools of {'(n_layers, ' if layers else '('}n_pages, kv_heads, page_size in {PAGE_SIZES}, {HEAD_DIM}), got {tuple(shape)}, {tuple(vc.shape)}")
    if kc.get_device() != dev or vc.get_device() != dev:
        raise ValueError(f"caches on {kc.device} / {vc.device}, GPU {dev} needed")
    packed = shape[1] * shape[2] * shape[3] * shape[4] if layers else 0
    for c in (kc, vc):
        if not layers and not c.is_contiguous():
            raise ValueError("the pages must be contiguous")
        if layers and (c.stride()[1:] != (shape[2] * shape[3] * HEAD_DIM, shape[3] * HEAD_DIM, HEAD_DIM, 1) or c.stride(0) < packed or c.stride(0) != kc.stride(0)):
            raise ValueError("the pages of a layer must be contiguous, and both pools' layers equally far apart")
    return shape


def rope_kv_paged(q, k, v, positions, rope, slots, k_cache, v_cache, out=None):
    """RoPE on the rows' q and k (``[rows][heads][64]``, views of a fused projection work as they are), k and v written into the
    pages: row r goes to slot ``slots[r]`` of ``k_cache`` / ``v_cache`` ``[n_pages][kv_heads][page_size][64]`` (a slot outside the
    pool, -1 for instance: not written; a slot named twice: either row).  ``rope`` fp32 ``[positions][32][2]`` = (cos, sin);
    positions outside the table take its nearest row.  Returns the rotated q (``out``, which may be q itself)."""
    dev, dtype = _gpu(q, "rope_kv_paged"), q.dtype
    dt = _CODE[dtype] if dtype in _CODE else L.dtype_code(dtype)
    n_pages, hkv, page, _ = _pools(k_cache, v_cache, dev, dtype)
    if out is q:
        out, q_rs = _out(out, q, dev)
        out_rs = q_rs
    else:
        q, q_rs = _heads("q", q, dev, dtype)
        out, out_rs = _out(out, q, dev)
    rows, H, _ = q.shape
    k, k_rs = _heads("k", k, dev, dtype, rows)
    v, v_rs = _heads("v", v, dev, dtype, rows)
    if k.shape[1] != hkv or v.shape[1] != hkv:
        raise ValueError(f"k, v have {k.shape[1]}, {v.shape[1]} heads, the cache {hkv}")
    if rope.dtype is not F32 or rope.get_device() != dev or rope.dim() != 3 or rope.shape[1:] != (HEAD_DIM // 2, 2) or not rope.is_contiguous():
        raise ValueError(f"rope: contiguous float32 (positions, {HEAD_DIM // 2}, 2) table on GPU {dev} needed")
    per_row = (rows,)
    if rows == 0:
        return out
    _call(dev, L.load().valle_rope_kv_paged, q.data_ptr(), q_rs, k.data_ptr(), k_rs, v.data_ptr(), v_rs, out.data_ptr(), out_rs,
          _ints("positions", positions, dev, per_row), rope.data_ptr(), len(rope), _ints("slots", slots, dev, per_row), rows, H, hkv, HEAD_DIM,
          k_cache.data_ptr(), v_cache.data_ptr(), n_pages, page, dt)
    return out


def attn_tree(q, k_cache, v_cache, block_table, ctx_len, cu_rows, tree_mask=None, max_nodes=None, max_ctx=None, softmax_scale=None, out=None):
    """Attention of each request's new rows over its pages: request b asks with rows ``cu_rows[b] .. cu_rows[b+1]`` of q
    (``[rows][heads][64]``, heads a multiple of the cache's kv_heads; up to 64 rows per request), which see all of its
    ``ctx_len[b]`` cached rows and, of the new rows (cached behind them), those whose bit is set in ``tree_mask[row]`` (None: a
    chain, row i sees rows 0 .. i; one row: a plain decode step).  A row that sees nothing is zero.  Requests with a negative
    ``ctx_len`` and rows behind ``cu_rows[-1]`` are left as they were (``out=`` to say what that is).  ``max_nodes``: the largest
    number of rows of a request (default: as many as can be; rows behind it are left), ``max_ctx``: the longest context, a hint
    for how to split the work."""
    dev, dtype = _gpu(q, "attn_tree"), q.dtype
    dt = _CODE[dtype] if dtype in _CODE else L.dtype_code(dtype)
    n_pages, hkv, page, _ = _pools(k_cache, v_cache, dev, dtype)
    q, q_rs = _heads("q", q, dev, dtype)
    rows, H, _ = q.shape
    if block_table.dim() != 2:
        raise ValueError(f"block_table: (requests, max_blocks) needed, got {tuple(block_table.shape)}")
    B, width = block_table.shape
    if H % hkv:
        raise ValueError(f"{H} heads over {hkv} kv heads")
    if max_nodes is None:
        max_nodes = max(1, min(MAX_NODES, rows))
    if not 0 < max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes {max_nodes}: 1 .. {MAX_NODES}")
    if max_ctx is None:
        max_ctx = width * page
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    tab, ctx, cu = _ints("block_table", block_table, dev, (B, width)), _ints("ctx_len", ctx_len, dev, (B,)), _ints("cu_rows", cu_rows, dev, (B + 1,))
    mask = None if tree_mask is None else _ints("tree_mask", tree_mask, dev, (rows,), I64)
    out, out_rs = _out(out, q, dev)
    if rows == 0 or B == 0:
        return out
    lib = L.load()
    size = lib.valle_attn_tree_workspace_bytes(rows, B, max_nodes, max_ctx, H, hkv, dt)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None    # of this call: two streams or graphs never share it
    _call(dev, lib.valle_attn_tree, q.data_ptr(), q_rs, k_cache.data_ptr(), v_cache.data_ptr(), n_pages, page, tab, width, ctx, cu, mask,
          out.data_ptr(), out_rs, rows, B, max_nodes, max_ctx, H, hkv, HEAD_DIM, scale, dt, ws.data_ptr() if size else None, size)
    return out


def kv_commit(k_cache, v_cache, block_table, ctx_len, path, n_accept):
    """The accepted nodes of every request's tree become context, in all layers: cached row ``ctx_len[b] + path[b][j]`` moves to
    ``ctx_len[b] + j`` for ``j < n_accept[b]`` (``path`` int32 [requests][up to 64], node numbers 0 .. 63; others stay where they
    are).  Caches ``[n_layers][n_pages][kv_heads][page_size][64]``, changed in place.  Returns the new lengths ``ctx_len + n_accept``
    (a negative ``ctx_len`` stays)."""
    dev, dtype = _gpu(k_cache, "kv_commit"), k_cache.dtype
    dt = _CODE[dtype] if dtype in _CODE else L.dtype_code(dtype)
    layers, n_pages, hkv, page, _ = _pools(k_cache, v_cache, dev, dtype, layers=True)
    if block_table.dim() != 2 or path.dim() != 2 or not 0 < path.shape[1] <= MAX_NODES:
        raise ValueError(f"block_table (requests, max_blocks) and path (requests, 1 .. {MAX_NODES}) needed, got {tuple(block_table.shape)}, {tuple(path.shape)}")
    (B, width), wide, per_request = block_table.shape, path.shape[1], ctx_len.shape
    if per_request != (B,):
        raise ValueError(f"ctx_len: {B} lengths needed, got {tuple(per_request)}")
    out = torch.empty_like(ctx_len)
    if B == 0:
        return out
    _call(dev, L.load().valle_paged_kv_commit, k_cache.data_ptr(), v_cache.data_ptr(), layers, k_cache.stride(0), _ints("block_table", block_table, dev, (B, width)),
          width, n_pages, page, _ints("ctx_len", ctx_len, dev, per_request), _ints("path", path, dev, (B, wide)), wide,
          _ints("n_accept", n_accept, dev, per_request), out.data_ptr(), B, hkv, HEAD_DIM, dt)
    return out
