"""The paged KV cache and its operators (vall_e_amd/paged.py, csrc/paged.hip, csrc/attn_tree.hip) against plain restatements: whole numbers
and moved rows exactly, RoPE and attention in 64 bits.

Tolerances.  u = eps / 2 of the type (bf16 2^-8, fp32 2^-24), u32 = 2^-24.
RoPE: two fp32 products and a sum, one rounding: |err| <= 3 u32 (|a| + |b|) + u |y|.
Attention: a score is 64 products summed in fp32 (64 u32 x sum |q k|), scaled and put into exp2 (a few u32 x |score|): ds = 70 u32 x
scale x max_t sum |q k| bounds it, a weight is off by the factor e^(2 ds) (its own score and the maximum's); sums over T weights add
(T + 64) u32; in bf16 the weights of the numerator are rounded once (u).  So |err| <= (2.2 ds + (T + 64) u32 + [bf16] u) x sum p |v| + u |y|.
"""
import math

import numpy as np
import pytest
import torch

from vall_e_amd import paged as P

gpu = pytest.mark.gpu
U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.bfloat16, torch.float32]


# --------------------------------------------------------------------------------------- plain restatements
def blocks(n, page):
    return -(-n // page)


def ref_plan(len_old, len_new, table, n_blocks, free_list, free_count, page, max_rows, parents=None):
    """The plan as a scheduler would write it: lists, one request after the other."""
    n, width = table.shape
    table, held, fl = table.copy(), list(n_blocks), free_list.copy()
    cap = width * page
    status, cu = [0] * n, [0]
    for b in range(n):
        lo, ln = len_old[b], len_new[b]
        if not (0 <= lo <= cap and 0 <= ln <= cap and 0 <= held[b] <= width) or (parents is not None and ln - lo > 64):
            status[b] = 2
        cu.append(cu[-1] + (max(0, ln - lo) if status[b] == 0 else 0))
        if status[b] == 0 and cu[-1] > max_rows:
            status[b] = 3
    stack = [int(v) for v in fl[:free_count]]
    back = [int(table[b, k]) for b in range(n) if status[b] == 0 for k in range(blocks(len_new[b], page), held[b])]
    stack += back[::-1]
    fl[:len(stack)] = stack
    dry = False
    out_blocks = list(held)
    for b in range(n):
        need = blocks(len_new[b], page) - held[b] if status[b] == 0 else 0
        if need > 0 and (dry or need > len(stack)):
            status[b], dry = 1, True
        elif status[b] == 0:
            for k in range(max(0, need)):
                table[b, held[b] + k] = stack.pop()
            out_blocks[b] = blocks(len_new[b], page)
    slots, pos, masks = np.full(max_rows, -1, np.int64), np.zeros(max_rows, np.int64), np.zeros(max_rows, np.uint64)
    for b in range(n):
        ms, depth = [], []
        for i in range(cu[b + 1] - cu[b]):
            r = cu[b] + i
            if r >= max_rows:
                break
            p = -1 if parents is None else int(parents[r])
            p = p if 0 <= p < i else -1
            ms.append((1 << i) | (ms[p] if p >= 0 else 0))
            depth.append(depth[p] + 1 if p >= 0 else 0)
            if status[b] == 0:
                slots[r] = table[b, (len_old[b] + i) // page] * page + (len_old[b] + i) % page
            pos[r] = len_old[b] + (i if parents is None else depth[i])
            masks[r] = ms[i] & (2 ** 64 - 1) if parents is not None else 0
    return dict(block_table=table, n_blocks=out_blocks, free_list=fl, free_count=[len(stack)], status=status, cu_rows=cu, slots=slots,
                positions=pos, tree_mask=masks.view(np.int64))


def ref_attn(q, kc, vc, table, ctx, cu, masks, scale):
    """fp64 attention per (row, head): (out, bound of the module's docstring without the rounding of the result)."""
    rows, H, _ = q.shape
    kv, page = kc.shape[1], kc.shape[2]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    unit = UNIT[q.dtype] if q.dtype == torch.bfloat16 else 0.0
    for b, c in enumerate(ctx):
        n = cu[b + 1] - cu[b]
        if c < 0 or n == 0:
            continue
        pages = torch.as_tensor(table[b][:blocks(c + n, page)]).long()
        k = kc[pages].double().permute(1, 0, 2, 3).reshape(kv, -1, 64)[:, :c + n]
        v = vc[pages].double().permute(1, 0, 2, 3).reshape(kv, -1, 64)[:, :c + n]
        for i in range(n):
            m = (1 << (i + 1)) - 1 if masks is None else int(masks[cu[b] + i]) & (2 ** 64 - 1)
            seen = list(range(c)) + [c + j for j in range(n) if (m >> j) & 1]
            if not seen:
                continue
            for h in range(H):
                kk, vv, qq = k[h * kv // H, seen], v[h * kv // H, seen], q[cu[b] + i, h].double()
                p = torch.softmax(kk @ qq * scale, 0)
                out[cu[b] + i, h] = p @ vv
                ds = 70 * U32 * scale * float((kk.abs() @ qq.abs()).max())
                bound[cu[b] + i, h] = (2.2 * ds + (len(seen) + 64) * U32 + unit) * (p @ vv.abs())
    return out, bound


def random_tree(n, rs):
    return [int(rs.integers(-1, i)) if i and rs.random() < 0.85 else -1 for i in range(n)]


def tree_masks(parents):
    ms = []
    for i, p in enumerate(parents):
        ms.append((1 << i) | (ms[p] if p >= 0 else 0))
    return ms


def as_i64(bits):
    return torch.from_numpy(np.array([b & (2 ** 64 - 1) for b in bits], dtype=np.uint64).view(np.int64))


def rope_table(rows):
    fr = torch.arange(rows, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))[None, :]
    return torch.stack((fr.cos(), fr.sin()), -1).float()


# --------------------------------------------------------------------------------------- refusals (no GPU needed)
def test_cpu_tensors_are_refused():
    from vall_e_amd._lib import ValleHipError
    t = P.PageTable(2, 4, 8, 16, 64, device="cpu")
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValleHipError):
        t.plan(z, z)
    x = torch.zeros(2, 4, 64)
    kc, vc = P.kv_cache(1, 8, 16, 4, torch.float32, "cpu")
    with pytest.raises(ValleHipError):
        P.rope_kv_paged(x, x, x, z, rope_table(4), z, kc[0], vc[0])
    with pytest.raises(ValleHipError):
        P.attn_tree(x, kc[0], vc[0], torch.zeros(2, 4, dtype=torch.int32), z, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValleHipError):
        P.kv_commit(kc, vc, torch.zeros(2, 4, dtype=torch.int32), z, torch.zeros(2, 3, dtype=torch.int32), z)


@pytest.mark.parametrize("bad", [dict(page_size=24), dict(page_size=8), dict(max_requests=0), dict(max_requests=4097), dict(max_rows=0), dict(n_pages=0),
                                 dict(n_pages=2 ** 27)])
def test_page_table_refuses_shapes(bad):
    kw = dict(max_requests=2, max_blocks=4, n_pages=8, page_size=16, max_rows=64)
    kw.update(bad)
    with pytest.raises(ValueError):
        P.PageTable(**kw, device="cpu")


def test_c_entries_refuse_bad_arguments():
    """Status and message before anything is enqueued (pointers are never followed: no GPU)."""
    import ctypes as C
    from vall_e_amd import _lib as L
    lib, p = L.load(), C.c_void_p(4096)

    def plan(**kw):
        a = dict(lo=p, B=2, page=16, width=4, n_pages=8, max_rows=64, parents=None, mask=None, ticket=p)
        a.update(kw)
        return lib.valle_page_plan(a["lo"], p, a["B"], a["page"], p, a["width"], p, p, p, a["n_pages"], p, p, p, p, p, p, a["max_rows"], a["parents"], a["mask"], a["ticket"], None)
    for kw in (dict(lo=None), dict(ticket=None), dict(B=0), dict(B=4097), dict(page=15), dict(page=512), dict(width=0), dict(width=2 ** 30), dict(n_pages=0), dict(n_pages=2 ** 30),
               dict(max_rows=0), dict(parents=p), dict(mask=p)):
        assert plan(**kw) == -1, kw
        assert b"valle_page_plan" in lib.valle_last_error()

    def rope(**kw):
        a = dict(q=p, rs=256, k=p, qo=p, qo_rs=256, rows=4, M=2, H=4, Hkv=2, Dh=64, n_pages=8, page=16, dt=1)
        a.update(kw)
        return lib.valle_rope_kv_paged(a["q"], a["rs"], a["k"], 128, p, 128, a["qo"], a["qo_rs"], p, p, a["rows"], p, a["M"], a["H"], a["Hkv"], a["Dh"], p, p,
                                       a["n_pages"], a["page"], a["dt"], None)
    for kw, rc in ((dict(k=None), -1), (dict(qo=None), -1), (dict(dt=2), -1), (dict(Dh=128), -2), (dict(M=-1), -1), (dict(rs=252), -1), (dict(k=C.c_void_p(4104)), -1),
                   (dict(rows=0), -1), (dict(page=20), -1), (dict(qo_rs=64), -1), (dict(n_pages=2 ** 28), -1)):
        assert rope(**kw) == rc, kw
    assert rope(M=0) == 0

    def attn(**kw):
        a = dict(q=p, rs=256, n_pages=8, page=16, width=4, out_rs=256, rows=4, B=2, mn=2, ctx=100, H=4, Hkv=2, Dh=64, scale=0.125, dt=1, ws=None, nb=0)
        a.update(kw)
        return lib.valle_attn_tree(a["q"], a["rs"], p, p, a["n_pages"], a["page"], p, a["width"], p, p, None, p, a["out_rs"], a["rows"], a["B"], a["mn"], a["ctx"], a["H"],
                                   a["Hkv"], a["Dh"], a["scale"], a["dt"], a["ws"], a["nb"], None)
    for kw, rc in ((dict(q=None), -1), (dict(Dh=128), -2), (dict(dt=3), -1), (dict(mn=0), -1), (dict(mn=65), -1), (dict(Hkv=3), -1), (dict(scale=0.0), -1),
                   (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(rs=250), -1), (dict(out_rs=64), -1), (dict(page=17), -1),
                   (dict(width=0), -1), (dict(B=65536), -1), (dict(B=1, ctx=100000, ws=None), -4), (dict(B=1, ctx=100000, ws=p, nb=64), -4), (dict(ctx=-1), -1)):
        assert attn(**kw) == rc, kw
    assert attn(rows=0) == 0
    assert lib.valle_attn_tree_workspace_bytes(4, 1, 2, 100000, 4, 2, 1) > 0 and lib.valle_attn_tree_workspace_bytes(64, 64, 1, 500, 16, 16, 1) == 0

    def commit(**kw):
        a = dict(k=p, layers=2, stride=8 * 16 * 2 * 64, page=16, ctx=p, mp=4, out=C.c_void_p(8192), Dh=64, dt=1, Hkv=2)
        a.update(kw)
        return lib.valle_paged_kv_commit(a["k"], p, a["layers"], a["stride"], p, 4, 8, a["page"], a["ctx"], p, a["mp"], p, a["out"], 2, a["Hkv"], a["Dh"], a["dt"], None)
    for kw, rc in ((dict(k=None), -1), (dict(out=p), -1), (dict(stride=64), -1), (dict(mp=65), -1), (dict(mp=0), -1), (dict(page=1), -1), (dict(Dh=32), -2), (dict(dt=7), -1),
                   (dict(layers=0), -1), (dict(k=C.c_void_p(4098)), -1)):
        assert commit(**kw) == rc, kw


def test_restated_plan_gives_back_what_it_takes():
    """Growing and shrinking by the same pages leaves pool and stack as they were (the rule the kernel's numbering implements)."""
    table, nb, fl = np.zeros((3, 8), np.int32), [0, 0, 0], np.arange(20)[::-1].copy()
    a = ref_plan([0, 0, 0], [40, 17, 100], table, nb, fl, 20, 16, 256)
    assert a["status"] == [0, 0, 0] and a["n_blocks"] == [3, 2, 7] and a["free_count"] == [8]
    b = ref_plan([40, 17, 100], [0, 0, 0], a["block_table"], a["n_blocks"], a["free_list"], 8, 16, 256)
    assert b["free_count"] == [20] and (b["free_list"] == fl).all()


# --------------------------------------------------------------------------------------- plan
def run_plan(dev, len_old, len_new, page, width, n_pages, max_rows, held=None, free=None, parents=None, in_place=True, seed=0):
    """A table with the requests' pages dealt out at random, one plan on the GPU, and its restatement."""
    rs = np.random.default_rng(seed)
    n = len(len_old)
    held = [blocks(max(0, c), page) for c in len_old] if held is None else held
    perm = rs.permutation(n_pages).astype(np.int32)
    table, at = np.full((n, width), 7, np.int32), 0
    for b, h in enumerate(held):
        k = min(max(h, 0), width)
        table[b, :k] = perm[at:at + k]
        at += k
    fl = np.zeros(n_pages, np.int32)
    free = n_pages - at if free is None else free
    fl[:free] = perm[at:at + free]
    t = P.PageTable(n, width, n_pages, page, max_rows, device=dev)
    for name, v in (("block_table", table), ("n_blocks", np.array(held, np.int32)), ("free_list", fl), ("free_count", np.array([free], np.int32))):
        getattr(t, name).copy_(torch.from_numpy(v))
    t.slots.fill_(-9), t.positions.fill_(-9), t.cu_rows.fill_(-9), t.status.fill_(-9)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    par = None
    if parents is not None:
        par = i32(list(parents) + [5] * (max_rows - len(parents)))
    want = ref_plan(len_old, len_new, table, held, fl, free, page, max_rows, None if par is None else par.cpu().numpy())
    t.plan(i32(len_old), i32(len_new), parents=par, in_place=in_place)
    return t, want


def check_plan(t, want, tree, in_place=True):
    for name, w in want.items():
        if name == "tree_mask" and not tree:
            continue
        g = getattr(t, name if in_place or name not in ("n_blocks", "free_count") else "next_" + name)
        assert g.cpu().tolist() == np.asarray(w).tolist(), name


PLANS = {
    "one_token_each": ([5, 16, 31, 32, 0], [6, 17, 32, 33, 1]),
    "ends_and_idle": ([40, 0, 100, 17], [0, 0, 3, 49]),
    "shrinks": ([64, 65, 300], [63, 1, 17]),
    "prompts": ([0, 0, 0], [1, 64, 333]),
    "one_request": ([0], [1]),
    "bad_lengths": ([5, -1, 9, 10 ** 6, 7], [6, 4, -3, 10 ** 6 + 1, 8]),
}


@gpu
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("name", sorted(PLANS))
def test_plan_lengths(gpu_device, name, page):
    lo, ln = PLANS[name]
    t, want = run_plan(gpu_device, lo, ln, page, 24, 120, 512, seed=1)
    check_plan(t, want, False)


@gpu
@pytest.mark.parametrize("max_rows", [300, 4096, 4097, 9000])
@pytest.mark.parametrize("n", [1, 63, 700])
def test_plan_random_batches_and_throwaway(gpu_device, n, max_rows):
    """One launch and two, more requests than threads of a wave; some rows do not fit, some requests find no pages."""
    rs = np.random.default_rng(n + max_rows)
    lo = [int(v) for v in rs.integers(0, 200, n)]
    ln = [0 if rs.random() < 0.2 else c + int(rs.integers(0, 30)) for c in lo]
    held = sum(blocks(c, 16) for c in lo)
    for free, in_place in ((held // 4, True), (0, True), (3, False)):
        t, want = run_plan(gpu_device, lo, ln, 16, 16, held + 2000, max_rows, free=free, in_place=in_place, seed=n)
        check_plan(t, want, False, in_place)
        if not in_place:
            assert t.n_blocks.tolist() == [blocks(c, 16) for c in lo] and t.free_count.item() == 3


@gpu
def test_plan_more_requests_than_threads(gpu_device):
    n = 4096
    lo = [i % 50 for i in range(n)]
    ln = [c + 1 + i % 3 if i % 7 else 0 for i, c in enumerate(lo)]
    t, want = run_plan(gpu_device, lo, ln, 16, 4, sum(blocks(c, 16) for c in lo) + 500, 12000, seed=3)
    check_plan(t, want, False)


@gpu
@pytest.mark.parametrize("max_rows", [512, 5000])
def test_plan_trees(gpu_device, max_rows):
    """Chains of 64, stars, random trees, parents that are no earlier node (children of the context), a request with 65 rows."""
    rs = np.random.default_rng(5)
    sizes = [64, 64, 1, 0, 26, 65, 17, 3]
    lo = [10, 0, 33, 12, 500, 4, 16, 7]
    par = list(range(-1, 63)) + [-1] * 64 + [-1] + random_tree(26, rs) + random_tree(17, rs) + [2, 1, -7]
    t, want = run_plan(gpu_device, lo, [c + k for c, k in zip(lo, sizes)], 16, 40, 300, max_rows, parents=par, seed=2)
    assert want["status"][5] == 2
    check_plan(t, want, True)
    t, want = run_plan(gpu_device, lo, [c + k for c, k in zip(lo, sizes)], 16, 40, 60, max_rows, free=3, parents=par, seed=2)
    assert 1 in want["status"]
    check_plan(t, want, True)


@gpu
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("n", [17, 40, 64, 65, 200, 512, 600])
def test_plan_one_table_over_many_steps(gpu_device, tree, n):
    """Batches whose rows or trees take several workgroups (the counters are written by the last one to have read them), planned in place
    step after step on one table, directly and through a graph: the state of every step is the restatement's."""
    rs = np.random.default_rng(n)
    page, width, max_rows, n_pages = 16, 300, n * 64 if tree else n * 140, n * 20
    t = P.PageTable(n, width, n_pages, page, max_rows, device=gpu_device)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=gpu_device)
    lo, ln, par = i32(n), i32(n), i32(max_rows) if tree else None
    t.plan(lo, ln, parents=par)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.plan(lo, ln, parents=par)
    state = dict(block_table=np.zeros((n, width), np.int32), n_blocks=[0] * n, free_list=np.arange(n_pages - 1, -1, -1, dtype=np.int32), free_count=[n_pages])
    length = [0] * n
    for step in range(7):
        new = [0 if rs.random() < 0.15 else c + int(rs.integers(0, 65 if tree else 200)) for c in length]
        parents = None
        if tree:
            parents = np.array([p for c, m in zip(length, new) for p in random_tree(max(0, m - c), rs)], np.int32)
            parents = np.concatenate((parents, np.full(max_rows - len(parents), 3, np.int32)))[:max_rows]
            par.copy_(torch.from_numpy(parents))
        lo.copy_(torch.tensor(length, dtype=torch.int32)), ln.copy_(torch.tensor(new, dtype=torch.int32))
        want = ref_plan(length, new, state["block_table"], state["n_blocks"], state["free_list"], state["free_count"][0], page, max_rows, parents)
        graph.replay() if step % 2 else t.plan(lo, ln, parents=par)
        got = t.block_table.cpu().numpy()
        for b in range(n):                                             # (entries behind n_blocks mean nothing)
            k = want["n_blocks"][b]
            assert (got[b, :k] == want["block_table"][b, :k]).all()
        check_plan(t, {k: v for k, v in want.items() if k not in ("block_table", "free_list")}, tree)
        assert (t.free_list.cpu().numpy()[:want["free_count"][0]] == want["free_list"][:want["free_count"][0]]).all()
        state = want
        length = [m if s == 0 else c for c, m, s in zip(length, new, want["status"])]
    assert 0 < want["free_count"][0] < n_pages


@gpu
def test_plan_there_and_back_keeps_every_page(gpu_device):
    """A random life of a batch: whatever it does, every page is in exactly one table or on the stack."""
    rs = np.random.default_rng(11)
    n, page, width, n_pages = 12, 16, 10, 70
    t = P.PageTable(n, width, n_pages, page, 4096, device=gpu_device)
    lens = [0] * n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    for step in range(12):
        new = [int(rs.integers(0, 161)) if rs.random() < 0.7 else 0 for _ in lens]
        want = ref_plan(lens, new, t.block_table.cpu().numpy(), t.n_blocks.tolist(), t.free_list.cpu().numpy(), t.free_count.item(), page, 4096)
        t.plan(i32(lens), i32(new))
        check_plan(t, want, False)
        lens = [w if s == 0 else c for c, w, s in zip(lens, new, want["status"])]
        nb, fc = t.n_blocks.tolist(), t.free_count.item()
        pages = [int(v) for b in range(n) for v in t.block_table[b, :nb[b]].tolist()] + t.free_list[:fc].tolist()
        assert sorted(pages) == list(range(n_pages))
        assert nb == [max(blocks(c, page), 0) for c in lens]


@gpu
@pytest.mark.parametrize("n,max_rows", [(1, 64), (5, 400), (64, 3000), (65, 3000), (512, 5000), (600, 3000), (600, 9000)])
def test_plain_plan_behind_a_tree_plan(gpu_device, n, max_rows):
    """One table, planned with trees and then without: no bit of the trees stays in tree_mask, which holds the chains that attn_tree takes for no
    mask; the same where a captured plan with trees was replayed in between."""
    rs = np.random.default_rng(n + max_rows)
    dev, page = gpu_device, 16
    t = P.PageTable(n, 12, n * 12, page, max_rows, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    zero, trees = i32([0] * n), i32([min(4, max_rows // n)] * n)
    par = i32([-1] * max_rows)                                  # stars: a node sees itself alone
    t.plan(zero, trees, parents=par, in_place=False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.plan(zero, trees, parents=par, in_place=False)
    lo = [int(v) for v in rs.integers(0, 90, n)]
    t.plan(zero, i32(lo))                                       # the contexts' pages
    for new in ([int(rs.integers(0, 100 if n < 10 else 3)) for _ in lo], [1] * n, [0] * n):
        graph.replay()
        nodes, star = int(trees[0]) * n, 2 ** (torch.arange(max_rows) % int(trees[0]))
        star[nodes:] = 0
        assert torch.equal(t.tree_mask.cpu(), star)
        t.plan(i32(lo), i32([a + b for a, b in zip(lo, new)]), in_place=False)
        rows = [min(i, 63) for k in new for i in range(k)][:max_rows]
        assert t.tree_mask.tolist() == [(1 << (i + 1)) - 1 if i < 63 else -1 for i in rows] + [0] * (max_rows - len(rows))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_plain_step_with_the_table_s_mask(gpu_device, dtype):
    """A drafted step, then a plain one, both as the module's documentation writes them: tree_mask handed on whatever the plan was."""
    dev, page = gpu_device, 16
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    t = P.PageTable(3, 8, 24, page, 128, device=dev)
    kc, vc = randn((24, 2, page, 64), dtype, 1, dev), randn((24, 2, page, 64), dtype, 2, dev)
    q = randn((128, 4, 64), dtype, 3, dev)
    length = i32([20, 0, 47])
    t.plan(i32([0, 0, 0]), length)
    t.plan(length, i32([23, 9, 50]), parents=i32([-1] * 128))
    drafted = P.attn_tree(q, kc, vc, t.block_table, length, t.cu_rows, t.tree_mask, 9)
    length, new = i32([21, 1, 48]), i32([1, 3, 1])
    t.plan(length, length + new)
    got = P.attn_tree(q, kc, vc, t.block_table, length, t.cu_rows, t.tree_mask, 3)
    want = P.attn_tree(q, kc, vc, t.block_table, length, t.cu_rows, None, 3)
    assert torch.equal(got[:5], want[:5]) and not torch.equal(got[:5], drafted[:5])
    check_attn(got[:5], (q[:5].cpu(), kc.cpu(), vc.cpu(), t.block_table.cpu().numpy(), length.tolist(), t.cu_rows.tolist(), None))


def test_masked_plan_entry_refuses_bad_arguments():
    import ctypes as C
    from vall_e_amd import _lib as L
    lib, p = L.load(), C.c_void_p(4096)

    def plan(lo=p, B=2, page=16, max_rows=64, mask=p):
        return lib.valle_page_plan_masked(lo, p, B, page, p, 4, p, p, p, 8, p, p, p, p, p, p, max_rows, None, mask, p, None)
    for kw in (dict(mask=None), dict(lo=None), dict(B=0), dict(page=24), dict(max_rows=0)):
        assert plan(**kw) == -1, kw
        assert b"valle_page_plan" in lib.valle_last_error()


# --------------------------------------------------------------------------------------- RoPE + write
def randn(shape, dtype, seed, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,kv,page,fused", [(1, 1, 1, 16, False), (3, 16, 16, 16, False), (37, 6, 2, 64, True), (130, 12, 3, 256, True), (16, 32, 8, 32, False)])
def test_rope_kv_paged(gpu_device, dtype, rows, heads, kv, page, fused):
    n_pages = blocks(rows, page) + 2
    qkv = randn((rows, heads + 2 * kv, 64), dtype, rows, gpu_device)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    rs = np.random.default_rng(rows)
    slots = rs.permutation(n_pages * page)[:rows].astype(np.int32)
    if rows > 2:
        slots[1], slots[2] = -1, n_pages * page                  # padding, and a slot behind the pool
    pos = rs.integers(0, 200, rows).astype(np.int32)
    pos[0] = 199
    rope = rope_table(200)
    kc, vc = randn((n_pages, kv, page, 64), dtype, 1, gpu_device), randn((n_pages, kv, page, 64), dtype, 2, gpu_device)
    k0, v0 = kc.clone(), vc.clone()
    dev = lambda a: torch.from_numpy(a).to(gpu_device)
    got = P.rope_kv_paged(q, k, v, dev(pos), rope.to(gpu_device), dev(slots), kc, vc)

    def turned(x):
        x = x.cpu().double()
        cs = rope.double()[torch.from_numpy(pos).long()][:, None]
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]), -1).flatten(-2)
        s = (a.abs() + b.abs()).repeat_interleave(2, -1)
        return y, 3 * U32 * s + UNIT[dtype] * y.abs()
    want, tol = turned(q)
    assert ((got.cpu().double() - want).abs() <= tol).all()
    wk, tk = turned(k)
    kc, vc, k0, v0 = kc.cpu(), vc.cpu(), k0.cpu(), v0.cpu()
    for r in range(rows):
        if 0 <= slots[r] < n_pages * page:
            p, o = divmod(int(slots[r]), page)
            assert ((kc[p, :, o].double() - wk[r]).abs() <= tk[r]).all() and torch.equal(vc[p, :, o], v[r].cpu())
            k0[p, :, o], v0[p, :, o] = kc[p, :, o], vc[p, :, o]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)           # nothing else was touched


@gpu
def test_rope_kv_paged_in_place_and_positions_outside_the_table(gpu_device):
    q, k, v = (randn((4, 2, 64), torch.float32, i, gpu_device) for i in range(3))
    kc, vc = P.kv_cache(1, 2, 16, 2, torch.float32, gpu_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    rope = rope_table(50).to(gpu_device)
    want = P.rope_kv_paged(q, k, v, i32([0, 49, 0, 49]), rope, i32([0, 1, 2, 3]), kc[0], vc[0])
    got = P.rope_kv_paged(q, k, v, i32([-5, 50, 0, 10 ** 9]), rope, i32([4, 5, 6, 7]), kc[0], vc[0], out=q)
    assert got is q and torch.equal(q, want)
    assert torch.equal(kc[0, 0, :, 0:4], kc[0, 0, :, 4:8])


@gpu
def test_rope_kv_paged_agrees_with_the_slot_cache_operator(gpu_device):
    """fp32: the same rotation as valle_rope_kv (which rounds its products apart): within 3 u32 (|a| + |b|)."""
    from vall_e_amd import _lib as L
    M, H = 9, 4
    qkv = randn((M, 3 * H * 64), torch.float32, 4, gpu_device)
    pos = torch.arange(M, dtype=torch.int32, device=gpu_device) * 7
    rope = rope_table(100).to(gpu_device)
    x = qkv.view(M, 3 * H, 64)
    kc, vc = P.kv_cache(1, 1, 16, H, torch.float32, gpu_device)
    q = P.rope_kv_paged(x[:, :H], x[:, H:2 * H], x[:, 2 * H:], pos, rope, torch.arange(M, dtype=torch.int32, device=gpu_device), kc[0], vc[0])
    ref = qkv.clone()
    L.check(L.load().valle_rope_kv(L.ptr(ref), L.ptr(pos), L.ptr(rope), None, 1, M, H, 64, None, None, 0, None, None, L.F32, L.stream_ptr(gpu_device)))
    ref = ref.view(M, 3 * H, 64)
    lim = 4 * U32 * 2 * qkv.abs().max()
    assert (q - ref[:, :H]).abs().max() <= lim and (kc[0, 0, :, :M].transpose(0, 1) - ref[:, H:2 * H]).abs().max() <= lim
    assert torch.equal(vc[0, 0, :, :M].transpose(0, 1), x[:, 2 * H:])


# --------------------------------------------------------------------------------------- attention
def attn_case(dev, dtype, ctx, nodes, H, kv, page, seed, masks="tree", poison=False, extra_rows=0, width=None):
    rs = np.random.default_rng(seed)
    total = [max(0, c) + n for c, n in zip(ctx, nodes)]
    need = [blocks(t, page) for t in total]
    n_pages = sum(need) + 3
    perm = rs.permutation(n_pages)
    table, at = np.full((len(ctx), width or max(1, max(need))), -1, np.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    cu = np.concatenate(([0], np.cumsum(nodes))).astype(np.int32)
    rows = int(cu[-1]) + extra_rows
    q = randn((rows, H, 64), dtype, seed, "cpu")
    kc, vc = randn((n_pages, kv, page, 64), dtype, seed + 1, "cpu"), randn((n_pages, kv, page, 64), dtype, seed + 2, "cpu")
    if poison:                                                   # everything behind the sequences, and the pages nobody has
        kp, vp = torch.full_like(kc, float("nan")), torch.full_like(vc, float("inf"))
        for b in range(len(ctx)):
            for t in range(total[b]):
                p, o = table[b, t // page], t % page
                kp[p, :, o], vp[p, :, o] = kc[p, :, o], vc[p, :, o]
        kc, vc = kp, vp
    ms = None
    if masks == "tree":
        ms = [m for n in nodes for m in tree_masks(random_tree(n, rs))]
    elif masks == "random":
        ms = [int(rs.integers(0, 2 ** 62)) & int(rs.integers(0, 2 ** 62)) | (int(rs.integers(0, 2)) << 63) for _ in range(int(cu[-1]))]
    elif masks == "none_seen":
        ms = [0] * int(cu[-1])
    d = lambda a: (torch.from_numpy(a) if isinstance(a, np.ndarray) else a).to(dev)
    mask = None if ms is None else d(as_i64(ms + [0] * extra_rows))
    args = (d(q), d(kc), d(vc), d(table), d(np.array(ctx, np.int32)), d(cu))
    return args, mask, (q, kc, vc, table, ctx, cu.tolist(), ms)


def check_attn(got, host, scale=0.125):
    q, kc, vc, table, ctx, cu, ms = host
    want, bound = ref_attn(q, kc, vc, table, ctx, cu, ms, scale)
    live = [r for b, c in enumerate(ctx) if c >= 0 for r in range(cu[b], cu[b + 1])]       # rows of finished requests hold whatever they held
    got, want, bound = got.cpu().double()[live], want[live], bound[live]
    err = (got - want).abs()
    lim = bound + UNIT[q.dtype] * want.abs()
    assert (err <= lim).all(), (float((err - lim).max()), float(err.max()))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,kv,page", [(1, 1, 16), (4, 4, 32), (6, 2, 16), (8, 1, 64), (5, 5, 256)])
@pytest.mark.parametrize("masks", ["tree", None, "random"])
def test_attn_tree_ragged_batches(gpu_device, dtype, H, kv, page, masks):
    """Contexts of nothing, one, a tile's edge and several pages; 1 to 64 nodes; pages that end inside a tile; NaN and infinities
    behind every sequence."""
    ctx, nodes = [0, 1, 15, 16, 31, 33, 100, 257], [1, 64, 17, 2, 5, 33, 9, 1]
    args, mask, host = attn_case(gpu_device, dtype, ctx, nodes, H, kv, page, 7, masks=masks, poison=True)
    check_attn(P.attn_tree(*args, tree_mask=mask), host)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,ctx,nodes,H,kv", [(1, 3000, 1, 2, 2), (1, 2049, 26, 4, 1), (2, 1500, 64, 2, 2), (3, 777, 3, 4, 2), (1, 4100, 64, 4, 1), (40, 70, 2, 16, 16)])
def test_attn_tree_split_keys(gpu_device, dtype, B, ctx, nodes, H, kv):
    """Key axes long enough to be split over workgroups; one request much shorter than the others (some parts are empty)."""
    c = [ctx - 13 * i for i in range(B)]
    if B > 1:
        c[-1] = 5
    args, mask, host = attn_case(gpu_device, dtype, c, [nodes] * B, H, kv, 16, 3, poison=True)
    check_attn(P.attn_tree(*args, tree_mask=mask, max_nodes=nodes, max_ctx=max(c)), host)
    check_attn(P.attn_tree(*args, tree_mask=mask), host)                              # defaults: other splits
    check_attn(P.attn_tree(*args, tree_mask=mask, max_nodes=nodes, max_ctx=1), host)  # a wrong hint costs time, not results


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attn_tree_rows_that_see_nothing_are_zero(gpu_device, dtype):
    args, mask, host = attn_case(gpu_device, dtype, [0, 0, 20], [3, 64, 5], 4, 2, 16, 5, masks="none_seen", poison=True)
    got = P.attn_tree(*args, tree_mask=mask)
    assert (got[:67] == 0).all()
    check_attn(got, host)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("val", [float("inf"), float("-inf"), float("nan")])
def test_attn_tree_siblings_with_infinities_and_nan(gpu_device, dtype, val):
    """A node whose key and value rows hold infinities or NaN: rows that do not see it keep their result bit for bit, rows that
    see its value get what the sum gives."""
    ctx, nodes = [30, 0, 200], [20, 40, 6]
    args, mask, host = attn_case(gpu_device, dtype, ctx, nodes, 4, 2, 16, 8)
    clean = P.attn_tree(*args, tree_mask=mask)
    table, ms = host[3], host[6]
    for which in ("k", "v"):
        q, kc, vc, *rest = args
        kc, vc = kc.clone(), vc.clone()
        node = 4
        for b, c in enumerate(ctx):
            p, o = table[b, (c + node) // 16], (c + node) % 16
            (kc if which == "k" else vc)[p, :, o, 5] = val
        got = P.attn_tree(q, kc, vc, *rest, tree_mask=mask)
        sees = torch.tensor([bool((m >> node) & 1) for m in ms])
        assert sees.any() and not sees.all()
        assert torch.equal(got[~sees.to(gpu_device)], clean[~sees.to(gpu_device)])
        if which == "v":
            hit = got[sees.to(gpu_device)][:, :, 5]
            assert (torch.isnan(hit) if math.isnan(val) else hit == val).all()
            rest_cols = [d for d in range(64) if d != 5]
            assert torch.equal(got[:, :, rest_cols], clean[:, :, rest_cols])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx", [[30, 5], [3000, 2100]])
def test_attn_tree_infinities_and_nan_that_are_seen_are_not_lost(gpu_device, dtype, ctx):
    """NaN in a query reaches that row alone; NaN in a context key every row of its request and kv head, an infinity in a context value
    every row's element of that dimension; nobody else's bits change.  (No key of a NaN query has a score with a maximum.)"""
    args, mask, host = attn_case(gpu_device, dtype, ctx, [6, 18], 4, 2, 16, 12)
    clean = P.attn_tree(*args, tree_mask=mask)
    q, kc, vc, *rest = args
    bad = q.clone()
    bad[2, 1, 7] = float("nan")
    got = P.attn_tree(bad, kc, vc, *rest, tree_mask=mask)
    assert got[2, 1].isnan().all()
    got[2, 1] = clean[2, 1]
    assert torch.equal(got, clean)
    for t in (0, 3, ctx[0] - 1):
        at = (int(host[3][0, t // 16]), 0, t % 16)
        bad = kc.clone()
        bad[at] = float("nan")
        got = P.attn_tree(q, bad, vc, *rest, tree_mask=mask)
        assert got[:6, :2].isnan().all() and torch.equal(got[:6, 2:], clean[:6, 2:]) and torch.equal(got[6:], clean[6:])
        bad = vc.clone()
        bad[at][9] = float("inf")
        got = P.attn_tree(q, kc, bad, *rest, tree_mask=mask)
        assert not got[:6, :2, 9].isfinite().any()
        got[:6, :2, 9] = clean[:6, :2, 9]
        assert torch.equal(got, clean)


@gpu
def test_attn_tree_leaves_other_rows(gpu_device):
    """Rows behind the last request, of finished requests (negative ctx_len) and behind max_nodes stay as they were."""
    for ctx in ([50, 70, 40], [3000, 4000, 3500]):
        args, mask, host = attn_case(gpu_device, torch.bfloat16, ctx, [4, 5, 6], 4, 4, 16, 4, extra_rows=7)
        args[4][1] = -1 - ctx[1]
        out = torch.full_like(args[0], 3.0)
        got = P.attn_tree(*args, tree_mask=mask, out=out)
        assert got is out and (out[4:9] == 3).all() and (out[15:] == 3).all() and not (out[:4] == 3).all()
        host[4][1] = -1
        want, bound = ref_attn(*host, 0.125)
        keep = [0, 1, 2, 3, 9, 10, 11, 12, 13, 14]
        assert ((out.cpu().double() - want).abs() <= bound + 2.0 ** -8 * want.abs())[keep].all()
        out.fill_(3.0)
        P.attn_tree(*args, tree_mask=mask, out=out, max_nodes=4)
        assert (out[13:] == 3).all() and (out[9:13] != 3).any()


@gpu
def test_attn_tree_views_scale_and_streams(gpu_device):
    """q as a view of a fused projection, out with padded rows, a scale of its own, on another stream than the current one."""
    args, mask, host = attn_case(gpu_device, torch.bfloat16, [40, 90], [3, 8], 4, 2, 32, 6)
    fused = torch.zeros(11, 8, 64, dtype=torch.bfloat16, device=gpu_device)
    fused[:, 2:6] = args[0]
    big = torch.zeros(11, 6, 64, dtype=torch.bfloat16, device=gpu_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        P.attn_tree(fused[:, 2:6], *args[1:], tree_mask=mask, softmax_scale=0.3, out=big[:, :4])
    torch.cuda.current_stream().wait_stream(s)
    assert (big[:, 4:] == 0).all()
    check_attn(big[:, :4], host, scale=0.3)
    odd = torch.zeros(11 * 256 + 1, dtype=torch.bfloat16, device=gpu_device)[1:].view(11, 4, 64)      # 2 bytes off: copied
    odd.copy_(args[0])
    check_attn(P.attn_tree(odd, *args[1:], tree_mask=mask), host)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,nodes,H,kv", [([40, 90], [30, 8], 8, 2), ([2500], [40], 4, 1), ([9, 0, 70], [1, 1, 1], 3, 3)])
def test_attn_tree_result_in_place_of_the_queries(gpu_device, dtype, ctx, nodes, H, kv):
    """out=q, with several query blocks and with split keys: the same bits as into a tensor of its own."""
    args, mask, host = attn_case(gpu_device, dtype, ctx, nodes, H, kv, 16, 14)
    want = P.attn_tree(*args, tree_mask=mask, max_nodes=max(nodes), max_ctx=max(ctx))
    q = args[0].clone()
    assert P.attn_tree(q, *args[1:], tree_mask=mask, max_nodes=max(nodes), max_ctx=max(ctx), out=q) is q and torch.equal(q, want)


@gpu
def test_attn_tree_more_heads_than_a_grid_of_small_blocks_holds(gpu_device):
    """20,480 heads in groups of 1,024, 64 nodes: query blocks are taken as large as the grid needs; too many are refused."""
    from vall_e_amd import _lib as L
    kc, vc = randn((2, 20, 16, 64), torch.bfloat16, 1, gpu_device), randn((2, 20, 16, 64), torch.bfloat16, 2, gpu_device)
    q = randn((64, 20 * 1024, 64), torch.bfloat16, 3, gpu_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    got = P.attn_tree(q, kc, vc, i32([[1, 0, 0, 0, 0]]), i32([16]), i32([0, 64]))
    rows, heads = [0, 1, 5], [0, 1023, 1024, 20479]                                      # a chain: row i sees itself and what lies before it
    for r in rows:
        for h in heads:
            k = torch.cat((kc[1, h // 1024], kc[0, h // 1024]))[:17 + r].double().cpu()
            v = torch.cat((vc[1, h // 1024], vc[0, h // 1024]))[:17 + r].double().cpu()
            w = torch.softmax(k @ q[r, h].double().cpu() * 0.125, 0)
            ds = 70 * U32 * 0.125 * float((k.abs() @ q[r, h].double().cpu().abs()).max())
            lim = (2.2 * ds + 81 * U32 + 2.0 ** -8) * (w @ v.abs()) + 2.0 ** -8 * (w @ v).abs()
            assert ((got[r, h].cpu().double() - w @ v).abs() <= lim).all()
    kc, vc = (torch.zeros(2, 63, 16, 64, device=gpu_device) for _ in range(2))
    with pytest.raises(L.ValleHipError, match="too many"):
        P.attn_tree(torch.zeros(64, 63 * 1024, 64, device=gpu_device), kc, vc, i32([[1, 0]]), i32([16]), i32([0, 64]))


@gpu
def test_attn_tree_one_token_equals_the_slot_cache_operator(gpu_device):
    """One node per request over pages == valle_attn_decode over slots, both within the bound of the fp64 result."""
    from vall_e_amd import _lib as L
    B, H, T = 5, 4, 96
    ctx = [95, 1, 33, 64, 17]
    kv = randn((2, B, H, T, 64), torch.bfloat16, 1, gpu_device)
    q = randn((B, H, 64), torch.bfloat16, 2, gpu_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    qkv = torch.cat((q.reshape(B, H * 64), torch.zeros(B, 2 * H * 64, dtype=torch.bfloat16, device=gpu_device)), 1).contiguous()
    slot_out = torch.empty(B, H, 64, dtype=torch.bfloat16, device=gpu_device)
    keys = [c + 1 for c in ctx]
    L.check(L.load().valle_attn_decode(L.ptr(qkv), L.ptr(kv[0]), L.ptr(kv[1]), L.ptr(i32(keys)), None, L.ptr(slot_out), B, H, 64, T, L.BF16, L.stream_ptr(gpu_device)))
    pages = kv.view(2, B, H, T // 32, 32, 64).transpose(2, 3).reshape(2, B * 3, H, 32, 64).contiguous()
    table = torch.arange(B * 3, dtype=torch.int32, device=gpu_device).view(B, 3)
    got = P.attn_tree(q, pages[0], pages[1], table, i32(ctx), torch.arange(B + 1, dtype=torch.int32, device=gpu_device))
    host = (q.cpu(), pages[0].cpu(), pages[1].cpu(), table.cpu().numpy(), ctx, list(range(B + 1)), None)
    check_attn(got, host)
    want, bound = ref_attn(*host, 0.125)
    assert ((slot_out.cpu().double() - got.cpu().double()).abs() <= 2 * (bound + 2.0 ** -8 * want.abs())).all()


@gpu
def test_attn_tree_pages_outside_the_pool_count_as_absent(gpu_device):
    args, mask, host = attn_case(gpu_device, torch.float32, [100, 64], [2, 2], 2, 2, 16, 9, masks=None)
    table = args[3].clone()
    table[0, 2], table[0, 4], table[1, 0] = -1, 10 ** 9, args[1].shape[0]
    got = P.attn_tree(*args[:3], table, *args[4:])
    q, kc, vc, tab, ctx, cu, _ = host
    for b, gone in ((0, {2, 4}), (1, {0})):
        for i in range(2):
            seen = [t for t in range(ctx[b] + i + 1) if t // 16 not in gone]
            for h in range(2):
                k = torch.stack([kc[tab[b, t // 16], h, t % 16] for t in seen]).double()
                v = torch.stack([vc[tab[b, t // 16], h, t % 16] for t in seen]).double()
                w = torch.softmax(k @ q[cu[b] + i, h].double() * 0.125, 0) @ v
                assert (got[cu[b] + i, h].cpu().double() - w).abs().max() < 1e-4       # fp32: far above the bound, far below a lost or extra row


@gpu
def test_attn_tree_offsets_pass_32_bits(gpu_device):
    """Pools of more than 2^31 elements and 2^32 bytes: the sequence lies in the last pages."""
    page, kv, n_pages = 256, 16, 8400
    kc = torch.empty(n_pages, kv, page, 64, dtype=torch.bfloat16, device=gpu_device)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31
    last = [n_pages - 1, n_pages - 3]
    q, k, v = (randn((400, kv, 64), torch.bfloat16, 20 + i, gpu_device) for i in range(3))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    slots = i32([last[t // page] * page + t % page for t in range(400)])
    rope = torch.zeros(1, 32, 2, device=gpu_device)
    rope[..., 0] = 1.0                                                                  # no rotation: rows arrive as they are
    P.rope_kv_paged(q, k, v, i32([0] * 400), rope, slots, kc, vc)
    got = P.attn_tree(q[397:], kc, vc, i32([last]), i32([397]), i32([0, 3]))
    small = (q[397:].cpu(), kc[last].cpu(), vc[last].cpu(), np.array([[0, 1]]), [397], [0, 3], None)
    assert torch.equal(small[1].transpose(1, 2).reshape(512, kv, 64)[:400], k.cpu())
    check_attn(got, small)


# --------------------------------------------------------------------------------------- commit
@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,kv,page", [(1, 1, 16), (3, 4, 32), (2, 3, 256)])
def test_kv_commit(gpu_device, dtype, layers, kv, page):
    """Overlapping sources and destinations, paths over page edges, rows that stay, nothing accepted, a finished request, all 64."""
    ctx = [0, 15, 31, 100, -5, 9, 40]
    path = [[0, 1, 2], [3, 4, 9], [63, 5, 7], [1, 2, 3], [4, 5, 6], [2, 64, -1], [5, 6, 7]]
    wide = np.zeros((7, 64), np.int32)
    for b, p in enumerate(path):
        wide[b, :3] = p
    wide[6] = np.arange(63, -1, -1)                                                     # the whole tree turned round
    acc = [3, 3, 3, 2, 3, 3, 64]
    need = [blocks(max(0, c) + 64, page) for c in ctx]
    n_pages = sum(need) + 1
    perm = np.random.default_rng(1).permutation(n_pages)
    table, at = np.zeros((7, max(need)), np.int32), 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    kc, vc = randn((layers, n_pages, kv, page, 64), dtype, 1, gpu_device), randn((layers, n_pages, kv, page, 64), dtype, 2, gpu_device)
    want = []
    for c in (kc.cpu(), vc.cpu()):
        new = c.clone()
        for b in range(7):
            for j in range(acc[b]):
                if ctx[b] >= 0 and 0 <= wide[b, j] < 64:
                    s, d = ctx[b] + int(wide[b, j]), ctx[b] + j
                    new[:, table[b, d // page], :, d % page] = c[:, table[b, s // page], :, s % page]
        want.append(new)
    i32 = lambda x: torch.from_numpy(np.asarray(x, dtype=np.int32)).to(gpu_device)
    out = P.kv_commit(kc, vc, i32(table), i32(ctx), i32(wide), i32(acc))
    assert out.tolist() == [3, 18, 34, 102, -5, 12, 104]
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


@gpu
def test_kv_commit_layer_slices_and_counts_out_of_range(gpu_device):
    """Two middle layers of a bigger cache; n_accept below 0 and above the path's width."""
    kc, vc = randn((4, 6, 2, 16, 64), torch.bfloat16, 1, gpu_device), randn((4, 6, 2, 16, 64), torch.bfloat16, 2, gpu_device)
    k0 = kc.clone()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    out = P.kv_commit(kc[1:3], vc[1:3], i32([[0, 1], [2, 3]]), i32([4, 4]), i32([[3, 5], [3, 5]]), i32([-2, 9]))
    assert out.tolist() == [4, 6]
    k0[1:3, 2, :, 4], k0[1:3, 2, :, 5] = k0[1:3, 2, :, 7].clone(), k0[1:3, 2, :, 9].clone()
    assert torch.equal(kc, k0)


def ref_commit(kc, vc, table, ctx, path, acc, page, n_blocks, status):
    """The commit as a scheduler would write it, request after request: (k, v, new lengths)."""
    out, lens = [c.clone() for c in (kc, vc)], []
    for b, c in enumerate(ctx):
        held, fine = (table.shape[1] if n_blocks is None else n_blocks[b]) * page, status is None or status[b] == 0
        n = min(max(acc[b], 0), len(path[b])) if fine else 0
        lens.append(c if c < 0 else min(c + n, held) if fine and n_blocks is not None else c + n)
        for j in range(n if c >= 0 else 0):
            s, d = c + int(path[b][j]), c + j
            if 0 <= path[b][j] < 64 and s < held and d < held:
                for new, old in zip(out, (kc, vc)):
                    new[:, table[b, d // page], :, d % page] = old[:, table[b, s // page], :, s % page]
    return out[0], out[1], lens


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_refused_request_leaves_the_pages_of_others(gpu_device, dtype):
    """A step in which the pool runs dry in front of one request, its drafted nodes accepted all the same (nothing is read back in between): its
    left-over table entry names page 0, another request's.  Every page but the served ones' rows stays bit for bit, its length too; a later plan
    serves it."""
    dev, page, layers, kv = gpu_device, 16, 2, 2
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = P.PageTable(3, 6, 7, page, 128, device=dev)
    table.plan(i32([0, 0, 0]), i32([30, 40, 10]))
    assert table.n_blocks.tolist() == [2, 3, 1] and table.free_count.item() == 1
    length = i32([30, 40, 10])
    kc, vc = randn((layers, 7, kv, page, 64), dtype, 1, dev), randn((layers, 7, kv, page, 64), dtype, 2, dev)
    nodes = [3, 20, 5]                                          # 33 rows need the last page, 60 rows one that is not there, 15 none
    table.plan(length, length + i32(nodes), parents=i32([-1, 0, 1] + [-1] * 20 + list(range(-1, 4)) + [0] * 100))
    assert table.status.tolist() == [0, 1, 0] and table.n_blocks.tolist() == [3, 3, 1] and table.block_table[1, 3].item() == 0 and table.block_table[0, 0].item() == 0
    rows = sum(nodes)
    q, k, v = (randn((rows, heads, 64), dtype, 3 + heads, dev) for heads in (4, kv, kv))
    for l in range(layers):
        k0, v0 = kc[l].clone(), vc[l].clone()
        t = P.rope_kv_paged(q, k, v, table.positions[:rows].contiguous(), rope_table(64).to(dev), table.slots[:rows].contiguous(), kc[l], vc[l])
        for s in table.slots[:rows].tolist():
            if s >= 0:
                k0[s // page, :, s % page], v0[s // page, :, s % page] = kc[l, s // page, :, s % page], vc[l, s // page, :, s % page]
        assert torch.equal(kc[l], k0) and torch.equal(vc[l], v0)
        P.attn_tree(t, kc[l], vc[l], table.block_table, length, table.cu_rows, table.tree_mask[:rows].contiguous(), max_nodes=20)
        assert torch.equal(kc[l], k0) and torch.equal(vc[l], v0)
    path = [[0, 1, 2] + [0] * 17, list(range(6, 20)) + [0] * 6, [1, 2, 4] + [0] * 17]
    acc = [3, 14, 3]
    want = ref_commit(kc.cpu(), vc.cpu(), table.block_table.cpu().numpy(), length.tolist(), path, acc, page, table.n_blocks.tolist(), table.status.tolist())
    out = P.kv_commit(kc, vc, table.block_table, length, i32(path), i32(acc), table.n_blocks, table.status)
    assert out.tolist() == want[2] == [33, 40, 13]
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    table.plan(out, i32([0, 41, 13]))                           # the first request ends: there is room again
    assert table.status.tolist() == [0, 0, 0] and table.n_blocks.tolist() == [0, 3, 1]
    table.plan(out, i32([0, 60, 13]))
    assert table.status.tolist() == [0, 0, 0] and table.n_blocks.tolist() == [0, 4, 1]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_kv_commit_inside_the_pages_held(gpu_device, dtype, page):
    """Any status, any n_accept and path, left-over entries that name the pages of others (or nothing): only the rows of served requests
    inside the pages they hold are read or written; both arguments alone and none of them too."""
    dev, layers, kv, n = gpu_device, 2, 3, 24
    rs = np.random.default_rng(page)
    width = 192 // page
    i32 = lambda v: torch.from_numpy(np.asarray(v, dtype=np.int32)).to(dev)
    held = [int(rs.integers(0, width + 1)) for _ in range(n)]
    ctx = [int(rs.integers(0, max(1, h * page))) if rs.random() < 0.9 else -2 for h in held]
    ctx[0], held[0] = 100, 0                                    # an ended request
    ctx[1], held[1] = 2 * page, 2                               # a full last page: its first new row would lie behind it
    pool = sum(held) + 2
    perm, at = rs.permutation(pool), 0
    table = rs.integers(-3, pool + 3, (n, width)).astype(np.int32)
    for b, h in enumerate(held):
        table[b, :h] = perm[at:at + h]
        at += h
    kc, vc = randn((layers, pool, kv, page, 64), dtype, 1, dev), randn((layers, pool, kv, page, 64), dtype, 2, dev)
    path = np.stack([rs.permutation(66)[:64] - 1 for _ in range(n)]).astype(np.int32)
    acc = [int(rs.integers(-2, 70)) for _ in range(n)]
    status = [int(rs.choice([0, 0, 0, 1, 2, 3])) for _ in range(n)]
    status[0] = status[1] = 0
    for nb, st in ((held, status), (held, None)):
        want = ref_commit(kc.cpu(), vc.cpu(), table, ctx, path, acc, page, nb, st)
        k, v = kc.clone(), vc.clone()
        out = P.kv_commit(k, v, i32(table), i32(ctx), i32(path), i32(acc), i32(nb), None if st is None else i32(st))
        assert out.tolist() == want[2] and want[2][0] == 0 and want[2][1] == 2 * page
        assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    none = [0 if s == 0 else a for s, a in zip(status, acc)]     # status alone: the served ones accept nothing here
    k, v = kc.clone(), vc.clone()
    assert P.kv_commit(k, v, i32(table), i32(ctx), i32(path), i32(none), status=i32(status)).tolist() == ctx and torch.equal(k, kc) and torch.equal(v, vc)
    for kw in (dict(n_blocks=i32(held[:-1])), dict(status=i32(status).long()), dict(n_blocks=i32(held).cpu()), dict(status=i32(status + [0]))):
        with pytest.raises(ValueError):
            P.kv_commit(k, v, i32(table), i32(ctx), i32(path), i32(acc), **kw)


def test_commit_entry_for_served_requests_refuses_bad_arguments():
    import ctypes as C
    from vall_e_amd import _lib as L
    lib, p, o = L.load(), C.c_void_p(4096), C.c_void_p(8192)

    def call(ctx=p, n_blocks=p, status=p, out=o, B=2, layers=2):
        return lib.valle_paged_kv_commit_served(p, p, layers, 8 * 16 * 2 * 64, p, 4, 8, 16, ctx, n_blocks, status, p, 4, p, out, B, 2, 64, 1, None)
    for kw in (dict(ctx=o), dict(n_blocks=o), dict(status=o), dict(ctx=None), dict(out=None), dict(layers=0), dict(B=-1)):
        assert call(**kw) == -1, kw
        assert b"valle_paged_kv_commit" in lib.valle_last_error()
    assert call(B=0) == 0 and call(B=0, n_blocks=None, status=None) == 0


@gpu
def test_empty_calls(gpu_device):
    """No rows, no requests: nothing to do, nothing touched."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu_device)
    kc, vc = randn((1, 3, 2, 16, 64), torch.float32, 1, gpu_device), randn((1, 3, 2, 16, 64), torch.float32, 2, gpu_device)
    k0 = kc.clone()
    q = torch.zeros(0, 2, 64, device=gpu_device)
    assert P.rope_kv_paged(q, q, q, i32(0), rope_table(4).to(gpu_device), i32(0), kc[0], vc[0]).shape == (0, 2, 64)
    assert P.attn_tree(q, kc[0], vc[0], i32(2, 1), i32(2), i32(3)).shape == (0, 2, 64)
    assert P.attn_tree(torch.zeros(3, 2, 64, device=gpu_device), kc[0], vc[0], i32(0, 1), i32(0), i32(1)).shape == (3, 2, 64)
    assert P.kv_commit(kc, vc, i32(0, 1), i32(0), i32(0, 2), i32(0)).shape == (0,) and torch.equal(kc, k0)


# --------------------------------------------------------------------------------------- refusals that need a device
@gpu
def test_gpu_refusals(gpu_device):
    dev = gpu_device
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    q, kc = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device=dev), torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16, device=dev)
    ok = dict(q=q, k_cache=kc, v_cache=kc, block_table=i32(2, 3), ctx_len=i32(2), cu_rows=i32(3))
    P.attn_tree(**ok)
    for kw, exc in ((dict(q=q.half()), Exception), (dict(q=q[:, :3]), ValueError), (dict(k_cache=kc.float()), TypeError), (dict(v_cache=kc[:2]), ValueError),
                    (dict(block_table=i32(2, 3).long()), ValueError), (dict(block_table=i32(3, 2).t()), ValueError), (dict(ctx_len=i32(3)), ValueError),
                    (dict(cu_rows=i32(2)), ValueError), (dict(ctx_len=i32(2).cpu()), ValueError), (dict(tree_mask=i32(4)), ValueError),
                    (dict(max_nodes=65), ValueError), (dict(max_nodes=0), ValueError), (dict(softmax_scale=-1.0), Exception), (dict(out=q[:2]), ValueError),
                    (dict(out=torch.zeros(4, 4, 64, device=dev)), ValueError), (dict(k_cache=kc.transpose(0, 1), v_cache=kc.transpose(0, 1)), ValueError),
                    (dict(q=torch.zeros(4, 4, 32, dtype=torch.bfloat16, device=dev)), ValueError)):
        with pytest.raises(exc):
            P.attn_tree(**{**ok, **kw})
    rope = rope_table(8).to(dev)
    okw = dict(q=q, k=q[:, :2], v=q[:, :2], positions=i32(4), rope=rope, slots=torch.arange(4, dtype=torch.int32, device=dev), k_cache=kc, v_cache=kc.clone())
    P.rope_kv_paged(**okw)
    for kw, exc in ((dict(k=q[:, :3]), ValueError), (dict(v=q[:3, :2]), ValueError), (dict(k=q[:, :2].float()), TypeError), (dict(rope=rope.double()), ValueError),
                    (dict(rope=rope[:, :16]), ValueError), (dict(slots=i32(3)), ValueError), (dict(positions=i32(4).long()), ValueError), (dict(out=q[:2]), ValueError)):
        with pytest.raises(exc):
            P.rope_kv_paged(**{**okw, **kw})
    k5 = kc[None]
    okc = dict(k_cache=k5, v_cache=k5.clone(), block_table=i32(2, 3), ctx_len=i32(2), path=i32(2, 4), n_accept=i32(2))
    P.kv_commit(**okc)
    for kw, exc in ((dict(k_cache=kc), ValueError), (dict(path=i32(2, 65)), ValueError), (dict(path=i32(3, 4)), ValueError), (dict(n_accept=i32(1)), ValueError)):
        with pytest.raises(exc):
            P.kv_commit(**{**okc, **kw})
    t = P.PageTable(2, 3, 6, 16, 64, device=dev)
    for a, b, par in ((i32(3), i32(2), None), (i32(2).long(), i32(2), None), (i32(2), i32(2), i32(63)), (i32(2).cpu(), i32(2), None)):
        with pytest.raises(ValueError):
            t.plan(a, b, parents=par)
