"""The serving operators of a paged KV cache and of 4-bit weights, with their plain forms in elementary torch operations.

Five operators that a speculating decode step calls one after the other:

* ``plan``    block tables, slot maps, positions and tree masks from the requests' lengths (``vall_e_amd.paged.PageTable.plan``)
* ``write``   RoPE on the step's q and k rows, k and v into the pages the slot map names (``vall_e_amd.paged.rope_kv_paged``)
* ``attend``  attention of each request's drafted tokens (one token: a plain decode step) over its pages
              (``vall_e_amd.paged.attn_tree``)
* ``commit``  the accepted path of each tree moved to the end of its context, all layers (``vall_e_amd.paged.kv_commit``)
* ``w4``      products of a step's few rows with 4-bit weights and group scales (``vall_e_amd.plugins.HipLinear4``)

Pages are ``[n_pages][kv_heads][page][64]``; slot = page * page size + offset in the page; q and k heads are pair-interleaved
(elements 2i and 2i + 1 rotate together).  The multiset of a case's lengths is fixed by the case, the seed deals them out.
"""
import math

import numpy as np
import torch

own = False

DH = 64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # every request of a batch of 16 plans a 26-node draft tree; two requests have just ended and give their pages back
        dict(name="plan_tree_step", op="plan", requests=16, page=16, ctx_lo=311, ctx_hi=761, new_lo=26, new_hi=26, tree=True, done=2, pool=1.0),
        # admission of 64 prompts of up to 761 rows at once: 0 -> 761 rows each, page by page
        dict(name="plan_admit_prompts", op="plan", requests=64, page=16, ctx_lo=0, ctx_hi=0, new_lo=305, new_hi=761, tree=False, done=0, pool=1.0),
        # the one new row of each of 16 utterances (16 heads of 64)
        dict(name="write_step", op="write", rows=16, heads=16, kv_heads=16, page=16, dtype="bf16"),
        # the prompt pass of 16 utterances x 761 rows into the pages
        dict(name="write_prompts", op="write", rows=12176, heads=16, kv_heads=16, page=16, dtype="bf16"),
        # a plain decode step: one token per utterance, contexts of the 450-frame run
        dict(name="attend_step", op="attend", requests=16, heads=16, kv_heads=16, page=16, ctx_lo=311, ctx_hi=761, nodes_lo=1, nodes_hi=1, dtype="bf16"),
        # verification of draft trees over long-form contexts (2,250 frames and their prompt), ragged trees
        dict(name="attend_tree_longform", op="attend", requests=32, heads=16, kv_heads=16, page=32, ctx_lo=1800, ctx_hi=2561, nodes_lo=9, nodes_hi=26, dtype="bf16"),
        # one very long context shared by grouped heads, the widest tree
        dict(name="attend_tree_one_long", op="attend", requests=1, heads=16, kv_heads=4, page=64, ctx_lo=130001, ctx_hi=130001, nodes_lo=64, nodes_hi=64, dtype="bf16"),
        # one request of the fp32 parity path takes over 3 drafted tokens in all 12 layers
        dict(name="commit_single", op="commit", requests=1, layers=12, kv_heads=16, page=16, ctx_lo=225, ctx_hi=225, nodes=26, accept_lo=3, accept_hi=3, dtype="f32"),
        # a batch of 16 takes over 0 to 5 drafted tokens each in all 12 layers
        dict(name="commit_batch", op="commit", requests=16, layers=12, kv_heads=16, page=16, ctx_lo=40, ctx_hi=225, nodes=26, accept_lo=0, accept_hi=5, dtype="bf16"),
        # down projection of one row of the fp32 path, residual added
        dict(name="w4_down_one_row", op="w4", rows=1, n=1024, k=4096, group=64, zeros=False, epilogue="resid", dtype="f32"),
        # interleaved gate / up rows of the MLP with GEGLU behind them, 16 utterances
        dict(name="w4_gate_up", op="w4", rows=16, n=8192, k=1024, group=64, zeros=True, epilogue="geglu", dtype="bf16"),
        # a wide layer for the rows of a draft tree
        dict(name="w4_wide_tree", op="w4", rows=40, n=8192, k=8192, group=128, zeros=True, epilogue="bias", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "commit", "w4", "w4"])
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    kv = rng.choice([1, 2, 4, 8, 12, 16])
    if op == "plan":
        tree = rng.random() < 0.6
        n = _log(rng, 1, 512)
        hi = rng.randint(1, 64) if tree else _log(rng, 1, max(2, min(2048, 48000 // n)))
        lo = rng.randint(1, hi)
        chi = _log(rng, 1, 4096)
        return dict(op=op, requests=n, page=page, ctx_lo=rng.randint(0, chi), ctx_hi=chi, new_lo=lo, new_hi=hi, tree=tree,
                    done=rng.randint(0, n // 3), pool=rng.choice([1.0, 1.0, 0.6]))
    if op == "write":
        return dict(op=op, rows=_log(rng, 1, 6000), heads=kv * rng.choice([h for h in (1, 2, 3, 4, 8) if kv * h <= 32]), kv_heads=kv, page=page, dtype=dtype)
    if op == "attend":
        n = _log(rng, 1, 48)
        chi = _log(rng, 1, max(2, 500000 // (n * kv)) if dtype == "bf16" else max(2, 120000 // (n * kv)))
        nhi = rng.choice([1, rng.randint(2, 16), rng.randint(2, 64)])
        return dict(op=op, requests=n, heads=kv * rng.choice([h for h in (1, 2, 3, 4, 8) if kv * h <= 32]), kv_heads=kv, page=page,
                    ctx_lo=rng.randint(0, chi), ctx_hi=chi, nodes_lo=rng.randint(1, nhi), nodes_hi=nhi, dtype=dtype)
    if op == "commit":
        n, layers = _log(rng, 1, 16), rng.randint(1, 12)
        nodes = rng.randint(8, 64)
        hi = rng.randint(1, nodes // 2)
        return dict(op=op, requests=n, layers=layers, kv_heads=kv, page=rng.choice([16, 32, 64]), ctx_lo=rng.randint(0, 100), ctx_hi=rng.randint(100, 225),
                    nodes=nodes, accept_lo=rng.randint(0, hi), accept_hi=hi, dtype=dtype)
    group = rng.choice([32, 64, 128])
    k = group * rng.randint(1, max(1, _log(rng, 256, 8192) // group))
    ep = rng.choice(["none", "bias", "resid", "geglu"])
    n = _log(rng, 24, 8192)
    return dict(op=op, rows=rng.choice([1, rng.randint(2, 16), rng.randint(2, 40)]), n=n + (n & 1 if ep == "geglu" else 0), k=k, group=group,
                zeros=rng.random() < 0.5, epilogue=ep, dtype=dtype)


# ------------------------------------------------------------------------------------------------- lengths and trees
def _spread(lo, hi, n):
    """n whole numbers spread evenly over lo .. hi."""
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _plan_lengths(case):
    n, done = case["requests"], case["done"]
    ctx = _spread(case["ctx_lo"], case["ctx_hi"], n)
    new = _spread(case["new_lo"], case["new_hi"], n)
    return [(c, 0 if i < done else c + k) for i, (c, k) in enumerate(zip(ctx, new))]


def _blocks(n, page):
    return (n + page - 1) // page


def _parents(n, rs):
    """A draft tree in topological order: the parent of node i is an earlier node or -1 (a child of the context)."""
    return [int(rs.integers(-1, i)) if i and rs.random() < 0.9 else -1 for i in range(n)]


def _mask_of(parents):
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else 0) | (1 << i))
    return out


def _i64(bits):
    return np.array([b - (1 << 64) if b >> 63 else b for b in bits], dtype=np.int64)


def _pages(lens, page, rs, spare=0):
    """A pool dealt out at random: (block table [len(lens)][max blocks], pages in the pool)."""
    need = [_blocks(n, page) for n in lens]
    total = sum(need) + spare
    perm = rs.permutation(total)
    tab = np.zeros((len(lens), max(max(need), 1)), dtype=np.int32)
    at = 0
    for b, k in enumerate(need):
        tab[b, :k] = perm[at:at + k]
        at += k
    return tab, max(total, 1)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, g, scale=1.0):
    t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
    return t if scale == 1.0 else t * scale


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


def _plan_state(case, seed):
    """What the scheduler holds in front of the step, as numpy arrays."""
    rs = np.random.default_rng(seed)
    pairs = _plan_lengths(case)
    pairs = [pairs[i] for i in rs.permutation(len(pairs))]
    page = case["page"]
    held = [_blocks(c, page) for c, _ in pairs]
    want = [_blocks(n, page) for _, n in pairs]
    grow = sum(max(0, w - h) for w, h in zip(want, held)) - sum(max(0, h - w) for w, h in zip(want, held))
    free = max(0, int(grow * case["pool"])) + (8 if case["pool"] == 1.0 else 0)
    total = max(1, sum(held) + free)
    perm = rs.permutation(total).astype(np.int32)
    width = max(1, max(max(w, h) for w, h in zip(want, held)))
    tab = np.zeros((len(pairs), width), dtype=np.int32)
    at = 0
    for b, h in enumerate(held):
        tab[b, :h] = perm[at:at + h]
        at += h
    fl = np.zeros(total, dtype=np.int32)
    fl[:total - at] = perm[at:]
    rows = sum(max(0, n - c) for c, n in pairs)
    st = dict(len_old=np.array([c for c, _ in pairs], np.int32), len_new=np.array([n for _, n in pairs], np.int32), block_table=tab,
              n_blocks=np.array(held, np.int32), free_list=fl, free_count=np.array([total - at], np.int32))
    max_rows = (rows + 63) // 64 * 64 if rows else 64
    if case["tree"]:
        par = np.full(max_rows, -1, np.int32)
        at = 0
        for c, n in pairs:
            k = max(0, n - c)
            par[at:at + k] = _parents(k, rs)
            at += k
        st["parents"] = par
    return st, max_rows


def _prepare_plan(case, seed):
    np_st, max_rows = _plan_state(case, seed)
    st = {k: _cuda(v) for k, v in np_st.items()}
    st.update(op="plan", page=case["page"], max_rows=max_rows)
    if own:
        from vall_e_amd.paged import PageTable
        n, width = np_st["block_table"].shape
        t = PageTable(n, width, len(np_st["free_list"]), case["page"], max_rows, device="cuda")
        for k in ("block_table", "n_blocks", "free_list", "free_count"):
            getattr(t, k).copy_(st[k])
        st["table"] = t
    return st


def _prepare_write(case, seed):
    rs, g, dt = np.random.default_rng(seed), _gen(seed), DTYPES[case["dtype"]]
    rows, h, kv, page = case["rows"], case["heads"], case["kv_heads"], case["page"]
    n_pages = _blocks(rows, page) + 4
    pages = rs.permutation(n_pages)
    r = np.arange(rows)
    slots = (pages[r // page] * page + r % page).astype(np.int32)
    rope_rows = 4096
    fr = np.arange(rope_rows)[:, None] * (10000.0 ** (-np.arange(0, DH, 2) / DH))[None, :]
    return dict(op="write", q=_randn((rows, h, DH), dt, g), k=_randn((rows, kv, DH), dt, g), v=_randn((rows, kv, DH), dt, g),
                positions=_cuda(rs.integers(0, rope_rows, rows).astype(np.int32)),
                rope=_cuda(np.stack((np.cos(fr), np.sin(fr)), axis=-1).astype(np.float32)), slots=_cuda(slots),
                kc=_randn((n_pages, kv, page, DH), dt, g), vc=_randn((n_pages, kv, page, DH), dt, g))


def _attend_lengths(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["requests"]), _spread(case["nodes_lo"], case["nodes_hi"], case["requests"])


def _prepare_attend(case, seed):
    rs, g, dt = np.random.default_rng(seed), _gen(seed), DTYPES[case["dtype"]]
    ctx, nodes = _attend_lengths(case)
    ctx = [ctx[i] for i in rs.permutation(len(ctx))]
    nodes = [nodes[i] for i in rs.permutation(len(nodes))]
    h, kv, page = case["heads"], case["kv_heads"], case["page"]
    tab, n_pages = _pages([c + n for c, n in zip(ctx, nodes)], page, rs, spare=2)
    mask = [m for n in nodes for m in _mask_of(_parents(n, rs))]
    return dict(op="attend", q=_randn((sum(nodes), h, DH), dt, g), kc=_randn((n_pages, kv, page, DH), dt, g), vc=_randn((n_pages, kv, page, DH), dt, g),
                block_table=_cuda(tab), ctx_len=_cuda(np.array(ctx, np.int32)), cu_rows=_cuda(np.concatenate(([0], np.cumsum(nodes))).astype(np.int32)),
                tree_mask=_cuda(_i64(mask)), max_nodes=max(nodes), max_ctx=max(ctx))


def _commit_lengths(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["requests"]), _spread(case["accept_lo"], case["accept_hi"], case["requests"])


def _prepare_commit(case, seed):
    rs, g, dt = np.random.default_rng(seed), _gen(seed), DTYPES[case["dtype"]]
    ctx, acc = _commit_lengths(case)
    ctx = [ctx[i] for i in rs.permutation(len(ctx))]
    acc = [acc[i] for i in rs.permutation(len(acc))]
    tab, n_pages = _pages([c + case["nodes"] for c in ctx], case["page"], rs, spare=2)
    width = max(1, max(acc))
    path = np.zeros((len(ctx), width), np.int32)
    for b, a in enumerate(acc):        # the accepted nodes lie behind the first a, so a second pass over the same pages moves the same rows
        path[b, :a] = np.sort(rs.choice(np.arange(a, case["nodes"]), a, replace=False))
    shape = (case["layers"], n_pages, case["kv_heads"], case["page"], DH)
    return dict(op="commit", kc=_randn(shape, dt, g), vc=_randn(shape, dt, g), block_table=_cuda(tab), ctx_len=_cuda(np.array(ctx, np.int32)),
                path=_cuda(path), n_accept=_cuda(np.array(acc, np.int32)))


def _prepare_w4(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    m, n, k, grp = case["rows"], case["n"], case["k"], case["group"]
    ep = case["epilogue"]
    q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)       # low nibble: even k
    scales = (torch.rand((n, k // grp), generator=g, device="cuda") * 0.5 + 0.75).mul(0.2 / math.sqrt(k)).to(dt)
    st = dict(op="w4", x=_randn((m, k), dt, g), q=q, scales=scales, zeros=None, bias=None, resid=None, group=grp, epilogue=ep)
    if case["zeros"]:
        st["zeros"] = torch.randint(5, 11, (n, k // grp), generator=g, device="cuda", dtype=torch.uint8)
    if ep == "bias":
        st["bias"] = _randn((n,), dt, g)
    if ep == "resid":
        st["resid"] = _randn((m, n), dt, g)
    if own:
        from vall_e_amd.plugins import HipLinear4
        st["lin"] = HipLinear4.from_quantized(q, scales, st["zeros"], group_size=grp, bias=st["bias"])
    return st


_PREPARE = {"plan": _prepare_plan, "write": _prepare_write, "attend": _prepare_attend, "commit": _prepare_commit, "w4": _prepare_w4}


# ------------------------------------------------------------------------------------------------- one pass
def run(st):
    return (_OWN if own else _PLAIN)[st["op"]](st)


def _own_plan(st):
    t = st["table"]
    t.plan(st["len_old"], st["len_new"], parents=st.get("parents"), in_place=False)
    out = [t.cu_rows, t.slots, t.positions, t.status, t.next_n_blocks, t.next_free_count, t.block_table, t.free_list]
    return out + [t.tree_mask] if "parents" in st else out


def _own_write(st):
    from vall_e_amd.paged import rope_kv_paged
    return [rope_kv_paged(st["q"], st["k"], st["v"], st["positions"], st["rope"], st["slots"], st["kc"], st["vc"]), st["kc"], st["vc"]]


def _own_attend(st):
    from vall_e_amd.paged import attn_tree
    return attn_tree(st["q"], st["kc"], st["vc"], st["block_table"], st["ctx_len"], st["cu_rows"], tree_mask=st["tree_mask"],
                     max_nodes=st["max_nodes"], max_ctx=st["max_ctx"])


def _own_commit(st):
    from vall_e_amd.paged import kv_commit
    return [kv_commit(st["kc"], st["vc"], st["block_table"], st["ctx_len"], st["path"], st["n_accept"]), st["kc"], st["vc"]]


def _own_w4(st):
    ep = st["epilogue"]
    return st["lin"](st["x"], resid=st["resid"], geglu=ep == "geglu")


def _plain_plan(st):
    lo, ln, held, page, max_rows = st["len_old"].long(), st["len_new"].long(), st["n_blocks"].long(), st["page"], st["max_rows"]
    tab, fl, fc = st["block_table"], st["free_list"], st["free_count"].long()
    n, width = tab.shape
    dev = tab.device
    valid = (lo >= 0) & (ln >= 0) & (lo <= width * page) & (ln <= width * page) & (held >= 0) & (held <= width)
    rows = (ln - lo).clamp(min=0)
    if "parents" in st:
        valid = valid & (rows <= 64)
    rows = rows * valid
    end = rows.cumsum(0)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device=dev), end))
    ok = valid & (end <= max_rows)
    needed = (ln + page - 1) // page
    freed, need = (held - needed).clamp(min=0) * ok, (needed - held).clamp(min=0) * ok
    f0, a1 = freed.cumsum(0) - freed, need.cumsum(0)
    total = fc + freed.sum()
    served = ok & ((need == 0) | (a1 <= total))
    j = torch.arange(width, device=dev)[None, :]
    back = ok[:, None] & (j >= needed[:, None]) & (j < held[:, None])
    dst = torch.where(back, total - 1 - (f0[:, None] + j - needed[:, None]), torch.full_like(j, fl.numel()))
    fl2 = torch.cat((fl, fl[:1])).index_put((dst.reshape(-1),), tab.reshape(-1))[:-1]
    take = served[:, None] & (j >= held[:, None]) & (j < needed[:, None])
    src = total - 1 - ((a1 - need)[:, None] + j - held[:, None])
    tab2 = torch.where(take, fl2[src.clamp(0, fl.numel() - 1)], tab)
    r = torch.arange(max_rows, device=dev)
    b = (r[:, None] >= end[None, :]).sum(1) if n * max_rows <= 1 << 24 else torch.searchsorted(end, r, right=True)
    live, b = r < cu[-1], b.clamp(max=n - 1)
    i = r - cu[b]
    p = lo[b] + i
    blk = (p // page).clamp(0, width - 1)
    slot = torch.where(live & served[b], tab2[b, blk].long() * page + p % page, torch.full_like(p, -1))
    status = torch.where(~valid, 2, torch.where(~ok, 3, torch.where(served, 0, 1)))
    out_blocks = torch.where(served, needed, held)
    left = total - (a1 * (served & (need > 0))).max()
    masks = None
    if "parents" in st:
        # pointer doubling over the ancestors: bits and depths of 1, 2, 4, ... 64 levels
        par = torch.where(live & (st["parents"] >= 0) & (st["parents"] < i), st["parents"].long(), torch.full_like(i, -1))
        up = torch.where(par >= 0, cu[b] + par, torch.full_like(par, -1))
        masks, depth = torch.where(live, torch.ones_like(i) << i.clamp(0, 63), torch.zeros_like(i)), (up >= 0).long()
        for _ in range(6):
            has, u = up >= 0, up.clamp(min=0)
            masks, depth, up = masks | (masks[u] * has), depth + depth[u] * has, torch.where(has, up[u], up)
        p = lo[b] + depth
    pos = torch.where(live, p, torch.zeros_like(p))
    out = [cu.int(), slot.int(), pos.int(), status.int(), out_blocks.int(), left.int(), tab2, fl2]
    return out + [masks] if masks is not None else out


def _plain_write(st):
    table = st["rope"][st["positions"].long()]                                       # [rows][32][2]
    cos, sin = table[:, None, :, 0], table[:, None, :, 1]

    def rot(x):
        x = x.float()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)

    kc, vc = st["kc"], st["vc"]
    page, off = st["slots"].long() // kc.shape[2], st["slots"].long() % kc.shape[2]
    kc[page, :, off] = rot(st["k"]).to(kc.dtype)
    vc[page, :, off] = st["v"]
    return [rot(st["q"]).to(kc.dtype), kc, vc]


def _plain_attend(st):
    q, kc, vc, tab, ctx, cu = st["q"], st["kc"], st["vc"], st["block_table"].long(), st["ctx_len"].long(), st["cu_rows"].long()
    n, width = tab.shape
    kv, page = kc.shape[1], kc.shape[2]
    h, grp, mn = q.shape[1], q.shape[1] // kv, st["max_nodes"]
    nodes = cu[1:] - cu[:-1]
    i = torch.arange(mn, device=q.device)
    live = i[None, :] < nodes[:, None]                                               # [n][mn]
    row = torch.where(live, cu[:-1, None] + i, torch.zeros_like(nodes[:, None]))
    qq = q.float()[row].view(n, mn, kv, grp, DH).permute(0, 2, 3, 1, 4).reshape(n, kv, grp * mn, DH)
    t = torch.arange(width * page, device=q.device)
    there = t[None, :] < (ctx + nodes)[:, None]                                      # [n][T]

    def gather(c):
        return c[tab].float().permute(0, 2, 1, 3, 4).reshape(n, kv, width * page, DH)

    k, v = gather(kc), gather(vc).masked_fill(~there[:, None, :, None], 0.0)
    s = torch.matmul(qq, k.transpose(-1, -2).contiguous()).view(n, kv, grp, mn, width * page) * (1.0 / math.sqrt(DH))
    node = t[None, :] - ctx[:, None]                                                 # [n][T]
    bit = (st["tree_mask"][row][:, :, None] >> node.clamp(0, 63)[:, None, :]) & 1
    seen = there[:, None, :] & ((node < 0)[:, None, :] | (bit != 0)) & live[:, :, None]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == float("-inf"), 0.0))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul((p / z.masked_fill(z == 0, 1.0)).view(n, kv, grp * mn, width * page), v).view(n, kv, grp, mn, DH)
    flat = o.permute(0, 3, 1, 2, 4).reshape(n * mn, h, DH)
    r = torch.arange(q.shape[0], device=q.device)
    b = (r[:, None] >= cu[None, 1:]).sum(1)
    return flat[b * mn + r - cu[b]].to(q.dtype)


def _plain_commit(st):
    kc, vc, tab, ctx, path, acc = st["kc"], st["vc"], st["block_table"].long(), st["ctx_len"].long(), st["path"].long(), st["n_accept"].long()
    page, n_pages = kc.shape[3], kc.shape[1]
    j = torch.arange(path.shape[1], device=kc.device)[None, :]
    live = j < acc[:, None]

    def place(at):
        at = at.clamp(0, tab.shape[1] * page - 1)
        return tab.gather(1, at // page), at % page

    sp, so = place(ctx[:, None] + path)
    dp, do = place(ctx[:, None] + j)
    sp, so = torch.where(live, sp, dp), torch.where(live, so, do)                    # a row that stays is written onto itself
    for c in (kc, vc):
        c[:, dp, :, do] = c[:, sp, :, so]
    return [(ctx + acc).int(), kc, vc]


def _plain_w4(st):
    q, grp = st["q"], st["group"]
    n = q.shape[0]
    w = torch.stack((q & 15, q >> 4), dim=-1).view(n, -1).float()
    z = st["zeros"].float().repeat_interleave(grp, 1) if st["zeros"] is not None else 8.0
    w = (w - z) * st["scales"].float().repeat_interleave(grp, 1)
    y = torch.matmul(st["x"].float(), w.t())
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["resid"] is not None:
        y = y + st["resid"].float()
    if st["epilogue"] == "geglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = 0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5))) * up
    return y.to(st["x"].dtype)


_OWN = {"plan": _own_plan, "write": _own_write, "attend": _own_attend, "commit": _own_commit, "w4": _own_w4}
_PLAIN = {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend, "commit": _plain_commit, "w4": _plain_w4}


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    es = 2 if case.get("dtype") == "bf16" else 4
    if op == "plan":
        pairs, page = _plan_lengths(case), case["page"]
        rows = sum(max(0, n - c) for c, n in pairs)
        moved = sum(abs(_blocks(n, page) - _blocks(c, page)) for c, n in pairs)
        return {"bytes": 24 * len(pairs) + 8 * moved + rows * (20 if case["tree"] else 8), "flops": rows}
    if op == "write":
        h, kv, rows = case["heads"], case["kv_heads"], case["rows"]
        return {"bytes": rows * (2 * (h + 2 * kv) * DH * es + 8 + min(DH * 4, 4096 * DH * 4 // max(1, rows))), "flops": rows * (h + kv) * DH * 3}
    if op == "attend":
        ctx, nodes = _attend_lengths(case)
        ctx, nodes = sorted(ctx), sorted(nodes)
        keys = sum(ctx) + sum(nodes)
        h, kv, page = case["heads"], case["kv_heads"], case["page"]
        mean = sum(ctx) / len(ctx)
        flops = 4 * DH * h * sum(n * (mean + (n + 1) / 2) for n in nodes)
        return {"bytes": 2 * keys * kv * DH * es + sum(nodes) * (2 * h * DH * es + 8) + 4 * keys // page + 8 * len(ctx), "flops": int(flops)}
    if op == "commit":
        _, acc = _commit_lengths(case)
        row = 2 * case["layers"] * case["kv_heads"] * DH * es
        return {"bytes": 2 * sum(acc) * row + 16 * len(acc) + 4 * sum(acc), "flops": len(acc)}
    m, n, k = case["rows"], case["n"], case["k"]
    meta = (n * k // case["group"]) * (es + (1 if case["zeros"] else 0))
    ep = case["epilogue"]
    out = m * (n // 2 if ep == "geglu" else n) * es
    return {"bytes": n * k // 2 + meta + m * k * es + out + (m * n * es if ep == "resid" else 0) + (n * es if ep == "bias" else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    return _EXACT[case["op"]](case, seed)


def _exact_plan(case, seed):
    st, max_rows = _plan_state(case, seed)
    page, width = case["page"], st["block_table"].shape[1]
    tab, held, fl = st["block_table"].copy(), [int(v) for v in st["n_blocks"]], st["free_list"].copy()
    pairs = list(zip(st["len_old"].tolist(), st["len_new"].tolist()))
    n = len(pairs)
    assert all(v <= width * page for p in pairs for v in p)
    cu = [0]
    for c, m in pairs:
        cu.append(cu[-1] + max(0, m - c))
    back = [int(tab[b, k]) for b, (_, m) in enumerate(pairs) for k in range(_blocks(m, page), held[b])]
    stack = [int(v) for v in fl[:int(st["free_count"][0])]] + back[::-1]             # the page given back first lies on top
    fl[:len(stack)] = stack
    status, out_blocks, full = [0] * n, [], False
    for b, (c, m) in enumerate(pairs):
        need = _blocks(m, page) - held[b]
        if need > 0 and (full or need > len(stack)):
            status[b], full = 1, True
            out_blocks.append(held[b])
            continue
        for k in range(max(0, need)):
            tab[b, held[b] + k] = stack.pop()
        out_blocks.append(_blocks(m, page))
    slots, pos, masks = [-1] * max_rows, [0] * max_rows, [0] * max_rows
    for b, (c, m) in enumerate(pairs):
        k = max(0, m - c)
        par = st["parents"][cu[b]:cu[b] + k].tolist() if case["tree"] else list(range(-1, k - 1))
        ms = _mask_of(par) if case["tree"] else None
        for i in range(k):
            if status[b] == 0:
                slots[cu[b] + i] = int(tab[b, (c + i) // page]) * page + (c + i) % page
            pos[cu[b] + i] = c + (bin(ms[i]).count("1") - 1 if case["tree"] else i)
            if case["tree"]:
                masks[cu[b] + i] = ms[i]
    i32 = lambda x: _cuda(np.asarray(x, dtype=np.int32).reshape(-1))
    out = [i32(cu), i32(slots), i32(pos), i32(status), i32(out_blocks), i32([len(stack)]), _cuda(tab), _cuda(fl)]
    return out + [_cuda(_i64(masks))] if case["tree"] else out


def _exact_write(case, seed):
    st = _prepare_write(case, seed)
    ang = st["rope"].double()[st["positions"].long()]
    z = torch.view_as_complex(ang.contiguous())[:, None, :]

    def turn(x):
        return torch.view_as_real(torch.view_as_complex(x.double().view(*x.shape[:-1], DH // 2, 2).contiguous()) * z).flatten(-2)

    kc, vc = st["kc"].double().transpose(1, 2).contiguous(), st["vc"].double().transpose(1, 2).contiguous()      # [page][offset][head][64]
    flat = lambda c: c.view(-1, *c.shape[2:])
    flat(kc)[st["slots"].long()] = turn(st["k"])
    flat(vc)[st["slots"].long()] = st["v"].double()
    return [turn(st["q"]), kc.transpose(1, 2), vc.transpose(1, 2)]


def _exact_attend(case, seed):
    st = _prepare_attend(dict(case), seed)
    ctx, cu = st["ctx_len"].tolist(), st["cu_rows"].tolist()
    h, kv, page = case["heads"], case["kv_heads"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    masks = st["tree_mask"].tolist()
    for b, c in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        total = c + hi - lo
        pages = st["block_table"][b, :_blocks(total, page)].long()
        see = torch.ones((hi - lo, total), dtype=torch.bool)
        for i in range(hi - lo):
            see[i, c:] = torch.tensor([(masks[lo + i] >> j) & 1 == 1 for j in range(hi - lo)])
        see = see.cuda()
        for head in range(h):
            k = st["kc"][pages, head * kv // h].double().reshape(-1, DH)[:total]
            v = st["vc"][pages, head * kv // h].double().reshape(-1, DH)[:total]
            s = (st["q"][lo:hi, head].double() @ k.t()) / 8.0
            out[lo:hi, head] = torch.softmax(s.masked_fill(~see, float("-inf")), dim=-1) @ v
    return out


def _exact_commit(case, seed):
    st = _prepare_commit(case, seed)
    page = case["page"]
    ctx, acc, path, tab = st["ctx_len"].tolist(), st["n_accept"].tolist(), st["path"].tolist(), st["block_table"].tolist()
    out = []
    for c in (st["kc"], st["vc"]):
        new = c.clone()
        for b in range(len(ctx)):
            for j in range(acc[b]):
                s, d = ctx[b] + path[b][j], ctx[b] + j
                new[:, tab[b][d // page], :, d % page] = c[:, tab[b][s // page], :, s % page]
        out.append(new.double())
    return [_cuda(np.array([a + b for a, b in zip(ctx, acc)], np.int32))] + out


def _exact_w4(case, seed):
    global own
    was, own = own, False
    try:
        st = _prepare_w4(case, seed)
    finally:
        own = was
    n, k, grp = case["n"], case["k"], case["group"]
    w = torch.empty((n, k), dtype=torch.float64, device="cuda")
    w[:, 0::2] = torch.remainder(st["q"].double(), 16)
    w[:, 1::2] = torch.div(st["q"].double(), 16, rounding_mode="floor")
    w = w.view(n, k // grp, grp)
    w = (w - (8.0 if st["zeros"] is None else st["zeros"].double()[:, :, None])) * st["scales"].double()[:, :, None]
    y = st["x"].double() @ w.view(n, k).t()
    if case["epilogue"] == "bias":
        y = y + st["bias"].double()
    if case["epilogue"] == "resid":
        y = y + st["resid"].double()
    if case["epilogue"] == "geglu":
        y = torch.nn.functional.gelu(y[:, 0::2]) * y[:, 1::2]
    return y


_EXACT = {"plan": _exact_plan, "write": _exact_write, "attend": _exact_attend, "commit": _exact_commit, "w4": _exact_w4}
