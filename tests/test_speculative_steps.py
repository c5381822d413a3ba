"""Steps of a serving loop with drafted trees: page plan, 4-bit projections, RoPE into the pages, tree attention and commit one after the other,
as vall_e_amd/paged.py describes them; eagerly against 64-bit formulas, and captured into graphs against the same steps run eagerly.

Every operator is held to its formula on the inputs that the operator before it made, with the bounds that test_paged_serving.py and
test_linear_w4.py derive; what attention has to see is kept beside the pages as plain lists of rows, which follow the accepted nodes."""
import numpy as np
import pytest
import torch

from test_linear_w4 import check as check_linear, expect
from test_paged_serving import DTYPES, U32, UNIT, as_i64, blocks, random_tree, ref_attn, rope_table, tree_masks
from vall_e_amd import paged as P
from vall_e_amd import plugins as PL

gpu = pytest.mark.gpu
H, KV, D, F = 4, 2, 256, 384
GROUP = 32


class Stack:
    """Layers of 4-bit projections with random weights; the quantised form is kept for the formulas."""

    def __init__(self, layers, dtype, dev, seed):
        g = torch.Generator().manual_seed(seed)

        def lin(n, k, zeros):
            q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
            s = ((torch.rand(n, k // GROUP, generator=g) + 0.5) * 0.15 / k ** 0.5).to(dtype)
            z = torch.randint(5, 11, (n, k // GROUP), generator=g, dtype=torch.uint8) if zeros else None
            m = PL.HipLinear4.from_quantized(q.to(dev), s.to(dev), None if z is None else z.to(dev), group_size=GROUP)
            m.packed = (q, s, z, GROUP)
            return m
        self.layers = [(lin((H + 2 * KV) * 64, D, True), lin(D, H * 64, False), lin(2 * F, D, True), lin(D, F, False)) for _ in range(layers)]

    def step(self, x, table, kc, vc, rope, ctx, tree, max_nodes):
        """One step's layers: (hidden rows, what each operator saw and made)."""
        log = []
        for l, (qkv, proj, gate_up, down) in enumerate(self.layers):
            t = qkv(x).view(-1, H + 2 * KV, 64)
            q = P.rope_kv_paged(t[:, :H], t[:, H:H + KV], t[:, H + KV:], table.positions, rope, table.slots, kc[l], vc[l])
            o = P.attn_tree(q, kc[l], vc[l], table.block_table, ctx, table.cu_rows, tree_mask=table.tree_mask if tree else None, max_nodes=max_nodes)
            mid = proj(o.view(-1, H * 64), resid=x)
            h = gate_up(mid, geglu=True)
            y = down(h, resid=mid)
            log.append((x, t, q, o, mid, h, y))
            x = y
        return x, log


def turn(rows, angles):
    """RoPE in 64 bits, and the bound of its error in front of the result's rounding."""
    a, b = rows.double()[..., 0::2], rows.double()[..., 1::2]
    c, s = angles.double()[:, None, :, 0], angles.double()[:, None, :, 1]
    y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return y, 3 * U32 * torch.stack((a.abs() + b.abs(), a.abs() + b.abs()), -1).flatten(-2)


def near(got, want, bound, dtype):
    e = (got.double() - want).abs()
    lim = bound + UNIT[dtype] * want.abs()
    assert (e <= lim).all(), float((e - lim).max())


def random_path(parents, rs):
    """The way from the context to a random node."""
    at, path = int(rs.integers(0, len(parents))), []
    while at >= 0:
        path.append(at)
        at = parents[at]
    return path[::-1]


# Per step and request: (kind, new rows): a prompt or drafted nodes, "end" gives the pages back, None: the request's place is idle
SCRIPT = [
    [("prompt", 37), ("prompt", 5), None, ("prompt", 20)],
    [("tree", 9), ("tree", 1), None, ("tree", 26)],
    [("tree", 5), ("end", 0), ("prompt", 30), ("tree", 12)],
    [("tree", 1), None, ("tree", 1), ("tree", 1)],
    [("tree", 64), ("prompt", 16), ("tree", 7), ("end", 0)],
    [("tree", 3), ("tree", 8), ("end", 0), ("prompt", 1)],
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_steps_against_the_formulas(gpu_device, dtype, page):
    dev, layers, B = gpu_device, 2, 4
    rs = np.random.default_rng(page)
    width, max_rows = -(-192 // page), 96
    n_pages = 18 if page == 16 else 7                                  # tight: pages of ended requests are needed again
    table = P.PageTable(B, width, n_pages, page, max_rows, device=dev)
    kc, vc = P.kv_cache(layers, n_pages, page, KV, dtype, dev)
    kc.fill_(float("nan")), vc.fill_(float("inf"))                     # what no request wrote must reach nothing
    rope = rope_table(256)
    stack = Stack(layers, dtype, dev, 11)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    length, kept = [0] * B, [[([], []) for _ in range(layers)] for _ in range(B)]
    for step in SCRIPT:
        parents, lens, trees = [], [], []
        for b, what in enumerate(step):
            kind, n = what or ("idle", 0)
            tr = list(range(-1, n - 1)) if kind == "prompt" else random_tree(n, rs) if n else []
            trees.append(tr)
            parents += tr
            lens.append(0 if kind == "end" else length[b] + n)
        cu = np.concatenate(([0], np.cumsum([len(t) for t in trees]))).tolist()
        rows = cu[-1]
        ctx = i32(length)
        table.plan(ctx, i32(lens), parents=i32(parents + [0] * (max_rows - rows)))
        assert table.status.tolist() == [0] * B and table.cu_rows.tolist() == cu
        masks = [m for t in trees for m in tree_masks(t)]
        assert torch.equal(table.tree_mask[:rows].cpu(), as_i64(masks)) and (table.slots[rows:] == -1).all()
        depth = [bin(m).count("1") - 1 for m in masks]
        base = [length[b] for b in range(B) for _ in trees[b]]
        assert table.positions[:rows].tolist() == [a + d for a, d in zip(base, depth)]
        tab, held = table.block_table.cpu(), table.n_blocks.tolist()
        assert held == [blocks(n, page) for n in lens]
        owned = [int(p) for b in range(B) for p in tab[b, :held[b]]] + table.free_list[:int(table.free_count)].tolist()
        assert sorted(owned) == list(range(n_pages))                   # every page has one owner
        x = torch.randn(max_rows, D, generator=torch.Generator().manual_seed(rows)).to(dtype)
        x[rows:] = float("nan")                                        # padding rows
        out, log = stack.step(x.to(dev), table, kc, vc, rope.to(dev), ctx, True, max(len(t) for t in trees))
        assert out.isfinite()[:rows].all()
        place = lambda b, t: (int(tab[b, t // page]), t % page)
        angles = rope[table.positions[:rows].cpu().long()]
        for l, (mods, made) in enumerate(zip(stack.layers, log)):
            x, t, q, o, mid, h, y = (v[:rows].cpu() for v in made)
            check_linear(t.reshape(rows, -1), *expect(x, *mods[0].packed), dtype)
            near(q, *turn(t[:, :H], angles), dtype)
            want_k, bound_k = turn(t[:, H:H + KV], angles)
            kh, vh = kc[l].cpu(), vc[l].cpu()
            for b in range(B):
                if lens[b] == 0:
                    kept[b][l] = ([], [])
                ks, vs = kept[b][l]
                for i in range(len(trees[b])):
                    r, (p, off) = cu[b] + i, place(b, length[b] + i)
                    near(kh[p, :, off], want_k[r], bound_k[r], dtype)
                    assert torch.equal(vh[p, :, off], t[r, H + KV:])
                    ks.append(kh[p, :, off].clone()), vs.append(vh[p, :, off].clone())
            # attention over the kept rows, packed one request after the other into one page each
            wide = 256
            dk, dv = torch.zeros(B, KV, wide, 64, dtype=dtype), torch.zeros(B, KV, wide, 64, dtype=dtype)
            for b in range(B):
                for s, d in ((kept[b][l][0], dk), (kept[b][l][1], dv)):
                    if s:
                        d[b, :, :len(s)] = torch.stack(s, 1)
            want_o, bound_o = ref_attn(q, dk, dv, np.arange(B)[:, None], length, cu, masks, 0.125)
            near(o, want_o, bound_o, dtype)
            check_linear(mid, *expect(o.reshape(rows, -1), *mods[1].packed, resid=x), dtype)
            check_linear(h, *expect(mid, *mods[2].packed, geglu=True), dtype)
            check_linear(y, *expect(h, *mods[3].packed, resid=mid), dtype)
        # prompts are taken over whole, trees up to a random node (now and then none)
        paths = []
        for b, what in enumerate(step):
            kind = what[0] if what else "idle"
            paths.append(list(range(len(trees[b]))) if kind == "prompt" else random_path(trees[b], rs) if trees[b] and rs.random() < 0.8 else [])
        after = [0 if lens[b] == 0 else length[b] for b in range(B)]
        new = P.kv_commit(kc, vc, table.block_table, i32(after), i32([p + [0] * (64 - len(p)) for p in paths]), i32([len(p) for p in paths]))
        length = [a + len(p) for a, p in zip(after, paths)]
        assert new.tolist() == length
        kh, vh = kc.cpu(), vc.cpu()
        for b in range(B):
            for l in range(layers):
                ks, vs = kept[b][l]
                n = after[b]
                kept[b][l] = (ks[:n] + [ks[n + j] for j in paths[b]], vs[:n] + [vs[n + j] for j in paths[b]])
                for t in range(length[b]):
                    p, off = place(b, t)
                    assert torch.equal(kh[l, p, :, off], kept[b][l][0][t]) and torch.equal(vh[l, p, :, off], kept[b][l][1][t])


class Loop:
    """A batch whose whole step -- plan, layers, commit, the new lengths -- runs on buffers that stay: eagerly, or as a graph."""

    def __init__(self, stack, dtype, dev, requests, seed):
        self.stack, self.dev, self.B, page = stack, dev, requests, 16
        self.table = P.PageTable(requests, 64, requests * 24, page, 160, device=dev)
        self.kc, self.vc = P.kv_cache(len(stack.layers), requests * 24, page, KV, dtype, dev)
        self.rope = rope_table(512).to(dev)
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
        self.length, self.new, self.parents, self.path, self.n_accept = z(requests), z(requests), z(160), z(requests, 64), z(requests)
        self.x, self.y = torch.zeros(160, D, dtype=dtype, device=dev), torch.zeros(160, D, dtype=dtype, device=dev)

    def feed(self, n_new, parents, x, paths):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)
        self.new.copy_(i32(n_new)), self.parents.copy_(i32(parents + [0] * (160 - len(parents))))
        self.x.zero_(), self.x[:len(x)].copy_(x)
        self.path.copy_(i32([p + [0] * (64 - len(p)) for p in paths])), self.n_accept.copy_(i32([len(p) for p in paths]))

    def tree_step(self):
        self.table.plan(self.length, self.length + self.new, parents=self.parents)
        y, _ = self.stack.step(self.x, self.table, self.kc, self.vc, self.rope, self.length, True, 64)
        self.y.copy_(y)
        self.length.copy_(P.kv_commit(self.kc, self.vc, self.table.block_table, self.length, self.path, self.n_accept))

    def token_step(self):
        self.table.plan(self.length, self.length + self.new)
        y, _ = self.stack.step(self.x, self.table, self.kc, self.vc, self.rope, self.length, False, 1)
        self.y.copy_(y)
        self.length.add_(self.new)

    def rows(self):
        """Everything that a request can see of itself."""
        tab, out = self.table.block_table.long(), []
        for b, n in enumerate(self.length.tolist()):
            t = torch.arange(n, device=self.dev)
            pg, off = tab[b, t // 16], t % 16
            out.append((self.kc[:, pg, :, off].clone(), self.vc[:, pg, :, off].clone()))
        return out


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests", [2, 70])
def test_captured_steps_equal_eager_steps(gpu_device, dtype, requests):
    """Two graphs of one batch (a drafted step and a plain one) replayed in turns, with eager work and synchronisations between them: every
    replay bit for bit what the same step gives when it is run eagerly on a batch of its own."""
    dev = gpu_device
    rs = np.random.default_rng(requests)
    stack = Stack(2, dtype, dev, 12)
    g, e = Loop(stack, dtype, dev, requests, 1), Loop(stack, dtype, dev, requests, 1)

    def inputs(tree):
        n_new, parents, paths = [], [], []
        for b in range(requests):
            n = int(rs.integers(1, 65 if requests < 8 else 3)) if tree else int(rs.integers(0, 2))
            tr = random_tree(n, rs) if tree else []
            n_new.append(n), parents.extend(tr)
            paths.append(random_path(tr, rs) if tr and rs.random() < 0.8 else [])
        rows = sum(n_new)
        x = torch.randn(rows, D, generator=torch.Generator().manual_seed(int(rs.integers(1 << 30)))).to(dtype)
        return rows, (n_new, parents, x, paths)

    graphs, side = {}, torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                      # both bodies once outside a capture, on no rows
        g.feed([0] * requests, [], torch.zeros(0, D, dtype=dtype), [[]] * requests)
        g.tree_step(), g.token_step()
    torch.cuda.current_stream().wait_stream(side)
    assert g.length.tolist() == [0] * requests
    for name in ("tree", "token"):
        graphs[name] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[name]):
            g.tree_step() if name == "tree" else g.token_step()
    torch.cuda.synchronize()
    for i, name in enumerate(["tree", "token", "tree", "tree", "token", "tree", "token", "token"]):
        rows, step = inputs(name == "tree")
        g.feed(*step), e.feed(*step)
        graphs[name].replay()
        e.tree_step() if name == "tree" else e.token_step()
        if i % 2:
            torch.cuda.synchronize()
        assert g.table.status.tolist() == [0] * requests
        assert torch.equal(g.y[:rows], e.y[:rows]) and e.y[:rows].isfinite().all()
        assert g.length.tolist() == e.length.tolist()
        for a, b in zip(g.rows(), e.rows()):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert max(g.length.tolist()) > 3


@gpu
def test_two_batches_on_two_streams(gpu_device):
    """Two batches step at the same time on streams of their own: nothing is shared between calls, workspaces least of all."""
    dev, dtype = gpu_device, torch.bfloat16
    rs = np.random.default_rng(5)
    stack = Stack(2, dtype, dev, 13)
    both, alone = [Loop(stack, dtype, dev, 2, s) for s in (1, 2)], [Loop(stack, dtype, dev, 2, s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in both]
    for _ in range(4):
        feeds = []
        for k in range(2):
            trees = [random_tree(int(rs.integers(20, 65)), rs) for _ in range(2)]
            x = torch.randn(sum(map(len, trees)), D, generator=torch.Generator().manual_seed(int(rs.integers(1 << 30)))).to(dtype)
            feeds.append(([len(t) for t in trees], trees[0] + trees[1], x, [random_path(t, rs) for t in trees]))
        for k in range(2):
            both[k].feed(*feeds[k]), alone[k].feed(*feeds[k])
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                both[k].tree_step()
        torch.cuda.synchronize()
        for k in range(2):
            alone[k].tree_step()
            torch.cuda.synchronize()
            rows = sum(feeds[k][0])
            assert torch.equal(both[k].y[:rows], alone[k].y[:rows]) and both[k].length.tolist() == alone[k].length.tolist()
