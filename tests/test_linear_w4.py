"""HipLinear4 / valle_linear_w4 (vall_e_amd/plugins.py, csrc/linear_w4.hip) against the definition in 64 bits.

Tolerance: the products x q are exact in fp32 (8-bit x 4-bit significands) for bf16 inputs and off by u32 = 2^-24 for fp32 ones; sums of K terms
and the per-group scale and subtraction add (K + 32) u32 of A = sum |x| scale (q + zero); the result is rounded once (u: bf16 2^-8,
fp32 2^-24); bias and residual add u32 of their own sums.  GEGLU: 1.13 is the largest slope of gelu, 4e-7 bounds the error of the erf
forms relative to |gate x up|."""
import math

import pytest
import torch

from vall_e_amd import plugins as PL

gpu = pytest.mark.gpu
U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(n, k, group, zeros, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((torch.rand(n, k // group, generator=g) + 0.5) / math.sqrt(k)).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def weights(q, s, z, group):
    n = q.shape[0]
    w = torch.stack((q & 15, q >> 4), -1).reshape(n, -1).double()
    zz = torch.full_like(s, 8).double() if z is None else z.double()
    zz, ss = zz.repeat_interleave(group, 1), s.double().repeat_interleave(group, 1)
    return (w - zz) * ss, (w + zz) * ss


def expect(x, q, s, z, group, bias=None, resid=None, geglu=False):
    w, a = weights(q, s, z, group)
    x = x.double()
    y, A = x @ w.T, x.abs() @ a.T
    err = (x.shape[-1] + 32) * U32 * A
    for t in (bias, resid):
        if t is not None:
            y = y + t.double()
            err = err + 2 * U32 * (y.abs() + t.double().abs())
    if geglu:
        g, u, eg, eu = y[..., 0::2], y[..., 1::2], err[..., 0::2], err[..., 1::2]
        y = torch.nn.functional.gelu(g) * u
        err = 1.13 * eg * (u.abs() + eu) + torch.nn.functional.gelu(g).abs() * eu + 4e-7 * (g * u).abs()
    return y, err


def check(got, want, err, dtype):
    e = (got.cpu().double() - want).abs()
    lim = err + UNIT[dtype] * want.abs()
    assert (e <= lim).all(), (float((e - lim).max()), float(e.max()))


def test_quantize_w4_is_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(24, 256, generator=g)
    w[3], w[4, :64] = 0.0, w[4, :64].abs()
    for sym in (False, True):
        q, s, z = PL.quantize_w4(w, 64, sym)
        assert q.dtype == torch.uint8 and q.shape == (24, 128) and s.shape == (24, 4) and (z is None) == sym
        back, _ = weights(q, s, z, 64)
        step = s.double().repeat_interleave(64, 1)
        slack = 0.5 if sym else 1.0                     # asymmetric: the zero point is rounded too, its range clipped by up to half a step
        assert ((back - w.double()).abs() <= slack * step * (1 + 1e-6) + 1e-9).all()


def test_quantize_w4_refuses_what_has_no_four_bits():
    for w, group in ((torch.randn(4, 100), 64), (torch.full((4, 64), float("nan")), 64), (torch.full((4, 64), float("inf")), 32)):
        with pytest.raises(ValueError):
            PL.quantize_w4(w, group)
    with pytest.raises(ValueError):
        PL.HipLinear4(64, 4).load_state_dict({"weight": torch.full((4, 64), float("nan")), "bias": torch.zeros(4)})
    with pytest.raises(ValueError):
        PL.HipLinear4(64, 4).load_state_dict({"weight": torch.zeros(4, 128), "bias": torch.zeros(4)})


def test_quantize_w4_refuses_a_range_without_a_finite_scale():
    """Finite weights of both signs near the type's end: their range, and with it the scale, would be infinite."""
    for dtype in (torch.float32, torch.bfloat16):
        w = torch.zeros(2, 64, dtype=dtype)
        w[1, 3], w[1, 9] = 3e38, -3e38
        with pytest.raises(ValueError):
            PL.quantize_w4(w, 64)
        with pytest.raises(ValueError):
            PL.HipLinear4(64, 2, dtype=dtype, bias=False).load_state_dict({"weight": w})
        q, s, z = PL.quantize_w4(w, 64, symmetric=True)             # one sign's range is finite
        assert torch.isfinite(s).all()
        w[1, 9] = 0.0
        assert torch.isfinite(PL.quantize_w4(w, 64)[1]).all()


def test_packed_layout_holds_every_weight():
    """The documented layout, element by element."""
    n, k, group = 18, 160, 32
    q, s, z = make(n, k, group, True, torch.float32, 3)
    m = PL.HipLinear4.from_quantized(q, s, z, group_size=group)
    nib = torch.stack((q & 15, q >> 4), -1).reshape(n, k)
    for col in range(n):
        for kk in range(0, k, 7):
            nt, fr, kb, r = col // 16, col % 16, kk // 128, kk % 128
            j, fq, i = r // 32, r % 32 // 8, r % 8
            byte = int(m.wq[nt, kb, fq * 16 + fr, j * 4 + i % 4])
            assert (byte >> 4 if i >= 4 else byte & 15) == int(nib[col, kk])
            assert m.scales[nt, kk // group, fr] == s[col, kk // group] and m.zeros[nt, kk // group, fr] == z[col, kk // group]
    assert (m.scales[1, :, 2:] == 0).all() and (m.scales[:, 5:] == 0).all()


def test_refusals_without_a_gpu():
    from vall_e_amd import _lib as L
    import ctypes as C
    for kw in (dict(in_features=100), dict(in_features=96, group_size=64), dict(in_features=128, group_size=48)):
        with pytest.raises(L.ValleHipError):
            PL.HipLinear4(out_features=8, **kw)
    with pytest.raises(L.ValleHipError):
        PL.HipLinear4(64, 8)(torch.zeros(1, 64))
    q, s, z = make(8, 64, 64, True, torch.float32, 0)
    for a in ((q.int(), s, z), (q, s[:4], z), (q, s, z.int())):
        with pytest.raises((ValueError, L.ValleHipError)):
            PL.HipLinear4.from_quantized(*a)
    lib, p = L.load(), C.c_void_p(4096)

    def call(**kw):
        a = dict(x=p, rs=128, wq=p, M=2, N=32, K=128, group=64, ldc=32, epi=0, dt=1, bias=None, resid=None)
        a.update(kw)
        return lib.valle_linear_w4(a["x"], a["rs"], a["wq"], p, None, a["bias"], a["resid"], p, a["M"], a["N"], a["K"], a["group"], a["ldc"], a["epi"], a["dt"], None)
    for kw, rc in ((dict(x=None), -1), (dict(dt=5), -1), (dict(group=16), -2), (dict(K=96), -1), (dict(N=0), -1), (dict(M=-1), -1), (dict(epi=1), -1), (dict(epi=6), -1),
                   (dict(epi=2, N=31), -1), (dict(epi=2, bias=p), -1), (dict(ldc=31), -1), (dict(x=C.c_void_p(4098)), -1), (dict(rs=127), -1)):
        assert call(**kw) == rc, kw
        assert b"valle_linear_w4" in lib.valle_last_error()
    assert call(M=0) == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,n,k,group", [(1, 1, 32, 32), (1, 16, 128, 64), (2, 40, 96, 32), (16, 33, 256, 128), (17, 64, 160, 32), (5, 1000, 1024, 64), (64, 48, 448, 64),
                                            (65, 100, 384, 128), (3, 256, 4096, 128), (150, 24, 256, 32), (33, 512, 2048, 64)])
def test_linear_w4(gpu_device, dtype, zeros, rows, n, k, group):
    q, s, z = make(n, k, group, zeros, dtype, rows + n)
    g = torch.Generator().manual_seed(k)
    x = torch.randn(rows, k, generator=g).to(dtype)
    bias, resid = torch.randn(n, generator=g).to(dtype), torch.randn(rows, n, generator=g).to(dtype)
    d = lambda t: None if t is None else t.to(gpu_device)
    m = PL.HipLinear4.from_quantized(d(q), d(s), d(z), group_size=group)
    check(m(d(x)), *expect(x, q, s, z, group), dtype)
    check(m(d(x), resid=d(resid)), *expect(x, q, s, z, group, resid=resid), dtype)
    if n % 2 == 0:
        check(m(d(x), geglu=True), *expect(x, q, s, z, group, geglu=True), dtype)
    mb = PL.HipLinear4.from_quantized(d(q), d(s), d(z), group_size=group, bias=d(bias))
    check(mb(d(x)), *expect(x, q, s, z, group, bias=bias), dtype)


@gpu
def test_linear_w4_shapes_views_and_rows_of_others(gpu_device):
    """Leading dimensions, strided and misaligned inputs, no rows; an infinity or NaN in one row stays in that row."""
    n, k, group = 72, 320, 64
    q, s, z = make(n, k, group, True, torch.bfloat16, 9)
    d = lambda t: t.to(gpu_device)
    m = PL.HipLinear4.from_quantized(d(q), d(s), d(z), group_size=group)
    big = torch.randn(24, 2 * k + 8, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu_device)
    x = big[:, 8:8 + k]
    want, err = expect(x.cpu(), q, s, z, group)
    check(m(x), want, err, torch.bfloat16)
    off = big[:, 3:3 + k]
    check(m(off), *expect(off.cpu(), q, s, z, group), torch.bfloat16)
    y = m(x.reshape(2, 3, 4, k))
    assert y.shape == (2, 3, 4, n) and torch.equal(y.reshape(24, n), m(x))
    assert m(x[0]).shape == (n,) and torch.equal(m(x[0]), m(x)[0])
    assert m(x[:0]).shape == (0, n)
    bad = x.clone()
    bad[5, 7], bad[9, 0] = float("nan"), float("inf")
    got = m(bad)
    keep = [i for i in range(24) if i not in (5, 9)]
    assert torch.equal(got[keep], m(x)[keep]) and torch.isnan(got[5]).all() and not torch.isfinite(got[9]).any()
    for exc, kw in ((TypeError, dict(x=x.float())), (ValueError, dict(x=x[:, :64])), (ValueError, dict(x=x, resid=x)), (ValueError, dict(x=x, geglu=True, resid=x))):
        with pytest.raises(exc):
            m(**kw)


@gpu
def test_linear_w4_rows_do_not_depend_on_their_neighbours(gpu_device):
    """A row's result is the same bits in a batch of 2, 16, 40 and 100, and in bf16 alone too (every output sums its k blocks in one order; a
    single fp32 row takes a form of its own, with an order of its own)."""
    for dtype in (torch.bfloat16, torch.float32):
        q, s, z = make(64, 1024, 64, True, dtype, 2)
        d = lambda t: t.to(gpu_device)
        m = PL.HipLinear4.from_quantized(d(q), d(s), d(z))
        x = torch.randn(100, 1024, generator=torch.Generator().manual_seed(3)).to(dtype).to(gpu_device)
        full = m(x)
        for rows in (1, 2, 16, 40) if dtype is torch.bfloat16 else (2, 16, 40):
            assert torch.equal(m(x[:rows]), full[:rows]), rows
        check(m(x[:1]), *expect(x[:1].cpu(), q, s, z, 64), dtype)


@gpu
def test_linear_w4_replaces_nn_linear(gpu_device):
    """klass of replace_linear: constructed like nn.Linear, filled from the replaced module's state dict."""
    torch.manual_seed(0)
    lin = torch.nn.Linear(256, 96).to(gpu_device, torch.float32)
    m = PL.HipLinear4(256, 96, bias=True, device=gpu_device, dtype=torch.float32)
    m.load_state_dict(lin.state_dict())
    same = PL.HipLinear4.from_linear(lin)
    x = torch.randn(2, 7, 256, device=gpu_device)
    assert torch.equal(m(x), same(x))
    q, s, z = PL.quantize_w4(lin.weight.cpu())
    check(m(x), *expect(x.cpu(), q, s, z, 64, bias=lin.bias.detach().cpu()), torch.float32)
    assert (m(x) - lin(x)).abs().max() < 0.5 * lin(x).abs().max()                       # 4 bits: near, not equal
    again = PL.HipLinear4(256, 96, bias=True, device=gpu_device, dtype=torch.float32)
    again.load_state_dict(m.state_dict())                                               # its own state dict, packed
    assert torch.equal(again(x), m(x))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,k,group", [(1, 1000, 4096, 64), (1, 72, 8320, 128), (1, 4100, 2336, 32), (1, 4112, 1216, 64), (40, 8200, 1408, 128), (33, 8192, 1216, 64),
                                            (20, 8192, 1184, 32), (7, 8194, 3264, 64), (48, 4096, 4224, 128), (97, 200, 1184, 32),
                                            (64, 8192, 1216, 64), (57, 8200, 1408, 128), (50, 8208, 2336, 32), (64, 8200, 992, 32), (120, 8256, 4224, 128)])
def test_linear_w4_long_and_wide(gpu_device, dtype, rows, n, k, group):
    """Several k blocks per wave in every form: last blocks that are no whole ones, an odd number of them, columns behind the last tile."""
    q, s, z = make(n, k, group, True, dtype, n + k)
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(k)).to(dtype)
    d = lambda t: t.to(gpu_device)
    m = PL.HipLinear4.from_quantized(d(q), d(s), d(z), group_size=group)
    want = expect(x, q, s, z, group)
    for _ in range(3):                                                                  # a race would differ
        check(m(d(x)), *want, dtype)
    pad = torch.full((rows, k + 8), float("nan"), dtype=dtype)
    pad[:, :k] = x
    check(m(d(pad)[:, :k]), *want, dtype)                                               # rows of a wider matrix: what lies between them is not theirs


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_linear_w4_c_entry_fp32_logits_and_wide_rows_of_c(gpu_device, dtype, rows):
    """What the module does not offer: fp32 results with an fp32 bias (heads), and C wider than N, with a bias and a residual; nothing is
    written between the rows."""
    from vall_e_amd import _lib as L
    n, k, group, ldc = 75, 352, 32, 90
    q, s, z = make(n, k, group, True, dtype, 21)
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(4)).to(dtype)
    d = lambda t: t.to(gpu_device)
    m = PL.HipLinear4.from_quantized(d(q), d(s), d(z), group_size=group)
    xd, code, stream = d(x), L.dtype_code(dtype), L.stream_ptr(gpu_device)

    def call(bias, resid, out, epi):
        L.check(L.load().valle_linear_w4(L.ptr(xd), k, L.ptr(m.wq), L.ptr(m.scales), L.ptr(m.zeros), L.ptr(bias), None if resid is None else L.ptr(resid), L.ptr(out), rows, n, k,
                                         group, ldc, epi, code, stream))
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5))
    out = torch.full((rows, ldc), 7.0, device=gpu_device)
    call(d(bias), None, out, 3)
    want, err = expect(x, q, s, z, group, bias=bias)
    assert (out[:, n:] == 7).all() and ((out[:, :n].cpu().double() - want).abs() <= err + U32 * want.abs()).all()
    bias, resid = bias.to(dtype), torch.randn(rows, ldc, generator=torch.Generator().manual_seed(6)).to(dtype)
    out = torch.full((rows, ldc), 7.0, dtype=dtype, device=gpu_device)
    bd, rd = d(bias), d(resid)
    call(bd, rd, out, 1)
    assert (out[:, n:] == 7).all()
    check(out[:, :n], *expect(x, q, s, z, group, bias=bias, resid=resid[:, :n]), dtype)


# --------------------------------------------------------------------------------------- every bf16 form
def form(rows, n):
    """(column tiles, row tiles) per workgroup that the dispatch takes for bf16; test_dispatch_rule_is_the_one_restated_here holds it to the source."""
    up = lambda a, b: -(-a // b)
    nt = 2 if up(n, 32) * up(rows, 48) >= 256 else 1
    gx = up(up(n, 16), nt)
    for mt in (1, 2, 3):
        if gx * up(rows, 16 * mt) <= 256:
            return nt, mt
    return nt, up(up(rows, up(rows, 64)), 16)


# rows x columns of every form: with rows and columns that end inside a tile, and whole ones
FORMS = {(1, 1): [(7, 4090), (16, 512)], (1, 2): [(23, 4090), (32, 4096)], (1, 3): [(37, 4090), (48, 4096)], (1, 4): [(57, 4060), (64, 4064)],
         (2, 1): [(7, 8186), (16, 8192)], (2, 2): [(23, 8186), (32, 8192)], (2, 3): [(37, 8186), (48, 8192)], (2, 4): [(57, 8200), (64, 8192)]}
# inputs by group: up to one k block of 128 per wave (eight waves), and several: an odd and an even number of blocks per wave, the last one whole and in part
INPUTS = {32: [96, 992, 1184, 2176], 64: [192, 960, 1216, 2176], 128: [384, 1024, 1408, 2176]}


def test_dispatch_rule_is_the_one_restated_here():
    """A changed rule has to change form() and FORMS with it, so that no form drops out of the test below."""
    from pathlib import Path
    src = (Path(PL.__file__).parent / "csrc" / "linear_w4.hip").read_text()
    for line in ("if ((long)ceil_div(a.N, 32) * ceil_div(a.M, 48) >= 256) w4_launch_bf16<G, 2>(a, s);",
                 "const int gx = ceil_div(ceil_div(a.N, 16), NT), mt = w4_row_tiles(a.M, gx, 4);",
                 "if ((long)gx * ceil_div(M, 16 * mt) <= 256) return mt;",
                 "return ceil_div(ceil_div(M, ceil_div(M, 16 * most)), 16);",
                 "if (mt == 1) linear_w4_kernel<G, NT, 1, 8><<<grid, 512, 0, s>>>(a);",
                 "if (a.KB <= NW) {"):
        assert line in src, line
    for want, shapes in FORMS.items():
        for rows, n in shapes:
            assert form(rows, n) == want and n % 2 == 0
    for group, ks in INPUTS.items():
        assert all(k % group == 0 for k in ks) and sum(-(-k // 128) <= 8 for k in ks) == 2


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("nt,mt", sorted(FORMS))
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_w4_every_form(gpu_device, group, nt, mt, zeros):
    """Every kernel that bf16 rows can reach -- group, column tiles, row tiles, one k block per wave or several -- with and without zero points and with
    every epilogue; each has its own count of loads under way, so each runs three times on memory that the others have just used."""
    from vall_e_amd import _lib as L
    dtype, dev = torch.bfloat16, gpu_device
    for i, k in enumerate(INPUTS[group]):
        rows, n = FORMS[nt, mt][i % 2]
        assert form(rows, n) == (nt, mt)
        q, s, z = (None if t is None else t.to(dev) for t in make(n, k, group, zeros, dtype, k + nt + mt))
        g = torch.Generator().manual_seed(k)
        x = torch.randn(rows, k, generator=g).to(dtype).to(dev)
        bias, resid = torch.randn(n, generator=g).to(dtype).to(dev), torch.randn(rows, n, generator=g).to(dtype).to(dev)
        plain, biased = PL.HipLinear4.from_quantized(q, s, z, group_size=group), PL.HipLinear4.from_quantized(q, s, z, group_size=group, bias=bias)
        y, err = expect(x, q, s, z, group)

        def held(got, want, err, unit):
            e = (got.double() - want).abs()
            lim = err + unit * want.abs()
            assert (e <= lim).all(), (rows, n, k, float((e - lim).max()), int((e > lim).sum()))
        logits = torch.empty(rows, n, device=dev)
        for _ in range(3):
            held(plain(x), y, err, UNIT[dtype])
            gate, up, eg, eu = y[:, 0::2], y[:, 1::2], err[:, 0::2], err[:, 1::2]
            act = torch.nn.functional.gelu(gate)
            held(plain(x, geglu=True), act * up, 1.13 * eg * (up.abs() + eu) + act.abs() * eu + 4e-7 * (gate * up).abs(), UNIT[dtype])
            b = y + bias.double()
            eb = err + 2 * U32 * (b.abs() + bias.double().abs())
            held(biased(x), b, eb, UNIT[dtype])
            r = b + resid.double()
            held(biased(x, resid=resid), r, eb + 2 * U32 * (r.abs() + resid.double().abs()), UNIT[dtype])
            L.check(L.load().valle_linear_w4(L.ptr(x), k, L.ptr(plain.wq), L.ptr(plain.scales), L.ptr(plain.zeros), None, None, L.ptr(logits), rows, n, k, group, n, L.EPI_F32OUT,
                                             L.BF16, L.stream_ptr(dev)))
            held(logits, y, err, U32)
