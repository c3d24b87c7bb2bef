"""add_rms_norm, its backward pass and add_rms_norm_mx against the 64-bit formulas.

Tolerances, from u = 2^-24 (half a step of fp32, relative) and half = finfo(type).eps / 2:
  sums of H squares run in chains of at most H / 32 + 16 fp32 additions of terms of one sign, so rstd is
  off by at most (H / 32 + 16) u, relative; y takes two more products and one rounding:
      |y - y64| <= half |y64| + (H / 32 + 20) u |y64|
  dx adds up dr, rstd g and rstd n mean(g n); each has an error of at most (H / 32 + 24) u of the sum of
  the magnitudes that went into it. dw is a sum of T terms: (T + 24) u sum |dy n|.
The stream r is one fp32 addition and one rounding: equal bits.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# rows x width: single rows, widths below a vector, odd, prime, wide; more rows than CTAs
SHAPES = [(1, 1), (1, 8192), (2, 7), (3, 8), (5, 33), (7, 250), (129, 1000), (64, 5003), (33, 4096), (3, 16384), (2, 65536),
          (1000, 136), (4099, 64), (700, 2560),
          # rows that start on no 16-byte boundary, in every plan: a CTA for a few rows, many, a warp to a row, 512 threads
          (1000, 137), (4099, 65), (700, 2561), (146, 1003), (148, 2050), (149, 6001), (300, 9001), (3, 10001), (1300, 1), (600, 15)]


def make(T, H, dtype, wdtype, residual, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * T + H)
    x = (torch.randn(T, H, generator=g) * torch.exp(0.7 * torch.randn(H, generator=g))).to(dtype)
    res = torch.randn(T, H, generator=g).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(H, generator=g)).to(wdtype)
    return x, res, w


def cu(t):
    return None if t is None else t.cuda()


def check_y(y, y64, H, dtype):
    err = (y.double().cpu() - y64).abs()
    tol = (HALF[dtype] + (H / 32 + 20) * U) * y64.abs() + 1e-38
    assert (err <= tol).all(), (err - tol).max().item()


def check_bwd(dx, dw, dy, dr, r, rstd, w, orc):
    T, H = r.shape
    dx64, dw64 = orc.add_rms_norm_bwd_ref(dy, dr, r, rstd, w)
    n = r.double() * rstd.double()[:, None]
    g = dy.double() * w.double()
    mag = rstd.double()[:, None] * (g.abs() + n.abs() * (g * n).abs().mean(dim=1, keepdim=True))
    if dr is not None:
        mag = mag + dr.double().abs()
    err = (dx.double().cpu() - dx64).abs()
    assert (err <= HALF[r.dtype] * dx64.abs() + (H / 32 + 24) * U * mag + 1e-37).all()
    err = (dw.double().cpu() - dw64).abs()
    assert (err <= HALF[w.dtype] * dw64.abs() + (T + 24) * U * (dy.double() * n).abs().sum(0) + 1e-37).all()


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("types", ["bf16-bf16", "bf16-f32", "f32-f32"])
@pytest.mark.parametrize("residual", [True, False])
def test_forward_and_backward(orc, T, H, types, residual):
    import tk_kernel as tk
    dtype, wdtype = (DT[t] for t in types.split("-"))
    x, res, w = make(T, H, dtype, wdtype, residual)
    y64, r_ref, rstd64 = orc.add_rms_norm_ref(x, res, w)
    dx_in = x.cuda()
    y, r, rstd = tk.add_rms_norm(dx_in, cu(res), w.cuda())
    torch.cuda.synchronize()
    assert torch.equal(r.cpu(), r_ref)
    if not residual:
        assert r is dx_in
    assert torch.equal(dx_in.cpu(), x)  # the input is left alone
    assert ((rstd.double().cpu() - rstd64).abs() <= (H / 32 + 18) * U * rstd64).all()
    check_y(y, y64, H, dtype)
    g = torch.Generator().manual_seed(T + H)
    dy = torch.randn(T, H, generator=g).to(dtype)
    dr = torch.randn(T, H, generator=g).to(dtype) if residual else None
    dx, dw = tk.add_rms_norm_bwd(dy.cuda(), cu(dr), r, rstd, w.cuda())
    assert dx.dtype == dtype and dw.dtype == wdtype
    check_bwd(dx, dw, dy, dr, r_ref, rstd.cpu(), w, orc)
    # the same bits again
    dx2, dw2 = tk.add_rms_norm_bwd(dy.cuda(), cu(dr), r, rstd, w.cuda())
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def check_mx(q, s, atoms, y64, orc):
    """Scales equal to floor(log2(amax)) of the 64-bit rows, except where the maximum lies within the fp32
    error of a power of two; values within half a step of e4m3 (2^-4 relative, 2^-10 of the scale below its
    normal range) plus the fp32 error."""
    T, H = y64.shape
    tol = (H / 32 + 20) * U
    blocks = y64.reshape(T, H // 32, 32)
    amax = blocks.abs().amax(2)
    lo, hi = ((torch.frexp(amax * (1 + d))[1] - 1 + 127).clamp(0, 254) for d in (-tol, tol))
    zero = amax == 0
    lo, hi = torch.where(zero, 0, lo), torch.where(zero, 0, hi)
    sc = s.cpu().to(torch.int32)
    assert ((sc >= lo) & (sc <= hi)).all()
    scale = torch.ldexp(torch.ones_like(amax), sc - 127)[:, :, None]
    got = q.cpu().view(torch.float8_e4m3fn).double().reshape(T, H // 32, 32) * scale
    err = (got - blocks).abs()
    assert (err <= (2.0 ** -4 + tol) * blocks.abs() + 2.0 ** -10 * scale).all()
    pad = torch.zeros((T + 127) // 128 * 128, H // 32, dtype=torch.uint8)
    pad[:T] = s.cpu()
    assert torch.equal(atoms.cpu().reshape(-1), orc.mx_sf_atoms(pad).reshape(-1))


@pytest.mark.parametrize("T,H", [(1, 128), (1, 8192), (3, 256), (127, 384), (128, 1024), (129, 4096), (257, 7168), (5, 65536),
                                 (2000, 640)])
@pytest.mark.parametrize("types", ["bf16-bf16", "bf16-f32", "f32-f32"])
@pytest.mark.parametrize("residual", [True, False])
def test_mx(orc, T, H, types, residual):
    import tk_kernel as tk
    dtype, wdtype = (DT[t] for t in types.split("-"))
    x, res, w = make(T, H, dtype, wdtype, residual, seed=5)
    w[H // 2:H // 2 + 32] = 0  # a block of zeros
    y64, r_ref, _ = orc.add_rms_norm_ref(x, res, w)
    q, s, atoms, r = tk.add_rms_norm_mx(x.cuda(), cu(res), w.cuda())
    torch.cuda.synchronize()
    assert torch.equal(r.cpu(), r_ref)
    assert q.shape == (T, H) and s.shape == (T, H // 32) and atoms.shape == ((T + 127) // 128, H // 128, 512)
    check_mx(q, s, atoms, y64, orc)


def test_mx_feeds_the_gemm(capi, orc):
    """norm -> MXFP8 GEMM: the bytes and scales are those mx_quant would hand over, so the product is the
    dequantised one."""
    import tk_kernel as tk
    x, res, w = make(200, 512, torch.bfloat16, torch.bfloat16, True)
    g = torch.Generator().manual_seed(3)
    b = torch.randn(136, 512, generator=g) / 512 ** 0.5
    q, s, atoms, _ = tk.add_rms_norm_mx(x.cuda(), res.cuda(), w.cuda())
    bq, bs, batoms = tk.mx_quant(b.cuda())
    c = tk.gemm_mxfp8(q, atoms, bq, batoms, True)
    torch.cuda.synchronize()
    want = orc.mx_gemm_ref(q.cpu(), s.cpu(), bq.cpu(), bs.cpu())
    assert orc.rel_fro(c.cpu(), want) <= 1e-5


@pytest.mark.parametrize("H", [96, 100, 8192])
def test_in_place_and_shared_inputs(orc, H):
    import tk_kernel as tk
    x, res, w = make(37, H, torch.bfloat16, torch.bfloat16, True)
    y64, r_ref, _ = orc.add_rms_norm_ref(x, res, w)
    d = res.cuda()
    y, r, _ = tk.add_rms_norm(x.cuda(), d, w.cuda(), 1e-6, True)
    assert r is d and torch.equal(d.cpu(), r_ref)
    check_y(y, y64, H, torch.bfloat16)
    # the same tensor as both summands, written over
    y64, r_ref, _ = orc.add_rms_norm_ref(x, x, w)
    d = x.cuda()
    y, r, _ = tk.add_rms_norm(d, d, w.cuda(), inplace=True)
    assert torch.equal(d.cpu(), r_ref)
    check_y(y, y64, H, torch.bfloat16)


def test_in_place_mx(orc):
    import tk_kernel as tk
    x, res, w = make(130, 1024, torch.float32, torch.float32, True)
    y64, r_ref, _ = orc.add_rms_norm_ref(x, res, w)
    d = res.cuda()
    q, s, atoms, r = tk.add_rms_norm_mx(x.cuda(), d, w.cuda(), inplace=True)
    assert r is d and torch.equal(d.cpu(), r_ref)
    check_mx(q, s, atoms, y64, orc)


@pytest.mark.parametrize("H", [64, 257, 4096])
def test_zero_rows_and_non_finite_rows(orc, H):
    """A row of zeros gives zeros; NaN and infinity stay in their rows."""
    import tk_kernel as tk
    x, _, w = make(6, H, torch.float32, torch.float32, False)
    x[1] = 0
    x[2, H // 2] = float("nan")
    x[4, 0] = float("inf")
    y, _, rstd = tk.add_rms_norm(x.cuda(), None, w.cuda())
    y64, _, _ = orc.add_rms_norm_ref(x, None, w)
    y = y.cpu()
    assert torch.isfinite(rstd.cpu()[[0, 1, 3, 5]]).all()
    assert (y[1] == 0).all()
    assert torch.isnan(y[2]).all() and torch.isnan(y[4, 0])
    for i in (0, 3, 5):
        check_y(y[i:i + 1].cuda(), y64[i:i + 1], H, torch.float32)
    if H % 128 == 0:
        q, s, _, _ = tk.add_rms_norm_mx(x.cuda(), None, w.cuda())
        v = q.cpu().view(torch.float8_e4m3fn).float()
        assert torch.isnan(v[2]).all() and torch.isfinite(v[[0, 1, 3, 5]]).all()
        assert (v[1] == 0).all() and (s.cpu()[1] == 0).all()


def test_no_rows():
    import tk_kernel as tk
    x, w = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), torch.ones(256, dtype=torch.bfloat16, device="cuda")
    y, r, rstd = tk.add_rms_norm(x, x, w)
    assert y.shape == (0, 256) and r.shape == (0, 256) and rstd.shape == (0,)
    q, s, atoms, _ = tk.add_rms_norm_mx(x, None, w)
    assert q.shape == (0, 256) and s.shape == (0, 8) and atoms.shape == (0, 2, 512)
    dx, dw = tk.add_rms_norm_bwd(y, None, x, rstd, w)
    assert dx.shape == (0, 256) and (dw == 0).all()


def test_unaligned_rows(orc):
    """Rows that start on 2 or 4 bytes only (a view into a larger buffer)."""
    import tk_kernel as tk
    for dtype, H in ((torch.bfloat16, 264), (torch.float32, 260)):
        x, res, w = make(9, H, dtype, dtype, True)
        buf = torch.empty(3 * 9 * H + H + 16, dtype=dtype, device="cuda")
        views, at = [], 1
        for t in (x, res, w):
            v = buf[at:at + t.numel()].view(t.shape)
            v.copy_(t)
            views.append(v)
            at += t.numel() + 1
        y, r, rstd = tk.add_rms_norm(*views)
        y64, r_ref, _ = orc.add_rms_norm_ref(x, res, w)
        assert torch.equal(r.cpu(), r_ref)
        check_y(y, y64, H, dtype)
        dx, dw = tk.add_rms_norm_bwd(views[0], views[1], r, rstd, views[2])
        check_bwd(dx, dw, x, res, r_ref, rstd.cpu(), w, orc)


def test_unaligned_rows_mx(orc):
    import tk_kernel as tk
    x, res, w = make(9, 256, torch.bfloat16, torch.bfloat16, True)
    buf = torch.empty(20 + 9 * 256, dtype=torch.bfloat16, device="cuda")
    v = buf[2:2 + 9 * 256].view(9, 256)
    v.copy_(x)
    q, s, atoms, r = tk.add_rms_norm_mx(v, res.cuda(), w.cuda())
    y64, r_ref, _ = orc.add_rms_norm_ref(x, res, w)
    assert torch.equal(r.cpu(), r_ref)
    check_mx(q, s, atoms, y64, orc)


@pytest.mark.parametrize("T", [1, 127, 128, 129])
@pytest.mark.parametrize("H,dtype", [(63, torch.float32), (65, torch.bfloat16), (512, torch.bfloat16), (5003, torch.float32),
                                     (8200, torch.bfloat16), (20000, torch.bfloat16)])
def test_few_rows_backward(orc, capi, T, H, dtype):
    """Both sides of the one-launch backward pass; guard words around its outputs, called through the C ABI."""
    x, res, w = make(T, H, dtype, torch.float32, True)
    dy = torch.randn(T, H, generator=torch.Generator().manual_seed(T + H)).to(dtype)
    rstd = 1 / (x.double().square().mean(1) + 1e-6).sqrt()
    rstd = rstd.float()
    bits, L = dtype.itemsize, capi.lib()
    wb = L.dk_add_rms_norm_bwd_workspace_bytes(T, H)
    assert (wb == 0) == (T <= 128)
    out = {k: torch.full((n + 512,), 0xA5, dtype=torch.uint8, device="cuda") for k, n in (("dx", T * H * bits), ("dw", 4 * H), ("ws", wb))}
    D, DR, R, S, W = dy.cuda(), res.cuda(), x.cuda(), rstd.cuda(), w.cuda()
    at = {k: b.data_ptr() + 256 for k, b in out.items()}
    capi.check(L.dk_add_rms_norm_bwd(D.data_ptr(), DR.data_ptr(), R.data_ptr(), S.data_ptr(), W.data_ptr(), int(bits == 4), 1, T, H,
                                     at["dx"], at["dw"], at["ws"] if wb else None, wb, capi._stream_ptr(None)))
    torch.cuda.synchronize()
    for k, b in out.items():
        assert (b[:256] == 0xA5).all() and (b[-256:] == 0xA5).all(), k
    check_bwd(out["dx"][256:-256].view(dtype).view(T, H), out["dw"][256:-256].view(torch.float32), dy, res, x, rstd, w, orc)


def test_nothing_is_written_outside(capi):
    """Guard words around every output, called through the C ABI."""
    T, H = 131, 384
    x, res, w = make(T, H, torch.bfloat16, torch.bfloat16, True)
    X, R, W = x.cuda(), res.cuda(), w.cuda()
    st = capi._stream_ptr(None)

    def guarded(nbytes):
        b = torch.full((nbytes + 512,), 0xA5, dtype=torch.uint8, device="cuda")
        return b, b.data_ptr() + 256

    sizes = dict(y=2 * T * H, r=2 * T * H, rstd=4 * T, q=T * H, s=T * H // 32, atoms=capi.lib().dk_mx_sf_bytes(T, H), dx=2 * T * H,
                 dw=2 * H, ws=capi.lib().dk_add_rms_norm_bwd_workspace_bytes(T, H))
    b = {k: guarded(n) for k, n in sizes.items()}
    L = capi.lib()
    capi.check(L.dk_add_rms_norm(X.data_ptr(), R.data_ptr(), W.data_ptr(), 0, 0, T, H, 1e-6, b["y"][1], b["r"][1], b["rstd"][1], st))
    capi.check(L.dk_add_rms_norm_mx(X.data_ptr(), R.data_ptr(), W.data_ptr(), 0, 0, T, H, 1e-6, b["q"][1], b["s"][1], b["atoms"][1],
                                    b["r"][1], st))
    capi.check(L.dk_add_rms_norm_bwd(X.data_ptr(), R.data_ptr(), b["r"][1], b["rstd"][1], W.data_ptr(), 0, 0, T, H, b["dx"][1],
                                     b["dw"][1], b["ws"][1], sizes["ws"], st))
    torch.cuda.synchronize()
    for k, (buf, _) in b.items():
        assert (buf[:256] == 0xA5).all() and (buf[256 + sizes[k]:] == 0xA5).all(), k


def test_more_than_2_31_elements(orc):
    """Offsets past 32 bits: rows beyond element 2^31 (bf16, 4.3 GB a tensor)."""
    import tk_kernel as tk
    H = 65536
    T = (1 << 31) // H + 3
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    row = torch.randn(2, H, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[-2:] = row.cuda()
    y, _, rstd = tk.add_rms_norm(x, None, w)
    y64, _, _ = orc.add_rms_norm_ref(row, None, w.cpu())
    check_y(y[-2:], y64, H, torch.bfloat16)
    assert (y[:4] == 0).all()
    q, s, _, _ = tk.add_rms_norm_mx(x, None, w)
    got = q[-2:].view(torch.float8_e4m3fn).float().reshape(2, -1, 32) * torch.exp2(s[-2:].float() - 127)[:, :, None]
    assert orc.rel_fro(got.reshape(2, H).cpu(), y64.float()) <= 2.0 ** -4
    dx, dw = tk.add_rms_norm_bwd(y, None, x, rstd, w)
    dx64, _ = orc.add_rms_norm_bwd_ref(y[-2:].cpu(), None, row, rstd[-2:].cpu(), w.cpu())
    n = row.double() * rstd[-2:].double().cpu()[:, None]
    mag = rstd[-2:].double().cpu()[:, None] * (y[-2:].double().cpu().abs() + n.abs())
    # |mean(g n)| <= 1.01 here (g is y, n is y up to its rounding): the bound of check_bwd
    assert ((dx[-2:].double().cpu() - dx64).abs() <= 2.0 ** -8 * dx64.abs() + (H / 32 + 24) * U * 1.02 * mag).all()
    del x, y, q, s, dx
    torch.cuda.empty_cache()


def test_side_stream_and_graph(orc):
    """On a stream of its own, and captured with its backward pass into a graph that is replayed on other inputs."""
    import tk_kernel as tk
    x, res, w = make(300, 520, torch.bfloat16, torch.bfloat16, True)
    X, R, W = x.cuda(), res.cuda(), w.cuda()
    DY = torch.randn(300, 520, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = tk.add_rms_norm(X, R, W)
        want = want + tk.add_rms_norm_bwd(DY, R, want[1], want[2], W)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    X0 = torch.zeros_like(X)
    with torch.cuda.graph(graph):
        y, r, rstd = tk.add_rms_norm(X0, R, W)
        dx, dw = tk.add_rms_norm_bwd(DY, R, r, rstd, W)
    for _ in range(2):
        X0.copy_(X)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((y, r, rstd, dx, dw), want):
            assert torch.equal(a, b)
        X0.zero_()


def test_refusals():
    import tk_kernel as tk
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    f = lambda *s: torch.zeros(*s, device="cuda")
    for call, what in [
        (lambda: tk.add_rms_norm(b(4, 8).t(), None, b(4)), "contiguous"),
        (lambda: tk.add_rms_norm(b(4, 8).half(), None, b(8)), "dtype"),
        (lambda: tk.add_rms_norm(b(4, 8), f(4, 8), b(8)), "Residual"),
        (lambda: tk.add_rms_norm(b(4, 8), b(4, 16), b(8)), "Residual"),
        (lambda: tk.add_rms_norm(b(4, 8), None, b(16)), "Weight"),
        (lambda: tk.add_rms_norm(f(4, 8), None, b(8)), "Weight"),
        (lambda: tk.add_rms_norm(b(8), None, b(8)), r"\[T, H\]"),
        (lambda: tk.add_rms_norm(b(4, 8), None, b(8), 0.0), "eps"),
        (lambda: tk.add_rms_norm(b(4, 8), None, b(8), float("nan")), "eps"),
        (lambda: tk.add_rms_norm(b(4, 8), None, b(8), 1e-6, True), "inplace"),
        (lambda: tk.add_rms_norm(b(1, 65537), None, b(65537)), "65536"),
        (lambda: tk.add_rms_norm_mx(b(4, 192), None, b(192)), "multiple of 128"),
        (lambda: tk.add_rms_norm_bwd(b(4, 8), None, b(4, 8), f(5), b(8)), "rstd"),
        (lambda: tk.add_rms_norm_bwd(b(4, 8), None, b(4, 8), b(4), b(8)), "rstd"),
        (lambda: tk.add_rms_norm_bwd(b(3, 8), None, b(4, 8), f(4), b(8)), "dY"),
        (lambda: tk.add_rms_norm_bwd(b(4, 8), b(4, 9), b(4, 8), f(4), b(8)), "dR"),
        (lambda: tk.add_rms_norm(b(4, 8), None, torch.zeros(8, dtype=torch.bfloat16)), "CUDA device"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call()
    torch.cuda.synchronize()
