"""gated_ffn and its backward pass against the 64-bit formulas, and the block with its norms as it is used.

Tolerances. A bf16 rounding is off by at most half a step, 2^-8 relative, spread evenly: its root mean square
is at most 2^-8 / sqrt(3) =: R of the value. Independent roundings add up in squares, and a product with
weights that know nothing of them keeps their relative size in the 2-norm:
  y, dw2      h and the result are rounded           sqrt(2) R
  dx, dw13    dgu and the result are rounded         sqrt(2) R
  h           the result is rounded                  R
with 2 % on top for fp32 accumulation and the spread of a finite sample.

A single value: with h = 2^-8 the largest rounding, and |.| taken of every factor,
  g, u      e_g = K 2^-23 |x||wg|^T (fp32 accumulation of K products); kept as they are
  h         e_h = 1.1 |u| e_g + |silu(g)| e_u + h|h|               |silu'| <= 1.1
  y         e_h |w2|^T + (F 2^-23) |h||w2|^T + h|y|
  dh        e_dh = H 2^-23 |dy||w2|
  dg, du    e = 0.5 |dh||u| e_g + 1.1 |dh| e_u + 1.1 |u| e_dh + h|dg|,  1.1 |dh| e_g + |silu(g)| e_dh + h|du|     |silu''| <= 0.5
  dx, dw13, dw2   the errors of the first factor times the second's magnitude, accumulation and rounding as for y
and 5 % on top for products of two errors. (With few rows a weight gradient is a single product: its errors are relative to
the value itself, not to the result's root mean square, so no bound by the latter holds.)
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
R = 2.0 ** -8 / 3 ** 0.5


@pytest.fixture(scope="module")
def ops(pkg):
    from distributed_hipkittens_b200 import torch_ops
    return torch.ops.dk_b200


def make(T, H, F, seed=0):
    g = torch.Generator().manual_seed(seed + T + 7 * H + 31 * F)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(torch.bfloat16)
    return n(T, H), n(2 * F, H, std=H ** -0.5), n(H, F, std=F ** -0.5), n(T, H)


def near(got, want, roundings, tol=None, spread=1.02):
    """`spread`: a sample of n values has a 2-norm that differs by up to about 4 / sqrt(n) from its expectation."""
    got = got.double().to(want.device)
    err, rms = (got - want).abs(), want.square().mean().sqrt()
    assert err.square().mean().sqrt() <= spread * (1 + 4 / want.numel() ** 0.5) * roundings ** 0.5 * R * rms
    if tol is not None:
        assert (err <= 1.05 * tol + 1e-30).all()


def bounds(x, w13, w2, dy):
    """The largest errors of gu, h, y, dx, dw13, dw2 by the rules above."""
    x, w13, w2, dy = (t.double() for t in (x, w13, w2, dy))
    (T, H), F, e, u = x.shape, w2.shape[1], 2.0 ** -8, 2.0 ** -23
    g, up = (x @ w13.t()).chunk(2, 1)
    s = torch.sigmoid(g)
    ag, au = (H * u * (x.abs() @ w13.abs().t())).chunk(2, 1)
    h = g * s * up
    eh = 1.1 * up.abs() * ag + (g * s).abs() * au + e * h.abs()
    y = eh @ w2.abs().t() + F * u * (h.abs() @ w2.abs().t()) + e * (h @ w2.t()).abs()
    dh, edh = dy @ w2, H * u * (dy.abs() @ w2.abs())
    dg, du = dh * up * (s + g * s * (1 - s)), dh * g * s
    eg = 0.5 * (dh * up).abs() * ag + 1.1 * dh.abs() * au + 1.1 * up.abs() * edh + e * dg.abs()
    eu = 1.1 * dh.abs() * ag + (g * s).abs() * edh + e * du.abs()
    d, ed = torch.cat([dg, du], 1), torch.cat([eg, eu], 1)
    prod = lambda a, ea, b: (ea + a.shape[1] * u * a.abs()) @ b.abs() + e * (a @ b).abs()
    return dict(gu=torch.cat([ag, au], 1), h=eh, y=y, dx=prod(d, ed, w13), dw13=prod(d.t(), ed.t(), x),
                dw2=prod(dy.t(), 0 * dy.t(), h) + dy.t().abs() @ eh)


# one token to several tiles; rows and widths that end inside a tile; single vectors
SHAPES = [(1, 512, 256), (2, 64, 64), (3, 8, 8), (5, 256, 72), (16, 1032, 136), (17, 520, 1000), (31, 2048, 4096), (33, 72, 2056),
          (64, 4096, 512), (65, 128, 128), (100, 512, 768), (127, 136, 264), (128, 256, 256), (129, 384, 640), (200, 1024, 136),
          (255, 264, 392), (257, 320, 1288), (513, 512, 520), (700, 2056, 1032),
          (1000, 4104, 1544), (1357, 2048, 3592), (600, 3592, 5128), (2100, 2056, 2568),
          # large weights: token tiles of more than 128, and the tile kernel from 257 rows on
          (150, 4104, 2056), (256, 2056, 4104), (260, 4104, 2056)]


@pytest.mark.parametrize("T,H,F", SHAPES)
def test_forward(orc, capi, T, H, F):
    import tk_kernel as tk
    x, w13, w2, dy = make(T, H, F)
    tol = bounds(*(t.cuda() for t in (x, w13, w2, dy)))
    y64, gu64, h64 = orc.gated_ffn_ref(x.cuda(), w13.cuda(), w2.cuda())
    y = tk.gated_ffn(x.cuda(), w13.cuda(), w2.cuda())
    y2, gu, h = tk.gated_ffn(x.cuda(), w13.cuda(), w2.cuda(), True)
    torch.cuda.synchronize()
    assert capi.device_status()[0] == 0
    near(y, y64, 2, tol["y"])
    assert gu.dtype == torch.float32 and ((gu - gu64).abs() <= tol["gu"] + 1e-30).all()
    near(h, h64, 1, tol["h"])
    assert torch.equal(y, y2)
    assert torch.equal(tk.gated_ffn(x.cuda(), w13.cuda(), w2.cuda()), y)  # the same bits again


@pytest.mark.parametrize("T,H,F", SHAPES)
def test_backward(orc, capi, T, H, F):
    import tk_kernel as tk
    x, w13, w2, dy = (t.cuda() for t in make(T, H, F, seed=1))
    want = orc.gated_ffn_bwd_ref(dy, x, w13, w2)
    _, gu, h = tk.gated_ffn(x, w13, w2, True)
    got = tk.gated_ffn_bwd(dy, x, w13, w2, gu, h)
    torch.cuda.synchronize()
    assert capi.device_status()[0] == 0
    tol = bounds(x, w13, w2, dy)
    for a, b, n, k in zip(got, want, (2, 2, 2), ("dx", "dw13", "dw2")):
        near(a, b, n, tol[k])
    for a, b in zip(got, tk.gated_ffn_bwd(dy, x, w13, w2, gu, h)):
        assert torch.equal(a, b)


def test_every_element_of_every_tile(orc):
    """Weights that route single inputs to single outputs: each value of y is one value of x, exactly, so a tile that
    is swapped, shifted or dropped shows. g = 32 (sigmoid(32) is 1 in fp32), u = x, h = 32 x, y = 32 x / 32."""
    import tk_kernel as tk
    for T, H in ((1, 512), (130, 640), (300, 264), (700, 264)):
        F = H - 8
        x = torch.randint(-64, 64, (T, H), generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
        x[:, -1] = 1
        w13 = torch.zeros(2 * F, H)
        w13[:F, -1] = 32.0
        perm = torch.randperm(F, generator=torch.Generator().manual_seed(H))
        w13[F + torch.arange(F), perm] = 1.0
        w2 = torch.zeros(H, F)
        w2[torch.arange(F), torch.arange(F)] = 1 / 32
        y = tk.gated_ffn(x.cuda(), w13.to(torch.bfloat16).cuda(), w2.to(torch.bfloat16).cuda())
        want = torch.zeros(T, H)
        want[:, :F] = x.float()[:, perm]
        assert torch.equal(y.float().cpu(), want)


def test_extreme_gates():
    """Large gates of both signs: silu(g) is g or 0, its derivative 1 or 0, nothing turns into NaN."""
    import tk_kernel as tk
    T, H, F = 40, 64, 64
    x = torch.zeros(T, H)
    x[:, 0] = torch.linspace(-200, 200, T)
    x[:, 1] = 1
    w13 = torch.zeros(2 * F, H)
    w13[:F, 0] = 4.0
    w13[F:, 1] = 1.0
    w2 = torch.eye(H, F)
    x, w13, w2 = (t.to(torch.bfloat16).cuda() for t in (x, w13, w2))
    y, gu, h = tk.gated_ffn(x, w13, w2, True)
    dx, dw13, dw2 = tk.gated_ffn_bwd(torch.ones_like(y), x, w13, w2, gu, h)
    g = 4 * x[:, 0].double()
    want = g * torch.sigmoid(g)
    assert ((h[:, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all()
    assert all(torch.isfinite(t.float()).all() for t in (y, dx, dw13, dw2))


def test_non_finite_rows_stay_in_their_rows(orc):
    import tk_kernel as tk
    for T in (6, 300, 700):
        x, w13, w2, _ = make(T, 256, 136)
        good = tk.gated_ffn(x.cuda(), w13.cuda(), w2.cuda())
        x[2, 5] = float("nan")
        x[4, 7] = float("inf")
        y = tk.gated_ffn(x.cuda(), w13.cuda(), w2.cuda())
        keep = [i for i in range(T) if i not in (2, 4)]
        assert torch.equal(y[keep], good[keep]) and torch.isnan(y[2]).all() and not torch.isfinite(y[4]).any()


def test_rows_do_not_depend_on_their_batch_neighbours(orc):
    """A row's result depends on that row and its place alone."""
    import tk_kernel as tk
    for T, H, F in ((7, 512, 264), (150, 512, 264), (400, 512, 264), (700, 512, 264), (1357, 2048, 1032)):
        x, w13, w2, _ = make(T, H, F)
        other = make(T, H, F, seed=1)[0]
        keep = torch.arange(0, T, 3)
        other[keep] = x[keep]
        a, b = (tk.gated_ffn(t.cuda(), w13.cuda(), w2.cuda()) for t in (x, other))
        assert torch.equal(a[keep], b[keep]) and not torch.equal(a, b)


def test_no_rows():
    import tk_kernel as tk
    b = lambda *s: torch.full(s, 3.0, dtype=torch.bfloat16, device="cuda")
    x, w13, w2 = b(0, 64), b(32, 64), b(64, 16)
    y, gu, h = tk.gated_ffn(x, w13, w2, True)
    assert y.shape == (0, 64) and gu.shape == (0, 32) and h.shape == (0, 16)
    dx, dw13, dw2 = tk.gated_ffn_bwd(y, x, w13, w2, gu, h)
    assert dx.shape == (0, 64) and (dw13 == 0).all() and (dw2 == 0).all() and dw13.shape == w13.shape and dw2.shape == w2.shape


@pytest.mark.parametrize("T,H,F", [(1, 136, 200), (37, 136, 200), (300, 136, 200), (1357, 2056, 1032)])
def test_nothing_is_written_outside(capi, T, H, F):
    x, w13, w2, dy = (t.cuda() for t in make(T, H, F))
    L, st = capi.lib(), capi._stream_ptr(None)
    sizes = dict(gu=8 * T * F, h=2 * T * F, y=2 * T * H, dgu=4 * T * F, dx=2 * T * H, dw13=4 * F * H, dw2=2 * F * H)
    bufs = {k: torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device="cuda") for k, n in sizes.items()}
    p = {k: b.data_ptr() + 4096 for k, b in bufs.items()}
    capi.check(L.dk_gated_ffn(x.data_ptr(), w13.data_ptr(), w2.data_ptr(), T, H, F, p["gu"], p["h"], p["y"], st))
    capi.check(L.dk_gated_ffn_bwd(dy.data_ptr(), x.data_ptr(), w13.data_ptr(), w2.data_ptr(), p["gu"], p["h"], T, H, F, p["dgu"],
                                  p["dx"], p["dw13"], p["dw2"], st))
    torch.cuda.synchronize()
    for k, b in bufs.items():
        assert (b[:4096] == 0xA5).all() and (b[4096 + sizes[k]:] == 0xA5).all(), k


def test_more_than_2_31_elements(capi):
    """Offsets past 32 bits: [g|u] and its gradient have 2.3e9 elements. The last rows of y and dx against the formulas, and some
    columns of the weight gradients, sums over all rows."""
    import tk_kernel as tk
    T, H, F = 70000, 64, 16384
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16)
    x, w13, w2, dy = n(T, H), n(2 * F, H, std=H ** -0.5), n(H, F, std=F ** -0.5), n(T, H)
    y, gu, h = tk.gated_ffn(x, w13, w2, True)
    dx, dw13, dw2 = tk.gated_ffn_bwd(dy, x, w13, w2, gu, h)
    torch.cuda.synchronize()
    assert capi.device_status()[0] == 0
    assert 2 * T * F > 1 << 31
    last = slice(T - 40, T)
    a = x[last].double()
    gate, up = (a @ w13.double().t()).chunk(2, 1)
    s = torch.sigmoid(gate)
    h64 = gate * s * up
    near(h[last], h64, 1)
    near(y[last], h64 @ w2.double().t(), 2)
    dh = dy[last].double() @ w2.double()
    dgu = torch.cat([dh * up * (s + gate * s * (1 - s)), dh * gate * s], 1)
    near(dx[last], dgu @ w13.double(), 2)
    cols = torch.tensor([0, 1, F // 2, F - 1], device="cuda")
    gate, up = (x.double() @ w13[c].double().t() for c in (cols, F + cols))
    s = torch.sigmoid(gate)
    dh = dy.double() @ w2[:, cols].double()
    near(dw2[:, cols], dy.double().t() @ (gate * s * up), 2)
    near(dw13[cols], (dh * up * (s + gate * s * (1 - s))).t() @ x.double(), 2)
    near(dw13[F + cols], (dh * gate * s).t() @ x.double(), 2)
    del y, gu, h, dx
    torch.cuda.empty_cache()


def test_operators_pass_opcheck(ops):
    x, w13, w2, dy = (t.cuda() for t in make(20, 128, 72))
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    y, r, rstd = ops.add_rms_norm(x, dy, w)
    _, gu, h = ops.gated_ffn_train(x, w13, w2)
    for op, args in ((ops.rms_norm, (x, w)), (ops.add_rms_norm, (x, dy, w)), (ops.add_rms_norm_bwd, (dy, None, r, rstd, w)),
                     (ops.add_rms_norm_mx, (x, dy, w)), (ops.gated_ffn, (x, w13, w2)), (ops.gated_ffn_train, (x, w13, w2)),
                     (ops.gated_ffn_bwd, (dy, x, w13, w2, gu, h))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("T", [4, 260, 700])
def test_two_streams_at_once_and_graph(T):
    """Two calls that overlap on the GPU, and a captured step replayed on other inputs."""
    import tk_kernel as tk
    sets = [tuple(t.cuda() for t in make(T, 1024, 512, seed=s)) for s in (1, 2)]

    def step(x, w13, w2, dy):
        y, gu, h = tk.gated_ffn(x, w13, w2, True)
        return (y,) + tuple(tk.gated_ffn_bwd(dy, x, w13, w2, gu, h))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = step(*sets[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    inputs = [torch.zeros_like(t) for t in sets[0]]
    graphs = []
    for _ in range(2):  # two graphs over the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*inputs)
        graphs.append((graph, out))
    for s, w in zip(sets, want):
        for t, v in zip(inputs, s):
            t.copy_(v)
        torch.cuda.synchronize()
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(u, v) for u, v in zip(out, w))


@pytest.mark.parametrize("T", [3, 260, 700])
def test_order_with_other_work(T):
    """The calls may set themselves up while earlier work runs, but read and write in order: after copies, memsets, torch's
    kernels and events of another stream, before torch's kernels, over buffers that are used again and again, eager and
    captured."""
    import tk_kernel as tk
    x, w13, w2, dy = (t.cuda() for t in make(T, 1024, 512, seed=5))
    w = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
    want = []
    for k in range(3):
        a, _, rstd = tk.add_rms_norm(x * (k + 1), None, w)
        torch.cuda.synchronize()
        y, gu, h = tk.gated_ffn(a, w13, w2, True)
        torch.cuda.synchronize()
        g = tk.gated_ffn_bwd(dy, a, w13, w2, gu, h)
        torch.cuda.synchronize()
        d = tk.add_rms_norm_bwd(g[0], None, x * (k + 1), rstd, w)
        torch.cuda.synchronize()
        want.append([t.clone() for t in (y, *g, *d)])
    side = torch.cuda.Stream()
    buf, wbuf = torch.empty_like(x), torch.empty_like(w13)

    def run(k):
        buf.zero_()
        wbuf.fill_(float("nan"))
        buf.copy_(x)                                 # a copy, not a kernel
        buf.mul_(k + 1)
        ready = torch.cuda.Event()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            wbuf.copy_(w13)
            ready.record(side)
        a, _, rstd = tk.add_rms_norm(buf, None, w)
        torch.cuda.current_stream().wait_event(ready)
        y, gu, h = tk.gated_ffn(a, wbuf, w2, True)
        g = tk.gated_ffn_bwd(dy, a, wbuf, w2, gu, h)
        wbuf.mul_(2)                                 # written right behind its last reader
        d = tk.add_rms_norm_bwd(g[0], None, buf, rstd, w)
        out = [t * 1 for t in (y, *g, *d)]
        buf.zero_()
        return out

    for _ in range(3):
        got = [run(k) for k in range(3)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [run(k) for k in range(3)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_weights_written_right_before(pkg):
    """Weights that a kernel of this library writes right before the call: the second product's early loads of W2 (and of W13 in
    the backward pass) come after that."""
    import tk_kernel as tk
    T, H, F = 5, 64, 8192
    x, w13, w2, dy = (t.cuda() for t in make(T, H, F, seed=8))
    ones, ones_h = (torch.ones(n, dtype=torch.bfloat16, device="cuda") for n in (F, H))
    w2_rows = [(w2 * (k + 1) + k) for k in range(4)]
    w13_rows = [(w13 * (k + 1) - k) for k in range(4)]
    want = []
    for a, b in zip(w2_rows, w13_rows):
        n2, n13 = tk.add_rms_norm(a, None, ones)[0], tk.add_rms_norm(b, None, ones_h)[0]
        torch.cuda.synchronize()
        y, gu, h = tk.gated_ffn(x, n13, n2, True)
        torch.cuda.synchronize()
        want.append([t.clone() for t in (y, *tk.gated_ffn_bwd(dy, x, n13, n2, gu, h))])
        torch.cuda.synchronize()
    L, st = capi_lib(), torch.cuda.current_stream().cuda_stream
    n2, n13, keep = torch.empty_like(w2), torch.empty_like(w13), torch.empty(F * 2, device="cuda")
    for _ in range(20):
        for k in range(4):
            # into the same two buffers every time
            assert L.dk_add_rms_norm(w13_rows[k].data_ptr(), None, ones_h.data_ptr(), 0, 0, 2 * F, H, 1e-6, n13.data_ptr(), None,
                                     keep.data_ptr(), st) == 0
            assert L.dk_add_rms_norm(w2_rows[k].data_ptr(), None, ones.data_ptr(), 0, 0, H, F, 1e-6, n2.data_ptr(), None,
                                     keep.data_ptr(), st) == 0
            y, gu, h = tk.gated_ffn(x, n13, n2, True)
            assert L.dk_add_rms_norm(w13_rows[k].data_ptr(), None, ones_h.data_ptr(), 0, 0, 2 * F, H, 1e-6, n13.data_ptr(), None,
                                     keep.data_ptr(), st) == 0
            got = (y, *tk.gated_ffn_bwd(dy, x, n13, n2, gu, h))
            for a, b in zip(got, want[k]):
                assert torch.equal(a, b)


def capi_lib():
    from distributed_hipkittens_b200 import capi
    return capi.lib()


def test_gradients_against_differences(orc):
    """The backward pass against central differences of the 64-bit forward along random directions."""
    import tk_kernel as tk
    x, w13, w2, dy = (t.cuda() for t in make(9, 128, 72, seed=3))
    _, gu, h = tk.gated_ffn(x, w13, w2, True)
    grads = tk.gated_ffn_bwd(dy, x, w13, w2, gu, h)
    g = torch.Generator().manual_seed(9)
    args = [x.double(), w13.double(), w2.double()]
    for i, grad in enumerate(grads):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64).cuda() * args[i].std()
        e = 1e-5
        up, down = ([a + s * e * d if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        slope = ((orc.gated_ffn_ref(*up)[0] - orc.gated_ffn_ref(*down)[0]) * dy.double()).sum() / (2 * e)
        got = (grad.double() * d).sum()
        # the rounded gradient's error is at most sqrt(2) R of its norm; along d that many standard deviations of d
        assert (got - slope).abs() <= 6 * 2 ** 0.5 * R * grad.double().norm() * args[i].std()


def test_the_block_as_it_is_trained(ops, orc):
    """norm with residual -> feed-forward -> added to the stream by the next norm, gradients through autograd, against
    the same in 64 bits. Roundings on the way: the stream twice, the normed rows twice, h and y; the gradients pass
    as many again. Each is R at most and enters once: sqrt(16) R bounds them together."""
    T, H, F = 150, 264, 520
    g = torch.Generator().manual_seed(4)
    n = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(torch.bfloat16).cuda()
    x, res, w13, w2, dout = n(T, H), n(T, H), n(2 * F, H, std=H ** -0.5), n(H, F, std=F ** -0.5), n(T, H)
    wa, wb = (1 + n(H, std=0.1).float()).to(torch.bfloat16), (1 + n(H, std=0.1).float()).to(torch.bfloat16)
    leaves = [t.clone().requires_grad_() for t in (x, res, wa, w13, w2, wb)]
    a, r, _ = ops.add_rms_norm(leaves[0], leaves[1], leaves[2])
    y, _, _ = ops.gated_ffn_train(a, leaves[3], leaves[4])
    out, r2, _ = ops.add_rms_norm(y, r, leaves[5])
    ((out * dout).sum() + r2.float().sum()).backward()

    ref = [t.double().requires_grad_() for t in (x, res, wa, w13, w2, wb)]
    norm = lambda v, w: v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w
    s = ref[0] + ref[1]
    a64 = norm(s, ref[2])
    gate, up = (a64 @ ref[3].t()).chunk(2, 1)
    y64 = (torch.nn.functional.silu(gate) * up) @ ref[4].t()
    out64 = norm(y64 + s, ref[5])
    ((out64 * dout.double()).sum() + (y64 + s).sum()).backward()
    assert orc.rel_fro(out.double().cpu(), out64.detach().cpu()) <= 4 * R
    for a, b in zip(leaves, ref):
        assert orc.rel_fro(a.grad.double().cpu(), b.grad.cpu()) <= 4 * R


def test_captured_gradients(ops):
    """A step through autograd captured when no eager graph of its leaves is alive, and explicit calls captured while one is."""
    leaves = [t.cuda().requires_grad_() for t in make(40, 64, 128)[:3]]
    dy = make(40, 64, 128)[3].cuda()
    y = ops.gated_ffn_train(*leaves)[0]
    y.backward(dy)
    want = [t.grad.clone() for t in leaves]
    del y
    for t in leaves:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gated_ffn_train(*leaves)[0].backward(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    alive = ops.gated_ffn_train(*leaves)[0]
    plain = [t.detach() for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, gu, h = ops.gated_ffn_train(*plain)
        got = ops.gated_ffn_bwd(dy, *plain, gu, h)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and alive.grad_fn is not None


def test_autograd_alone(ops, orc):
    """rms_norm and gated_ffn_train with an expanded incoming gradient, and an output nobody uses."""
    x, w13, w2, dy = (t.cuda() for t in make(20, 64, 128))
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    xr = x.clone().requires_grad_()
    y, rstd = ops.rms_norm(xr, w)
    assert not rstd.requires_grad
    y.sum().backward()
    dx64, dw64 = orc.add_rms_norm_bwd_ref(torch.ones(20, 64), None, x.cpu(), rstd.cpu(), torch.ones(64))
    assert orc.rel_fro(w.grad.double().cpu(), dw64) <= 2.0 ** -8
    a, r, _ = ops.add_rms_norm(xr, x, w)
    gx, = torch.autograd.grad(r.sum(), [xr])           # only the stream is used
    assert (gx == 1).all()


def test_serving_run(capi, orc):
    """A step as it is served: norm -> feed-forward, the next norm straight into MXFP8 and its GEMM, the stream updated in
    place; every stage against the 64-bit form of its own inputs."""
    import tk_kernel as tk
    for T in (1, 48, 300):
        x, w13, w2, _ = (t.cuda() for t in make(T, 512, 768))
        w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
        stream = x.flip(0).contiguous()
        r_ref = (x.float() + stream.float()).to(torch.bfloat16)
        a, r, _ = tk.add_rms_norm(x, stream, w, 1e-6, True)
        assert r is stream and torch.equal(stream, r_ref)
        y = tk.gated_ffn(a, w13, w2)
        near(y, orc.gated_ffn_ref(a, w13, w2)[0], 2)
        before = stream.clone()
        q, s, atoms, _ = tk.add_rms_norm_mx(y, stream, w, 1e-6, True)
        assert torch.equal(stream, (y.float() + before.float()).to(torch.bfloat16))
        bq, bs, batoms = tk.mx_quant(w2)
        c = tk.gemm_mxfp8(q, atoms, tk.mx_quant(w13)[0], tk.mx_quant(w13)[2], True)
        want = orc.mx_gemm_ref(q.cpu(), s.cpu(), *(t.cpu() for t in tk.mx_quant(w13)[:2]))
        assert orc.rel_fro(c.cpu(), want) <= 1e-5


def test_refusals():
    import tk_kernel as tk
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    x, w13, w2 = b(4, 64), b(48, 64), b(64, 24)
    for call, what in [
        (lambda: tk.gated_ffn(x.float(), w13, w2), "bfloat16"),
        (lambda: tk.gated_ffn(x, w13.half(), w2), "bfloat16"),
        (lambda: tk.gated_ffn(x, w13[:46], w2), "expected X"),
        (lambda: tk.gated_ffn(x, b(48, 56), w2), "expected X"),
        (lambda: tk.gated_ffn(x, w13, b(56, 24)), "expected X"),
        (lambda: tk.gated_ffn(x.t(), w13, w2), "contiguous"),
        (lambda: tk.gated_ffn(x[0], w13, w2), "expected X"),
        (lambda: tk.gated_ffn(x.cpu(), w13, w2), "CUDA device"),
        (lambda: tk.gated_ffn(b(4, 60), b(48, 60), b(60, 24)), "multiples of 8"),
        (lambda: tk.gated_ffn(x, b(40, 64), b(64, 20)), "multiples of 8"),
        (lambda: tk.gated_ffn(b(4 * 64 + 4)[4:].view(4, 64), w13, w2), "16-byte"),
        (lambda: tk.gated_ffn_bwd(b(5, 64), x, w13, w2, b(4, 48).float(), b(4, 24)), "expected dY"),
        (lambda: tk.gated_ffn_bwd(x, x, w13, w2, b(4, 24).float(), b(4, 24)), "expected dY"),
        (lambda: tk.gated_ffn_bwd(x, x, w13, w2, b(4, 48).float(), b(4, 48)), "expected dY"),
        (lambda: tk.gated_ffn_bwd(x, x, w13, w2, b(4, 48), b(4, 24)), "float32"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call()
    torch.cuda.synchronize()
