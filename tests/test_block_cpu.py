"""Norm and gated feed-forward block without a GPU: the 64-bit formulas the GPU tests hold the kernels to, checked
against autograd and differences; argument checks of the C ABI and of tk_kernel; shape functions."""
import ctypes as C

import pytest
import torch


def _p(n):
    return C.c_void_p(n)


def test_norm_formulas_against_autograd(orc):
    g = torch.Generator().manual_seed(0)
    r, w, dy, dr = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((5, 12), (12,), (5, 12), (5, 12)))
    rr, ww = r.clone().requires_grad_(), w.clone().requires_grad_()
    y = rr / torch.sqrt(rr.square().mean(1, keepdim=True) + 1e-6) * ww
    ((y * dy).sum() + (rr * dr).sum()).backward()
    y64, _, rstd = orc.add_rms_norm_ref(r, None, w)
    assert torch.allclose(y64, y.detach(), rtol=1e-12, atol=1e-12)
    dx, dw = orc.add_rms_norm_bwd_ref(dy, dr, r, rstd, w)
    assert torch.allclose(dx, rr.grad, rtol=1e-10, atol=1e-10) and torch.allclose(dw, ww.grad, rtol=1e-10, atol=1e-10)


def test_ffn_formulas_against_autograd_and_differences(orc):
    g = torch.Generator().manual_seed(1)
    x, w13, w2, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 6), (8, 6), (6, 4), (3, 6)))
    leaves = [t.clone().requires_grad_() for t in (x, w13, w2)]
    y = orc.gated_ffn_ref(*leaves)[0]
    (y * dy).sum().backward()
    got = orc.gated_ffn_bwd_ref(dy, x, w13, w2)
    for a, b in zip(got, leaves):
        assert torch.allclose(a, b.grad, rtol=1e-10, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: orc.gated_ffn_ref(*a)[0], [t.clone().requires_grad_() for t in (x, w13, w2)])


def test_stream_is_rounded_before_the_norm(orc):
    x, res = torch.tensor([[256.0, 1.0]]).to(torch.bfloat16), torch.tensor([[1.0, 1.0]]).to(torch.bfloat16)
    _, r, rstd = orc.add_rms_norm_ref(x, res, torch.ones(2))
    assert r[0, 0] == 256.0  # 257 lies between two bf16 values
    assert abs(rstd.item() - ((256.0 ** 2 + 4) / 2 + 1e-6) ** -0.5) < 1e-12


def test_c_abi_argument_errors(capi):
    L, one = capi.lib(), _p(4096)
    norm = lambda T=4, H=64, x=one, w=one, xf=0, wf=0, eps=1e-6, y=one, res=None, r=None: L.dk_add_rms_norm(
        x, res, w, xf, wf, T, H, eps, y, r, one, None)
    bad = [norm(T=-1), norm(T=(1 << 30) + 1), norm(H=0), norm(H=65537), norm(x=None), norm(w=None), norm(y=None), norm(xf=1, wf=0), norm(eps=0.0),
           norm(eps=-1.0), norm(eps=float("nan")), norm(eps=float("inf")), norm(res=one), norm(r=one), norm(x=_p(4097)), norm(y=_p(4097)), norm(w=_p(4097)), norm(x=_p(4098), xf=1, wf=1)]
    assert bad == [capi.ERR_ARG] * len(bad)
    assert norm(T=0, x=None, y=None) == 0
    mx = lambda T=4, H=128, q=one, s=one, a=one, res=None, r=None: L.dk_add_rms_norm_mx(one, res, one, 0, 0, T, H, 1e-6, q, s, a,
                                                                                      r, None)
    bad = [mx(H=64), mx(H=192), mx(q=None), mx(s=None), mx(a=None), mx(res=one), mx(q=_p(4100)), mx(a=_p(4104)), mx(s=_p(4097))]
    assert bad == [capi.ERR_ARG] * len(bad)
    assert mx(T=0, q=None) == 0
    wb = L.dk_add_rms_norm_bwd_workspace_bytes(200, 64)
    assert wb >= 64 * 4 and L.dk_add_rms_norm_bwd_workspace_bytes(128, 64) == 0 and L.dk_add_rms_norm_bwd_workspace_bytes(-1, 64) == 0 and L.dk_add_rms_norm_bwd_workspace_bytes(4, 0) == 0
    bwd = lambda dy=one, r=one, rstd=one, w=one, dx=one, dw=one, ws=one, n=wb: L.dk_add_rms_norm_bwd(
        dy, None, r, rstd, w, 0, 0, 200, 64, dx, dw, ws, n, None)
    bad = [bwd(dy=None), bwd(r=None), bwd(rstd=None), bwd(w=None), bwd(dx=None), bwd(dw=None), bwd(ws=None), bwd(n=wb - 1),
           bwd(ws=_p(4100)), bwd(dy=_p(4097)), bwd(dx=_p(4097)), bwd(rstd=_p(4098)), bwd(dw=_p(4097))]
    assert bad == [capi.ERR_ARG] * len(bad)
    ffn = lambda T=4, H=64, F=32, x=one, w13=one, w2=one, h=one, y=one: L.dk_gated_ffn(x, w13, w2, T, H, F, None, h, y, None)
    bad = [ffn(T=-1), ffn(H=0), ffn(F=0), ffn(H=60), ffn(F=20), ffn(x=None), ffn(w13=None), ffn(w2=None), ffn(h=None), ffn(y=None),
           ffn(T=(1 << 24) + 1), ffn(H=(1 << 20) + 8), ffn(x=_p(4104)), ffn(w2=_p(4100)), ffn(y=_p(4104))]
    assert bad == [capi.ERR_ARG] * len(bad)
    assert ffn(T=0, x=None, h=None, y=None) == 0
    for k in range(10):
        args = [one] * 6 + [4, 64, 32] + [one] * 4
        args[k if k < 6 else k + 3] = None
        assert L.dk_gated_ffn_bwd(*args, None) == capi.ERR_ARG, k
        args[k if k < 6 else k + 3] = _p(4104)
        assert L.dk_gated_ffn_bwd(*args, None) == capi.ERR_ARG, k


def test_tk_kernel_argument_errors():
    import tk_kernel as tk
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.bfloat16)
    for call in (lambda: tk.add_rms_norm(x, None, w), lambda: tk.add_rms_norm_mx(x, None, w), lambda: tk.gated_ffn(x, x, x),
                 lambda: tk.add_rms_norm_bwd(x, None, x, w, w), lambda: tk.gated_ffn_bwd(x, x, x, x, x, x)):
        with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
            call()
    with pytest.raises(RuntimeError, match="Expected a torch.Tensor"):
        tk.add_rms_norm([1.0], None, w)
    with pytest.raises(RuntimeError, match="Tensor must be contiguous"):
        tk.gated_ffn(x.t(), x, x)


def test_shape_functions_and_gradients_on_meta(pkg):
    from distributed_hipkittens_b200 import torch_ops
    ops = torch.ops.dk_b200
    for name in torch_ops.OPS:
        assert hasattr(ops, name)
    b = lambda *s, grad=False: torch.empty(*s, dtype=torch.bfloat16, device="meta", requires_grad=grad)
    q, s, atoms, r = ops.add_rms_norm_mx(b(200, 256), b(200, 256), b(256))
    assert q.shape == (200, 256) and s.shape == (200, 8) and atoms.shape == (2, 2, 512) and r.dtype == torch.bfloat16
    x, res, w = b(5, 64, grad=True), b(5, 64, grad=True), b(64, grad=True)
    y, r, rstd = ops.add_rms_norm(x, res, w)
    assert y.shape == (5, 64) and rstd.shape == (5,) and rstd.dtype == torch.float32 and not rstd.requires_grad
    w13, w2 = b(48, 64, grad=True), b(64, 24, grad=True)
    out, gu, h = ops.gated_ffn_train(y, w13, w2)
    assert out.shape == (5, 64) and gu.shape == (5, 48) and h.shape == (5, 24)
    assert not gu.requires_grad and not h.requires_grad
    (out.sum() + r.sum()).backward()
    for t in (x, res, w, w13, w2):
        assert t.grad.shape == t.shape and t.grad.dtype == torch.bfloat16
    assert ops.gated_ffn(y.detach(), w13.detach(), w2.detach()).shape == (5, 64)
    with pytest.raises(RuntimeError, match="expected x"):
        ops.gated_ffn(b(5, 64), b(48, 64), b(64, 32))
