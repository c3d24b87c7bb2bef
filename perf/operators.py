"""The dense half of a decoder layer around the framework's GEMMs: what is measured of it.

Operators, by a case's "op":

  norm        add_rms_norm: the residual's addition and the root-mean-square norm
  norm_train  the same with its backward pass
  norm_mx     add_rms_norm_mx: the norm leaves as MXFP8 (e4m3 with a power-of-two scale per 32 values), the
              scales row-major and as the tensor core's atoms
  ffn         gated_ffn: gate and up projection, SiLU, product, down projection
  ffn_train   the same with its backward pass

With `own` false, run() is the plain form: elementary torch operations in 32 bits, rounded once at the end.
With `own` true it makes the framework's calls.
"""
import os
import sys

import torch

own = False

EPS = 1e-6
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def listed():
    return [
        # one sequence being answered: latency
        dict(name="norm, one token", op="norm", tokens=1, hidden=8192, dtype="bfloat16", residual=True),
        # a long prompt, or several packed into one pass
        dict(name="norm, prompt", op="norm", tokens=16384, hidden=8192, dtype="bfloat16", residual=True),
        # a training step of a narrow layer of odd width in 32 bits, the first of its stack (no residual yet)
        dict(name="norm step, odd width", op="norm_train", tokens=1021, hidden=5003, dtype="float32", residual=False),
        # a training step
        dict(name="norm step", op="norm_train", tokens=8192, hidden=7168, dtype="bfloat16", residual=True),
        # ragged prompts of a layer whose stream is kept in 32 bits
        dict(name="norm to 8 bits, ragged", op="norm_mx", tokens=3001, hidden=4096, dtype="float32", residual=True),
        # the largest pass of a serving step
        dict(name="norm to 8 bits, prompt", op="norm_mx", tokens=32768, hidden=7168, dtype="bfloat16", residual=True),
        # one sequence being answered: the weights are read for one row
        dict(name="ffn, one token", op="ffn", tokens=1, hidden=4096, inner=14336),
        # a batch of sequences being answered, one rank of eight of a tensor-parallel layer
        dict(name="ffn, 48 sequences", op="ffn", tokens=48, hidden=8192, inner=3584),
        # prompts of odd length
        dict(name="ffn, ragged prompts", op="ffn", tokens=1357, hidden=7168, inner=2048),
        # a long prompt
        dict(name="ffn, prompt", op="ffn", tokens=8192, hidden=4096, inner=14336),
        # a small training step of odd length, inner width no multiple of a tile
        dict(name="ffn step, small", op="ffn_train", tokens=513, hidden=2048, inner=1416),
        # a training step, one rank of four of a tensor-parallel layer
        dict(name="ffn step", op="ffn_train", tokens=4096, hidden=8192, inner=7168),
    ]


def _log_int(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "norm_mx", "ffn", "ffn_train"])
    if op in ("ffn", "ffn_train"):
        hidden, inner = 8 * _log_int(rng, 32, 1024), 8 * _log_int(rng, 32, 1792)
        tokens = _log_int(rng, 1, 8192 if op == "ffn" else 4096)
        most = 8192 * 4096 * 14336 if op == "ffn" else 4096 * 8192 * 7168  # the largest listed ones
        return dict(op=op, tokens=max(1, min(tokens, most // (hidden * inner))), hidden=hidden, inner=inner)
    case = dict(op=op, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), residual=rng.random() < 0.75)
    if op == "norm_mx":
        hidden, tokens, most = 128 * _log_int(rng, 1, 64), _log_int(rng, 1, 32768), 32768 * 7168
    elif op == "norm_train":
        hidden, tokens, most = _log_int(rng, 64, 8192), _log_int(rng, 1, 8192), 8192 * 7168
    else:
        hidden, tokens, most = _log_int(rng, 64, 8192), _log_int(rng, 1, 16384), 16384 * 8192
    if op != "norm_mx" and rng.random() < 0.7:  # widths are multiples of 8 more often than not
        hidden = max(64, hidden // 8 * 8)
    if case["dtype"] == "float32":
        most //= 2
    return dict(case, tokens=max(1, min(tokens, most // hidden)), hidden=hidden)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    t, h = case["tokens"], case["hidden"]
    if case["op"] in ("ffn", "ffn_train"):
        f = case["inner"]
        state = dict(x=normal(t, h), w13=normal(2 * f, h, std=h ** -0.5), w2=normal(h, f, std=f ** -0.5))
        if case["op"] == "ffn_train":
            state["dy"] = normal(t, h)
    else:
        dtype = getattr(torch, case["dtype"])
        # some channels of a residual stream are much larger than others
        channel = torch.exp(0.7 * torch.randn(h, generator=gen, device="cuda"))
        state = dict(x=(torch.randn(t, h, generator=gen, device="cuda") * channel).to(dtype),
                     weight=(1 + 0.2 * torch.randn(h, generator=gen, device="cuda")).to(dtype), residual=None)
        if case["residual"]:
            state["residual"] = (2 * torch.randn(t, h, generator=gen, device="cuda") * channel).to(dtype)
        if case["op"] == "norm_train":
            state["dy"] = normal(t, h, dtype=dtype)
            state["dr"] = normal(t, h, dtype=dtype) if case["residual"] else None
    state["op"] = case["op"]
    return state


# ------------------------------------------------------------------------------------ plain forms
def _norm(state):
    """The stream r in its type (x itself without a residual), r in 32 bits, 1/rms, the normed values in 32 bits."""
    x, residual = state["x"], state["residual"]
    r = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    r32 = r.float()
    rstd = 1.0 / torch.sqrt(r32.square().mean(dim=1) + EPS)
    n = r32 * rstd[:, None]
    return r, rstd, n


def _plain_norm(state):
    r, rstd, n = _norm(state)
    y = (n * state["weight"].float()).to(r.dtype)
    return dict(y=y, r=r, rstd=rstd) if state["residual"] is not None else dict(y=y, rstd=rstd)


def _plain_norm_train(state):
    r, rstd, n = _norm(state)
    w, dy = state["weight"].float(), state["dy"].float()
    y = (n * w).to(r.dtype)
    g = dy * w
    dx = rstd[:, None] * (g - n * (g * n).mean(dim=1, keepdim=True))
    if state["dr"] is not None:
        dx = dx + state["dr"].float()
    dw = (dy * n).sum(dim=0)
    return dict(y=y, dx=dx.to(r.dtype), dw=dw.to(r.dtype))


def _plain_norm_mx(state):
    r, _, n = _norm(state)
    y = n * state["weight"].float()
    t, h = y.shape
    blocks = y.reshape(t, h // 32, 32)
    amax = blocks.abs().amax(dim=2)
    # amax = m * 2^e with m in [0.5, 1): floor(log2(amax)) = e - 1
    s = torch.where(amax == 0, 0, (torch.frexp(amax)[1] - 1 + 127).clamp(0, 254)).to(torch.int32)
    scaled = torch.ldexp(blocks, (127 - s)[:, :, None]).reshape(t, h)
    q = scaled.to(torch.float8_e4m3fn)
    rows = torch.zeros((t + 127) // 128 * 128, h // 32, dtype=torch.uint8, device=y.device)
    rows[:t] = s.to(torch.uint8)
    # atom of 128 rows x 4 scales: byte 16 * (row % 32) + 4 * (row // 32) + scale
    atoms = rows.reshape(-1, 4, 32, h // 128, 4).permute(0, 3, 2, 1, 4).reshape(-1, h // 128, 512)
    e8m0 = torch.float8_e8m0fnu
    out = dict(q=q, s=rows[:t].view(e8m0), atoms=atoms.contiguous().view(e8m0))
    return dict(out, r=r) if state["residual"] is not None else out


def _ffn(state):
    x, w13, w2 = state["x"].float(), state["w13"].float(), state["w2"].float()
    f = w2.shape[1]
    gu = x @ w13.t()
    g, u = gu[:, :f], gu[:, f:]
    sig = 1.0 / (1.0 + torch.exp(-g))
    return x, w13, w2, g, u, sig, g * sig * u


def _plain_ffn(state):
    _, _, w2, _, _, _, h = _ffn(state)
    return (h @ w2.t()).to(state["x"].dtype)


def _plain_ffn_train(state):
    x, w13, w2, g, u, sig, h = _ffn(state)
    dtype = state["x"].dtype
    y = (h @ w2.t()).to(dtype)
    dy = state["dy"].float()
    dh = dy @ w2
    dgu = torch.cat([dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig], dim=1)
    return dict(y=y, dx=(dgu @ w13).to(dtype), dw13=(dgu.t() @ x).to(dtype), dw2=(dy.t() @ h).to(dtype))


# ------------------------------------------------------------------------------------ the framework's calls
def _kernels():
    path = os.path.join(ROOT, "distributed-hipkittens_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tk_kernel
    return tk_kernel


def _own(state):
    tk = sys.modules.get("tk_kernel") or _kernels()
    op = state["op"]
    if op == "ffn":
        return tk.gated_ffn(state["x"], state["w13"], state["w2"])
    if op == "ffn_train":
        x, w13, w2 = state["x"], state["w13"], state["w2"]
        y, gu, h = tk.gated_ffn(x, w13, w2, True)
        dx, dw13, dw2 = tk.gated_ffn_bwd(state["dy"], x, w13, w2, gu, h)
        return dict(y=y, dx=dx, dw13=dw13, dw2=dw2)
    x, residual, weight = state["x"], state["residual"], state["weight"]
    if op == "norm_mx":
        q, s, atoms, r = tk.add_rms_norm_mx(x, residual, weight, EPS)
        e8m0 = torch.float8_e8m0fnu
        out = dict(q=q.view(torch.float8_e4m3fn), s=s.view(e8m0), atoms=atoms.view(e8m0))
        return dict(out, r=r) if residual is not None else out
    y, r, rstd = tk.add_rms_norm(x, residual, weight, EPS)
    if op == "norm":
        return dict(y=y, r=r, rstd=rstd) if residual is not None else dict(y=y, rstd=rstd)
    dx, dw = tk.add_rms_norm_bwd(state["dy"], state["dr"], r, rstd, weight)
    return dict(y=y, dx=dx, dw=dw)


PLAIN = dict(norm=_plain_norm, norm_train=_plain_norm_train, norm_mx=_plain_norm_mx, ffn=_plain_ffn,
             ffn_train=_plain_ffn_train)


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["op"]](state)


def work(case):
    t, h = case["tokens"], case["hidden"]
    if case["op"] in ("ffn", "ffn_train"):
        f = case["inner"]
        if case["op"] == "ffn":
            return dict(bytes=2 * (2 * t * h + 3 * h * f), flops=6 * t * h * f)
        return dict(bytes=2 * (4 * t * h + 6 * h * f), flops=18 * t * h * f)
    b = 2 if case["dtype"] == "bfloat16" else 4
    rows, res = t * h * b, 1 if case["residual"] else 0
    if case["op"] == "norm":  # x, residual, r, y, weight, rstd
        return dict(bytes=(2 + 2 * res) * rows + h * b + 4 * t, flops=5 * t * h)
    if case["op"] == "norm_train":  # x, residual, y, dy, dr, dx, weight, its gradient
        return dict(bytes=(4 + 2 * res) * rows + 2 * h * b, flops=16 * t * h)
    atoms = (t + 127) // 128 * 128 * (h // 32)
    return dict(bytes=(1 + 2 * res) * rows + t * h + t * h // 32 + atoms + h * b, flops=8 * t * h)


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("ffn", "ffn_train"):
        x, w2 = state["x"].double(), state["w2"].double()
        wg, wu = state["w13"].double().split(case["inner"])
        gate, up = x.matmul(wg.T), x.matmul(wu.T)
        s = torch.sigmoid(gate)
        hidden = gate.mul(s).mul(up)
        y = hidden.matmul(w2.T)
        if case["op"] == "ffn":
            return y
        dy = state["dy"].double()
        dh = dy.matmul(w2)
        dgate = dh * up * (s + gate * s * (1 - s))
        dup = dh * gate * s
        return dict(y=y, dx=dgate.matmul(wg) + dup.matmul(wu),
                    dw13=torch.cat([dgate.T.matmul(x), dup.T.matmul(x)]), dw2=dy.T.matmul(hidden))
    # the stream is kept in the inputs' type, and what is kept is what is normed
    stream = state["x"] if state["residual"] is None else (state["x"].double() + state["residual"].double()).to(state["x"].dtype)
    r, w = stream.double(), state["weight"].double()
    norm = torch.linalg.vector_norm(r, dim=1, keepdim=True)
    rstd = (norm * norm / r.shape[1] + EPS) ** -0.5
    y = r * rstd * w
    if case["op"] == "norm":
        out = dict(y=y, rstd=rstd.squeeze(1))
        return out if state["residual"] is None else dict(out, r=r)
    if case["op"] == "norm_train":
        dy = state["dy"].double()
        a = dy * w
        dx = a * rstd - r * rstd ** 3 * torch.einsum("th,th->t", a, r)[:, None] / r.shape[1]
        if state["dr"] is not None:
            dx += state["dr"].double()
        return dict(y=y, dx=dx, dw=torch.einsum("th,th->h", dy, r * rstd))
    t, h = y.shape
    top = y.unflatten(1, (-1, 32)).abs().max(dim=2).values
    power = torch.floor(torch.log2(top)).clamp(-127, 127)
    power = torch.where(top == 0, -127.0, power)
    scale = torch.exp2(power)
    q = (y.unflatten(1, (-1, 32)) / scale[:, :, None]).flatten(1)
    padded = torch.full(((t + 127) // 128 * 128, h // 32), 2.0 ** -127, dtype=torch.float64, device=y.device)
    padded[:t] = scale
    row = torch.arange(128, device=y.device).reshape(4, 32).T.reshape(-1)  # atom order: row % 32, then row // 32
    atoms = padded.reshape(-1, 128, h // 128, 4)[:, row].transpose(1, 2).reshape(-1, h // 128, 512)
    out = dict(q=q, s=scale, atoms=atoms)
    return out if state["residual"] is None else dict(out, r=r)
