"""The training-step operators around the attention and its matrix products: what they compute, on which sizes.

Five operators, all bound by the bytes that they move:

* ``rotary``: rotary positions on q and k, half or interleaved pairs, the whole head or its first part, angles from
  64-bit frequencies (scaled for long contexts by the caller's table of frequencies and its attention factor).
  ``serve`` writes the rotated keys into a KV cache's slots, ``train`` runs forward and backward.
* ``pack``: an activation to 8 bits (e4m3 with one power-of-two scale for 32 values) and back.
* ``swiglu``: z = silu(g) * u with (g, u) kept in 8 bits, and the backward pass from them, which gives z again.
* ``norm``: residual add (a sum of the inputs' type) + RMSNorm of that sum with the sum kept in 8 bits, and the
  backward pass from it, which gives y again.
* ``loss``: mean next-token cross entropy over the vocabulary with its gradient.

``run`` takes the plain form (elementary torch operations in 32 bits) or, where ``own`` is set, the framework's
entry points.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
GROUP = 32  # values that share a scale


# -- cases --------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 sequences with 65,536 cached tokens each: launch latency
        dict(name="rotary_decode", op="rotary", mode="serve", B=64, L=1, H=32, Hk=8, D=128, rd=128, pairs="half",
             dtype="bfloat16", scaling="yarn", pos0=65536),
        # the prompt of 131,072 tokens of the 4096-wide layer, keys into the cache
        dict(name="rotary_prompt_128k", op="rotary", mode="serve", B=1, L=131072, H=32, Hk=8, D=128, rd=128,
             pairs="half", dtype="bfloat16", scaling="ntk", pos0=0),
        # a training batch with packed documents, half of each head rotated, pairs side by side
        dict(name="rotary_train_partial", op="rotary", mode="train", B=2, L=8191, H=32, Hk=8, D=128, rd=64,
             pairs="interleaved", dtype="bfloat16", scaling="llama3", pos0=0),
        # the 2048-token fp32 layer (8/2 heads of 64), training
        dict(name="rotary_train_fp32", op="rotary", mode="train", B=1, L=2048, H=8, Hk=2, D=64, rd=64, pairs="half",
             dtype="float32", scaling="none", pos0=0),
        # the residual stream of a small fp32 model, a ragged number of tokens
        dict(name="pack_small", op="pack", rows=191, n=500, dtype="float32"),
        # the residual stream of 32,768 tokens of the 4096-wide model
        dict(name="pack_32k", op="pack", rows=32768, n=4096, dtype="bfloat16"),
        # the MLP of a small model (d_ffn 512) on 2 x 96 tokens
        dict(name="swiglu_small", op="swiglu", rows=192, n=512, dtype="bfloat16"),
        # the MLP of the 4096-wide model (d_ffn 11008) on 16,384 tokens
        dict(name="swiglu_16k", op="swiglu", rows=16384, n=11008, dtype="bfloat16"),
        # the norm of the 512-wide fp32 model on 2047 tokens
        dict(name="norm_small", op="norm", rows=2047, n=512, dtype="float32"),
        # the norm of the 4096-wide model on 32,768 tokens
        dict(name="norm_32k", op="norm", rows=32768, n=4096, dtype="bfloat16"),
        # the loss of a small model: 384 tokens in the vocabulary
        dict(name="loss_small", op="loss", B=2, L=96, V=384, dtype="float32"),
        # the loss of the 4096-wide model: 128,256 tokens in the vocabulary, 8192 positions
        dict(name="loss_8k", op="loss", B=1, L=8192, V=128256, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "pack", "swiglu", "norm", "loss"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    wide = 2 if dtype == "float32" else 1
    if op == "rotary":
        mode = rng.choice(["serve", "train"])
        H, Hk = rng.choice([(32, 8), (8, 2), (16, 16), (20, 4), (9, 3), (5, 1)])
        D = rng.choice([32, 64, 80, 96, 128, 256])
        rd = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        most = 131072 * 40 * 128 // (wide * (2 if mode == "train" else 1))
        tokens = _log_int(rng, 1, max(1, most // ((H + Hk) * D)) if (H + Hk) * D * 131072 > most else 131072)
        B = _log_int(rng, 1, min(64, tokens))
        return dict(op=op, mode=mode, B=B, L=max(1, tokens // B), H=H, Hk=Hk, D=D, rd=rd,
                    pairs=rng.choice(["half", "interleaved"]), dtype=dtype,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), pos0=_log_int(rng, 1, 1000000))
    if op == "loss":
        V = _log_int(rng, 2, 128256)
        tokens = _log_int(rng, 2, max(2, min(131072, 8192 * 128256 // (V * wide))))
        B = _log_int(rng, 1, min(16, tokens // 2))
        return dict(op=op, B=B, L=max(2, tokens // B), V=V, dtype=dtype)
    most = (16384 * 11008 if op == "swiglu" else 32768 * 4096) // wide
    n = _log_int(rng, 1, 16384)
    if rng.random() < 0.5:
        n = max(16, n // 16 * 16)
    return dict(op=op, rows=_log_int(rng, 1, max(1, min(131072, most // n))), n=n, dtype=dtype)


# -- inputs -------------------------------------------------------------------------------------
def _frequencies(rd, scaling, base=10000.0):
    """([rd/2] frequencies in 64 bits, attention factor), as a checkpoint's configuration gives them."""
    f = [base ** (-2.0 * i / rd) for i in range(rd // 2)]
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return [v / 4.0 for v in f], 1.0
    if scaling == "ntk":
        b = base * 8.0 ** (rd / (rd - 2)) if rd > 2 else base
        return [b ** (-2.0 * i / rd) for i in range(rd // 2)], 1.0
    if scaling == "yarn":
        out = []
        for i, v in enumerate(f):
            turns = 4096 * v / (2 * math.pi)  # of this frequency in the trained context
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            out.append(v * keep + v / 16.0 * (1.0 - keep))
        return out, 0.1 * math.log(16.0) + 1.0
    out = []  # llama3: low frequencies divided, high ones kept, a ramp between
    for v in f:
        turns = 8192 * v / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
        out.append(v * keep + v / 8.0 * (1.0 - keep))
    return out, 1.0


def _randn(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=gen, dtype=torch.float32) * scale).to(dtype)


def _activation(gen, rows, n, dtype):
    """Rows of a residual stream: channels of unlike size, some far larger than the rest."""
    chan = torch.exp(torch.randn(n, device=DEV, generator=gen))
    x = torch.randn(rows, n, device=DEV, generator=gen, dtype=torch.float32)
    x *= chan
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    s = dict(case)
    if case["op"] == "rotary":
        B, L, H, Hk, D = (case[k] for k in ("B", "L", "H", "Hk", "D"))
        freq, s["factor"] = _frequencies(case["rd"], case["scaling"])
        s["inv_freq"] = torch.tensor(freq, dtype=torch.float64, device=DEV)
        s["q"] = _randn(gen, B, L, H, D, dtype=dt)
        s["k"] = _randn(gen, B, L, Hk, D, dtype=dt)
        if case["mode"] == "serve":
            # sequences of unlike length: each starts at its own position
            start = case["pos0"] + torch.randint(0, 64, (B, 1), device=DEV, generator=gen)
            s["positions"] = start + torch.arange(L, device=DEV)
            s["q_out"] = torch.empty_like(s["q"])
            cache = torch.zeros(B, L + 8, 2, Hk, D, device=DEV, dtype=dt)
            s["k_out"] = cache[:, 5:5 + L, 0]
        else:
            # packed documents: positions start again at 0
            cut = torch.randint(0, max(1, L // 2) + 1, (B, 1), device=DEV, generator=gen)
            at = torch.arange(L, device=DEV).expand(B, L)
            s["positions"] = torch.where(at < cut, at, at - cut) + case["pos0"]
            s["dq"] = _randn(gen, B, L, H, D, dtype=dt)
            s["dk"] = _randn(gen, B, L, Hk, D, dtype=dt)
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
    elif case["op"] == "pack":
        s["x"] = _activation(gen, case["rows"], case["n"], dt)
    elif case["op"] == "swiglu":
        s["gu"] = _randn(gen, case["rows"], 2 * case["n"], dtype=dt, scale=1.5)
        s["dz"] = _randn(gen, case["rows"], case["n"], dtype=dt)
    elif case["op"] == "norm":
        s["x"] = _activation(gen, case["rows"], case["n"], dt)
        s["a"] = _randn(gen, case["rows"], case["n"], dtype=dt)
        s["weight"] = (1 + 0.1 * torch.randn(case["n"], device=DEV, generator=gen)).to(dt)
        s["dy"] = _randn(gen, case["rows"], case["n"], dtype=dt)
        s["dh"] = _randn(gen, case["rows"], case["n"], dtype=dt)
        s["eps"] = 1e-5
    else:
        B, L, V = case["B"], case["L"], case["V"]
        s["logits"] = torch.randn(B, L, V, device=DEV, generator=gen, dtype=dt).mul_(3.0)
        labels = torch.randint(0, V, (B, L), device=DEV, generator=gen)
        # a prompt of up to a quarter of each sequence does not count
        skip = torch.randint(0, L // 4 + 1, (B, 1), device=DEV, generator=gen)
        s["labels"] = labels.masked_fill(torch.arange(L, device=DEV) < skip, -100)
        s["logits"].requires_grad_(True)
    return s


# -- the plain forms ----------------------------------------------------------------------------
def _turn(x, cos, sin, rd, pairs):
    y = x.float()
    out = y.clone()
    if pairs == "half":
        a, b = y[..., :rd // 2], y[..., rd // 2:rd]
        out[..., :rd // 2] = a * cos - b * sin
        out[..., rd // 2:rd] = b * cos + a * sin
    else:
        a, b = y[..., 0:rd:2], y[..., 1:rd:2]
        out[..., 0:rd:2] = a * cos - b * sin
        out[..., 1:rd:2] = b * cos + a * sin
    return out.to(x.dtype)


def _rotary(s):
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"]
    cos = (angle.cos() * s["factor"]).float().unsqueeze(2)
    sin = (angle.sin() * s["factor"]).float().unsqueeze(2)
    rd, pairs = s["rd"], s["pairs"]
    q, k = _turn(s["q"], cos, sin, rd, pairs), _turn(s["k"], cos, sin, rd, pairs)
    if s["mode"] == "serve":
        s["q_out"].copy_(q)
        s["k_out"].copy_(k)
        return s["q_out"], s["k_out"]
    return q, k, _turn(s["dq"], cos, -sin, rd, pairs), _turn(s["dk"], cos, -sin, rd, pairs)


def _eight_bits(x):
    """x [..., n] in 32 bits as 8 bits hold it: e4m3 values times the least power of two that brings each group of 32
    to at most 448."""
    n = x.shape[-1]
    pad = -n % GROUP
    g = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, GROUP))
    mant, exp = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = torch.where(mant > 0.875, exp - 8, exp - 9).clamp_(min=-127).float()
    q = (g * torch.exp2(-e)).to(torch.float8_e4m3fn).float()
    return (q * torch.exp2(e)).flatten(-2)[..., :n]


def _pack(s):
    return _eight_bits(s["x"].float()).to(s["x"].dtype)


def _swiglu(s):
    n, dt = s["n"], s["gu"].dtype
    gu = s["gu"].float()
    g, u = gu[:, :n], gu[:, n:]
    z = (g * torch.sigmoid(g) * u).to(dt)
    g, u, dz = _eight_bits(g), _eight_bits(u), s["dz"].float()
    sig = torch.sigmoid(g)
    silu = g * sig
    dg = dz * u * (sig * (1 + g * (1 - sig)))
    return z, torch.cat([dg, dz * silu], -1).to(dt), (silu * u).to(dt)


def _norm(s):
    dt = s["x"].dtype
    # the residual stream is a tensor of its type: the norm and the checkpoint are of what it holds
    h = (s["x"].float() + s["a"].float()).to(dt).float()
    w = s["weight"].float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"])
    y = (h * rstd * w).to(dt)
    xhat = _eight_bits(h) * rstd
    dy = s["dy"].float()
    dxhat = dy * w
    dx = rstd * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True)) + s["dh"].float()
    return h.to(dt), y, dx.to(dt), (dy * xhat).sum(0).to(dt), (xhat * w).to(dt)


def _loss(s):
    logits, labels = s["logits"], s["labels"]
    x = logits[:, :-1].float()
    t = labels[:, 1:]
    keep = t != -100
    count = keep.sum()
    at = t.clamp(min=0).unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    nll = (total.log() + top - x.gather(-1, at)).squeeze(-1)
    loss = (torch.where(keep, nll, 0.0).double().sum() / count).float()
    del x
    p /= total
    p.scatter_add_(-1, at, torch.full_like(at, -1, dtype=p.dtype))
    p *= (keep / count).float().unsqueeze(-1)
    grad = torch.zeros_like(logits)
    grad[:, :-1] = p.to(logits.dtype)
    return loss, grad


_PLAIN = {"rotary": _rotary, "pack": _pack, "swiglu": _swiglu, "norm": _norm, "loss": _loss}


# -- the framework's calls ----------------------------------------------------------------------
def _package():
    at = str(Path.cwd() / "gated-sparse-attention_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import gsa_b200
    return gsa_b200


def _own(s):
    gsa = _package()
    op = s["op"]
    if op == "rotary":
        turn = dict(attention_factor=s["factor"], interleaved=s["pairs"] == "interleaved")
        if s["mode"] == "serve":
            return gsa.apply_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], out=(s["q_out"], s["k_out"]), **turn)
        q, k = gsa.apply_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], **turn)
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return q.detach(), k.detach(), dq, dk
    if op == "pack":
        return gsa.pack_activation(s["x"]).unpack()
    if op == "swiglu":
        z, packed = gsa.ops.silu_mul_packed(s["gu"])
        dgu, z_again = gsa.ops.silu_mul_packed_backward(s["dz"], packed, want_z=True)
        return z, dgu, z_again
    if op == "norm":
        h, y, packed, rstd = gsa.ops.add_rmsnorm_packed(s["x"], s["a"], s["weight"], s["eps"])
        dx, dw, y_again = gsa.ops.rmsnorm_packed_backward(s["dy"], packed, rstd, s["weight"], dh=s["dh"], want_y=True)
        return h, y, dx, dw, y_again
    loss = gsa.fused_next_token_loss(s["logits"], s["labels"])
    grad, = torch.autograd.grad(loss, s["logits"])
    return loss.detach(), grad


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["op"]](state)


# -- work and exact values ----------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotary":
        n = case["B"] * case["L"] * (case["H"] + case["Hk"]) * case["D"]
        turns = case["B"] * case["L"] * (case["H"] + case["Hk"]) * case["rd"]
        passes = 2 if case["mode"] == "train" else 1
        return {"bytes": passes * 2 * n * e + 8 * case["B"] * case["L"], "flops": passes * 3 * turns}
    if case["op"] == "loss":
        n = case["B"] * case["L"] * case["V"]
        return {"bytes": 2 * n * e + 8 * case["B"] * case["L"], "flops": 5 * n}
    n = case["rows"] * case["n"]
    held = 1 + 1 / GROUP  # bytes of a value in 8 bits, written once and read once
    if case["op"] == "pack":
        return {"bytes": n * (2 * e + 2 * held), "flops": 3 * n}
    if case["op"] == "swiglu":  # gu, z out | dz, dgu, z out | (g, u) in 8 bits
        return {"bytes": n * (3 * e + 4 * e + 4 * held), "flops": 20 * n}
    # x, a, h, y | dy, dh, dx, y | the sum in 8 bits
    return {"bytes": n * (8 * e + 2 * held), "flops": 16 * n}


def _round_e4m3(v):
    """v (64 bits, at most 448 in size) to the nearest multiple of its binade's eighth, ties to even."""
    _, ex = torch.frexp(v)
    step = torch.exp2((ex - 1).clamp(min=-6).double() - 3)
    return torch.round(v / step) * step


def _exact_eight(x):
    rows, n = x.shape
    out = torch.zeros(rows, -(-n // GROUP) * GROUP, dtype=torch.float64, device=x.device)
    out[:, :n] = x
    out = out.view(rows, -1, GROUP)
    top = out.abs().amax(-1, keepdim=True)
    # the least e with top <= 448 * 2^e
    e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -127)))
    e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e).clamp(min=-127)
    unit = torch.exp2(e)
    return (_round_e4m3(out / unit) * unit).view(rows, -1)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s)


def _exact_rotary(s):
    B, L = s["B"], s["L"]
    rd, D = s["rd"], s["D"]
    angle = s["positions"].double().view(B, L, 1, 1) * s["inv_freq"]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)  # factor * e^(i angle)

    def go(x, w):
        head, rest = x[..., :rd].double(), x[..., rd:].double()
        if s["pairs"] == "half":
            z = torch.complex(head[..., :rd // 2], head[..., rd // 2:]) * w
            head = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(head.reshape(B, L, -1, rd // 2, 2).contiguous()) * w
            head = torch.view_as_real(z).reshape(B, L, -1, rd)
        return torch.cat([head, rest], -1) if rd < D else head

    out = [go(s["q"], turn), go(s["k"], turn)]
    if s["mode"] == "train":
        out += [go(s["dq"], turn.conj()), go(s["dk"], turn.conj())]
    return tuple(out)


def _exact_pack(s):
    return _exact_eight(s["x"].double())


def _exact_swiglu(s):
    n = s["n"]
    gu, dz = s["gu"].double(), s["dz"].double()
    z = gu[:, :n] / (1 + torch.exp(-gu[:, :n])) * gu[:, n:]
    g, u = _exact_eight(gu[:, :n]), _exact_eight(gu[:, n:])
    up = 1 + torch.exp(-g)
    # d/dg of g / (1 + e^-g)
    slope = 1 / up + g * torch.exp(-g) / up.square()
    return z, torch.cat([dz * u * slope, dz * g / up], -1), g / up * u


def _exact_norm(s):
    h = (s["x"].double() + s["a"].double()).to(s["x"].dtype).double()
    w, n = s["weight"].double(), s["n"]
    size = torch.sqrt(h.square().sum(-1, keepdim=True) / n + s["eps"])
    xhat = _exact_eight(h) / size
    dy = s["dy"].double()
    along = (dy * w * xhat).sum(-1, keepdim=True) / n
    dx = (dy * w - xhat * along) / size + s["dh"].double()
    return h, h / size * w, dx, (dy * xhat).sum(0), xhat * w


def _exact_loss(s):
    logits, labels = s["logits"].detach(), s["labels"]
    B, L, V = logits.shape
    count = int((labels[:, 1:] != -100).sum())
    grad = torch.zeros(B, L, V, dtype=torch.float64, device=DEV)
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for b in range(B):
        for i in range(0, L - 1, 1024):
            j = min(L - 1, i + 1024)
            t = labels[b, i + 1:j + 1]
            keep = t != -100
            logp = torch.log_softmax(logits[b, i:j].double(), -1)
            total -= logp[torch.arange(j - i, device=DEV), t.clamp(min=0)][keep].sum()
            g = logp.exp()
            g[torch.arange(j - i, device=DEV), t.clamp(min=0)] -= 1
            grad[b, i:j] = g * (keep.double() / count).unsqueeze(-1)
    return total / count, grad


_EXACT = {"rotary": _exact_rotary, "pack": _exact_pack, "swiglu": _exact_swiglu, "norm": _exact_norm,
          "loss": _exact_loss}
