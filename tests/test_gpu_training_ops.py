"""The training-step operators (rotary positions, activations in 8 bits with the norm and SwiGLU that use them, the
next-token loss) against their formulas in 64 bits.

Tolerances count roundings: an output of type t is off by at most half a step of it (eps/2 of its size) plus what the 32-bit
arithmetic before that rounding loses (each test derives it).  Packed values are compared for equality: the
scale is a power of two, so the one rounding of a value is the same in any arithmetic."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=_gen(seed)) * scale).to(dtype)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _near(got, want, slack, what=""):
    """|got - want| <= half a step of got's type at want + slack (a tensor or number), elementwise."""
    bound = _half_step(got.dtype) * (want.abs() + slack) + slack + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs() - bound
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert not bool(torch.isnan(off).any()) and float(off.max() if off.numel() else 0) <= 0, (
        what, float(off.max()), int(off.argmax()))


# -- rotary -------------------------------------------------------------------------------------
def _rotary_oracle(x, positions, freq, factor, interleaved, inverse=False):
    """x [B, L, H, D] turned in 64 bits, and |x0| + |x1| of each value's pair."""
    rd = 2 * freq.numel()
    ang = positions.double().view(-1, x.shape[1], 1, 1) * freq
    c, s = factor * ang.cos(), factor * ang.sin() * (-1 if inverse else 1)
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    i = torch.arange(rd // 2, device=x.device)
    i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
    x0, x1 = x.double()[..., i0], x.double()[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    size[..., i0] = size[..., i1] = x0.abs() + x1.abs()
    return y, size


ROTARY = [
    # B, L, H, Hk, D, rd, interleaved
    (1, 1, 1, 1, 2, 2, False),
    (64, 1, 32, 8, 128, 128, False),
    (2, 77, 8, 2, 64, 64, False),
    (2, 19, 6, 2, 80, 40, False),
    (2, 300, 4, 1, 96, 24, True),
    (2, 33, 32, 8, 128, 64, True),
    (3, 19, 9, 3, 80, 80, False),
    (3, 19, 9, 3, 80, 20, True),
    (1, 65, 5, 1, 96, 34, False),
    (1, 7, 3, 1, 10, 6, True),
    (1, 5, 2, 2, 33, 2, False),
    (1, 40, 16, 16, 256, 256, True),
    (1, 3, 1000, 24, 16, 16, False),
    (1, 3, 2, 1, 1024, 1024, False),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,Hk,D,rd,interleaved", ROTARY)
def test_rotary_forward_and_backward(cuda_ok, dtype, B, L, H, Hk, D, rd, interleaved):
    import gsa_b200 as gsa

    q, k = _randn(1, B, L, H, D, dtype=dtype), _randn(2, B, L, Hk, D, dtype=dtype)
    pos = torch.randint(0, 1 << 20, (B, L), device=DEV, generator=_gen(3))
    freq, factor = gsa.rotary_frequencies(rd, scaling=dict(type="linear", factor=2.0, attention_factor=1.25),
                                          device=DEV)
    q.requires_grad_(True)
    k.requires_grad_(True)
    q2, k2 = gsa.apply_rotary(q, k, pos, freq, factor, interleaved)
    dq, dk = _randn(4, B, L, H, D, dtype=dtype), _randn(5, B, L, Hk, D, dtype=dtype)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk))
    # sine and cosine of a 32-bit fraction of a turn: pi U each from the fraction's rounding, 2 steps from the function,
    # the product with the factor, a product and a sum: under 12 U of factor (|x0| + |x1|)
    for got, x, inv in ((q2, q, False), (k2, k, False), (gq, dq, True), (gk, dk, True)):
        want, size = _rotary_oracle(x.detach(), pos, freq, factor, interleaved, inv)
        _near(got.detach(), want, 12 * U * factor * size)
    # the pass-through part is copied bit for bit
    assert torch.equal(q2.detach()[..., rd:], q.detach()[..., rd:])


def test_rotary_gradient_is_that_of_differences(cuda_ok):
    """<R x, g> differenced in x against the backward pass: R is linear, so any step gives it, to 32-bit rounding."""
    import gsa_b200 as gsa

    q = _randn(1, 1, 6, 2, 16).requires_grad_(True)
    freq, _ = gsa.rotary_frequencies(8, device=DEV)
    pos = torch.arange(6, device=DEV) * 1000
    g = _randn(2, 1, 6, 2, 16)
    y, _ = gsa.apply_rotary(q, None, pos, freq, interleaved=True)
    (grad,) = torch.autograd.grad(y, q, g)
    v = _randn(3, 1, 6, 2, 16)
    with torch.no_grad():
        up = gsa.apply_rotary(q + v, None, pos, freq, interleaved=True)[0].double()
        down = gsa.apply_rotary(q - v, None, pos, freq, interleaved=True)[0].double()
    diff = float(((up - down) / 2 * g.double()).sum())
    # 192 terms, each of size about 1, off by under 16 U
    assert abs(diff - float((grad.double() * v.double()).sum())) < 192 * 16 * U * 8


def test_rotary_layouts_strides_and_outputs(cuda_ok):
    """Slices of a fused projection, [B, H, L, D] storage, shared and int32 positions, cache slots, in place, only q,
    a gradient for one of the two, expanded gradients."""
    import gsa_b200 as gsa

    B, L, H, Hk, D = 2, 21, 4, 2, 64
    freq, _ = gsa.rotary_frequencies(D, device=DEV)
    pos = torch.randint(0, 4096, (L,), device=DEV, generator=_gen(1))
    proj = _randn(2, B, L, (H + 2 * Hk) * D + 3, dtype=torch.bfloat16)
    q = proj[..., 1:1 + H * D].view(B, L, H, D)      # rows at odd element offsets
    k = proj[..., 1 + H * D:1 + (H + Hk) * D].view(B, L, Hk, D)
    want_q, _ = gsa.apply_rotary(q.contiguous(), None, pos, freq)
    want_k, _ = gsa.apply_rotary(k.contiguous(), None, pos, freq)
    got = gsa.apply_rotary(q, k, pos.int(), freq)
    assert torch.equal(got[0], want_q) and torch.equal(got[1], want_k)
    # heads before tokens in memory, and a stride between values
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(gsa.apply_rotary(qt, k, pos.view(1, L), freq)[0], want_q)
    wide = torch.empty(B, L, H, 2 * D, device=DEV, dtype=torch.bfloat16)
    wide[..., ::2] = q
    assert torch.equal(gsa.apply_rotary(wide[..., ::2], None, pos, freq)[0], want_q)
    # K into the slots of a cache, its neighbours left as they were
    kv = torch.full((B, L + 9, 2, Hk, D), 7.0, device=DEV, dtype=torch.bfloat16)
    slot = kv[:, 4:4 + L, 0]
    out = gsa.apply_rotary(q, k, pos, freq, out=(torch.empty_like(want_q), slot))
    assert out[1].data_ptr() == slot.data_ptr() and torch.equal(slot, want_k)
    assert bool((kv[:, :4] == 7).all() and (kv[:, 4 + L:] == 7).all() and (kv[:, :, 1] == 7).all())
    # in place, inside the projection
    keep = proj.clone()
    gsa.apply_rotary(q, k, pos, freq, out=(q, k))
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(proj[..., (H + Hk) * D + 1:], keep[..., (H + Hk) * D + 1:])
    assert torch.equal(proj[..., 0], keep[..., 0])
    # in place with a part of the head: the rest is not written
    half, _ = gsa.rotary_frequencies(16, device=DEV)
    x = _randn(5, 1, 3, 2, D)
    y = gsa.apply_rotary(x, None, pos[:3], half)[0]
    gsa.apply_rotary(x, None, pos[:3], half, out=(x, None))
    assert torch.equal(x, y)
    # gradients: k alone, and an expanded one
    q32, k32 = _randn(6, B, L, H, D).requires_grad_(True), _randn(7, B, L, Hk, D).requires_grad_(True)
    q2, k2 = gsa.apply_rotary(q32, k32, pos, freq)
    (gk,) = torch.autograd.grad(k2.sum(), k32, retain_graph=True)
    want, size = _rotary_oracle(torch.ones_like(k32), pos.view(1, L), freq, 1.0, False, True)
    _near(gk, want, 12 * U * size)
    gq, gk2 = torch.autograd.grad(q2.sum(), (q32, k32), allow_unused=True)
    assert gk2 is None and bool(torch.isfinite(gq).all())
    # a broadcast head: its gradient is the sum over the places it stands in
    one = _randn(8, B, L, 1, D).requires_grad_(True)
    y = gsa.apply_rotary(one.expand(B, L, H, D), None, pos, freq)[0]
    g = _randn(9, B, L, H, D)
    (g1,) = torch.autograd.grad(y, one, g)
    want, size = _rotary_oracle(g, pos.view(1, L), freq, 1.0, False, True)
    _near(g1, want.sum(2, keepdim=True), (12 + H) * U * size.sum(2, keepdim=True))


def test_rotary_far_positions_and_tables(cuda_ok):
    """Positions past 2^31 keep their angle; the tables of RotaryEmbedding give torch's bits for its transpose; a position
    outside the tables is reported and gives NaN."""
    import gsa_b200 as gsa
    from gsa_b200 import _lib, ops
    from gsa_b200.attention import _rope_backward

    freq, _ = gsa.rotary_frequencies(64, device=DEV)
    x = _randn(1, 1, 8, 3, 64)
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 31) + 5, 1 << 33, -3, 12345678901], device=DEV).view(1, 8)
    y, _ = gsa.apply_rotary(x, None, pos, freq)
    want, size = _rotary_oracle(x, pos, freq, 1.0, False)
    # the 64-bit angle itself is off by up to p 2^-53 on either side: 2^34 2^-52 = 2^-18 for the largest
    _near(y, want, size * (12 * U + 2.0 ** -52 * pos.abs().double().view(1, 8, 1, 1)))
    for dt in (torch.float32, torch.bfloat16):
        emb = gsa.RotaryEmbedding(64, 512).to(DEV).to(dt)
        p = torch.randint(0, 512, (2, 8), device=DEV, generator=_gen(4))
        dy = _randn(5, 2, 8, 3, 64)
        want = _rope_backward(dy.view(16, 3, 64), emb.cos_cached[p.view(-1)], emb.sin_cached[p.view(-1)])
        got, _ = ops.rotary(dy, None, p, tables=(emb.cos_cached, emb.sin_cached), rotary_dim=64, inverse=True)
        assert torch.equal(got.view(16, 3, 64), want)
    p[1, 3] = 512
    got, _ = ops.rotary(dy, None, p, tables=(emb.cos_cached, emb.sin_cached), rotary_dim=64)
    assert bool(torch.isnan(got[1, 3]).all()) and not bool(torch.isnan(got[0]).any())
    with pytest.raises(_lib.GSAError):
        ops.check_device_error()
    ops.check_device_error()


def test_rotary_empty_inputs(cuda_ok):
    import gsa_b200 as gsa

    freq, _ = gsa.rotary_frequencies(8, device=DEV)
    for B, L in ((0, 5), (2, 0)):
        q = torch.empty(B, L, 2, 8, device=DEV)
        y, k = gsa.apply_rotary(q, q, torch.zeros(B, L, device=DEV, dtype=torch.long), freq)
        assert y.shape == q.shape and k.shape == q.shape


# -- 8 bits -------------------------------------------------------------------------------------
def _eight(x):
    """x [..., n] (64 bits) as 8 bits hold it, by the definition: per group of 32 the least e >= -127 with
    max finite |x| <= 448 2^e, each value to the nearest of e4m3's multiples (ties to even); NaN for NaN and inf."""
    n = x.shape[-1]
    g = torch.nn.functional.pad(x, (0, -n % 32)).unflatten(-1, (-1, 32))
    top = torch.where(torch.isfinite(g), g.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for cand in range(120, -128, -1):  # the last candidate that still holds the group is the least
        e = torch.where(top <= 448 * 2.0 ** cand, torch.full_like(e, cand), e)
    v = g / torch.exp2(e)
    ex = torch.frexp(torch.where(torch.isfinite(v), v, 0.0))[1] - 1
    step = torch.exp2(ex.clamp(min=-6).double() - 3)
    q = torch.where(torch.isfinite(v), torch.round(v / step) * step, math.nan) * torch.exp2(e)
    return q.flatten(-2)[..., :n], e.squeeze(-1)


def _same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (5, 31), (4, 32), (3, 33), (2, 7, 48), (3, 1000), (17, 4096), (2, 11008), (1000, 16),
                                   (7, 160), (9,)])
def test_pack_and_unpack_are_the_definition(cuda_ok, dtype, shape):
    import gsa_b200 as gsa

    x = (_randn(1, *shape) * torch.exp(_randn(2, *shape) * 6)).to(dtype)
    p = gsa.pack_activation(x)
    want, e = _eight(x.double())
    got = p.unpack()
    assert got.dtype == dtype and got.shape == x.shape
    assert torch.equal(p.unpack(torch.float32).double(), want)
    assert torch.equal(p.scales.view(e.shape).double() - 127, e)
    n = shape[-1]
    assert p.nbytes == x.numel() // n * ((n + 15) // 16 * 16 + (n + 31) // 32)
    # what 8 bits promise: within 2^-4 of the value, or 2^-17 of the group's largest (half a step of 2^-9 2^e against more than 224 2^e)
    big = torch.nn.functional.pad(x.double().abs(), (0, -n % 32)).unflatten(-1, (-1, 32))
    big = big.amax(-1, keepdim=True).expand_as(big).flatten(-2)[..., :n]
    assert bool(((want - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, big * 2.0 ** -17)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 37])
def test_pack_special_values(cuda_ok, dtype, n):
    """Zeros, the type's smallest and largest numbers, NaN and infinities beside ordinary values, ties, borders
    of the scale."""
    import gsa_b200 as gsa

    rows = []
    fi = torch.finfo(dtype)
    for fill in ([0.0], [-0.0], [fi.max], [fi.max, fi.tiny], [fi.tiny], [fi.smallest_normal / 64], [448.0, 2.0 ** -10, 2.0 ** -11],
                 [449.0, 1.0], [450.0, 17.0, 18.0, 19.0, 21.0], [1.75, 1.0625, 1.1875], [1.7578125, 1.0625],
                 [math.nan, 1.0], [math.inf, 1.0, 3.0], [-math.inf, math.nan], [math.nan], [2.0 ** -120, 2.0 ** -126],
                 [-3.5, 2.0 ** -9 * 3.5, 2.0 ** -16 * 3.5, 2.0 ** -20]):
        rows.append([fill[i % len(fill)] for i in range(n)])
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).to(DEV)
    got = gsa.pack_activation(x).unpack(torch.float32).double()
    # the packed value of the largest numbers is 256 * 2^120 = 2^128, which fp32 holds as infinity
    want = _eight(x.double())[0].float().double()
    assert _same(got, want), (got - want).abs().max()


def test_pack_strided_and_empty(cuda_ok):
    import gsa_b200 as gsa

    base = _randn(1, 12, 200, dtype=torch.bfloat16)
    for x in (base[:, 3:99], base[::2, :96], base.t(), base[:, ::2], base[:1].expand(5, 200), base[:, :64].unflatten(1, (2, 32))):
        assert torch.equal(gsa.pack_activation(x).unpack(), gsa.pack_activation(x.contiguous()).unpack())
    for shape in ((0, 64), (4, 0), (2, 0, 32)):
        p = gsa.pack_activation(torch.empty(shape, device=DEV))
        assert p.unpack().shape == torch.Size(shape) and p.nbytes == 0


ROWS = [(1, 1), (3, 16), (2, 31), (5, 33), (192, 512), (7, 1376), (1, 4096), (33, 1000), (3, 11008), (300, 48)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", ROWS)
def test_swiglu_forward_and_backward(cuda_ok, dtype, rows, n):
    import gsa_b200 as gsa

    gu = _randn(1, rows, 2 * n, dtype=dtype, scale=2.0)
    dz = _randn(2, rows, n, dtype=dtype)
    z, p = gsa.ops.silu_mul_packed(gu)
    g, u = gu.double()[:, :n], gu.double()[:, n:]
    # the sigmoid is off by 8 U of itself (exp 2 steps, sum, reciprocal), each product by U
    _near(z, g * torch.sigmoid(g) * u, 12 * U * (g * u).abs())
    want, _ = _eight(gu.double().view(rows, 2, n))
    assert torch.equal(p.unpack(torch.float32).double(), want)
    dgu, z2 = gsa.ops.silu_mul_packed_backward(dz, p, want_z=True)
    g, u, d = want[:, 0], want[:, 1], dz.double()
    sig = torch.sigmoid(g)
    size = (d * u).abs() * sig * (1 + g.abs())
    _near(dgu[:, :n], d * u * sig * (1 + g * (1 - sig)), 24 * U * size)
    _near(dgu[:, n:], d * g * sig, 12 * U * (d * g).abs())
    _near(z2, g * sig * u, 12 * U * (g * u).abs())
    none = gsa.ops.silu_mul_packed_backward(dz, p)
    assert none[1] is None and torch.equal(none[0], dgu)
    # through autograd
    leaf = gu.clone().requires_grad_(True)
    y = gsa.packed_silu_mul(leaf)
    (grad,) = torch.autograd.grad(y, leaf, dz)
    assert torch.equal(y.detach(), z) and torch.equal(grad, dgu) and torch.equal(gsa.packed_silu_mul(gu), z)


def test_swiglu_gradient_is_that_of_differences(cuda_ok):
    """At values that 8 bits hold exactly, central differences of the 64-bit formula along a direction."""
    import gsa_b200 as gsa

    gu = _eight(_randn(1, 4, 96).double())[0]
    v, dz = _randn(2, 4, 96).double(), _randn(3, 4, 48)

    def f(x):
        return (torch.nn.functional.silu(x[:, :48]) * x[:, 48:] * dz.double()).sum()

    h = 1e-6
    diff = float((f(gu + h * v) - f(gu - h * v)) / (2 * h))
    leaf = gu.float().requires_grad_(True)
    gsa.packed_silu_mul(leaf).backward(dz)
    # 384 terms of size about 1 at 32 U, and h^2 of the third derivative
    assert abs(float((leaf.grad.double() * v).sum()) - diff) < 384 * 32 * U + 1e-8


def test_swiglu_extreme_gates(cuda_ok):
    """Gates far out (sigmoid 0 or 1), infinite and NaN ones."""
    import gsa_b200 as gsa

    g = torch.tensor([-1e30, -200.0, -88.0, 88.0, 200.0, 1e30, 0.0, -0.0], device=DEV).repeat(4)
    gu = torch.cat([g, torch.ones(32, device=DEV)]).view(1, 64)
    z, p = gsa.ops.silu_mul_packed(gu)
    want = torch.nn.functional.silu(g.double())
    _near(z[0], want, 12 * U * want.abs())
    dgu, z2 = gsa.ops.silu_mul_packed_backward(torch.ones(1, 32, device=DEV), p, want_z=True)
    assert bool(torch.isfinite(dgu).all() and torch.isfinite(z2).all())
    gu[0, 3], gu[0, 40] = math.nan, math.inf
    z, p = gsa.ops.silu_mul_packed(gu)
    dgu, _ = gsa.ops.silu_mul_packed_backward(torch.ones(1, 32, device=DEV), p)
    assert bool(torch.isnan(z[0, 3])) and bool(torch.isnan(dgu[0, 3])) and bool(torch.isnan(dgu[0, 8]))
    assert int(torch.isnan(dgu).sum()) <= 4  # and in no other column


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("add", [True, False])
@pytest.mark.parametrize("rows,d", ROWS + [(2, 16384), (1, 20000), (700, 256), (5, 4112), (2000, 8)])
def test_norm_forward_and_backward(cuda_ok, dtype, add, rows, d):
    import gsa_b200 as gsa

    x = _randn(1, rows, d, dtype=dtype, scale=2.0)
    a = _randn(2, rows, d, dtype=dtype) if add else None
    w = (1 + 0.2 * _randn(3, d)).to(dtype)
    eps = 1e-5
    h, y, p, rstd = gsa.ops.add_rmsnorm_packed(x, a, w, eps)
    hd = (x.double() + a.double()).to(dtype).double() if add else x.double()
    assert (h is None) == (not add) and (h is None or torch.equal(h.double(), hd))
    # a sum of d squares in 32 bits: at most d / 32 + 16 additions follow one another in any lane and the tree
    lose = (d / 32 + 16) * U
    r = 1 / torch.sqrt(hd.square().mean(-1, keepdim=True) + eps)
    assert float((rstd.double() / r.view(-1) - 1).abs().max()) <= lose + 8 * U
    wd = w.double()
    want = hd * r * wd
    _near(y, want, (lose + 12 * U) * want.abs())
    held, _ = _eight(hd)
    assert torch.equal(p.unpack(torch.float32).double(), held)
    dy, dh = _randn(4, rows, d, dtype=dtype), _randn(5, rows, d, dtype=dtype)
    xh = held * r
    for extra in (dh, None):
        dx, dw, y2 = gsa.ops.rmsnorm_packed_backward(dy, p, rstd, w, dh=extra, want_y=extra is not None)
        dyw = dy.double() * wd
        along = (dyw * xh).mean(-1, keepdim=True)
        ref = r * (dyw - xh * along)
        size = r * (dyw.abs() + xh.abs() * (dyw * xh).abs().mean(-1, keepdim=True))
        if extra is not None:
            ref, size = ref + extra.double(), size + extra.double().abs()
        _near(dx, ref, (3 * lose + 24 * U) * size, "dx")
        _near(dw, (dy.double() * xh).sum(0), (rows + 16 + lose / U) * U * (dy.double() * xh).abs().sum(0), "dw")
        if extra is not None:
            _near(y2, xh * wd, (lose + 12 * U) * (xh * wd).abs(), "y")
    assert y2 is None
    assert gsa.ops.rmsnorm_packed_backward(dy, p, rstd, w, want_dw=False)[1] is None
    # the same sums in the same order every time
    again = gsa.ops.rmsnorm_packed_backward(dy, p, rstd, w)
    assert torch.equal(again[1], dw) and torch.equal(again[0], dx)


def test_norm_autograd_and_differences(cuda_ok):
    """packed_add_rmsnorm under autograd at values that 8 bits hold exactly, against central differences of the
    64-bit formula; h's own gradient, unused outputs, no addend."""
    import gsa_b200 as gsa

    x = _eight(_randn(1, 3, 64).double())[0]
    w = 1 + 0.1 * _randn(2, 64)
    gy, gh = _randn(3, 3, 64), _randn(4, 3, 64)
    zero = torch.zeros(3, 64, device=DEV)

    def f(x, w):
        return (x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w * gy.double()).sum() + (x * gh.double()).sum()

    lx, la, lw = x.float().requires_grad_(True), zero.requires_grad_(True), w.clone().requires_grad_(True)
    h, y = gsa.packed_add_rmsnorm(lx, la, lw, 1e-5)
    torch.autograd.backward((h, y), (gh, gy))
    assert torch.equal(lx.grad, la.grad)
    vx, vw, e = _randn(5, 3, 64).double(), _randn(6, 64).double(), 1e-6
    diff = float((f(x + e * vx, w.double() + e * vw) - f(x - e * vx, w.double() - e * vw)) / (2 * e))
    got = float((lx.grad.double() * vx).sum() + (lw.grad.double() * vw).sum())
    assert abs(got - diff) < 400 * 64 * U + 1e-7
    # y alone, h alone, and x alone without an addend
    h, y = gsa.packed_add_rmsnorm(lx, la, lw, 1e-5)
    g1 = torch.autograd.grad(y, lx, gy, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(h, lx, gh)[0], gh)
    h, y = gsa.packed_add_rmsnorm(lx, None, lw, 1e-5)
    assert h is lx and torch.equal(torch.autograd.grad(y, lx, gy)[0], g1)


def test_norm_special_rows(cuda_ok):
    """Rows of zeros, of one huge value, with NaN, strided rows, a broadcast row, no rows."""
    import gsa_b200 as gsa

    d = 96
    x = torch.zeros(5, d, device=DEV)
    x[1, 7] = 1e18
    x[2, 3] = math.nan
    x[3] = _randn(1, d)
    w = torch.ones(d, device=DEV)
    h, y, p, rstd = gsa.ops.add_rmsnorm_packed(x, torch.zeros_like(x), w, 1e-5)
    assert bool((y[0] == 0).all()) and abs(float(rstd[0]) - 1e-5 ** -0.5) < 1e-3
    assert abs(float(y[1, 7]) - math.sqrt(d)) < 1e-3 and bool(torch.isnan(y[2]).all())
    dx, dw, _ = gsa.ops.rmsnorm_packed_backward(torch.ones_like(x), p, rstd, w)
    assert bool(torch.isfinite(dx[[0, 1, 3, 4]]).all()) and bool(torch.isnan(dx[2]).all())
    base = _randn(2, 6, 2 * d + 1, dtype=torch.bfloat16)
    wb = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    xs, as_ = base[:, 1:1 + d], base[:1, d:2 * d].expand(6, d)
    for got, want in zip(gsa.ops.add_rmsnorm_packed(xs, as_, wb, 1e-5)[:2],
                         gsa.ops.add_rmsnorm_packed(xs.contiguous(), as_.contiguous(), wb, 1e-5)[:2]):
        assert torch.equal(got, want)
    empty = torch.empty(0, d, device=DEV)
    h, y, p, rstd = gsa.ops.add_rmsnorm_packed(empty, empty, w, 1e-5)
    dx, dw, _ = gsa.ops.rmsnorm_packed_backward(empty, p, rstd, w)
    assert y.shape == (0, d) and bool((dw == 0).all())


# -- loss ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 7, 15, 17, 31, 33, 95, 250, 511, 513, 1003, 8193, 16381])
def test_rows_at_any_offset(cuda_ok, dtype, n):
    """Rows that start at every offset within 32 bytes, NaN around them, give the bits of contiguous ones; outputs
    with gaps between their rows leave the gaps, and what lies before and behind, as they were."""
    import gsa_b200 as gsa
    from gsa_b200 import _lib

    ops, lib, rows, guard = gsa.ops, _lib.lib(), 3, 7777.0

    def spread(t, off, gap):
        """t's rows at that element offset and distance in storage of NaN."""
        ld = t.shape[-1] + gap
        v = torch.full((off + t.shape[0] * ld + 64,), math.nan, device=DEV, dtype=dtype).as_strided(t.shape, (ld, 1), off)
        return v.copy_(t)

    def holes(width, off, ld):
        """An output for rows of that width, and what tells whether the rest of its storage is as it was."""
        base = torch.full((off + rows * ld + 64,), guard, device=DEV, dtype=dtype)
        out = base.as_strided((rows, width), (ld, 1), off)
        return out, lambda: bool((base.as_strided((rows, ld - width), (ld, 1), off + width) == guard).all()) and bool(
            (base[:off] == guard).all()) and bool((base[off + rows * ld:] == guard).all())

    x, a, dh = (_randn(i, rows, n, dtype=dtype) for i in (1, 2, 3))
    gu, w = _randn(4, rows, 2 * n, dtype=dtype), _randn(5, 1, n, dtype=dtype)
    want_p = ops.pack_e4m3(x)
    want_x = ops.unpack_e4m3(want_p)
    want_z, pgu = ops.silu_mul_packed(gu)
    want_dgu, want_z2 = ops.silu_mul_packed_backward(x, pgu, want_z=True)
    want_h, want_y, ph, rstd = ops.add_rmsnorm_packed(x, a, w[0], 1e-5)
    want_dx, want_dw, want_y2 = ops.rmsnorm_packed_backward(x, ph, rstd, w[0], dh=dh, want_y=True)
    t = _lib.DTYPE_BF16 if dtype is torch.bfloat16 else _lib.DTYPE_F32
    stream = torch.cuda.current_stream().cuda_stream
    c_ld, s_ld = (n + 15) // 16 * 16, (n + 31) // 32
    for off in range(32 // x.element_size()):
        xs, as_, dhs, gus, ws = (spread(v, off, gap) for v, gap in ((x, 3), (a, 1), (dh, 2), (gu, 5), (w, 0)))
        p = ops.pack_e4m3(xs)
        assert torch.equal(p.scales, want_p.scales)
        assert torch.equal(p.codes.view(torch.uint8)[:, :n], want_p.codes.view(torch.uint8)[:, :n])
        z, q = ops.silu_mul_packed(gus)
        assert torch.equal(z, want_z) and torch.equal(q.unpack(), pgu.unpack())
        dgu, z = ops.silu_mul_packed_backward(xs, pgu, want_z=True)
        assert torch.equal(dgu, want_dgu) and torch.equal(z, want_z2)
        h, y, q, r = ops.add_rmsnorm_packed(xs, as_, ws[0], 1e-5)
        assert torch.equal(h, want_h) and torch.equal(y, want_y) and torch.equal(q.unpack(), ph.unpack())
        assert torch.equal(r, rstd)
        dx, dw, y = ops.rmsnorm_packed_backward(xs, ph, rstd, ws[0], dh=dhs, want_y=True)
        assert torch.equal(dx, want_dx) and torch.equal(dw, want_dw) and torch.equal(y, want_y2)
        # outputs at that offset, by the C entries
        ld = n + 5
        out, kept = holes(n, off, ld)
        codes, scales = want_p.codes.data_ptr(), want_p.scales.data_ptr()
        assert lib.gsa_unpack_e4m3(t, rows, n, codes, c_ld, scales, s_ld, out.data_ptr(), ld, stream) == 0
        assert torch.equal(out, want_x) and kept()
        out, kept = holes(n, off, ld)
        q = gsa.PackedActivation.empty((rows, 2, n), dtype, DEV)
        qc, qs = q.codes.data_ptr(), q.scales.data_ptr()
        assert lib.gsa_silu_mul_pack(t, rows, n, gu.data_ptr(), 2 * n, out.data_ptr(), ld, qc, c_ld, qs, s_ld, stream) == 0
        assert torch.equal(out, want_z) and torch.equal(q.unpack(), pgu.unpack()) and kept()
        out, kept = holes(2 * n, off, ld + n)
        out2, kept2 = holes(n, off, ld)
        assert lib.gsa_silu_mul_packed_backward(t, rows, n, x.data_ptr(), n, pgu.codes.data_ptr(), c_ld, pgu.scales.data_ptr(),
                                                s_ld, out.data_ptr(), ld + n, out2.data_ptr(), ld, stream) == 0
        assert torch.equal(out.reshape(want_dgu.shape), want_dgu) and torch.equal(out2, want_z2) and kept() and kept2()
        out, kept = holes(n, off, ld)
        out2, kept2 = holes(n, off, ld)
        q, r = gsa.PackedActivation.empty((rows, n), dtype, DEV), torch.empty(rows, device=DEV)
        assert lib.gsa_add_rmsnorm_pack(t, rows, n, x.data_ptr(), n, a.data_ptr(), n, w.data_ptr(), 1e-5, out.data_ptr(), ld,
                                        out2.data_ptr(), ld, q.codes.data_ptr(), c_ld, q.scales.data_ptr(), s_ld,
                                        r.data_ptr(), stream) == 0
        assert torch.equal(out, want_h) and torch.equal(out2, want_y) and torch.equal(r, rstd) and kept() and kept2()
        out, kept = holes(n, off, ld)
        out2, kept2 = holes(n, off, ld)
        assert lib.gsa_rmsnorm_packed_backward(t, rows, n, x.data_ptr(), n, dh.data_ptr(), n, w.data_ptr(), ph.codes.data_ptr(),
                                               c_ld, ph.scales.data_ptr(), s_ld, rstd.data_ptr(), out.data_ptr(), ld,
                                               out2.data_ptr(), ld, None, None, 0, stream) == 0
        assert torch.equal(out, want_dx) and torch.equal(out2, want_y2) and kept() and kept2()


def _loss_oracle(logits, labels, ignore=-100):
    x = logits.double()[:, :-1]
    t = labels[:, 1:]
    keep = t != ignore
    logp = torch.log_softmax(x, -1)
    at = t.clamp(min=0).unsqueeze(-1)
    nll = torch.where(keep, -logp.gather(-1, at).squeeze(-1), 0.0)
    count = keep.sum()
    p = logp.exp()
    grad = torch.zeros_like(logits, dtype=torch.float64)
    grad[:, :-1] = torch.where(keep.unsqueeze(-1), (p - torch.zeros_like(p).scatter(-1, at, 1.0)) / count, 0.0)
    size = torch.zeros_like(grad)  # |softmax| / count + onehot / count, with the distance from the row's largest
    size[:, :-1] = (p + torch.zeros_like(p).scatter(-1, at, 1.0)) / count
    far = (x.amax(-1, keepdim=True) - x).clamp(max=200.0)
    loss_size = torch.where(keep, x.abs().amax(-1) + nll.abs(), 0.0).sum() / count
    return nll.sum() / count, grad, size, torch.nn.functional.pad(far, (0, 0, 0, 1)), loss_size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,V", [(1, 2, 1), (1, 2, 2), (3, 700, 9), (2, 300, 64), (1, 50, 257), (4, 9, 2047), (2, 96, 384), (3, 17, 1000), (1, 33, 4097), (2, 5, 128256), (1, 600, 31),
                                   (1, 3, 32768), (700, 2, 8), (1, 9, 50257), (2, 200, 32768), (1, 3, 20000),
                                   (1, 150, 65544), (1, 3, 131072), (1, 2, 262152)])
def test_loss_and_gradient(cuda_ok, dtype, B, L, V):
    import gsa_b200 as gsa

    logits = _randn(1, B, L, V, dtype=dtype, scale=3.0)
    labels = torch.randint(0, V, (B, L), device=DEV, generator=_gen(2))
    labels[torch.rand(B, L, device=DEV, generator=_gen(3)) < 0.3] = -100
    labels[0, 1] = V - 1
    loss, grad = gsa.ops.next_token_loss(logits, labels)
    want, g, size, far, loss_size = _loss_oracle(logits, labels)
    # sum of V exponentials, at most V / 32 + 16 additions after one another; each exponential off by 4 U and by U of its
    # argument; the loss a difference of numbers of the logits' size
    lose = (V / 32 + 32) * U
    _near(loss, want, (lose + 8 * U) * (1 + loss_size))
    _near(grad, g, size * (lose + (far + 16) * U))
    leaf = logits.clone().requires_grad_(True)
    out = gsa.fused_next_token_loss(leaf, labels)
    out.backward()
    assert torch.equal(out.detach(), loss) and torch.equal(leaf.grad, grad)
    assert torch.equal(gsa.fused_next_token_loss(logits, labels), loss)
    # a scaled loss scales the gradient (by a power of two: exactly)
    leaf.grad = None
    (gsa.fused_next_token_loss(leaf, labels) * 0.25).backward()
    assert torch.equal(leaf.grad, (grad.float() * 0.25).to(dtype))


def test_loss_gradient_is_that_of_differences(cuda_ok):
    import gsa_b200 as gsa

    logits, labels = _randn(1, 2, 5, 40), torch.randint(0, 40, (2, 5), device=DEV, generator=_gen(2))
    v, e = _randn(3, 2, 5, 40).double(), 1e-6
    up, down = _loss_oracle(logits.double() + e * v, labels)[0], _loss_oracle(logits.double() - e * v, labels)[0]
    _, grad = gsa.ops.next_token_loss(logits, labels)
    assert abs(float((grad.double() * v).sum() - (up - down) / (2 * e))) < 400 * 16 * U


@pytest.mark.parametrize("V", [70, 500, 3000, 4099, 32768, 65536, 128256])
def test_loss_special_rows(cuda_ok, V):
    """Masked (-inf) logits, a target among them, large and equal logits, rows that do not count, no row that counts, another
    ignore_index, a label out of range, NaN."""
    import gsa_b200 as gsa
    from gsa_b200 import _lib, ops

    x = _randn(1, 1, 6, V)
    x[0, 0, 5:60] = -math.inf
    x[0, 1] = 1000.0
    x[0, 2] = -1000.0
    x[0, 3, 1:] = torch.finfo(torch.float32).min
    labels = torch.tensor([[9, 2, 3, 4, 0, 64]], device=DEV)
    want, g, size, far, loss_size = _loss_oracle(x, labels)
    loss, grad = ops.next_token_loss(x, labels)
    # a sum of V terms (V / 32 additions after one another at most), and 2^(x log2 e - M) at |x| of 1000: 256 U
    _near(loss, want, (V / 32 + 64) * U * (1 + loss_size))
    _near(grad, g, size * (V / 32 + 256) * U)
    assert bool((grad[0, 0, 5:60] == 0).all()) and bool((grad[0, 5] == 0).all())
    # the target itself masked: an infinite loss, a finite gradient
    hit = labels.clone()
    hit[0, 1] = 30
    loss, grad = ops.next_token_loss(x, hit)
    assert float(loss) == math.inf and bool(torch.isfinite(grad).all())
    # nothing counts
    for lab, ign in ((torch.full_like(labels, -100), -100), (torch.full_like(labels, 7), 7)):
        loss, grad = ops.next_token_loss(x, lab, ign)
        assert bool(torch.isnan(loss)) and bool((grad == 0).all())
    loss, grad = ops.next_token_loss(x[:, :1], labels[:, :1])
    assert bool(torch.isnan(loss)) and bool((grad == 0).all())
    # NaN and +inf take their row, a NaN among masked values too, and no other
    for bad in (math.nan, math.inf):
        for row, at in ((1, 3), (0, 30), (0, V - 1)):
            y = x.clone()
            y[0, row, at] = bad
            loss, grad = ops.next_token_loss(y, labels)
            assert bool(torch.isnan(loss)) and bool(torch.isnan(grad[0, row]).all()), (bad, row, at)
            assert bool(torch.isfinite(grad[0, [r for r in range(6) if r != row]]).all())
    # rows masked throughout: the type's lowest value is as good as any other, -inf is not
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype, copy=True)
        y[0, 2] = torch.finfo(dtype).min
        y[0, 4, ::2] = torch.finfo(dtype).min
        y[0, 4, 1::2] = -math.inf
        loss, grad = ops.next_token_loss(y, labels)
        assert bool(torch.isfinite(loss)) and bool(torch.isfinite(grad[0, [0, 1, 2, 3]]).all())
        even = torch.arange(V, device=DEV) % 2 == 0
        for row, p, on in ((2, 1 / V, torch.ones_like(even)), (4, 1 / ((V + 1) // 2), even)):
            want = torch.where(on, p, 0.0).double()
            want[labels[0, row + 1]] -= 1
            _near(grad[0, row], want / 5, 16 * U * (want.abs() + p) / 5)
        y[0, 3] = -math.inf
        loss, grad = ops.next_token_loss(y, labels)
        assert bool(torch.isnan(loss)) and bool(torch.isnan(grad[0, 3]).all()) and bool(torch.isfinite(grad[0, 4]).all())
    ops.check_device_error()
    wrong = labels.clone()
    wrong[0, 2] = V
    loss, grad = ops.next_token_loss(x, wrong)
    assert bool(torch.isnan(loss)) and bool(torch.isnan(grad[0, 1]).all()) and bool(torch.isfinite(grad[0, 0]).all())
    with pytest.raises(_lib.GSAError):
        ops.check_device_error()
    # an ignored label may be anything
    wrong[0, 2] = 12345678
    loss, _ = ops.next_token_loss(x, wrong, ignore_index=12345678)
    assert bool(torch.isfinite(loss))
    ops.check_device_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 8, 16, 31, 60, 64, 100])
def test_loss_special_short_rows(cuda_ok, dtype, V):
    """Rows that two to eight lanes hold, special ones beside ordinary ones in a warp."""
    from gsa_b200 import _lib, ops

    L = 40
    x = _randn(1, 1, L, V, dtype=dtype)
    x[0, 1, 1:] = -math.inf
    x[0, 4] = torch.finfo(dtype).min
    x[0, 9, 0] = -math.inf
    x[0, 17] = 500.0
    labels = torch.randint(0, V, (1, L), device=DEV, generator=_gen(2))
    labels[0, 2] = labels[0, 5] = 0
    labels[0, 10] = V - 1
    labels[0, 20:23] = -100
    want, g, size, far, _ = _loss_oracle(x, labels)
    plain = x.clone()
    plain[0, 4] = 0.0  # its loss is log V too, which the value's size does not enter
    loss_size = _loss_oracle(plain, labels)[-1]
    loss, grad = ops.next_token_loss(x, labels)
    # two lanes at least: V / 2 additions after one another, and 2^(x log2 e - M) as above
    _near(loss, want, (V / 2 + 256) * U * (1 + loss_size))
    _near(grad, g, size * (V / 2 + 256) * U)
    assert bool((grad[0, 19:22] == 0).all()) and bool((grad[0, -1] == 0).all()) and bool((grad[0, 1, 1:] == 0).all())
    # a row without any probability, a NaN and labels out of range make their rows NaN, and no other
    y, bad = x.clone(), labels.clone()
    y[0, 6] = -math.inf
    y[0, 11, V // 2] = math.nan
    bad[0, 31], bad[0, 33] = V, -1
    loss, other = ops.next_token_loss(y, bad)
    assert math.isnan(float(loss))
    for t in range(L):
        assert bool(torch.isnan(other[0, t]).all()) if t in (6, 11, 30, 32) else torch.equal(other[0, t], grad[0, t]), t
    with pytest.raises(_lib.GSAError):
        ops.check_device_error()
    ops.check_device_error()


def test_loss_strides_types_and_second_backward(cuda_ok):
    import gsa_b200 as gsa

    B, L, V = 2, 9, 130
    wide = _randn(1, B, L + 3, 2 * V + 1, dtype=torch.bfloat16)
    labels = torch.randint(0, V, (L, B), device=DEV, generator=_gen(2)).t()
    for x in (wide[:, 2:2 + L, 1:1 + V], wide[:, :L, :2 * V:2], wide[:, :L].transpose(0, 1).contiguous().transpose(0, 1)[..., :V],
              wide[:1, :L, :V].expand(B, L, V)):
        a, b = gsa.ops.next_token_loss(x, labels), gsa.ops.next_token_loss(x.contiguous(), labels.contiguous().int())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[1].is_contiguous()
    leaf = wide[:, :L, :V].clone().requires_grad_(True)
    loss = gsa.fused_next_token_loss(leaf, labels)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="earlier backward"):
        loss.backward()


# -- streams, graphs ----------------------------------------------------------------------------
def _step(q, k, pos, freq, x, a, w, gu, logits, labels):
    import gsa_b200 as gsa

    q2, k2 = gsa.ops.rotary(q, k, pos, freq)
    h, y, p, rstd = gsa.ops.add_rmsnorm_packed(x, a, w, 1e-5)
    dx, dw, y2 = gsa.ops.rmsnorm_packed_backward(y, p, rstd, w, dh=h, want_y=True)
    z, pg = gsa.ops.silu_mul_packed(gu)
    dgu, z2 = gsa.ops.silu_mul_packed_backward(z, pg, want_z=True)
    loss, grad = gsa.ops.next_token_loss(logits, labels)
    return q2, k2, h, y, dx, dw, y2, z, dgu, z2, loss, grad


def _step_inputs(seed):
    import gsa_b200 as gsa

    bf = torch.bfloat16
    return (_randn(seed, 2, 50, 8, 64, dtype=bf), _randn(seed + 1, 2, 50, 2, 64, dtype=bf),
            torch.randint(0, 5000, (2, 50), device=DEV, generator=_gen(seed)), gsa.rotary_frequencies(64, device=DEV)[0],
            _randn(seed + 2, 100, 512, dtype=bf), _randn(seed + 3, 100, 512, dtype=bf), _randn(seed + 4, 512, dtype=bf),
            _randn(seed + 5, 100, 1024, dtype=bf), _randn(seed + 6, 2, 50, 1000, dtype=bf),
            torch.randint(0, 1000, (2, 50), device=DEV, generator=_gen(seed)))


def test_ops_on_a_side_stream_and_in_two_graphs(cuda_ok):
    """The same bits on another stream, and from two captured graphs that are replayed on new inputs, at once."""
    sets = [_step_inputs(10), _step_inputs(30)]
    want = [_step(*s) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(*sets[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for s in sets:
        held = tuple(t.clone() for t in s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*held)
        graphs.append((g, held, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for i, (g, held, _) in enumerate(graphs):
            for t, v in zip(held, sets[(i + turn) % 2]):
                t.copy_(v)
        torch.cuda.synchronize()
        for st, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(i + turn) % 2])), (turn, i)


def test_captured_training_step(cuda_ok):
    """Forward and backward through autograd, captured and replayed: the eager step's bits."""
    import gsa_b200 as gsa

    def step(x, w, wl, labels):
        h, y = gsa.packed_add_rmsnorm(x, None, w, 1e-5)
        z = gsa.packed_silu_mul(y)
        loss = gsa.fused_next_token_loss(z @ wl, labels)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w, wl)))

    def leaves():
        return [_randn(i, *s).requires_grad_(True) for i, s in ((1, (2, 16, 128)), (2, (128,)), (3, (64, 90)))]

    labels = torch.randint(0, 90, (2, 16), device=DEV, generator=_gen(4))
    want = step(*leaves(), labels)
    ins = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ins, labels)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*ins, labels)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda_ok):
    """What does not fit together is refused before any launch: shapes, dtypes, devices, overlapping outputs, second
    derivatives, an output under autograd."""
    import gsa_b200 as gsa
    from gsa_b200 import _lib, ops

    q, k = _randn(1, 2, 6, 4, 16), _randn(2, 2, 6, 2, 16)
    pos = torch.arange(6, device=DEV)
    freq, _ = gsa.rotary_frequencies(16, device=DEV)
    bad = [
        (q[0], k, pos, freq), (q, k[:, :5], pos, freq), (q, k[..., :8], pos, freq), (q, k.bfloat16(), pos, freq),
        (q, k, pos[:5], freq), (q, k, pos.expand(3, 6), freq), (q, k, pos.float(), freq), (q, k, pos > 2, freq),
        (q, k, pos, freq.view(2, 4)), (q, k, pos, gsa.rotary_frequencies(18, device=DEV)[0]), (q, k, pos, freq[:0]),
        (q[:, :, :0], k, pos, freq), (_randn(3, 1, 6, 1000, 16), _randn(3, 1, 6, 25, 16), pos, freq),
        (_randn(3, 1, 6, 1, 1026), None, pos, freq),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            gsa.apply_rotary(*args)
    o = torch.empty_like(q)
    for out in ((o, None), (o[:1].expand_as(q), torch.empty_like(k)), (o.bfloat16(), torch.empty_like(k)), (o[..., :8], torch.empty_like(k)),
                (o.transpose(2, 3).contiguous().transpose(2, 3), torch.empty_like(k)),
                (torch.empty(400, device=DEV).as_strided(q.shape, (96, 16, 8, 1)), torch.empty_like(k))):
        with pytest.raises(ValueError):
            gsa.apply_rotary(q, k, pos, freq, out=out)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gsa.apply_rotary(q, k, pos.cpu(), freq)
    with pytest.raises(NotImplementedError):
        gsa.apply_rotary(q.half(), None, pos, freq)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        gsa.apply_rotary(leaf, k, pos, freq, out=(o, torch.empty_like(k)))
    with pytest.raises(ValueError):
        ops.rotary(q, k, pos, tables=(torch.ones(8, 4, device=DEV), torch.ones(8, 4, device=DEV)), rotary_dim=16)
    x, w = _randn(4, 5, 32), torch.ones(32, device=DEV)
    for call in (lambda: gsa.pack_activation(x.half()), lambda: gsa.packed_silu_mul(x.half()),
                 lambda: gsa.packed_add_rmsnorm(x.half(), None, w.half(), 1e-5),
                 lambda: gsa.pack_activation(x).unpack(torch.float16),
                 lambda: gsa.fused_next_token_loss(x.half()[None], torch.zeros(1, 5, device=DEV, dtype=torch.long))):
        with pytest.raises(NotImplementedError):
            call()
    p = gsa.pack_activation(x)
    z, pg = ops.silu_mul_packed(x)
    h, y, ph, rstd = ops.add_rmsnorm_packed(x, x, w, 1e-5)
    lg, lab = _randn(5, 2, 6, 10), torch.zeros(2, 6, device=DEV, dtype=torch.long)
    for call in (lambda: gsa.pack_activation(x[0, 0]), lambda: gsa.PackedActivation(p.data[:-1], p.shape, p.dtype).unpack(),
                 lambda: gsa.PackedActivation(p.data, (), p.dtype).unpack(), lambda: gsa.packed_silu_mul(x[:, :31]),
                 lambda: ops.silu_mul_packed_backward(x, pg), lambda: ops.silu_mul_packed_backward(z.bfloat16(), pg),
                 lambda: ops.silu_mul_packed_backward(z, p), lambda: gsa.packed_add_rmsnorm(x, x[:4], w, 1e-5),
                 lambda: gsa.packed_add_rmsnorm(x, None, w[:31], 1e-5), lambda: gsa.packed_add_rmsnorm(x, None, w.bfloat16(), 1e-5),
                 lambda: gsa.packed_add_rmsnorm(x[:, :0], None, w[:0], 1e-5), lambda: ops.rmsnorm_packed_backward(y[:4], ph, rstd, w),
                 lambda: ops.rmsnorm_packed_backward(y, ph, rstd[:4], w), lambda: ops.rmsnorm_packed_backward(y, ph, rstd.double(), w),
                 lambda: ops.rmsnorm_packed_backward(y, ph, rstd, w, dh=y[:4]), lambda: gsa.fused_next_token_loss(lg[0], lab),
                 lambda: gsa.fused_next_token_loss(lg, lab[:, :5]), lambda: gsa.fused_next_token_loss(lg, lab.float()),
                 lambda: gsa.fused_next_token_loss(lg[..., :0], lab), lambda: ops.scale_(lg[..., ::2], rstd[0]),
                 lambda: ops.scale_(lg, rstd)):
        with pytest.raises(ValueError):
            call()
    # a packed buffer off the alignment of its codes
    odd = torch.empty(p.data.numel() + 1, device=DEV, dtype=torch.uint8)[1:]
    with pytest.raises(_lib.GSAError):
        gsa.PackedActivation(odd, p.shape, p.dtype).unpack()
    # second derivatives
    gu = _randn(6, 3, 64).requires_grad_(True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(gsa.packed_silu_mul(gu).sum(), gu, create_graph=True)
    ops.check_device_error()


def test_tensors_written_in_place_are_noticed(cuda_ok):
    """A tensor that another graph saved and apply_rotary then overwrites: that graph's backward pass refuses."""
    import gsa_b200 as gsa

    q = _randn(1, 1, 4, 2, 16)
    w = torch.ones_like(q).requires_grad_(True)
    y = (w * q).sum()
    freq, _ = gsa.rotary_frequencies(16, device=DEV)
    with torch.no_grad():
        gsa.apply_rotary(q, None, torch.arange(4, device=DEV), freq, out=(q, None))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_offsets_past_32_bits(cuda_ok):
    """The last rows of tensors of more than 2^31 elements, and tokens 2^31 elements apart."""
    import gsa_b200 as gsa

    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    bf = torch.bfloat16
    rows, n = 140000, 16384
    x = torch.zeros(rows, n, device=DEV, dtype=bf)
    x[-3:] = _randn(1, 3, n, dtype=bf)
    p = gsa.pack_activation(x)
    assert torch.equal(p.unpack()[-3:], gsa.pack_activation(x[-3:].clone()).unpack())
    z, pg = gsa.ops.silu_mul_packed(x)
    z2, pg2 = gsa.ops.silu_mul_packed(x[-3:].clone())
    assert torch.equal(z[-3:], z2)
    dgu, _ = gsa.ops.silu_mul_packed_backward(z, pg)
    assert torch.equal(dgu[-3:], gsa.ops.silu_mul_packed_backward(z2, pg2)[0])
    del dgu, z, pg
    w = torch.ones(n, device=DEV, dtype=bf)
    _, y, ph, rstd = gsa.ops.add_rmsnorm_packed(x, None, w, 1e-5)
    _, y2, ph2, rstd2 = gsa.ops.add_rmsnorm_packed(x[-3:].clone(), None, w, 1e-5)
    assert torch.equal(y[-3:], y2) and torch.equal(rstd[-3:], rstd2)
    dx = gsa.ops.rmsnorm_packed_backward(y, ph, rstd, w, want_dw=False)[0]
    assert torch.equal(dx[-3:], gsa.ops.rmsnorm_packed_backward(y2, ph2, rstd2, w, want_dw=False)[0])
    del dx, y, ph, p
    logits = x.view(1, -1)[:, :128256 * 17000].view(1, 17000, 128256)
    logits[0, -2] = _randn(2, 128256, dtype=bf)
    labels = torch.full((1, 17000), -100, device=DEV)
    labels[0, -1] = 77
    loss, grad = gsa.ops.next_token_loss(logits, labels)
    loss2, grad2 = gsa.ops.next_token_loss(logits[:, -2:].clone(), labels[:, -2:])
    assert torch.equal(loss, loss2) and torch.equal(grad[:, -2:], grad2) and bool((grad[0, 5] == 0).all())
    del logits, grad, x
    far = torch.zeros((1 << 32) + 4096, device=DEV, dtype=bf)
    q = far.as_strided((1, 3, 2, 64), (0, 1 << 31, 64, 1))
    q.copy_(_randn(3, 1, 3, 2, 64, dtype=bf))
    pos, (freq, _) = torch.arange(3, device=DEV) * 999, gsa.rotary_frequencies(64, device=DEV)
    want = gsa.apply_rotary(q.clone(), None, pos, freq)[0]
    assert torch.equal(gsa.apply_rotary(q, None, pos, freq)[0], want)
    gsa.apply_rotary(q, None, pos, freq, out=(q, None))
    assert torch.equal(q, want)


# -- together -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,n", [(5, 48, 33), (64, 256, 512)])
def test_packed_mlp_block(cuda_ok, dtype, rows, d, n):
    """The block's output and every gradient against the 64-bit formulas at the values that the kernels keep (the packed
    tensors of the same calls): matrix products of k terms lose up to k U and a half step of each operand in between."""
    import gsa_b200 as gsa

    x, a = _randn(1, rows, d, dtype=dtype), _randn(2, rows, d, dtype=dtype)
    w = (1 + 0.1 * _randn(3, d)).to(dtype)
    wg, wu, wd = (_randn(4 + i, *s, dtype=dtype, scale=s[1] ** -0.5) for i, s in enumerate(((n, d), (n, d), (d, n))))
    dout = _randn(8, rows, d, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, a, w, wg, wu, wd)]
    out = gsa.packed_mlp_block(*leaves, 1e-5)
    grads = torch.autograd.grad(out, leaves, dout)
    # the same kernels by hand, for what they keep
    h, y, ph, rstd = gsa.ops.add_rmsnorm_packed(x, a, w, 1e-5)
    gu = torch.empty(rows, 2 * n, device=DEV, dtype=dtype)
    torch.mm(y, wg.t(), out=gu[:, :n])
    torch.mm(y, wu.t(), out=gu[:, n:])
    z, pgu = gsa.ops.silu_mul_packed(gu)
    D = lambda t: t.double()
    hh, guh, r = D(ph.unpack(torch.float32)), D(pgu.unpack(torch.float32)), D(rstd).unsqueeze(-1)
    g, u = guh[:, 0], guh[:, 1]
    sig = torch.sigmoid(g)
    yk, zk = hh * r * D(w), g * sig * u
    dz = D(dout) @ D(wd)
    dg, du = dz * u * sig * (1 + g * (1 - sig)), dz * g * sig
    dy = dg @ D(wg) + du @ D(wu)
    xh = hh * r
    dx = r * (dy * D(w) - xh * (dy * D(w) * xh).mean(-1, keepdim=True)) + D(dout)
    want = [dx, dx, (dy * xh).sum(0), dg.t() @ yk, du.t() @ yk, D(dout).t() @ zk]
    # sums of absolute values: what each result is made of; every rounded operand in between is off by half a step
    e = _half_step(dtype)
    ab = torch.abs
    mdz = ab(D(dout)) @ ab(D(wd))
    mdg, mdu = mdz * ab(u) * sig * (1 + ab(g)), mdz * ab(g) * sig
    mdy = mdg @ ab(D(wg)) + mdu @ ab(D(wu))
    mdx = r * (mdy * ab(D(w)) + ab(xh) * (mdy * ab(D(w) * xh)).mean(-1, keepdim=True)) + ab(D(dout))
    made = [mdx, mdx, (mdy * ab(xh)).sum(0), mdg.t() @ ab(yk), mdu.t() @ ab(yk), ab(D(dout)).t() @ ab(zk)]
    for name, got, ref, m in zip(("x", "a", "w", "gate", "up", "down"), grads, want, made):
        _near(got, ref, m * (6 * e + (n + d + rows + 64) * U), name)
    # the down product is the matrix library's, which may round the product, and partial sums of it, to the type before h
    # is added (torch allows bf16 reductions by default): a half step of the terms' sizes for each of the two
    ref, made = D(h) + D(z) @ D(wd).t(), ab(D(z)) @ ab(D(wd)).t()
    _near(out.detach(), ref, (ab(D(h)) + made) * (n + 8) * U + 2 * e * made, "out")
    # frozen parts get no gradient, the others the same
    some = [t.clone().requires_grad_(i in (0, 3)) for i, t in enumerate((x, a, w, wg, wu, wd))]
    got = torch.autograd.grad(gsa.packed_mlp_block(*some, 1e-5), (some[0], some[3]), dout)
    assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[3])


def _lm(dtype, layers=2):
    from gsa_b200 import GSAConfig, GSALlamaForCausalLM

    cfg = GSAConfig(d_model=256, n_heads=4, n_kv_heads=2, d_indexer=32, n_indexer_heads=4, k_base=24, k_min=8, k_max=48,
                    n_layers=layers, d_ffn=512, vocab_size=384, max_position_embeddings=512)
    torch.manual_seed(0)
    return GSALlamaForCausalLM(cfg).to(DEV).to(dtype).train()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_causal_lm_packed_training_step(cuda_ok, dtype):
    """The model's training step with packed activations and the fused loss: the loss is the torch one, every trainable
    parameter gets a gradient near the unpacked step's.  Each kept value is within 2^-4 of its value and a term of a
    gradient has at most four of them, so gradients differ by less than 4 / 16 in norm."""
    m = _lm(dtype)
    ids = torch.randint(0, 384, (2, 64), generator=torch.Generator().manual_seed(2)).to(DEV)
    plain = m(ids, labels=ids)
    plain.loss.backward()
    ref = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}
    m.zero_grad(set_to_none=True)
    m.enable_packed_training()
    out = m(ids, labels=ids)
    out.loss.backward()
    assert out.loss.dtype == torch.float32
    exact = torch.nn.functional.cross_entropy(out.logits.double()[:, :-1].reshape(-1, 384), ids[:, 1:].reshape(-1))
    assert abs(float(out.loss.detach()) - float(exact.detach())) < 1e-5 * float(exact.detach())
    for name, p in m.named_parameters():
        if ".indexer." in name:
            assert p.grad is None, name
            continue
        assert p.grad is not None and p.grad.dtype == dtype and bool(torch.isfinite(p.grad).all()), name
        off = float((p.grad.double() - ref[name].double()).norm() / ref[name].double().norm())
        assert off < 0.25, (name, off)
    # without autograd, and switched off again, the model is what it was
    with torch.no_grad():
        a = m(ids).logits
    m.enable_packed_training(False)
    with torch.no_grad():
        assert torch.equal(m(ids).logits, a)
    m.zero_grad(set_to_none=True)
    again = m(ids, labels=ids)
    assert torch.equal(again.loss, plain.loss)


def test_packed_training_with_gradient_checkpointing(cuda_ok):
    """Recomputing the layers in the backward pass gives the same gradients."""
    m = _lm(torch.float32)
    m.enable_packed_training()
    ids = torch.randint(0, 384, (2, 32), generator=torch.Generator().manual_seed(2)).to(DEV)
    grads = []
    for again in (False, True):
        m.model.gradient_checkpointing = again
        m.zero_grad(set_to_none=True)
        m(ids, labels=ids).loss.backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for name, g in grads[0].items():
        # dK and dV of the sparse attention are added by atomics, in an order of their own each time
        assert float((grads[1][name] - g).norm()) <= 1e-4 * float(g.norm()), name


def test_packed_training_holds_less(cuda_ok):
    """Memory that the graph of a step keeps (allocated after the forward pass, above the weights)."""
    m = _lm(torch.bfloat16, layers=4)
    ids = torch.randint(0, 384, (4, 512), generator=torch.Generator().manual_seed(2)).to(DEV)
    kept = []
    for packed in (False, True):
        m.enable_packed_training(packed)
        m(ids)  # caches of the layers
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = m.model(ids).last_hidden_state
        torch.cuda.synchronize()
        kept.append(torch.cuda.memory_allocated() - before)
        del out
    # what the layers keep beside the attention goes from 16- and 32-bit copies to 33/32 bytes a value
    assert kept[1] < 0.75 * kept[0], kept
