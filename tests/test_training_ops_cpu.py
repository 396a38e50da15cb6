"""Rotary frequencies against their formulas, and what the training-step operators refuse (nothing here touches a GPU: the C entry
points return before any launch, the Python ones before any call)."""

import ctypes as C
import math

import pytest
import torch


def test_rotary_frequencies_match_the_embedding():
    """None, ntk and yarn are RotaryEmbedding's frequencies, in 64 bits (its own are 32-bit: off by a few 2^-24)."""
    import gsa_b200 as gsa

    for scaling in (None, dict(type="ntk", factor=4.0), dict(type="yarn", factor=16.0, original_max_position_embeddings=4096),
                    dict(type="yarn", factor=8.0, original_max_position_embeddings=8192, beta_fast=16, beta_slow=2)):
        for dim, base in ((128, 10000.0), (64, 500000.0)):
            f, m = gsa.rotary_frequencies(dim, base, scaling)
            old = gsa.RotaryEmbedding(dim, 4, base, scaling).inv_freq.double()
            assert f.dtype == torch.float64 and f.shape == (dim // 2,) and m == 1.0
            assert float((f / old - 1).abs().max()) < 8 * 2.0 ** -24


def test_rotary_frequency_scalings():
    import gsa_b200 as gsa

    std, _ = gsa.rotary_frequencies(64)
    assert abs(float(std[1]) - 10000.0 ** (-2 / 64)) < 1e-15
    lin, m = gsa.rotary_frequencies(64, scaling=dict(rope_type="linear", factor=4.0, attention_factor=1.5))
    assert torch.equal(lin, std / 4) and m == 1.5
    dyn = dict(type="dynamic_ntk", factor=2.0, original_max_position_embeddings=1000)
    assert torch.equal(gsa.rotary_frequencies(64, scaling=dyn, seq_len=1000)[0], std)
    assert torch.equal(gsa.rotary_frequencies(64, scaling=dyn)[0], std)
    far = gsa.rotary_frequencies(64, scaling=dyn, seq_len=3000)[0]
    assert abs(float(far[3]) - (10000.0 * 5.0 ** (64 / 62)) ** (-6 / 64)) < 1e-15  # 2 * 3 - 1 = 5
    l3, _ = gsa.rotary_frequencies(128, 500000.0, dict(type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                       original_max_position_embeddings=8192))
    f, _ = gsa.rotary_frequencies(128, 500000.0)
    for a, b in zip(f.tolist(), l3.tolist()):
        wave = 2 * math.pi / a
        if wave < 8192 / 4:
            assert a == b
        elif wave > 8192:
            assert abs(b * 8 / a - 1) < 1e-12
        else:
            s = (8192 / wave - 1) / 3
            assert abs(b - ((1 - s) * a / 8 + s * a)) < 1e-12 * a
    assert gsa.rotary_frequencies(2, scaling=dict(type="ntk", factor=4.0))[0].tolist() == [1.0]
    for dim in (0, 3, -2):
        with pytest.raises(ValueError):
            gsa.rotary_frequencies(dim)
    with pytest.raises(ValueError, match="unknown"):
        gsa.rotary_frequencies(64, scaling=dict(type="other"))
    with pytest.raises(ValueError):
        gsa.rotary_frequencies(64, scaling=dict(type="llama3", low_freq_factor=4.0, high_freq_factor=4.0))


def test_cpu_tensors_are_refused():
    import gsa_b200 as gsa

    x = torch.zeros(2, 4, 2, 8)
    pos = torch.zeros(2, 4, dtype=torch.long)
    for call in (lambda: gsa.apply_rotary(x, x, pos, gsa.rotary_frequencies(8)[0]), lambda: gsa.pack_activation(x),
                 lambda: gsa.packed_silu_mul(x), lambda: gsa.packed_add_rmsnorm(x, x, torch.ones(8), 1e-5),
                 lambda: gsa.fused_next_token_loss(x[0], pos[:, :2])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_packed_layout():
    """33/32 bytes a value: codes of whole 16-byte pieces, then a byte for each group."""
    import gsa_b200 as gsa

    p = gsa.PackedActivation.empty((3, 2, 40), torch.bfloat16, "cpu")
    assert p.rows == 6 and p.n == 40 and p.nbytes == 6 * (48 + 2)
    assert p.codes.shape == (6, 48) and p.scales.shape == (6, 2)
    assert p.codes.data_ptr() == p.data.data_ptr() and p.scales.data_ptr() == p.data.data_ptr() + 6 * 48
    assert gsa.PackedActivation.empty((0, 8), torch.float32, "cpu").nbytes == 0


def _p():
    return C.c_void_p(256)  # a stand-in pointer: every case returns before using it


def test_rotary_entry_point_refuses():
    from gsa_b200 import _lib

    lib, p = _lib.lib(), _p()

    def call(dtype=1, B=1, L=4, D=64, rd=64, q=(256, 256, 2, 512, 128, 64, 512, 128, 64), k=None, pos=p, freq=p, cos=None, sin=None,
             tab_dtype=0, tab_ld=64, rows=16):
        return lib.gsa_rotary(dtype, B, L, D, rd, C.byref(_lib.RotarySide(*q)) if q else None,
                              C.byref(_lib.RotarySide(*k)) if k else None, pos, 4, 1, freq, cos, sin, tab_dtype, tab_ld, rows, 1.0,
                              0, 0, None)

    good = (256, 256, 2, 512, 128, 64, 512, 128, 64)
    assert call(dtype=2) == 1 and call(B=-1) == 1
    assert call(rd=63) == 1 and call(rd=0) == 1 and call(rd=66) == 1          # odd, empty, wider than the head
    assert call(D=1026, rd=1026) == 1                                         # wider than a head may be
    assert call(q=None) == 1 and call(q=(None,) + good[1:]) == 1 and call(q=(256, None) + good[2:]) == 1
    assert call(q=(256, 256, 0) + good[3:]) == 1                              # no heads
    assert call(q=good[:8] + (32,)) == 1                                      # heads of the output overlap
    assert call(k=(256, 256, 1023, 0, 0, 0, 1 << 20, 1 << 20, 64)) == 1       # more than 1024 heads together
    assert call(pos=None) == 1 and call(freq=None) == 1                       # no positions; no angles at all
    assert call(freq=None, cos=p, sin=p, tab_ld=31) == 1 and call(freq=None, cos=p, sin=p, rows=0) == 1
    assert call(freq=None, cos=p, sin=p, tab_dtype=5) == 1 and call(freq=None, cos=p) == 1
    assert call(B=0) == 0 and call(L=0) == 0                                  # nothing to do


def test_packed_entry_points_refuse():
    from gsa_b200 import _lib

    lib, p = _lib.lib(), _p()
    odd = C.c_void_p(264)
    # pack / unpack: type, sizes, pointers, rows of codes, alignment, rows of scales
    for name, lead in (("gsa_pack_e4m3", True), ("gsa_unpack_e4m3", False)):
        def call(dtype=1, rows=4, n=40, x=p, x_ld=40, codes=p, c_ld=48, scales=p, s_ld=2):
            tail = (x, x_ld, codes, c_ld, scales, s_ld) if lead else (codes, c_ld, scales, s_ld, x, x_ld)
            return getattr(lib, name)(dtype, rows, n, *tail, None)

        assert call(dtype=3) == 1 and call(rows=-1) == 1 and call(x=None) == 1 and call(codes=None) == 1
        assert call(scales=None) == 1 and call(c_ld=40) == 1 and call(c_ld=50) == 1 and call(s_ld=1) == 1
        assert call(codes=odd) == 1
        assert call(rows=0) == 0 and call(n=0) == 0
    assert lib.gsa_unpack_e4m3(1, 4, 40, p, 48, p, 2, p, 39, None) == 1       # output rows overlap
    assert lib.gsa_silu_mul_pack(1, 4, 40, p, 80, p, 39, p, 48, p, 2, None) == 1
    assert lib.gsa_silu_mul_pack(1, 4, 40, None, 80, p, 40, p, 48, p, 2, None) == 1
    assert lib.gsa_silu_mul_packed_backward(1, 4, 40, p, 40, p, 48, p, 2, p, 79, None, 0, None) == 1
    assert lib.gsa_silu_mul_packed_backward(1, 4, 40, p, 40, p, 48, p, 2, p, 80, p, 39, None) == 1
    assert lib.gsa_silu_mul_packed_backward(1, 0, 40, None, 40, None, 48, None, 2, None, 80, None, 0, None) == 0

    def norm(rows=4, x=p, a=p, w=p, h=p, h_ld=40, y=p, y_ld=40, rstd=p, c_ld=48):
        return lib.gsa_add_rmsnorm_pack(1, rows, 40, x, 40, a, 40, w, 1e-5, h, h_ld, y, y_ld, p, c_ld, p, 2, rstd, None)

    assert norm(x=None) == 1 and norm(w=None) == 1 and norm(y=None) == 1 and norm(rstd=None) == 1 and norm(c_ld=32) == 1
    assert norm(h_ld=39) == 1 and norm(y_ld=39) == 1 and norm(a=None) == 1    # a sum to write and nothing to add
    assert norm(rows=0) == 0 and norm(rows=1 << 31) == 1

    def back(rows=4, dy=p, dx_ld=40, y=None, dw=p, ws=p, nbytes=1 << 30, rstd=p):
        return lib.gsa_rmsnorm_packed_backward(1, rows, 40, dy, 40, None, 0, p, p, 48, p, 2, rstd, p, dx_ld, y, 39, dw, ws, nbytes,
                                               None)

    assert back(dy=None) == 1 and back(dx_ld=39) == 1 and back(y=p) == 1 and back(rstd=None) == 1
    assert back(ws=None) == 3 and back(nbytes=159) == 3                       # a row of partial sums is 160 bytes
    assert back(rows=0, dw=None) == 0
    assert lib.gsa_rmsnorm_packed_workspace_size(1, 40) >= 160 and lib.gsa_rmsnorm_packed_workspace_size(0, 40) == 0


def test_loss_entry_points_refuse():
    from gsa_b200 import _lib

    lib, p = _lib.lib(), _p()

    def call(dtype=1, B=2, L=4, V=10, x=p, labels=p, loss=p, grad=p, g_b=40, g_l=10, ws=p, nbytes=1 << 20):
        return lib.gsa_next_token_loss(dtype, B, L, V, x, 40, 10, labels, 4, 1, -100, loss, grad, g_b, g_l, ws, nbytes, None)

    assert call(dtype=9) == 1 and call(B=-1) == 1 and call(V=0) == 1 and call(x=None) == 1 and call(labels=None) == 1
    assert call(loss=None) == 1 and call(g_l=9) == 1 and call(g_b=9) == 1
    assert call(ws=None) == 3 and call(nbytes=lib.gsa_next_token_loss_workspace_size() - 1) == 3
    assert call(ws=C.c_void_p(264)) == 3
    assert lib.gsa_scale(1, -1, p, p, None) == 1 and lib.gsa_scale(1, 4, None, p, None) == 1
    assert lib.gsa_scale(4, 4, p, p, None) == 1 and lib.gsa_scale(1, 0, None, None, None) == 0
