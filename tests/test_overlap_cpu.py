"""Which strided tensors share memory: what apply_rotary refuses of its outputs, against the sets of elements themselves."""

import random

import pytest
import torch


def _overlap():
    from gsa_b200 import _lib

    return _lib.native().overlap


def _elements(t):
    at = torch.tensor(t.storage_offset())
    for size, stride in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(size) * stride
    return set(at.flatten().tolist())


def test_overlap_is_that_of_the_elements():
    rng = random.Random(0)
    base = torch.zeros(4096)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        views = []
        shared = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 48, 64, 96, 200]) for _ in range(4)]
        for _ in range(2):
            sizes = [rng.randint(1, 5) for _ in range(4)]
            strides = shared if rng.random() < 0.7 else [rng.choice([0, 1, 2, 3, 5, 7, 8, 16, 40, 64, 130]) for _ in range(4)]
            views.append(base.as_strided(sizes, strides, rng.randint(0, 300)))
        a, b = views
        want = bool(_elements(a) & _elements(b))
        seen[want] += 1
        assert _overlap()(a, b) == want and _overlap()(b, a) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(),
                                                                        b.storage_offset())
    assert min(seen.values()) > 500


def test_overlap_of_the_layouts_in_use():
    overlap = _overlap()
    B, L, H, Hk, D = 2, 700, 32, 8, 128
    proj = torch.zeros(B, L, (H + 2 * Hk) * D + 7, dtype=torch.bfloat16)
    q = proj[..., :H * D].view(B, L, H, D)
    k = proj[..., H * D:(H + Hk) * D].view(B, L, Hk, D)
    assert not overlap(q, k) and overlap(q, q) and overlap(q[:, 3:], q[:, :-3]) and not overlap(q[:, 3:], q[:, :3])
    assert overlap(q, q[..., 64:]) and overlap(q[..., 60:], q[..., :64]) and not overlap(q[..., 64:], q[..., :64])
    kv = torch.zeros(B, L + 9, 2, Hk, D)
    assert not overlap(kv[:, :L, 0], kv[:, :L, 1]) and not overlap(kv[:, :5, 0], kv[:, 5:9, 0])
    assert overlap(kv[:, 0:L, 0], kv[:, 1:L + 1, 0])  # a shift by one slot
    heads = torch.zeros(B, H + Hk, L, D)
    qt, kt = heads[:, :H].transpose(1, 2), heads[:, H:].transpose(1, 2)
    assert not overlap(qt, kt) and overlap(qt, heads[:, H - 1:].transpose(1, 2))
    assert not overlap(q[:0], q) and not overlap(torch.zeros(3), torch.zeros(3))
    # one element off by a part of itself
    raw = torch.zeros(64, dtype=torch.uint8)
    assert overlap(raw[:32].view(torch.float32), raw[4:36].view(torch.float32))
    # strides that have nothing in common, over many elements: an answer in bounded time
    big = torch.zeros(1 << 22)
    a = big.as_strided((40, 41, 42, 43), (4001, 977, 101, 7), 3)
    assert overlap(a, big.as_strided((39, 38, 37, 36), (3989, 1009, 103, 11), 1)) in (True, False)


@pytest.mark.gpu
def test_rotary_refuses_outputs_that_share_memory(cuda_ok):
    """Outputs that overlap each other, or an input without being it; what is apart, or the input itself, is taken."""
    import gsa_b200 as gsa

    B, L, H, D = 1, 6, 2, 16
    pos, (freq, _) = torch.arange(L, device="cuda"), gsa.rotary_frequencies(D, device="cuda")
    buf = torch.randn(B, L + 2, 3 * H, D, device="cuda")
    keep = buf.clone()
    q, k, free = buf[:, :L, :H], buf[:, :L, H:2 * H], buf[:, :L, 2 * H:]
    other = torch.empty(B, L, H, D, device="cuda")
    for args, out in (((q, None), (buf[:, 1:L + 1, :H], None)),      # one slot further
                      ((q, None), (buf[:, :L, 1:H + 1], None)),      # one head further
                      ((q, k), (other, other)),                      # both in one place
                      ((q, k), (free, buf[:, 1:L + 1, 2 * H:])),     # two outputs that overlap in part
                      ((q, k), (k, other)),                          # q where k still is
                      ((q, k), (other, q)),                          # k where q still is
                      ((q, k), (k, q)),                              # exchanged
                      ((q, q), (q, q)),
                      ((q.transpose(1, 2).contiguous().transpose(1, 2), k), (k, other))):
        with pytest.raises(ValueError, match="overlap"):
            gsa.apply_rotary(*args, pos, freq, out=out)
    torch.cuda.synchronize()
    assert torch.equal(buf, keep)
    want = gsa.apply_rotary(q, k, pos, freq)
    got = gsa.apply_rotary(q, k, pos, freq, out=(free, other))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    gsa.apply_rotary(q, k, pos, freq, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    # an input that is laid out anew first may lie anywhere: here every second value, turned into itself
    wide = torch.randn(B, L, H, 2 * D, device="cuda")
    want = gsa.apply_rotary(wide[..., ::2].contiguous(), None, pos, freq)[0]
    gsa.apply_rotary(wide[..., ::2], None, pos, freq, out=(wide[..., :D], None))
    assert torch.equal(wide[..., :D], want)
