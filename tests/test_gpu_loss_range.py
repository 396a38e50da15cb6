"""The next-token loss over the whole range of its logits' type: rows whose largest value is far from zero, masks of any
finite size beside ordinary logits, labels on masked values.

Every row is also a call of its own, so that the mean hides nothing.  The oracle is the definition in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative

# one size for each number of threads that a row may have, by its bytes
BYTES = [40, 200, 900, 4000, 15000, 40000, 100000, 256512, 400000]


def _ordinary(seed, V, dtype):
    return (torch.randn(V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)) * 3).to(dtype)


def _oracle(x, labels):
    """Losses [R] and d loss / dx [R, V] of rows x under their labels, in 64 bits, and each value's distance from the largest."""
    xd = x.double()
    top = xd.amax(-1, keepdim=True)
    far = top - xd
    e = torch.exp(-far)
    s = e.sum(-1, keepdim=True)
    at = labels.view(-1, 1)
    loss = (s.log() + far.gather(-1, at)).squeeze(-1)
    p = e / s
    grad = p.clone()
    grad.scatter_add_(-1, at, torch.full_like(at, -1, dtype=torch.float64))
    return loss, grad, p + torch.zeros_like(p).scatter(-1, at, 1.0), far


def _check_rows(rows, labels):
    from gsa_b200 import ops

    x, labels = torch.stack(rows), torch.tensor(labels, device=DEV)
    R, V = x.shape
    want, grad, size, far = _oracle(x, labels)
    half = torch.finfo(x.dtype).eps / 2
    # V exponentials are added, at most V / 32 + 80 after one another; each is off by 4 U and by U and a half of its
    # argument, to which a rounding of the row's largest scaled value adds up to 4; log2 of the sum by U of its size
    lose = (V / 32 + 80) * U

    def near(got, i, count):
        bound = half * grad[i].abs() / count + size[i] / count * (lose + (1.5 * far[i].clamp(max=200) + 64) * U) * (1 + half)
        off = (got.double() - grad[i] / count).abs() - bound - 2.0 ** -120
        return not bool(torch.isnan(off).any()) and float(off.max()) <= 0

    # all of them as one sequence of rows, a last position behind them
    lab = torch.cat([labels.new_zeros(1), labels]).view(1, -1)
    many = torch.cat([x, x[:1]]).unsqueeze(0)
    _, together = ops.next_token_loss(many, lab)
    for i in range(R):
        loss, g = ops.next_token_loss(x[i].expand(1, 2, V), torch.stack([labels[i], labels[i]]).view(1, 2))
        bound = U * want[i].abs() + lose + (1.5 * far[i, labels[i]] + 64) * U
        what = (i, rows[i].dtype, V, float(loss), float(want[i]))
        largest = torch.finfo(torch.float32).max
        if float(want[i]) > largest:
            assert float(loss) == math.inf, what
        else:
            assert math.isfinite(float(loss)) and abs(float(loss) - float(want[i])) <= float(bound), what
        assert near(g[0, 0], i, 1), what
        assert near(together[0, i], i, R), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nbytes", BYTES)
def test_loss_rows_far_from_zero(cuda_ok, dtype, nbytes):
    """Rows whose largest value is anything up to the type's largest, of either sign."""
    V = nbytes * 8 // torch.finfo(dtype).bits
    big = torch.finfo(dtype).max
    rows, labels = [], []
    for v in (2.0 ** 26, 2.0 ** 27, 2.0 ** 28, 1e9, 1e10, 1e15, 1e30, 9e37, 2.3e38, 2.4e38, 3e38, big):
        for sign in (1.0, -1.0):
            rows.append(torch.full((V,), sign * v, device=DEV).to(dtype))
            labels.append((7 * len(labels)) % V)
    # one of them above ordinary ones, the label or not; neighbouring values of the type near the borders between methods
    for v in (9e7, 1e8, 1e10, 2.4e38, big):
        for hit in (True, False):
            row = _ordinary(len(rows), V, dtype)
            row[V // 2] = v
            rows.append(row)
            labels.append(V // 2 if hit else 1)
    for v in (-2.0 ** 28, -9.3e7, 9.3e7, 1e6):
        edge = torch.tensor(v, device=DEV).to(dtype)
        step = float(edge.abs()) * torch.finfo(dtype).eps
        rows.append((float(edge) + step * (torch.arange(V, device=DEV) % 5 - 2)).to(dtype))
        labels.append(3)
    _check_rows(rows, labels)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nbytes", BYTES)
def test_loss_masks_of_any_size(cuda_ok, dtype, nbytes):
    """Parts of a row masked with a finite value: a half, all but one, all but the edges, every second one."""
    V = nbytes * 8 // torch.finfo(dtype).bits
    i = torch.arange(V, device=DEV)
    rows, labels = [], []
    for mask in (-1e8, -2.0 ** 28, -1e9, -1e10, -1e12, -1e20, -1e30, -9e37, -1.1e38, torch.finfo(dtype).min):
        for keep in (i >= V // 2, i < V // 3 + 1, i == V - 1, i == 0, (i < 2) | (i == V - 1), i % 2 == 0):
            row = _ordinary(len(rows), V, dtype)
            row[~keep] = mask
            rows.append(row)
            labels.append(int(keep.nonzero()[0]))
    _check_rows(rows, labels)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nbytes", BYTES)
def test_loss_of_labels_far_below(cuda_ok, dtype, nbytes):
    """The label's own logit masked with a finite value: the loss is its distance, as far as fp32 holds it, and also where
    the mean over several rows does."""
    from gsa_b200 import ops

    V = nbytes * 8 // torch.finfo(dtype).bits
    low = torch.finfo(dtype).min
    rows, labels = [], []
    for v in (-1e9, -1e10, -1e30, -2.3e38, -2.4e38, -3e38, low):
        row = _ordinary(len(rows), V, dtype)
        row[V // 2] = v
        rows.append(row)
        labels.append(V // 2)
    for v, other in ((1e10, -1e10), (1e38, -1e38), (1.5e38, -1.5e38), (low, low)):
        row = torch.full((V,), v, device=DEV).to(dtype)
        row[V // 2] = other
        rows.append(row)
        labels.append(V // 2)
    _check_rows(rows, labels)
    # a row's loss past fp32's largest, and a mean that is not
    x = torch.zeros(1, 6, V, device=DEV, dtype=dtype)
    x[0, 2, 0], x[0, 2, 1] = -low, low
    lab = torch.tensor([[0, 0, 0, 1, 0, 0]], device=DEV)
    loss, grad = ops.next_token_loss(x, lab)
    want = (-2 * low + 4 * math.log(V)) / 5
    assert math.isfinite(float(loss)) and abs(float(loss) - want) <= 4 * U * want and bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("factor", [1 / 3, 0.1, 1e-4, 7.0, -3.0, 0.0])
def test_scaled_loss_is_rounded_twice_at_most(cuda_ok, dtype, factor):
    """The gradient of a scaled loss is within the unscaled one's half step and one more of the exact one."""
    import gsa_b200 as gsa

    V, L = 1000, 40
    logits = (torch.randn(1, L, V, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * 3).to(dtype)
    labels = torch.randint(0, V, (1, L), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    want, grad, size, far = _oracle(logits[0, :-1], labels[0, 1:])
    leaf = logits.clone().requires_grad_(True)
    (gsa.fused_next_token_loss(leaf, labels) * factor).backward()
    exact, size = grad * factor / (L - 1), size * abs(factor) / (L - 1)
    half = torch.finfo(dtype).eps / 2
    # two roundings to the type, the factor's own and the arithmetic's of the unscaled gradient (as for the rows above)
    bound = (2 * half + 2 * half * half) * exact.abs() + size * ((V / 32 + 80) + 1.5 * far + 70) * U * (1 + 2 * half) + 2.0 ** -120
    assert bool(((leaf.grad[0, :-1].double() - exact).abs() <= bound).all())
    assert bool((leaf.grad[0, -1] == 0).all())
