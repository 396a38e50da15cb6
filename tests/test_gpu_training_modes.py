"""The training-step operators in the modes that torch has beside plain reverse mode: adapters and hooks on a packed model's
modules, autocast, forward-mode derivatives, gradients that the operators do not give."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)) * scale).to(dtype)


# -- modules that are not what the packed path knows ---------------------------------------------
class _Adapter(torch.nn.Module):
    """base(x) + x A B, with base frozen."""

    def __init__(self, base, rank=4):
        super().__init__()
        self.base = base.requires_grad_(False)
        self.a = torch.nn.Parameter(torch.randn(base.in_features, rank, device=DEV) * 0.1)
        self.b = torch.nn.Parameter(torch.randn(rank, base.out_features, device=DEV) * 0.1)

    @property
    def weight(self):
        return self.base.weight

    def forward(self, x):
        return self.base(x) + x @ self.a @ self.b


class _LinearChild(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def _model():
    from gsa_b200 import GSAConfig, GSALlamaForCausalLM

    cfg = GSAConfig(d_model=256, n_heads=4, n_kv_heads=2, d_indexer=32, n_indexer_heads=4, k_base=24, k_min=8, k_max=48,
                    n_layers=2, d_ffn=512, vocab_size=384, max_position_embeddings=512)
    torch.manual_seed(0)
    return GSALlamaForCausalLM(cfg).to(DEV).train()


def _bias(m):
    mlp = m.model.layers[1].mlp
    new = torch.nn.Linear(512, 256, bias=True, device=DEV)
    with torch.no_grad():
        new.weight.copy_(mlp.down_proj.weight)
    mlp.down_proj = new


def _child(m):
    mlp = m.model.layers[0].mlp
    new = _LinearChild(256, 512, bias=False, device=DEV)
    with torch.no_grad():
        new.weight.copy_(mlp.up_proj.weight)
    mlp.up_proj = new


def _instance_forward(m):
    mlp = m.model.layers[1].mlp
    plain = mlp.forward
    mlp.forward = lambda x: 0.5 * plain(x)


def _parametrization(m):
    up = torch.nn.utils.parametrizations.weight_norm(m.model.layers[1].mlp.up_proj)
    with torch.no_grad():
        up.parametrizations.weight.original0.mul_(2)


STANDINS = {
    "adapter": lambda m: setattr(m.model.layers[0].mlp, "gate_proj", _Adapter(m.model.layers[0].mlp.gate_proj)),
    "bias": _bias,
    "subclass": _child,
    "instance forward": _instance_forward,
    "parametrization": _parametrization,
    "hook on a projection": lambda m: m.model.layers[0].mlp.gate_proj.register_forward_hook(lambda mod, a, out: 2 * out),
    "hook on the MLP": lambda m: m.model.layers[1].mlp.register_forward_pre_hook(lambda mod, a: (a[0] * 0.5,)),
    "hook on the first norm": lambda m: m.model.layers[0].input_layernorm.register_forward_hook(lambda mod, a, out: 2 * out),
    "hook on the second norm": lambda m: m.model.layers[0].post_attention_layernorm.register_forward_hook(
        lambda mod, a, out: 2 * out),
    "another last norm": lambda m: setattr(m.model, "norm", torch.nn.LayerNorm(256, device=DEV)),
    "hook on the last norm": lambda m: m.model.norm.register_forward_hook(lambda mod, a, out: 2 * out),
}


@pytest.mark.parametrize("what", STANDINS)
def test_packed_training_calls_what_is_there(cuda_ok, what):
    """With a module replaced or hooked, a packed training step is the step without packing: the logits alike to fp32 rounding
    through two layers, a gradient for the same parameters, and near it (a kept value is within 2^-4 and a term of a gradient
    has at most four of them)."""
    ids = torch.randint(0, 384, (2, 48), generator=torch.Generator().manual_seed(2)).to(DEV)
    m = _model()
    before = m(ids).logits.detach()
    STANDINS[what](m)
    got = []
    for packed in (False, True):
        m.enable_packed_training(packed)
        m.zero_grad(set_to_none=True)
        out = m(ids, labels=ids)
        out.loss.backward()
        got.append((out.logits.detach(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}))
    (plain, ref), (logits, grads) = got
    change = float((plain - before).norm())
    assert change > 0  # the stand-in does something
    # the sparse selection may differ in a row for a rounding's sake; the stand-in's own effect is far larger
    assert float((logits - plain).norm()) < 0.01 * change
    assert grads.keys() == ref.keys()
    for name, g in grads.items():
        assert float((g - ref[name]).norm()) <= 0.25 * float(ref[name].norm()), name


def test_backward_hooks_fire(cuda_ok):
    m = _model()
    m.enable_packed_training()
    seen = []
    m.model.layers[0].mlp.register_full_backward_hook(lambda mod, gi, go: seen.append("mlp"))
    m.model.layers[0].post_attention_layernorm.register_full_backward_pre_hook(lambda mod, go: seen.append("norm"))
    ids = torch.randint(0, 384, (1, 32), generator=torch.Generator().manual_seed(2)).to(DEV)
    m(ids, labels=ids).loss.backward()
    assert sorted(seen) == ["mlp", "norm"]


# -- autocast -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_mlp_block_under_autocast(cuda_ok, dtype):
    """The block computes in its tensors' type whatever autocast says, forward and backward, inside its context or out."""
    import gsa_b200 as gsa

    rows, d, n = 24, 64, 96
    shapes = ((rows, d), (rows, d), (d,), (n, d), (n, d), (d, n))
    leaves = [_randn(i, *s, scale=s[-1] ** -0.5).requires_grad_(True) for i, s in enumerate(shapes)]
    dout = _randn(9, rows, d)
    out = gsa.packed_mlp_block(*leaves, 1e-5)
    want = torch.autograd.grad(out, leaves, dout)
    for inside in (False, True):
        with torch.autocast("cuda", dtype=dtype):
            got = gsa.packed_mlp_block(*leaves, 1e-5)
            # the residual stream keeps its type: the next norm takes it
            again = gsa.packed_add_rmsnorm(got, None, leaves[2], 1e-5)[1]
            if inside:
                grads = torch.autograd.grad(got, leaves, dout)
        if not inside:
            grads = torch.autograd.grad(got, leaves, dout)
        assert got.dtype == again.dtype == torch.float32 and torch.equal(got, out)
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_packed_training_under_autocast(cuda_ok):
    """An fp32 model's packed step under bf16 autocast (its backward pass inside the context, as the attention's needs it): a gradient
    for the same parameters as without packing, in their type, near it.  Kept values as above; the two differ by bf16 roundings in
    the MLP beside that, of 2^-8 a product."""
    ids = torch.randint(0, 384, (2, 48), generator=torch.Generator().manual_seed(2)).to(DEV)
    got = []
    for packed in (False, True):
        m = _model()
        m.enable_packed_training(packed)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = m(ids, labels=ids)
            out.loss.backward()
        assert bool(torch.isfinite(out.loss))
        got.append({n: p.grad for n, p in m.named_parameters() if p.grad is not None})
    assert got[0].keys() == got[1].keys()
    for name, g in got[1].items():
        ref = got[0][name]
        assert g.dtype == ref.dtype == torch.float32 and bool(torch.isfinite(g).all()), name
        assert float((g - ref).norm()) <= (0.25 + 8 * 2.0 ** -8) * float(ref.norm()), name


# -- derivatives that there are not -------------------------------------------------------------
def test_forward_mode_is_refused(cuda_ok):
    """A tangent is not dropped in silence, whether or not anything requires a gradient."""
    import gsa_b200 as gsa
    from torch.autograd import forward_ad as fw

    freq, _ = gsa.rotary_frequencies(16, device=DEV)
    pos = torch.arange(6, device=DEV)
    w = torch.ones(16, device=DEV)
    lab = torch.zeros(2, 6, device=DEV, dtype=torch.long)
    mats = [_randn(20 + i, *s) for i, s in enumerate(((8, 16), (8, 16), (16, 8)))]
    calls = {
        "rotary": lambda t: gsa.apply_rotary(t, None, pos, freq),
        "rotary k": lambda t: gsa.apply_rotary(_randn(2, 2, 6, 2, 16), t, pos, freq),
        "pack": lambda t: gsa.pack_activation(t),
        "silu": lambda t: gsa.packed_silu_mul(t),
        "norm": lambda t: gsa.packed_add_rmsnorm(t, None, w, 1e-5),
        "norm addend": lambda t: gsa.packed_add_rmsnorm(_randn(3, 2, 6, 2, 16), t, w, 1e-5),
        "block": lambda t: gsa.packed_mlp_block(t, None, w, *mats, 1e-5),
        "loss": lambda t: gsa.fused_next_token_loss(t[:, :, 0], lab),
    }
    for name, call in calls.items():
        for grad in (False, True):
            x = _randn(1, 2, 6, 2, 16).requires_grad_(grad)
            with fw.dual_level():
                dual = fw.make_dual(x, torch.ones_like(x))
                with pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                    call(dual)
                with torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError), match="forward|jvp"):
                    call(dual)
            call(x)  # and without one it is computed
    x = _randn(1, 2, 6, 2, 16)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            gsa.packed_add_rmsnorm(x, None, fw.make_dual(w, torch.ones_like(w)), 1e-5)
        with pytest.raises(NotImplementedError, match="forward"):
            gsa.apply_rotary(x, None, pos, fw.make_dual(freq, torch.ones_like(freq)))


def test_frequencies_have_no_gradient(cuda_ok):
    """Frequencies that want a gradient are refused rather than left without one."""
    import gsa_b200 as gsa

    freq, _ = gsa.rotary_frequencies(16, device=DEV)
    freq.requires_grad_(True)
    pos = torch.arange(6, device=DEV)
    for grad in (False, True):
        q = _randn(1, 2, 6, 2, 16).requires_grad_(grad)
        with pytest.raises(NotImplementedError, match="inv_freq"):
            gsa.apply_rotary(q, None, pos, freq)
        with torch.no_grad():
            gsa.apply_rotary(q, None, pos, freq)
        gsa.apply_rotary(q, None, pos, freq.detach())


def test_tensors_with_a_graph_are_not_overwritten(cuda_ok):
    """Writing into a tensor that requires a gradient is refused while gradients are recorded, as torch's in-place operations
    refuse a leaf; without recording it is done."""
    import gsa_b200 as gsa

    freq, _ = gsa.rotary_frequencies(16, device=DEV)
    pos = torch.arange(6, device=DEV)
    q, k = _randn(1, 2, 6, 2, 16), _randn(2, 2, 6, 2, 16)
    leaf = torch.zeros_like(q).requires_grad_(True)
    inner = leaf * 2
    for outs in ((leaf, torch.empty_like(k)), (torch.empty_like(q), inner)):
        with pytest.raises(NotImplementedError, match="without autograd"):
            gsa.apply_rotary(q, k, pos, freq, out=outs)
    for t in (leaf, inner):
        assert bool((t.detach() == 0).all())
        with pytest.raises(NotImplementedError, match="without autograd"):
            gsa.ops.scale_(t, torch.full((1,), 2.0, device=DEV))
    want = gsa.apply_rotary(q, None, pos, freq)[0]
    with torch.no_grad():
        gsa.apply_rotary(q, None, pos, freq, out=(leaf, None))
    assert torch.equal(leaf.detach(), want)
