"""Forward-mode derivatives, which the operators do not have: a call on a dual tensor says so instead of returning a
result without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from vmonarch_b200 import PackedSequences, gated_residual_norm, packed_attention

pytestmark = pytest.mark.gpu


def rows(*shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch.bfloat16)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_packed_attention_refuses_duals(which, grad):
    x = [rows(40, 2, 64) for _ in range(3)]
    seqs = PackedSequences([30, 10])
    want = packed_attention(*x, seqs)
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        assert torch.equal(packed_attention(*x, seqs), want)  # no dual among the inputs
        x[which] = fwad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward"):
            packed_attention(*x, seqs)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["x", "y", "gate", "scale", "shift", "weight", "post_weight"])
def test_gated_norm_refuses_duals(name, grad):
    t = dict(x=rows(9, 64), y=rows(9, 64), **{n: rows(1, 64) for n in ("gate", "scale", "shift")}, weight=rows(64),
             post_weight=rows(64))
    want = gated_residual_norm(**t)
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        for a, b in zip(gated_residual_norm(**t), want):
            assert torch.equal(a, b)
        t[name] = fwad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match="forward"):
            gated_residual_norm(**t)
