"""Group normalisation where its numbers are hardest to keep: the tails of the smooth activations, and sums over long
maps.  u = 2^-24 is half a unit of float32."""
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    """A dual tensor needs no gradient of its own, so it has to be looked for: its tangent must not get lost."""
    from mmsa_amd.norm import GroupNormAct, group_norm_act
    x, t = torch.randn(2, 8, 5, device=DEV), torch.randn(2, 8, 5, device=DEV)
    w = torch.ones(8, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, t)
        for args in ((dual, 2), (x, 2, torch.autograd.forward_ad.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(RuntimeError, match="jvp|forward"):
                group_norm_act(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp|forward"):
                group_norm_act(*args)
        # plain tensors pass at such a level, with and without a gradient
        plain = group_norm_act(x, 2, w)
    assert torch.equal(plain, group_norm_act(x, 2, w))
    m = GroupNormAct(2, 8).to(DEV)
    with torch.autograd.forward_ad.dual_level():
        y = m(x)
    assert y.requires_grad
