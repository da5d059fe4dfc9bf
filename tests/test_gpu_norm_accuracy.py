"""Group normalisation where its numbers are hardest to keep: the tails of the smooth activations, and sums over long
maps.  u = 2^-24 is half a unit of float32."""
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24


LONG = (1, 2 ** 24, 64, 8)          # one sample of 2^30 float32 values: a thread walks about a thousand rows of its block


@pytest.mark.gpu
def test_statistics_of_a_long_map_whose_first_rows_stand_apart():
    """The first rows, from which every thread takes its origin, are 0 and all others 0.7.  In a run of 64 rows about
    that origin the sum of squares 63 c^2 rounds to 64 u of itself at most, against a thread's whole sum of squares about
    its mean of c^2: 64 * 64 u of the variance.  Later runs have an origin among their own values; sixteen of them are
    joined in 32 bits, then all threads in 64.  The mean: a run's sum 64 u, sixteen joins, its own rounding."""
    import mmsa_amd.torch_ops  # noqa: F401
    B, P, C, G = LONG
    x = torch.full((B, P, C), 0.7, device=DEV)
    x[:, :P // 1024] = 0
    y, stats = torch.empty_like(x), torch.empty(B, G, 2, dtype=torch.float64, device=DEV)
    torch.ops.mmsa.group_norm_act_fwd(x, None, None, y, stats, G, 0.0, "none")
    c, share = x[0, -1, 0].double().item(), 1 / 1024
    assert float((stats[..., 0] / (c * (1 - share)) - 1).abs().max()) <= 84 * U
    var = stats[..., 1] ** -2
    assert float((var / (c * c * share * (1 - share)) - 1).abs().max()) <= 64 * 68 * U


@pytest.mark.gpu
def test_parameter_gradients_of_a_long_map():
    """Sums of equal addends, the case in which a long chain of 32-bit additions drifts: runs of 64 rows (64 u at most),
    sixteen runs a thread (16 u), the rest in 64 bits with a rounding of each chunk's and the final sum; rstd's own 2 u."""
    import mmsa_amd.torch_ops  # noqa: F401
    B, P, C, G = LONG
    sign = torch.ones(P, device=DEV)
    sign.view(-1, 2, P // 1024)[:, 1] = -1                # whole rows of one sign: mean 0, variance 1, both exact
    x = sign.view(1, P, 1).expand(B, P, C).contiguous()
    y, stats = torch.empty_like(x), torch.empty(B, G, 2, dtype=torch.float64, device=DEV)
    torch.ops.mmsa.group_norm_act_fwd(x, None, None, y, stats, G, 1e-5, "none")
    dw, db = torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    dy = torch.full_like(y, 0.7)
    c = dy[0, 0, 0].double().item()
    torch.ops.mmsa.group_norm_act_bwd(dy, x, None, None, stats, None, dw, db, G, "none")
    assert float((db.double() / (c * P) - 1).abs().max()) <= 84 * U
    torch.mul(x, 0.7, out=dy)
    torch.ops.mmsa.group_norm_act_bwd(dy, x, None, None, stats, None, dw, db, G, "none")
    assert float((dw.double() / (c * P / math.sqrt(1 + 1e-5)) - 1).abs().max()) <= 88 * U


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
