"""Group normalisation where its numbers are hardest to keep: the tails of the smooth activations, and sums over long
maps.  u = 2^-24 is half a unit of float32."""
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24


def pointwise64(z, act):
    """The activation and its slope in 64 bits, each with the bound of a good 32-bit evaluation's error at 32-bit z and
    of a 16-bit map's.

    Phi(z) is erfc(-z / sqrt 2) / 2: its argument carries two roundings, which z < 0 magnifies by z^2 + 1, erfc itself
    4 u.  exp(-z^2 / 2) rounds its argument (z^2 / 2 of it) and itself.  sigmoid: exp 2 u, sum u, quotient u.  For 16-bit
    maps the normal tail is a polynomial good to 4e-6 of it, and exponentials take their argument times log2 e (three
    roundings of it)."""
    z = z.double()
    if act == "silu":
        s = torch.sigmoid(z)
        y, slope = z * s, s * (1 + z * (1 - s))
        r32, r16 = 8 * U * torch.ones_like(z), (2 * z.abs() + 10) * U
        return y, slope, [(r * y.abs(), r * (slope.abs() + s * (1 + z.abs()))) for r in (r32, r16)]
    phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    hill = z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    y, slope = z * phi, phi + hill
    r32, r16 = (2 * z * z + 10) * U, 4e-6 + (1.5 * z * z + 12) * U
    return y, slope, [(r * y.abs(), r * (phi + hill.abs())) for r in (r32, r16)]


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [2, 3000])                       # in registers, and cut into chunks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_keep_their_digits_in_the_tails(act, dtype, positions):
    """A weight of zero puts every channel's value at its bias, so that the activation and (as the bias gradient of one
    unit in one place) its slope can be read off: relative accuracy from -12 to 12."""
    from mmsa_amd.norm import group_norm_act
    C = 1024
    z = torch.linspace(-12, 12, C, device=DEV)
    x = torch.randn(1, positions, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dtype)
    bias = z.clone().requires_grad_()
    y = group_norm_act(x.transpose(1, 2), 1, torch.zeros(C, device=DEV), bias, 1e-5, act)
    dy = torch.zeros_like(y)
    dy[0, :, 0] = 1
    slope, = torch.autograd.grad(y, bias, dy)
    want, want_slope, bounds = pointwise64(z, act)
    ey, es = bounds[0 if dtype == torch.float32 else 1]
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    off = (y.detach().double() - want.view(1, C, 1)).abs()
    assert bool((off <= (ey + half * want.abs() + tiny).view(1, C, 1)).all()), \
        float((off / (ey + half * want.abs() + tiny).view(1, C, 1)).max())
    off = (slope.double() - want_slope).abs()
    assert bool((off <= es).all()), float((off / es).max())


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_module_converted_to_16_bits(dtype):
    """model.to(bfloat16) converts the parameters too: they are taken at their values, and their gradients come in their
    type."""
    from mmsa_amd.norm import GroupNormAct, group_norm_act
    torch.manual_seed(3)
    m = GroupNormAct(4, 24, activation="silu").to(DEV)
    with torch.no_grad():
        m.weight.normal_(1, 0.2)
        m.bias.normal_(0, 0.2)
    m.to(dtype)
    x = torch.randn(3, 24, 7, 9, device=DEV, dtype=dtype, requires_grad=True)
    dy = torch.randn(3, 24, 7, 9, device=DEV, dtype=dtype)
    w, b = (p.detach().float().requires_grad_() for p in (m.weight, m.bias))
    want = group_norm_act(x, 4, w, b, 1e-5, "silu")
    got = m(x)
    assert got.dtype == dtype and torch.equal(got, want)
    for g, v in zip(torch.autograd.grad(got, (x, m.weight, m.bias), dy), torch.autograd.grad(want, (x, w, b), dy)):
        assert g.dtype == dtype and torch.equal(g, v.to(dtype))
    with pytest.raises(TypeError):                       # 64 bits would be narrowed
        m.double()(x)


def test_channel_counts_that_32_bits_cannot_hold_are_refused():
    from mmsa_amd import _lib, ops
    for C in (2 ** 31, 2 ** 32 + 8):
        with pytest.raises(_lib.MmsaError, match="limit"):
            ops._group_norm_check(C, 1, "none", None, None, 0)
