"""Group normalisation with an activation (mmsa_amd.norm, torch.ops.mmsa.group_norm_act_*) against its formulas in
64 bits.  u = 2^-24 is half a unit of float32; the coefficients count roundings: a value passes through about a dozen
32-bit operations, a thread sums at most 32 values and a block at most 512 such sums before they are joined in 64 bits."""
import math

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def act64(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def formula(x, w, b, groups, eps, act, dy=None):
    """x [B, P, C] float64; returns y (dx, dw, db) and the bounds of their 32-bit roundings."""
    B, P, C = x.shape
    xg = x.view(B, P, groups, C // groups)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    var = (xg - mean).square().mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = ((xg - mean) * rstd).view(B, P, C)
    mr = (mean.abs() * rstd).expand(B, 1, groups, C // groups).reshape(B, 1, C)
    z = xh * w + b
    y, slope = act64(z, act)
    # |error of z|: a dozen roundings of the product, the mean's own rounding, the statistics' summation
    ez = U * (48 * (xh * w).abs() + 4 * mr * w.abs() + 48 * w.abs() + 4 * b.abs())
    ey = 1.2 * ez + 12 * U * (z.abs() + 1) * (act in ("silu", "gelu"))
    if dy is None:
        return y, ey
    dz = dy * slope
    q = dz * w

    def gm(t):
        return t.view(B, P, groups, -1).mean(dim=(1, 3), keepdim=True).expand(B, 1, groups, C // groups).reshape(B, 1, C)
    r = rstd.expand(B, 1, groups, C // groups).reshape(B, 1, C)
    dx = r * (q - gm(q) - xh * gm(q * xh))
    smooth = act in ("silu", "gelu")
    eslope = (1.2 * ez + 16 * U * (1 + z.abs())) * smooth
    exh = U * (48 * xh.abs() + 4 * mr + 48)
    edz = dy.abs() * eslope + 4 * U * dz.abs()
    eq = edz * w.abs() + 4 * U * q.abs()
    edx = r * (eq + gm(eq) + xh.abs() * gm(eq * xh.abs() + q.abs() * exh) + exh * gm((q * xh).abs())
               + 600 * U * (gm(q.abs()) + xh.abs() * gm((q * xh).abs()))) + 64 * U * dx.abs()
    dw, db = (dz * xh).sum((0, 1)), dz.sum((0, 1))
    edw = (edz * xh.abs() + dz.abs() * exh + 600 * U * (dz * xh).abs()).sum((0, 1))
    edb = (edz + 600 * U * dz.abs()).sum((0, 1))
    return (y, ey), (dx, edx), (dw, edw), (db, edb)


def within(got, want, bound, dtype=torch.float32):
    """|got - want| <= bound + half a unit of the output type."""
    g = got.double()
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    tol = bound * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + tiny
    bad = (g - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((g - want).abs() - tol).max()), float(tol.min()))


def data(B, P, C, dtype, seed=0, offset=0.5, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(B, P, C, device=DEV, generator=g) * scale
         + offset * torch.randn(C, device=DEV, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(C, device=DEV, generator=g)
    b = 0.3 * torch.randn(C, device=DEV, generator=g)
    dy = torch.randn(B, P, C, device=DEV, generator=g).to(dtype)
    return x, w, b, dy


SIZES = [  # B, P, C, groups
    (1, 1, 8, 1), (1, 1, 8, 8), (2, 3, 1, 1), (3, 7, 5, 1), (2, 9, 12, 4), (1, 128, 256, 32), (3, 1961, 60, 12),
    (5, 33, 61, 61), (2, 101, 999, 27), (2, 17, 1500, 10), (2, 40, 4096, 64), (300, 5, 24, 3), (2, 2080, 64, 8),
    (1, 40001, 20, 5), (4, 64, 40, 8), (1, 2, 2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients_match_the_formulas(size, dtype):
    from mmsa_amd.norm import group_norm_act
    B, P, C, G = size
    x, w, b, dy = data(B, P, C, DT[dtype], seed=P + C)
    for act in ("none", "relu", "silu", "gelu"):
        leaves = [t.detach().requires_grad_() for t in (x.transpose(1, 2), w, b)]
        y = group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, act)
        assert y.dtype == DT[dtype] and y.shape == (B, C, P)
        dx, dw, db = torch.autograd.grad(y, leaves, dy.transpose(1, 2))
        want = formula(x.double(), w.double(), b.double(), G, 1e-5, act, dy.double())
        within(y.detach().transpose(1, 2), *want[0], DT[dtype])
        within(dx.transpose(1, 2), *want[1], DT[dtype])
        within(dw, *want[2])
        within(db, *want[3])
        with torch.no_grad():
            assert torch.equal(group_norm_act(x.transpose(1, 2), G, w, b, 1e-5, act), y)


@pytest.mark.gpu
def test_odd_channel_counts_up_to_the_limit_and_beyond():
    from mmsa_amd import _lib
    from mmsa_amd.norm import group_norm_act
    x, w, b, _ = data(2, 19, 1535, torch.bfloat16)
    y = group_norm_act(x.transpose(1, 2), 5, w, b)
    within(y.transpose(1, 2), *formula(x.double(), w.double(), b.double(), 5, 1e-5, "none"), torch.bfloat16)
    for C, dtype in ((1537, torch.bfloat16), (4097, torch.float32)):
        with pytest.raises(_lib.MmsaError, match="limit"):
            group_norm_act(torch.zeros(1, C, 4, device=DEV, dtype=dtype), 1)


@pytest.mark.gpu
def test_memory_orders_give_the_same_values():
    from mmsa_amd.norm import GroupNormAct, group_norm_act
    torch.manual_seed(1)
    x = torch.randn(3, 32, 9, 11, device=DEV)
    w, b = torch.randn(32, device=DEV), torch.randn(32, device=DEV)
    cl = x.to(memory_format=torch.channels_last)
    y = group_norm_act(cl, 4, w, b, 1e-5, "silu")
    assert y.is_contiguous(memory_format=torch.channels_last)
    big = torch.randn(3, 48, 9, 22, device=DEV)
    big[:, 8:40, :, ::2] = x
    for other in (x, big[:, 8:40, :, ::2], x.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(group_norm_act(other, 4, w, b, 1e-5, "silu"), y)
    m = GroupNormAct(4, 32, activation="silu").to(DEV)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    assert torch.equal(m(cl), y) and list(m.state_dict()) == ["weight", "bias"]
    # a gradient that arrives in another order
    xr = cl.detach().requires_grad_()
    g = torch.randn(3, 32, 9, 11, device=DEV)
    a, = torch.autograd.grad(group_norm_act(xr, 4, w, b, 1e-5, "silu"), xr, g)
    c, = torch.autograd.grad(group_norm_act(xr, 4, w, b, 1e-5, "silu"), xr, g.to(memory_format=torch.channels_last))
    assert torch.equal(a, c)
    # rank 2 (no positions) and rank 5
    v = torch.randn(5, 32, device=DEV)
    within(group_norm_act(v, 4, w, b).view(5, 1, 32), *formula(v.double().view(5, 1, 32), w.double(), b.double(), 4,
                                                               1e-5, "none"))
    assert group_norm_act(torch.randn(2, 8, 3, 4, 5, device=DEV), 2).shape == (2, 8, 3, 4, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["x", "weight", "bias", "none_affine"])
def test_only_the_wanted_gradients(way):
    from mmsa_amd.norm import group_norm_act
    x, w, b, dy = data(3, 50, 24, torch.float32)
    want = formula(x.double(), w.double(), b.double(), 3, 1e-5, "gelu", dy.double())
    if way == "none_affine":
        xr = x.detach().requires_grad_()
        y = group_norm_act(xr.transpose(1, 2), 3, None, None, 1e-5, "gelu")
        one, zero = torch.ones_like(w).double(), torch.zeros_like(b).double()
        want = formula(x.double(), one, zero, 3, 1e-5, "gelu", dy.double())
        within(torch.autograd.grad(y, xr, dy.transpose(1, 2))[0], *want[1])
        return
    leaf = {"x": x, "weight": w, "bias": b}[way].detach().requires_grad_()
    args = {"x": x, "weight": w, "bias": b, way: leaf}
    y = group_norm_act(args["x"].transpose(1, 2), 3, args["weight"], args["bias"], 1e-5, "gelu")
    within(torch.autograd.grad(y, leaf, dy.transpose(1, 2))[0], *want[{"x": 1, "weight": 2, "bias": 3}[way]])


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional derivative of a 64-bit sum of the 32-bit outputs: central differences, h^2 truncation of order 1e-4."""
    from mmsa_amd.norm import group_norm_act
    x, w, b, dy = data(2, 300, 24, torch.float32, seed=3)
    v = torch.randn_like(x)
    xr = x.detach().requires_grad_()
    dx, = torch.autograd.grad(group_norm_act(xr.transpose(1, 2), 3, w, b, 1e-5, "silu"), xr, dy.transpose(1, 2))
    h = 2.0 ** -7

    def loss(t):
        return float((group_norm_act(t.transpose(1, 2), 3, w, b, 1e-5, "silu").transpose(1, 2).double() * dy.double()).sum())
    diff = (loss(x + h * v) - loss(x - h * v)) / (2 * h)
    got = float((dx.double() * v.double()).sum())
    scale = float((dx.double() * v.double()).norm())
    # truncation h^2/6 of a third derivative of order one per element, and the roundings of the two sums over 2 h
    assert abs(diff - got) <= scale * (h * h * 4 + 64 * U / h), (diff, got, scale)


@pytest.mark.gpu
def test_a_mean_far_above_the_spread():
    """mean = 4096 spreads: the statistics lose nothing, the only loss is the float32 input's own grid and the mean's
    rounding (4 mr in the bound)."""
    from mmsa_amd.norm import group_norm_act
    x = 4096.0 + torch.randn(2, 5000, 16, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    w, b = torch.ones(16, device=DEV), torch.zeros(16, device=DEV)
    within(group_norm_act(x.transpose(1, 2), 2, w, b).transpose(1, 2),
           *formula(x.double(), w.double(), b.double(), 2, 1e-5, "none"))
    # an outlier as the very first value
    x[:, 0, :] = -1e6
    within(group_norm_act(x.transpose(1, 2), 2, w, b).transpose(1, 2),
           *formula(x.double(), w.double(), b.double(), 2, 1e-5, "none"))


@pytest.mark.gpu
def test_relu_decides_its_side_of_zero_in_64_bits():
    """Four million values, of which several lie within a float32 rounding of the border: every gradient element is on
    the side the 64-bit formula puts it (an element on the wrong side would be off by its whole size)."""
    from mmsa_amd.norm import group_norm_act
    x, w, b, dy = data(8, 8192, 64, torch.float32, seed=11)
    xr = x.detach().requires_grad_()
    dx, = torch.autograd.grad(group_norm_act(xr.transpose(1, 2), 8, w, b, 1e-5, "relu"), xr, dy.transpose(1, 2))
    within(dx, *formula(x.double(), w.double(), b.double(), 8, 1e-5, "relu", dy.double())[1])
    # a constant group sits exactly on the border: no gradient passes
    c = torch.full((1, 8, 40), 2.0, device=DEV, requires_grad=True)
    one = torch.ones(8, device=DEV, requires_grad=True)
    y = group_norm_act(c, 2, one, torch.zeros(8, device=DEV), 1e-5, "relu")
    g = torch.autograd.grad(y, (c, one), torch.randn(1, 8, 40, device=DEV))
    assert float(y.detach().abs().max()) == 0.0 and float(g[0].abs().max()) == 0.0 and float(g[1].abs().max()) == 0.0


@pytest.mark.gpu
def test_a_nan_or_infinity_stays_in_its_group():
    from mmsa_amd.norm import group_norm_act
    for act in ("none", "relu", "silu", "gelu"):
        x, w, b, _ = data(3, 70, 16, torch.float32)
        clean = group_norm_act(x.transpose(1, 2), 4, w, b, 1e-5, act)
        x[1, 5, 6] = float("nan")
        x[2, 69, 15] = float("inf")
        y = group_norm_act(x.transpose(1, 2), 4, w, b, 1e-5, act)
        hit = torch.zeros_like(y, dtype=torch.bool)
        hit[1, 4:8] = True
        hit[2, 12:] = True
        assert torch.equal(y[~hit], clean[~hit])
        assert bool(y[1, 4:8].isnan().all()) and bool(y[2, 12:].isnan().all())


@pytest.mark.gpu
def test_empty_maps():
    from mmsa_amd.norm import group_norm_act
    w = torch.ones(8, device=DEV, requires_grad=True)
    for shape in ((0, 8, 4, 4), (3, 8, 0), (0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = group_norm_act(x, 2, w, None, 1e-5, "relu")
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros(shape, device=DEV))
        assert gx.shape == shape and float(gw.abs().max()) == 0.0


@pytest.mark.gpu
def test_results_do_not_depend_on_other_samples_or_repetition():
    from mmsa_amd.norm import group_norm_act
    x, w, b, dy = data(7, 777, 20, torch.bfloat16)
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()

    def both():
        y = group_norm_act(xr.transpose(1, 2), 4, wr, b, 1e-5, "silu")
        return [y.detach(), *torch.autograd.grad(y, (xr, wr), dy.transpose(1, 2))]
    a, c = both(), both()
    assert all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.gpu
def test_another_stream_and_a_replayed_graph():
    from mmsa_amd.norm import group_norm_act
    x, w, b, dy = data(4, 500, 32, torch.float32)
    xr, wr, br = (t.detach().requires_grad_() for t in (x, w, b))

    def both():
        y = group_norm_act(xr.transpose(1, 2), 4, wr, br, 1e-5, "relu")
        return [y.detach(), *torch.autograd.grad(y, (xr, wr, br), dy.transpose(1, 2))]
    want = both()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            got = both()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        held = both()
    for k in range(4):
        with torch.no_grad():
            xr.copy_(x * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        eager = both()
        assert all(torch.equal(p, q) for p, q in zip(eager, held)), k


@pytest.mark.gpu
def test_operators_write_into_the_callers_tensors():
    import mmsa_amd.torch_ops  # noqa: F401
    x, w, b, dy = data(2, 90, 16, torch.float16)
    y, stats = torch.empty_like(x), torch.empty(2, 4, 2, dtype=torch.float64, device=DEV)
    torch.ops.mmsa.group_norm_act_fwd(x, w, b, y, stats, 4, 1e-5, "gelu")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    torch.ops.mmsa.group_norm_act_bwd(dy, x, w, b, stats, dx, dw, db, 4, "gelu")
    want = formula(x.double(), w.double(), b.double(), 4, 1e-5, "gelu", dy.double())
    for got, (val, err), dt in zip((y, dx, dw, db), want, (torch.float16, torch.float16, torch.float32, torch.float32)):
        within(got, val, err, dt)
    mean = x.double().view(2, 90, 4, 4).mean(dim=(1, 3))
    assert float((stats[..., 0] - mean).abs().max()) < 64 * U


@pytest.mark.gpu
def test_more_than_two_to_the_31_values():
    from mmsa_amd.norm import group_norm_act
    C, P = 64, 2 ** 25 + 3
    row = torch.arange(1021 * C, device=DEV).remainder(251).view(1021, C).to(torch.bfloat16)   # exact in 8 bits
    x = torch.empty(1, P, C, device=DEV, dtype=torch.bfloat16)
    whole = P // 1021 * 1021
    x[0, :whole].view(-1, 1021, C).copy_(row)
    x[0, whole:] = row[:P - whole]
    y = group_norm_act(x.transpose(1, 2), 4).transpose(1, 2)[0]
    n = float(P) * 16
    r = row.double().view(1021, 4, 16)
    tail = r[:P - whole]
    mean = (r.sum((0, 2)) * (P // 1021) + tail.sum((0, 2))) / n
    sq = ((r - mean[:, None]).square().sum((0, 2)) * (P // 1021) + (tail - mean[:, None]).square().sum((0, 2))) / n
    want = (r - mean[:, None]) / torch.sqrt(sq[:, None] + 1e-5)
    # statistics: a thread sums a few hundred values here, hence 512 u of a spread
    for lo in (0, whole - 1021, whole // 2 // 1021 * 1021):
        within(y[lo:lo + 1021].view(1021, 4, 16), want, 1024 * U * (1 + want.abs()), torch.bfloat16)
    within(y[whole:].view(-1, 4, 16), want[:P - whole], 1024 * U * (1 + want[:P - whole].abs()), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(3, 6, 8, 4), (2, 4096, 64, 2)])          # in registers, and cut
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_closed_relu_lets_no_infinity_or_nan_of_dy_through(size, bad):
    from mmsa_amd.norm import group_norm_act
    B, P, C, G = size
    x, w, b, dy = data(B, P, C, torch.float32, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x.transpose(1, 2), w, b)]
    y = group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, "relu")
    clean = torch.where(y.detach() > 0, dy.transpose(1, 2), 0.0)
    dirty = torch.where(y.detach() > 0, dy.transpose(1, 2), bad)
    want = torch.autograd.grad(y, leaves, clean, retain_graph=True)
    got = torch.autograd.grad(y, leaves, dirty)
    for g, v in zip(got, want):
        assert torch.equal(g, v)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from mmsa_amd import _lib
    from mmsa_amd.norm import group_norm_act
    x = torch.zeros(2, 8, 4, device=DEV)
    with pytest.raises(_lib.MmsaError, match="cpu"):
        group_norm_act(x, 2, torch.ones(8))
    with pytest.raises(TypeError):
        group_norm_act(x.double(), 2)
    with pytest.raises(TypeError):
        group_norm_act(x, 2, torch.ones(8, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        group_norm_act(x, 2, torch.ones(16, device=DEV)[::2])
    for groups in (0, 3, -2):
        with pytest.raises(ValueError):
            group_norm_act(x, groups)
    with pytest.raises(RuntimeError):                    # no gradient of a gradient
        y = x.clone().requires_grad_()
        g, = torch.autograd.grad(group_norm_act(y, 2).sum(), y, create_graph=True)
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(2, 1500, 256, 1), (2, 1500, 260, 2), (3, 700, 195, 3), (2, 4096, 64, 32),
                                  (40, 600, 66, 33), (1, 9000, 1024, 8), (5, 300, 128, 2)])
def test_groups_of_many_and_of_two_channels(size, dtype):
    """More than 64 channels a group, groups that are no multiple of 64 or of a vector, and groups of two channels over
    many positions: the ways in which the sums of chunks are joined."""
    from mmsa_amd.norm import group_norm_act
    B, P, C, G = size
    x, w, b, dy = data(B, P, C, dtype, seed=C)
    leaves = [t.detach().requires_grad_() for t in (x.transpose(1, 2), w, b)]
    y = group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, "silu")
    got = torch.autograd.grad(y, leaves, dy.transpose(1, 2))
    want = formula(x.double(), w.double(), b.double(), G, 1e-5, "silu", dy.double())
    within(y.detach().transpose(1, 2), *want[0], dtype)
    within(got[0].transpose(1, 2), *want[1], dtype)
    within(got[1], *want[2])
    within(got[2], *want[3])


@pytest.mark.gpu
def test_more_values_than_32_bits_count():
    """33 samples of 2^26 values, 2.2 billion in all: the first and the last sample against the formula."""
    from mmsa_amd.norm import group_norm_act
    B, P, C, G = 33, 1 << 20, 64, 8
    x = torch.randn(B, P, C, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(B, P, C, device=DEV, dtype=torch.bfloat16)
    w, b = torch.linspace(0.5, 1.5, C, device=DEV), torch.linspace(-1.0, 1.0, C, device=DEV)
    leaf = x.transpose(1, 2).requires_grad_()
    y = group_norm_act(leaf, G, w, b, 1e-5, "silu")
    dx, = torch.autograd.grad(y, leaf, dy.transpose(1, 2))
    for i in (0, B - 1):
        want = formula(x[i:i + 1].detach().double(), w.double(), b.double(), G, 1e-5, "silu", dy[i:i + 1].double())
        within(y[i:i + 1].detach().transpose(1, 2), *want[0], torch.bfloat16)
        within(dx[i:i + 1].transpose(1, 2), *want[1], torch.bfloat16)


@pytest.mark.gpu
def test_a_batch_of_many_tiny_samples_and_one_of_few_long_ones():
    """The two ends of how a map is cut: 20 000 blocks of one row, and one sample that a whole launch shares."""
    from mmsa_amd.norm import group_norm_act
    for size in ((20000, 1, 16, 4), (20000, 3, 6, 2), (1, 300000, 8, 8)):
        B, P, C, G = size
        x, w, b, dy = data(B, P, C, torch.bfloat16, seed=C)
        leaves = [t.detach().requires_grad_() for t in (x.transpose(1, 2), w, b)]
        y = group_norm_act(leaves[0], G, leaves[1], leaves[2], 1e-5, "relu")
        got = torch.autograd.grad(y, leaves, dy.transpose(1, 2))
        want = formula(x.double(), w.double(), b.double(), G, 1e-5, "relu", dy.double())
        within(y.detach().transpose(1, 2), *want[0], torch.bfloat16)
        within(got[0].transpose(1, 2), *want[1], torch.bfloat16)
        # a thread of the long sample sums up to 40 values here, a block up to 512 of those: within the 600 u counted
        within(got[1], *want[2])
        within(got[2], *want[3])


def test_refusals():
    from mmsa_amd import _lib, ops
    from mmsa_amd.norm import GroupNormAct, group_norm_act
    lib = _lib.load()
    with pytest.raises(_lib.MmsaError, match="GPU"):
        group_norm_act(torch.zeros(2, 8, 4), 2)
    with pytest.raises(ValueError):
        group_norm_act(torch.zeros(8), 2)
    with pytest.raises(ValueError):
        GroupNormAct(3, 8)
    with pytest.raises(ValueError):
        GroupNormAct(2, 8, activation="tanh")
    with pytest.raises(ValueError):
        GroupNormAct(2, 8)(torch.zeros(2, 6, 4))
    x = torch.zeros(2, 4, 8)
    st = torch.zeros(2, 2, 2, dtype=torch.float64)
    for bad in (dict(groups=3), dict(groups=0), dict(act="tanh"), dict(gamma=torch.zeros(7)), dict(x=torch.zeros(2, 8)),
                dict(y=torch.zeros(2, 4, 9)), dict(stats=torch.zeros(2, 3, 2, dtype=torch.float64))):
        kw = dict(x=x, gamma=None, beta=None, y=torch.zeros(2, 4, 8), stats=st, groups=2)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.group_norm_act_fwd(**kw)
    with pytest.raises(TypeError):
        ops.group_norm_act_fwd(x.double(), None, None, x.double(), st, 2)
    with pytest.raises(_lib.MmsaError, match="GPU"):
        ops.group_norm_act_fwd(x, None, None, x.clone(), st, 2)
    with pytest.raises(ValueError):
        ops.group_norm_act_bwd(x, x, None, None, st, x[:1], None, None, 2)
    one = 1 << 12
    q = lib.mmsa_group_norm_act_scratch_bytes
    for backward in (0, 1):
        assert q(1, 1, 8, 3, 0, backward) == -1 and q(0, 1, 8, 2, 0, backward) == -1 and q(1, 1, 8, 2, 3, backward) == -1
        assert q(1, 1, 4097, 1, 0, backward) == -3 and q(5_000_000, 1, 8, 1, 0, backward) == -3
        assert q(1, 1, 1537, 1, 1, backward) == -3 and q(2, 100000, 64, 8, 1, backward) > 0
    assert q(2, 100, 64, 8, 1, 0) == 0 and q(2, 100, 64, 8, 1, 1) == 2 * 64 * 8      # a sample's groups fit a block each
    assert lib.mmsa_group_norm_act_fwd(one, None, None, one, None, None, 2, 100000, 64, 8, 1e-5, 0, 1, None) == -1
    assert lib.mmsa_group_norm_act_fwd(None, None, None, one, one, one, 1, 1, 8, 2, 1e-5, 0, 0, None) == -1
    assert lib.mmsa_group_norm_act_fwd(one, None, None, one, one, one, 1, 1, 8, 3, 1e-5, 0, 0, None) == -1
    assert lib.mmsa_group_norm_act_fwd(one, None, None, one, one, one, 1, 1, 8, 2, 1e-5, 4, 0, None) == -1
    assert lib.mmsa_group_norm_act_bwd(one, one, None, None, one, one, None, None, None, 1, 1, 8, 2, 0, 0, None) == -1
