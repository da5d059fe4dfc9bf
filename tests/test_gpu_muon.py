"""Newton-Schulz orthogonalisation and the Muon step (mmsa_amd.muon) against their formulas in 64 bits.

Tolerance of an orthogonalised matrix, relative in the Frobenius norm: one step's products round to about
u (4 + sqrt(K) / 4) (u = 2^-24: three roundings of the operand pairs and of the dropped low product, and partial sums
over K values whose errors add up at random); x -> a x + b x^3 + c x^5 passes an error on with a factor between 0 and
max|p'| = 4, about 2 in the mean, so five steps collect 1 + 2 + ... + 16 = 31 of them."""
import copy

import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
A, B, C = 3.4445, -4.775, 2.0315


def ns64(u, steps=5, eps=1e-7):
    x = u.double()
    x = x / max(float(x.norm()), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        s = x @ x.T
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.T if tall else x


def tol(shape, dtype=torch.float32, steps=5):
    k = max(shape)
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U
    return (2 ** steps - 1) * U * (4 + k ** 0.5 / 4) + half


def close(got, want, rel):
    """Frobenius distance; no single element further off than the whole may be (times its share, 16 over the mean)."""
    d = got.double() - want
    assert bool(torch.isfinite(got).all())
    size = float(want.norm())
    assert float(d.norm()) <= rel * size + 1e-300, (float(d.norm()), rel * size)
    assert float(d.abs().max()) <= rel * (16 * size / want.numel() ** 0.5 + float(want.abs().max())) + 1e-300


def grad(m, n, seed=0, dtype=torch.float32, scale=1e-3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = max(1, min(m, n) // 4)
    low = torch.randn(m, k, device=DEV, generator=g) @ torch.randn(k, n, device=DEV, generator=g) / k ** 0.5
    return ((low + 0.2 * torch.randn(m, n, device=DEV, generator=g)) * scale).to(dtype)


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (31, 33), (64, 64), (65, 64), (64, 65), (63, 200), (128, 128), (129, 257),
          (300, 70), (64, 288), (256, 2304), (1000, 130), (513, 513), (5, 5000), (640, 1100), (1537, 1023)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize_matches_the_formula(shape, dtype):
    from mmsa_amd.muon import orthogonalize
    g = grad(*shape, seed=sum(shape), dtype=dtype)
    o = orthogonalize(g)
    assert o.dtype == dtype and o.shape == g.shape and o.data_ptr() != g.data_ptr()
    close(o, ns64(g), tol(shape, dtype))
    assert torch.equal(o, orthogonalize(g))


@pytest.mark.gpu
@pytest.mark.parametrize("longest", [256, 257, 512, 513, 768, 769])
def test_lists_of_small_matrices(longest):
    """Up to 64 rows and 768 columns (or the transpose) a matrix is one block's work, if all of its list are; one longer
    matrix sends the list the general way."""
    from mmsa_amd.muon import muon_step, orthogonalize
    shapes = [(64, longest), (longest, 3), (1, 1), (33, 32), (50, 64), (64, 64), (17, 255)] + [(5 + i, 40) for i in range(30)]
    gs = [grad(*s, seed=i) for i, s in enumerate(shapes)]
    gs[3][7, 7] = float("nan")
    gs[4].zero_()
    for s, g, o in zip(shapes, gs, orthogonalize(gs)):
        if s == (33, 32):
            assert bool(o.isnan().all())
        elif s == (50, 64):
            assert float(o.abs().max()) == 0.0
        else:
            close(o, ns64(g), tol(s))
    for g, tiny in ((gs[0], 1e-9), (gs[1], 1e-12)):
        close(orthogonalize(g * tiny), ns64(g * tiny), tol(shapes[0]))
    p, m = gs[0].clone(), gs[0] * 0.5
    want, mom, o = muon64(p, gs[0], m, 0.02, 0.1, 0.9, True)
    muon_step([p], [gs[0]], [m], lr=0.02, weight_decay=0.1, momentum=0.9)
    assert float((p.double() - want).norm()) <= 0.02 * (tol(shapes[0]) + 248 * U) * float(o.norm()) + 4 * U * float(want.norm())
    assert float((m.double() - mom).abs().max()) <= 4 * U * float(gs[0].abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(65, 6000)], [(700, 700)], [(96, 20011)], [(130, 2600)], [(200, 30000)], [(385, 768)],
                                    [(128, 1152)] * 30, [(200, 64), (70, 3000), (520, 520), (66, 66), (3, 4000)],
                                    [(2600, 1300)]], ids=lambda v: "-".join("x".join(map(str, s)) for s in v[:5]))
def test_tiles_and_splits(shapes):
    """Sizes for which the symmetric products come in tiles of 32, 64 and 128, whole and with their K split, in one
    launch with others."""
    from mmsa_amd.muon import orthogonalize
    gs = [grad(*s, seed=sum(s) + i) for i, s in enumerate(shapes)]
    for s, g, o in zip(shapes, gs, orthogonalize(gs)):
        close(o, ns64(g), tol(s))


@pytest.mark.gpu
def test_a_large_matrix():
    from mmsa_amd.muon import orthogonalize
    for shape in ((2048, 2100), (4097, 700)):
        g = grad(*shape, seed=1)
        close(orthogonalize(g), ns64(g), tol(shape))


@pytest.mark.gpu
def test_a_list_gives_each_matrix_what_it_gets_alone():
    """More matrices than one set of launches takes, of very different sizes.  A tile size or a split of the long axis
    may differ with the company a matrix is in, so equality is to rounding; the same list twice gives the same bits."""
    from mmsa_amd.muon import orthogonalize
    shapes = [(1 + 13 * i % 90, 1 + 29 * i % 130) for i in range(55)] + [(700, 900), (64, 3000), (2000, 32)]
    gs = [grad(*s, seed=i) for i, s in enumerate(shapes)]
    os_ = orthogonalize(gs)
    for s, g, o in zip(shapes, gs, os_):
        close(o, ns64(g), tol(s))
    assert all(torch.equal(a, b) for a, b in zip(os_, orthogonalize(gs)))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 5, 8, 16])
def test_number_of_steps(steps):
    from mmsa_amd.muon import orthogonalize
    g = grad(70, 150, seed=steps)
    # beyond five steps the singular values wander inside [0.68, 1.2025], where errors stay what they are (|p'| < 2)
    close(orthogonalize(g, steps=steps), ns64(g, steps), 4 * tol((70, 150), steps=min(steps, 6)))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-12, 1e-9, 3e-8, 1e-7, 1.0, 1e15, 1e30])
def test_any_scale_of_the_input(scale):
    """Norms from far below eps (the matrix then only grows by a per step) to squares beyond float32's range."""
    from mmsa_amd.muon import orthogonalize
    g = grad(96, 160, seed=4, scale=1.0) * scale
    want = ns64(g)
    # results below the smallest normal float32 keep an absolute grid
    close(orthogonalize(g), want, tol((96, 160)) + 2.0 ** -149 * 96 / max(float(want.norm()), 1e-45))
    z = orthogonalize(torch.zeros(40, 70, device=DEV))
    assert float(z.abs().max()) == 0.0


@pytest.mark.gpu
def test_low_rank_and_orthogonal_inputs():
    from mmsa_amd.muon import orthogonalize
    u = torch.randn(200, 1, device=DEV) @ torch.randn(1, 300, device=DEV)
    # the empty directions hold the input's own rounding noise, which grows by a per step in either evaluation: 64-bit
    # rounding of the float32 product leaves it at u of the one strong direction, times a^5 = 485, over 200 directions
    got, want = orthogonalize(u), ns64(u)
    assert float((got.double() - want).norm()) <= (485 * U * 8 + tol((200, 300))) * float(want.norm())
    q, _ = torch.linalg.qr(torch.randn(128, 128, device=DEV, dtype=torch.float64))
    close(orthogonalize(q.float()), ns64(q.float()), tol((128, 128)))
    s = torch.linalg.svdvals(orthogonalize(grad(100, 300, seed=2)).double())
    assert float(s.max()) < 1.2025 * (1 + 1e-5) and float(s.min()) > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_nan_or_infinity_does_not_reach_the_other_matrices(bad):
    from mmsa_amd.muon import orthogonalize
    gs = [grad(64, 96, seed=i) for i in range(3)]
    clean = orthogonalize(gs)
    gs[1][5, 7] = bad
    o = orthogonalize(gs)
    assert torch.equal(o[0], clean[0]) and torch.equal(o[2], clean[2]) and bool(o[1].isnan().all())


@pytest.mark.gpu
def test_inputs_in_other_orders_and_in_place():
    from mmsa_amd import ops
    from mmsa_amd.muon import orthogonalize
    g = grad(90, 120, seed=9)
    o = orthogonalize(g)
    assert torch.equal(orthogonalize(g.T.contiguous().T), o)
    wide = torch.zeros(90, 240, device=DEV)
    wide[:, ::2] = g
    assert torch.equal(orthogonalize(wide[:, ::2]), o)
    same = g.clone()
    ops.orthogonalize([same], [same])
    assert torch.equal(same, o)
    pad = torch.zeros(90 * 120 + 1, device=DEV)            # a matrix that starts at no multiple of 16 bytes
    pad[1:] = g.flatten()
    assert torch.equal(orthogonalize(pad[1:].view(90, 120)), o)
    p = g.clone().requires_grad_()
    assert not orthogonalize(p).requires_grad
    assert orthogonalize([]) == []


def muon64(p, g, m, lr, wd, mu, nesterov):
    m = m.double() + (1 - mu) * (g.double() - m.double())
    u = g.double() + mu * (m - g.double()) if nesterov else m
    rows, cols = p.shape[0], p[0].numel()
    o = ns64(u.reshape(rows, cols)).view(p.shape)
    return p.double() * (1 - lr * wd) - lr * max(1.0, rows / cols) ** 0.5 * o, m, o


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_step_matches_the_formula(nesterov):
    from mmsa_amd.muon import muon_step
    shapes = [(64, 32, 3, 3), (128, 64, 1, 1), (128, 256, 5), (300, 40), (1, 50), (7, 1), (256, 1152)]
    torch.manual_seed(0)
    ps = [torch.randn(s, device=DEV) * 0.1 for s in shapes]
    gs = [torch.randn(s, device=DEV) * 1e-3 for s in shapes]
    ms = [torch.randn(s, device=DEV) * 1e-3 for s in shapes]
    p0, m0 = [p.clone() for p in ps], [m.clone() for m in ms]
    v0 = [p._version for p in ps]
    muon_step(ps, gs, ms, lr=0.02, weight_decay=0.1, momentum=0.95, nesterov=nesterov)
    for p, g, m, a, b, v in zip(ps, gs, ms, p0, m0, v0):
        want, mom, o = muon64(a, g, b, 0.02, 0.1, 0.95, nesterov)
        assert float((m.double() - mom).abs().max()) <= 4 * U * float(b.abs().max() + g.abs().max())
        rows, cols = a.shape[0], a[0].numel()
        rate = 0.02 * max(1.0, rows / cols) ** 0.5
        d = p.double() - want
        # update: orthogonalisation of a direction known to a few u; parameter: three roundings
        assert float(d.norm()) <= rate * (tol((rows, cols)) + 31 * 8 * U) * float(o.norm()) + 4 * U * float(a.norm())
        assert p._version > v


@pytest.mark.gpu
def test_optimizer_follows_the_formula_over_steps_and_a_scheduler():
    from mmsa_amd.muon import Muon
    torch.manual_seed(2)
    w = torch.nn.Parameter(torch.randn(48, 80, device=DEV) * 0.1)
    k = torch.nn.Parameter(torch.randn(32, 16, 3, 3, device=DEV) * 0.1)
    idle = torch.nn.Parameter(torch.randn(4, 4, device=DEV))
    idle0 = idle.detach().clone()
    opt = Muon([{"params": [w, idle]}, {"params": [k], "lr": 0.005, "nesterov": False}], lr=0.02, weight_decay=0.05)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda e: 1.0 / (1 + e))
    ref = [(w.detach().double(), torch.zeros_like(w).double()), (k.detach().double(), torch.zeros_like(k).double())]
    for it in range(3):
        opt.zero_grad()
        for p in (w, k):
            p.grad = torch.randn_like(p) * 1e-2
        ref = [muon64(r[0], p.grad, r[1], lr / (1 + it), 0.05, 0.95, nest)[:2]
               for r, p, lr, nest in zip(ref, (w, k), (0.02, 0.005), (True, False))]
        opt.step()
        sched.step()
    for p, (want, mom) in zip((w, k), ref):
        # three updates of entries below lr, each to the tolerance of its orthogonalisation, and three roundings each
        assert float((p.detach().double() - want).norm()) <= 3 * (0.02 * (tol((48, 144)) + 248 * U) * 8 + 4 * U * float(want.norm()))
        assert float((opt.state[p]["momentum_buffer"].double() - mom).abs().max()) <= 16 * U * float(mom.abs().max() + 0.05)
    assert torch.equal(idle, idle0) and idle not in opt.state
    # a state that travels through state_dict continues with the same bits (a copy, as through a file: torch's
    # load_state_dict adopts the tensors it is given, and two optimisers would update one momentum buffer)
    w2, k2, i2 = (torch.nn.Parameter(t.detach().clone()) for t in (w, k, idle))
    opt2 = Muon([{"params": [w2, i2]}, {"params": [k2]}])
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    for a, b in ((w, w2), (k, k2)):
        a.grad = torch.randn_like(a)
        b.grad = a.grad.clone()
    opt.step()
    opt2.step()
    assert torch.equal(w, w2) and torch.equal(k, k2)


@pytest.mark.gpu
def test_another_stream_two_streams_at_once_and_replayed_graphs():
    from mmsa_amd.muon import muon_step, orthogonalize
    gs = [grad(*s, seed=i) for i, s in enumerate([(64, 288), (256, 600), (1000, 64)])]
    want = orthogonalize(gs)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(3):
                last = orthogonalize(gs)
            got.append(last)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(want, g))
    # two graphs of the same operator, replayed side by side: their scratch is their own
    ps = [[torch.randn(g.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)) for g in gs]
          for i in range(2)]
    ms = [[torch.zeros_like(g) for g in gs] for _ in range(2)]
    eager = [[p.clone() for p in side_ps] for side_ps in ps]
    eager_m = [[m.clone() for m in side_ms] for side_ms in ms]
    graphs = []
    for p, m in zip(ps, ms):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            muon_step(p, gs, m, lr=0.02, weight_decay=0.01)
        graphs.append(graph)
    for k in range(4):
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        for p, m in zip(eager, eager_m):
            muon_step(p, gs, m, lr=0.02, weight_decay=0.01)
        torch.cuda.synchronize()
        for a, b in zip(ps + ms, eager + eager_m):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), k


@pytest.mark.gpu
def test_group_norm_blocks_trained_by_muon():
    """The two operators as they are used together: a small stack of the package's own layers (linear maps over
    positions on the HIP dense kernel, GroupNormAct between them), its gradients against 64 bits, then a Muon step."""
    from mmsa_amd.model import _LinearFn
    from mmsa_amd.muon import Muon
    from mmsa_amd.norm import GroupNormAct
    torch.manual_seed(5)
    Bn, P, Cin, Ch = 4, 60, 32, 64
    w1 = torch.nn.Parameter(torch.randn(Ch, Cin, device=DEV) * Cin ** -0.5)
    w2 = torch.nn.Parameter(torch.randn(Ch, Ch, device=DEV) * Ch ** -0.5)
    norms = [GroupNormAct(8, Ch, activation="silu").to(DEV) for _ in range(2)]
    opt = Muon([w1, w2], lr=0.02)
    x = torch.randn(Bn * P, Cin, device=DEV)
    t = torch.randn(Bn, Ch, device=DEV)

    def gn64(h, gamma, beta):
        z = torch.nn.functional.group_norm(h.view(Bn, P, Ch).transpose(1, 2), 8, gamma, beta, 1e-5)
        return torch.nn.functional.silu(z).transpose(1, 2).reshape(Bn * P, Ch)

    zero = torch.zeros(Ch, device=DEV)
    for _ in range(2):
        opt.zero_grad()
        h = x
        for w, n in zip((w1, w2), norms):
            h = _LinearFn.apply(h.contiguous(), w, zero)
            h = n(h.view(Bn, P, Ch).transpose(1, 2)).transpose(1, 2).reshape(Bn * P, Ch)
        loss = ((h.view(Bn, P, Ch).mean(1) - t) ** 2).mean()
        loss.backward()
        ws = [w.detach().double().requires_grad_() for w in (w1, w2)]
        h = x.double()
        for w in ws:
            h = gn64(h @ w.T, torch.ones(Ch, device=DEV).double(), torch.zeros(Ch, device=DEV).double())
        want = torch.autograd.grad(((h.view(Bn, P, Ch).mean(1) - t.double()) ** 2).mean(), ws)
        for w, g in zip((w1, w2), want):
            # two normalised layers deep: a few dozen roundings a value, sums of 240 rows
            assert float((w.grad.double() - g).norm()) <= 400 * U * float(g.norm())
        before = [w.detach().clone() for w in (w1, w2)]
        moms = [opt.state[w]["momentum_buffer"].clone() if w in opt.state else torch.zeros_like(w) for w in (w1, w2)]
        opt.step()
        for w, b, m in zip((w1, w2), before, moms):
            p, _, o = muon64(b, w.grad, m, 0.02, 0.0, 0.95, True)
            assert float((w.detach().double() - p).norm()) <= 0.02 * 2 ** 0.5 * (tol((64, 64)) + 248 * U) * float(o.norm()) + 4 * U * float(b.norm())


def test_refusals():
    from mmsa_amd import _lib, ops
    from mmsa_amd.muon import Muon, muon_step, orthogonalize
    lib = _lib.load()
    z = torch.zeros(4, 4)
    with pytest.raises(_lib.MmsaError, match="GPU"):
        orthogonalize(z)
    with pytest.raises(_lib.MmsaError, match="GPU"):
        muon_step([z], [z], [z], lr=0.1)
    for kw in (dict(steps=0), dict(steps=17), dict(steps=2.5), dict(eps=0.0)):
        with pytest.raises(ValueError):
            ops.orthogonalize([z], [z.clone()], **kw)
    with pytest.raises(ValueError):
        ops.orthogonalize([z], [])
    with pytest.raises(ValueError):
        ops.orthogonalize([z], [torch.zeros(4, 5)])
    with pytest.raises(ValueError):
        ops.orthogonalize([torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(ValueError):
        ops.orthogonalize([torch.zeros(0, 4)], [torch.zeros(0, 4)])
    with pytest.raises(TypeError):
        ops.orthogonalize([z.double()], [z.double()])
    with pytest.raises(ValueError):
        ops.muon_step([z], [z], [], 0.1, 0.0, 0.9)
    for bad in (torch.zeros(4), torch.zeros(4, 4, dtype=torch.float16)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(bad)])
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0), dict(eps=0.0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(z)], **kw)
    import ctypes
    ints = (ctypes.c_int * 1)
    q = lib.mmsa_orthogonalize_scratch_bytes
    assert q(None, None, 1) == -1 and q(ints(4), ints(0), 1) == -1 and q(ints(4), ints(4), 0) == -1
    assert q(ints(2 ** 20 + 1), ints(4), 1) == -3 and q(ints(2 ** 17), ints(2 ** 17), 1) == -3
    assert q(ints(64), ints(288), 1) > 0
    ptr = (ctypes.c_void_p * 1)(4096)
    null = (ctypes.c_void_p * 1)(None)
    call = lib.mmsa_orthogonalize
    assert call(null, ptr, ints(4), ints(4), 1, 0, 5, 1e-7, 4096, None) == -1
    assert call(ptr, ptr, ints(4), ints(4), 1, 3, 5, 1e-7, 4096, None) == -1
    assert call(ptr, ptr, ints(4), ints(4), 1, 0, 0, 1e-7, 4096, None) == -1
    assert call(ptr, ptr, ints(4), ints(4), 1, 0, 5, 0.0, 4096, None) == -1
    assert call(ptr, ptr, ints(4), ints(4), 1, 0, 5, 1e-7, 4097, None) == -1
    assert lib.mmsa_muon_step(ptr, ptr, null, ints(4), ints(4), 1, 0.1, 0.0, 0.9, 1, 5, 1e-7, 4096, None) == -1


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    from mmsa_amd.muon import Muon, muon_step
    p, g, m = (torch.zeros(8, 8, device=DEV) for _ in range(3))
    for args in (([p, p], [g, g], [m, m.clone()]), ([p], [p], [m]), ([p], [g], [g]), ([p], [g], [p])):
        with pytest.raises(ValueError, match="twice"):
            muon_step(*args, lr=0.1)
    with pytest.raises(ValueError, match="contiguous"):
        muon_step([torch.zeros(8, 16, device=DEV)[:, ::2]], [g], [m], lr=0.1)
    q = torch.nn.Parameter(torch.zeros(8, 4, 3, 3, device=DEV).to(memory_format=torch.channels_last))
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError, match="contiguous"):
        Muon([q]).step()
