"""Newton-Schulz orthogonalisation and the Muon step: the largest tiles in every result type, lists that take more than
one set of launches, and what the optimiser does before, during and instead of a step.

Tolerance, relative in the Frobenius norm, u = 2^-24.  An operand is a pair of fp16 values, off by 2 u at most and by
2 u / sqrt 12 or so in the mean; the product of the two low halves, left out, is below 4 u and 0.7 u in the mean where
both factors are the same value (the diagonal of X X^T); a sum over K values in one 32-bit accumulator is rounded three
times for 16 of them, with errors that add up at random: sqrt(3 K / 16) u.  Together u (4 + sqrt(K) / 2) covers a step's
products.  x -> a x + b x^3 + c x^5 passes an error on with a factor between 0 and max |p'| = 4, about 2 in the mean:
five steps collect 1 + 2 + ... + 16 = 31 of them."""
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
A, B, C = 3.4445, -4.775, 2.0315


def ns64(u, steps=5, eps=1e-7):
    x = u.double()
    x = x / max(float(x.norm()), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if tall else x
    for _ in range(steps):
        s = x @ x.T
        x = A * x + (B * s + C * (s @ s)) @ x
    return x.T if tall else x


def tol(shape, dtype=torch.float32):
    return 31 * U * (4 + max(shape) ** 0.5 / 2) + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U)


def grad(m, n, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = max(1, min(m, n) // 4)
    low = torch.randn(m, k, device=DEV, generator=g) @ torch.randn(k, n, device=DEV, generator=g) / k ** 0.5
    return ((low + 0.2 * torch.randn(m, n, device=DEV, generator=g)) * 1e-3).to(dtype)


def close(got, want, rel):
    d = got.double() - want
    assert bool(torch.isfinite(got).all())
    assert float(d.norm()) <= rel * float(want.norm()), (float(d.norm()) / float(want.norm()), rel)
    # no single place stands out: 16 times a place's share of the whole
    assert float(d.abs().max()) <= rel * (16 * float(want.norm()) / want.numel() ** 0.5 + float(want.abs().max()))


# sizes for which the general product comes in tiles of 128 and of 256, wide and tall, neither side a multiple of a tile
LARGE = [(2000, 2101), (2101, 2000), (2500, 4999), (4999, 2500)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large_tiles_in_every_type(shape, dtype):
    from mmsa_amd.muon import orthogonalize
    g = grad(*shape, seed=sum(shape), dtype=dtype)
    o = orthogonalize(g)
    want = ns64(g)
    close(o, want, tol(shape, dtype))
    if dtype != torch.float32:
        # every place is the rounding of a value that float32 products leave near the exact one
        near = tol(shape) * (16 * float(want.norm()) / want.numel() ** 0.5 + want.abs())
        half = torch.finfo(dtype).eps / 2 * (want.abs() + near) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
        assert bool(((o.double() - want).abs() <= near + half).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large_tiles_into_a_parameter(shape):
    from mmsa_amd.muon import muon_step
    p, g, m = torch.randn(shape, device=DEV) * 0.02, grad(*shape, seed=1), grad(*shape, seed=2)
    p0, mom = p.double(), m.double() + (1 - 0.95) * (g.double() - m.double())
    o = ns64(g.double() + 0.95 * (mom - g.double()))
    rate = 0.02 * max(1.0, shape[0] / shape[1]) ** 0.5
    want = p0 * (1 - 0.02 * 0.1) - rate * o
    muon_step([p], [g], [m], lr=0.02, weight_decay=0.1)
    assert float((m.double() - mom).abs().max()) <= 4 * U * float(mom.abs().max() + g.abs().max())
    # the direction is known to a few u, which the iteration magnifies 31 times; the parameter is rounded three times
    bound = rate * (tol(shape) + 31 * 8 * U) * float(o.norm()) + 4 * U * float(p0.norm())
    assert float((p.double() - want).norm()) <= bound


def scratch_bytes(shapes):
    from mmsa_amd import ops
    n = len(shapes)
    return ops._lib.query("mmsa_orthogonalize_scratch_bytes", ops._iarr([s[0] for s in shapes]),
                          ops._iarr([s[1] for s in shapes]), n)


def test_the_scratch_of_a_list_is_bounded():
    """A list of large matrices is worked off in sets of launches that fill the chip, not all at once."""
    one = scratch_bytes([(4096, 14336)])
    assert scratch_bytes([(4096, 14336)] * 24) <= one + 2 ** 30 + 2 ** 20
    assert scratch_bytes([(4096, 4096)] * 100) <= 2 ** 31
    small = scratch_bytes([(256, 1152)])
    assert 20 * small < scratch_bytes([(256, 1152)] * 24) < 30 * small         # these still go together


@pytest.mark.gpu
def test_lists_of_large_matrices():
    """More than one set of launches because of their size, with small ones between them."""
    from mmsa_amd.muon import muon_step, orthogonalize
    shapes = [(2048, 8192), (70, 200), (4096, 4100), (4096, 4096), (33, 64), (2048, 8192), (130, 40)]
    gs = [grad(*s, seed=i) for i, s in enumerate(shapes)]
    wants = [ns64(g) for g in gs]
    for s, o, w in zip(shapes, orthogonalize(gs), wants):
        close(o, w, tol(s))
    ps, ms = [torch.zeros_like(g) for g in gs], [g.clone() for g in gs]
    muon_step(ps, gs, ms, lr=0.5)
    for s, p, w in zip(shapes, ps, wants):
        rate = 0.5 * max(1.0, s[0] / s[1]) ** 0.5
        close(p, -rate * w, tol(s) + 31 * 8 * U)


def test_sizes_that_32_bits_cannot_hold_are_refused():
    from mmsa_amd import _lib, ops
    for shape in ((2 ** 32 + 64, 64), (64, 2 ** 32 + 64), (2 ** 16, 2 ** 16), (2 ** 20 + 1, 2), (1, 2 ** 20 + 1)):
        with pytest.raises(_lib.MmsaError, match="limit"):
            ops._sizes([torch.empty(4, 4, device="meta"), torch.empty(shape, device="meta")])
    rows, cols = ops._sizes([torch.empty(2 ** 20, 2 ** 11, device="meta"), torch.empty(8, 4, 3, 3, device="meta")])
    assert list(rows) == [2 ** 20, 8] and list(cols) == [2 ** 11, 36]


@pytest.mark.gpu
def test_operands_that_share_memory_are_refused():
    from mmsa_amd import ops
    from mmsa_amd.muon import muon_step
    flat = torch.zeros(64, 8, device=DEV)
    a, over, apart = flat[:32], flat[31:63], torch.zeros(32, 8, device=DEV)
    g, m, n = (torch.zeros(32, 8, device=DEV) for _ in range(3))
    for args in (([a, over], [g, g], [m, n]), ([a], [over], [m]), ([a], [g], [over]), ([m, n], [g, g], [a, over])):
        with pytest.raises(ValueError, match="share"):
            muon_step(*args, lr=0.1)
    for srcs, dsts in (([a, apart], [m, m]), ([a, apart], [apart, m]), ([a], [over])):
        with pytest.raises(ValueError, match="share"):
            ops.orthogonalize(srcs, dsts)
    ops.orthogonalize([a, apart], [a, m])                   # in its own place
    muon_step([flat[:32], flat[32:]], [g, g], [m, n], lr=0.1)          # neighbours, one gradient for both


def test_the_check_for_shared_memory_against_every_pair():
    import random

    from mmsa_amd import ops
    memory, rng = torch.zeros(4000), random.Random(1)

    def some(k):
        at = [rng.randrange(3000) for _ in range(k)]
        return [(t.data_ptr(), t) for t in (memory[a:a + rng.randrange(1, 400)] for a in at)]

    def meet(x, y):
        return x[0] < y[0] + y[1].nbytes and y[0] < x[0] + x[1].nbytes
    refused = 0
    for _ in range(2000):
        writes, reads = some(rng.randrange(4)), some(rng.randrange(4))
        if writes and reads and rng.random() < 0.2:
            reads[0] = writes[0]
        want = any(meet(x, y) for i, x in enumerate(writes) for y in writes[:i] + reads)
        try:
            ops._apart(writes, reads, "a tensor")
            assert not want
        except ValueError as e:
            assert want and "share" in str(e)
            refused += 1
    assert 200 < refused < 1800


def _params(*shapes):
    gen = torch.Generator(device=DEV).manual_seed(7)
    ps = [torch.nn.Parameter(torch.randn(s, device=DEV, generator=gen)) for s in shapes]
    for p in ps:
        p.grad = torch.randn(p.shape, device=DEV, generator=gen)
    return ps


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["cpu", "sparse", "order"])
def test_a_refused_step_leaves_everything_as_it_was(bad):
    from mmsa_amd import _lib
    from mmsa_amd.muon import Muon
    good, q = _params((8, 8), (8, 4, 3, 3))
    if bad == "cpu":
        q = torch.nn.Parameter(torch.randn(8, 36))
        q.grad = torch.randn(8, 36)
    opt = Muon([{"params": [good]}, {"params": [q]}], lr=0.1)
    if bad == "sparse":
        q.grad = torch.zeros(8, 4, 3, 3, device=DEV).to_sparse()
    if bad == "order":
        q.data = q.data.to(memory_format=torch.channels_last)
    before = good.detach().clone()
    with pytest.raises((_lib.MmsaError, RuntimeError, ValueError)):
        opt.step()
    assert torch.equal(good, before) and not opt.state


@pytest.mark.gpu
def test_parameters_in_another_order_are_refused_when_they_are_given():
    from mmsa_amd.muon import Muon
    good, q = _params((8, 8), (8, 4, 3, 3))
    q.data = q.data.to(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="contiguous"):
        Muon([good, q])
    opt = Muon([good])
    with pytest.raises(ValueError, match="contiguous"):
        opt.add_param_group({"params": [q]})
    opt.step()
    assert len(opt.param_groups) == 1


@pytest.mark.gpu
def test_an_empty_parameter_is_left_alone():
    from mmsa_amd.muon import Muon
    good, empty = _params((8, 8), (0, 4))
    before = good.detach().clone()
    Muon([good, empty], lr=0.1).step()
    assert not torch.equal(good, before) and empty.shape == (0, 4)


@pytest.mark.gpu
def test_momentum_is_not_made_inside_a_graph():
    """A buffer made and cleared while a graph is recorded would be cleared again by every replay: the first step is an
    eager one, and replays then follow eager steps."""
    from mmsa_amd.muon import Muon
    ps, qs = _params((48, 80), (7, 300)), _params((48, 80), (7, 300))
    opt, ref = Muon(ps, lr=0.02), Muon(qs, lr=0.02)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), pytest.raises(RuntimeError, match="eager"):
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            opt.step()
    torch.cuda.synchronize()
    assert not opt.state and all(torch.equal(p, q) for p, q in zip(ps, qs))
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        opt.step()
    for k in range(4):
        for p, q in zip(ps, qs):
            p.grad.normal_()
            q.grad.copy_(p.grad)
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k


@pytest.mark.gpu
def test_muon_and_adamw_train_the_model_together():
    """The package's own model: its hidden weight matrices with Muon, the embedding, the classifier's last layer and all
    vectors with AdamW; every parameter is updated once, by its own rule, over steps with changing gradients.

    Some of these gradients have a low rank (the two rows of the attention over two modalities are opposite), and what
    lies in their empty directions grows by a = 3.4445 in every step.  A rounding of the iteration is magnified at most
    1 + a + ... + a^4 = 198 times there, one of the direction a^5 = 485 times.  The direction's own: every step rounds the
    factor 1 - momentum, g - m and m; then the factor momentum, m - g and u are rounded."""
    from conftest import SMALL_VOCAB, batch_tensors, model_inputs, seeded_model
    from mmsa_amd.muon import Muon
    m = seeded_model("both", vocab=SMALL_VOCAB).to(DEV).train()
    apart = {m.text_model.embedding.weight, m.classifier[-1].weight}
    matrices = [p for p in m.parameters() if p.dim() >= 2 and p not in apart]
    others = [p for p in m.parameters() if p.dim() < 2 or p in apart]
    assert len(matrices) == 24 and len(matrices) + len(others) == len(list(m.parameters()))
    opts = [Muon(matrices, lr=0.02, weight_decay=0.01), torch.optim.AdamW(others, lr=1e-3)]
    mom = [torch.zeros_like(p, dtype=torch.float64) for p in matrices]
    most_g, most_m = [0.0] * len(matrices), [0.0] * len(matrices)
    for it in range(3):
        b = batch_tensors(8 * it, 8, vocab=SMALL_VOCAB, device=DEV)
        for o in opts:
            o.zero_grad()
        m(**model_inputs("both", b), labels=b["label"])["loss"].backward()
        before = [p.detach().double() for p in matrices]
        rest = [p.detach().clone() for p in others]
        for o in opts:
            o.step()
        for k, (p, p0) in enumerate(zip(matrices, before)):
            g = p.grad.double()
            mom[k] = mom[k] + (1 - 0.95) * (g - mom[k])
            most_g[k], most_m[k] = max(most_g[k], float(g.norm())), max(most_m[k], float(mom[k].norm()))
            rows, cols = p.shape[0], p[0].numel()
            u = g + 0.95 * (mom[k] - g)
            o = ns64(u.view(rows, cols)).reshape(p.shape)
            rate = 0.02 * max(1.0, rows / cols) ** 0.5
            both, size = most_g[k] + most_m[k], float(u.norm())
            direction = U * ((it + 1) * (0.1 * both + most_m[k]) + 2 * both + size) / size
            iteration = 198 * U * (4 + max(rows, cols) ** 0.5 / 2) * max(1.0, float(o.norm()))
            off = float((p.detach().double() - (p0 * (1 - 0.02 * 0.01) - rate * o)).norm())
            assert off <= rate * (iteration + 485 * direction) + 4 * U * float(p0.norm()), (k, p.shape)
        assert sum(not torch.equal(p, r) for p, r in zip(others, rest)) >= len(others) - 1
