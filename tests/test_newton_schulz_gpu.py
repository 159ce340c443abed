"""The Newton-Schulz kernels against the 64-bit statement.

Bounds of the result's error, relative in the 2-norm.  A rounding is off by at most half a step, 2^-8 of a value for the bf16 result
and 2^-11 for the f16 operands, and evenly spread: by half a step over the square root of 3 in the mean square (2.3e-3, 2.8e-4).
x, G and P round once per step, and what a rounding leaves grows by at most 3.4445 in the step where the result, which grows
alike, takes it up.

* Many entries (d >= 16): roundings are independent and their squares add up; five steps: sqrt(2.3e-3^2 + 15 (3.4445 2.8e-4)^2) =
  4.4e-3, and 5.2e-3 with a margin for the correlation of an entry's three roundings (a factor sqrt(1.5) on their part).
* Fewer: nothing averages out in the few singular directions, and the largest errors add up:
  2^-8 + 15 * 3.4445 * 2^-11 = 2.9e-2.

The derivative applies the steps' products with the same P and f16 roundings: the same bounds."""
import math

import pytest
import torch

from dttt_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BOUND, FEW = 5.2e-3, 2.9e-2


@pytest.fixture(autouse=True)
def _status():
    yield
    from dttt_b200.ops import _lib
    torch.cuda.synchronize()
    _lib.check_status()


def make(shape, dtype, seed=0, scale=1e-3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = 2 * min(shape[-2:])
    h = torch.randn(*shape[:-2], t, shape[-2], generator=gen, device="cuda")
    d = torch.randn(*shape[:-2], t, shape[-1], generator=gen, device="cuda") * torch.rand(*shape[:-2], t, 1, generator=gen, device="cuda")
    return (h.mT @ d * scale).to(dtype), torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)


def off(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


SHAPES = [(127, 511), (512, 128), (3, 129, 300), (2, 128, 513), (5, 40, 1), (8, 8), (64, 64), (1, 65, 127), (3, 128, 256), (2, 256, 128), (5, 100, 36), (257, 256), (256, 257), (2, 509, 1283), (1283, 509),
          (2, 2, 130, 700), (512, 2048), (1024, 1000), (12, 96, 96), (768, 64), (17, 4096),
          (3, 128, 4096), (4090, 127), (2, 100, 2049), (5, 1100, 64), (129, 1032), (64, 4097),
          (16, 30, 2049), (20, 100, 701), (1024, 64), (128, 1088)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_direction_and_derivative(shape, dtype, steps):
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make(shape, dtype, sum(shape))
    want, norms, polys = ref.newton_schulz(g, steps, torch.float64)
    bound = BOUND if min(shape[-2:]) >= 16 else FEW
    y = newton_schulz(g, steps)
    assert y.dtype == torch.bfloat16 and y.shape == g.shape and off(y, want) <= bound
    leaf = g.clone().requires_grad_(True)
    out = newton_schulz(leaf, steps)
    assert out.equal(y)
    got, = torch.autograd.grad(out, leaf, gy)
    assert got.dtype == dtype and off(got, ref.newton_schulz_apply(gy, norms, polys)) <= bound


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (3, 5), (2, 3), (7, 33)])
def test_tiny_matrices(shape):
    """A handful of entries, rows and columns of one element."""
    from dttt_b200.ops.newton_schulz import newton_schulz
    for steps in (1, 5):
        g, gy = make(shape, torch.float32, 3)
        leaf = g.clone().requires_grad_(True)
        want, norms, polys = ref.newton_schulz(g, steps, torch.float64)
        y = newton_schulz(leaf, steps)
        assert off(y, want) <= FEW
        assert off(torch.autograd.grad(y, leaf, gy)[0], ref.newton_schulz_apply(gy, norms, polys)) <= FEW


def test_derivative_against_differences():
    """The map is linear in g once its matrix is held: a difference of the 64-bit map along a direction is the derivative."""
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make((200, 320), torch.bfloat16, 4)
    _, norms, polys = ref.newton_schulz(g, 5, torch.float64)
    leaf = g.clone().requires_grad_(True)
    got, = torch.autograd.grad(newton_schulz(leaf), leaf, gy)
    for seed in (1, 2):
        _, d = make((200, 320), torch.bfloat16, seed)
        step = lambda e: ref.newton_schulz_apply(g.double() + e * d.double(), norms, polys)
        slope = ((step(0.5) - step(-0.5)) * gy.double()).sum()
        mine = (got.double() * d.double()).sum()
        assert abs(mine - slope) <= BOUND * got.double().norm() * d.double().norm()


def test_twice_differentiable_scale_zero_and_special_values():
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make((3, 150, 90), torch.float32, 5)
    leaf, cot = g.clone().requires_grad_(True), gy.clone().requires_grad_(True)
    gx, = torch.autograd.grad(newton_schulz(leaf, 3), leaf, cot, create_graph=True)
    c, _ = make((3, 150, 90), torch.float32, 6)
    back, = torch.autograd.grad(gx, cot, c)
    _, norms, polys = ref.newton_schulz(g, 3, torch.float64)
    assert back.dtype == torch.bfloat16 and off(back, ref.newton_schulz_apply(c, norms, polys)) <= BOUND
    assert newton_schulz(g * 2.0 ** 90).equal(newton_schulz(g)) and newton_schulz(g * 2.0 ** -90).equal(newton_schulz(g))
    z = g.clone()
    z[1] = 0
    z[2, 3, 4] = float("nan")
    leaf = z.requires_grad_(True)
    y = newton_schulz(leaf)
    assert y[0].equal(newton_schulz(g[0])) and y[1].eq(0).all() and y[2].isnan().all()
    gx, = torch.autograd.grad(y, leaf, gy)
    assert gx[1].eq(0).all() and gx[0].isfinite().all()


def test_concentrated_cotangent_and_spectrum():
    """One entry of the cotangent alone, and a matrix whose singular values span three decades (the f16 roundings of the first step
    leave 3 * 2.8e-4 of the largest values in the directions of the smallest, which grow up to 485 times to results near 1:
    relative to those at most 0.4, and to the whole, where the larger ones weigh as much, a quarter of it)."""
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make((128, 384), torch.float32, 7)
    one = torch.zeros_like(gy)
    one[5, 7] = 1e4
    leaf = g.clone().requires_grad_(True)
    got, = torch.autograd.grad(newton_schulz(leaf), leaf, one)
    _, norms, polys = ref.newton_schulz(g, 5, torch.float64)
    assert got.isfinite().all() and off(got, ref.newton_schulz_apply(one, norms, polys)) <= BOUND
    u, _, vt = torch.linalg.svd(g, full_matrices=False)
    sharp = u @ (torch.logspace(0, -3, 128, device="cuda")[:, None] * vt)
    assert newton_schulz(sharp).isfinite().all()
    assert off(newton_schulz(sharp), ref.newton_schulz(sharp, 5, torch.float64)[0]) <= 0.1


def test_views_repeats_streams_graphs_and_empty():
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make((4, 300, 200), torch.bfloat16, 8)
    first = newton_schulz(g)
    assert all(newton_schulz(g).equal(first) for _ in range(3))
    assert newton_schulz(g.mT.contiguous().mT).equal(first) and newton_schulz(g[1:3]).equal(first[1:3])
    cut = g[:, 3:290, 5:150]
    assert newton_schulz(cut).equal(newton_schulz(cut.contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = newton_schulz(g)
    torch.cuda.current_stream().wait_stream(side)
    assert other.equal(first) and newton_schulz(g[:0]).shape == (0, 300, 200)
    # forward and backward in one graph, replayed on other values; the leaf has no eager graph alive
    leaf = g.clone().requires_grad_(True)
    cot = gy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = newton_schulz(leaf)
        gx, = torch.autograd.grad(y, leaf, cot)
    g2, gy2 = make((4, 300, 200), torch.bfloat16, 9)
    with torch.no_grad():
        leaf.copy_(g2)
    cot.copy_(gy2)
    graph.replay()
    want = g2.clone().requires_grad_(True)
    y2 = newton_schulz(want)
    assert y.equal(y2) and gx.equal(torch.autograd.grad(y2, want, gy2)[0])


def test_the_write_rule_on_the_kernels():
    """The direction that the inner step takes: norms over a sequence's matrices kept, every matrix near-orthogonal."""
    from dttt_b200.ttt import inner as IN
    g = [make((2, 256, 512), torch.bfloat16, 1)[0], make((2, 512, 256), torch.float32, 2)[0]]
    u = IN.direction(g, "muon5")
    assert torch.allclose(IN.seq_norm(u), IN.seq_norm(g), rtol=1e-3)
    for t in u:
        s = torch.linalg.svdvals(t.float())
        assert (s.amax(-1) / s.amin(-1) < 2.5).all()


@pytest.mark.parametrize("shape", [(4, 300, 200), (2, 64, 100)])
def test_capture_on_a_thread_that_has_not_called_before(shape):
    """Autograd's thread, or one of the user's, may meet the device for the first time inside a capture."""
    import threading
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, _ = make(shape, torch.bfloat16, 8)
    want, got = newton_schulz(g), []
    torch.cuda.synchronize()

    def work():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = newton_schulz(g)
        graph.replay()
        torch.cuda.synchronize()
        got.append(y.clone())

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert len(got) == 1 and got[0].equal(want)


# ------------------------------------------------------------------------------------------------------------ many steps
def plan_of(rows, cols, steps):
    """(iterations, alpha) of every group, as the launcher groups them: pairs at both ends of long large matrices."""
    a, b, c = ref.NEWTON_SCHULZ
    d, n = min(rows, cols), max(rows, cols)
    q = lambda l: a + b * l + c * l * l
    l, k, out = 1.0 / d, 0, []
    while k < steps:
        two = d >= 512 and n >= 2 * d and ((k == 0 and steps >= 2) or (k == steps - 2 and k >= 3))
        l2 = l * q(l) ** 2
        out.append((2, q(l) * q(l2)) if two else (1, q(l)))
        l, k = (l2 * q(l2) ** 2, k + 2) if two else (l2, k + 1)
    return out


def maps_of(maps, shape, steps):
    """The kept matrices of every group in 64 bits with their diagonal, and the largest growth in each."""
    d = min(shape[-2:])
    ms = [maps[k, :, :, :d].double() / 4096 + alpha * torch.eye(d, dtype=torch.float64, device=maps.device)
          for k, (_, alpha) in enumerate(plan_of(*shape[-2:], steps))]
    return ms, [torch.linalg.eigvalsh(m.mT @ m)[:, -1] for m in ms]


def apply_of(ms, most, norms, r):
    """What the kept matrices of a forward say the derivative is, in 64 bits, and the error that f16 roundings of the cotangent may
    leave: a step rounds by 2^-11 over the square root of 3 in the mean square, and what it leaves grows like a part of the cotangent
    in the direction that grows most."""
    x = torch.where(norms[:, None, None] == 0, 0.0, r.double() / norms[:, None, None])
    off2 = torch.zeros(r.shape[0], dtype=torch.float64, device=r.device)
    for m, top in zip(reversed(ms), reversed(most)):
        off2 = top * (off2 + (2.0 ** -11 / 3 ** 0.5) ** 2 * x.pow(2).sum((-2, -1)))
        x = m.mT @ x if r.shape[-2] <= r.shape[-1] else x @ m.mT
    return x, off2.sqrt()


@pytest.mark.parametrize("shape", [(64, 200), (1, 48, 40), (2, 128, 1024), (512, 128), (2, 129, 300), (300, 200), (512, 1024), (1100, 520)])
@pytest.mark.parametrize("steps", [7, 8, 12, 32])
def test_derivative_of_many_steps(shape, steps):
    """Directions without a singular value grow 3.4445-fold a step in the cotangent: 10^4 at eight steps, 10^17 at 32.  Against the kept
    matrices themselves, so that what many steps do to the forward's roundings is not part of it.  The bound: that of the roundings,
    in the norm (they are many and independent: a factor of two over the mean square is never met), and the result's own."""
    from dttt_b200.ops import kernels
    from dttt_b200.ops.newton_schulz import newton_schulz
    full, gy = make(shape if len(shape) == 3 else (1, *shape), torch.float32, 2)
    d = min(shape[-2:])
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    lean = r(*full.shape[:-1], max(1, d // 3)) @ r(full.shape[0], max(1, d // 3), full.shape[-1])
    gap = full.clone()
    (gap[:, 3] if shape[-2] <= shape[-1] else gap[:, :, 3]).zero_()
    one = torch.zeros_like(gy)
    one[:, 3, 5] = 0.7
    for g in (full, lean, gap, torch.zeros_like(full)):
        _, norms, maps = kernels.newton_schulz(g, steps, True)
        ms, growth = maps_of(maps, shape, steps)
        for c in (gy, one, gy * 1e20):
            want, off2 = apply_of(ms, growth, norms, c)
            for dtype in (torch.float32, torch.bfloat16):
                got = kernels.newton_schulz_apply(c, norms, maps, steps, dtype)
                most = want.norm(dim=(-2, -1))
                if most.max() > 1e37:                                       # (f32 itself ends)
                    continue
                assert got.isfinite().all()
                lost = 2.0 ** -24 if dtype is torch.float32 else 2.0 ** -8
                assert ((got.double() - want).norm(dim=(-2, -1)) <= 2 * off2 + lost * most).all()
    leaf = torch.zeros_like(full).requires_grad_(True)
    gx, = torch.autograd.grad(newton_schulz(leaf, steps), leaf, gy)
    assert gx.eq(0).all()


# ------------------------------------------------------------------------------------------------- fewer tokens than rows
@pytest.mark.parametrize("shape", [(64, 100), (2, 128, 256), (256, 128), (3, 100, 900), (1024, 64), (128, 2048), (260, 300), (2, 509, 1283), (1283, 509),
                                   (512, 2048), (1200, 600)])
@pytest.mark.parametrize("tokens", [1, 8, 0.25, 0.5, 1.0])
@pytest.mark.parametrize("steps", [2, 5, 8])
def test_matrices_of_low_rank(shape, tokens, steps):
    """The gradient of a write has at most the rank of its chunk's tokens.  Roundings of G, of P and of x inside P x stay in the row or
    the column space of x: they turn singular vectors, by at most |P| / |a + P| <= 4.4 of themselves a step, and nothing amplifies
    that: the bound above.  What lies outside both spaces grows 3.4445-fold a step, and that is only what x loses when it is
    stored: half a step of 2^-11 of what a step of 2^-11 leaves, evenly spread both (2^-22 / 3), and the few 2^-24 of f32 arithmetic,
    1e-7 of |x_0| = 1 together, relative to a result of at least 0.68 (one singular value); a factor of two over the mean square.
    The last group takes x in one half: 2.8e-4 of it, 3.4445-fold (11.9-fold by a pair), independent of the rest."""
    from dttt_b200.ops.newton_schulz import newton_schulz
    d = min(shape[-2:])
    t = tokens if isinstance(tokens, int) else int(tokens * d)
    gen = torch.Generator(device="cuda").manual_seed(sum(shape) + t)
    h = torch.randn(*shape[:-2], t, shape[-2], generator=gen, device="cuda")
    e = torch.randn(*shape[:-2], t, shape[-1], generator=gen, device="cuda") * torch.rand(*shape[:-2], t, 1, generator=gen, device="cuda")
    gy = torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)
    lost = plan_of(*shape[-2:], steps)[-1][0]
    for g in (h.mT @ e * 1e-3, (h.mT @ e * 1e-3).to(torch.bfloat16)):
        want, norms, polys = ref.newton_schulz(g, steps, torch.float64)
        before = (ref.newton_schulz(g, steps - lost, torch.float64)[0].norm() / want.norm()).item()
        bound = math.hypot(BOUND, 2.0 ** -11 / 3 ** 0.5 * 3.4445 ** lost * before) + 2 * 1e-7 * 3.4445 ** steps / 0.68
        leaf = g.clone().requires_grad_(True)
        y = newton_schulz(leaf, steps)
        assert newton_schulz(g, steps).equal(y) and off(y, want) <= bound
        got, = torch.autograd.grad(y, leaf, gy)
        assert off(got, ref.newton_schulz_apply(gy, norms, polys)) <= bound


def test_launches_are_counted():
    """What the calls say they launch, against the profiler."""
    from dttt_b200.ops import kernels
    from torch.profiler import ProfilerActivity, profile
    for shape in [(2, 64, 100), (3, 129, 300), (1, 512, 1100), (2, 2048, 3100)]:
        g, gy = make(shape, torch.float32, 1)
        for steps in (1, 5, 9):
            y, norms, maps = kernels.newton_schulz(g, steps, True)
            for call in (lambda: kernels.newton_schulz(g, steps, False), lambda: kernels.newton_schulz_apply(gy, norms, maps, steps, torch.float32)):
                n = kernels.LAUNCHES
                with profile(activities=[ProfilerActivity.CUDA]) as prof:
                    call()
                    torch.cuda.synchronize()
                seen = sum(e.count for e in prof.key_averages() if "ns_" in e.key and "kernel" in e.key)
                if not seen:
                    pytest.skip("no device events from the profiler here")
                assert kernels.LAUNCHES - n == seen, (shape, steps)


@pytest.mark.parametrize("shape,one", [((24, 84, 915), True), ((23, 84, 915), False), ((25, 100, 701), True), ((2, 127, 2049), False), ((40, 3001), True),
                                       ((2, 65, 601), False), ((3, 64, 601), True), ((4096, 128), True), ((2, 4095, 127), True), ((1500, 128), True),
                                       ((2, 3000, 50), True), ((4097, 16), False), ((129, 129), False), ((128, 4104), False), ((3, 1, 4095), True)])
def test_both_sides_of_the_one_launch_rule(shape, one):
    from dttt_b200.ops import kernels
    n = kernels.LAUNCHES
    kernels.newton_schulz(make(shape, torch.float32)[0].reshape(-1, *shape[-2:]), 2, False)
    assert (kernels.LAUNCHES - n == 1) == one
    for dtype in (torch.float32, torch.bfloat16):
        test_direction_and_derivative(shape, dtype, 5)


@pytest.mark.parametrize("shape", [(2, 64, 100), (2, 300, 200)])
def test_kept_matrices_move_with_saved_tensor_hooks(shape):
    from dttt_b200.ops.newton_schulz import newton_schulz
    g, gy = make(shape, torch.float32, 3)
    leaf = g.requires_grad_(True)
    want, = torch.autograd.grad(newton_schulz(leaf), leaf, gy)
    with torch.autograd.graph.save_on_cpu():
        y = newton_schulz(leaf)
    assert torch.autograd.grad(y, leaf, gy)[0].equal(want)


# ------------------------------------------------------------------------------------------------------------ the write
def write_rule(g, steps=5):
    """``ttt.inner.direction(g, "muon5")`` of 64-bit leaves, differentiable in all but the polynomials."""
    y = []
    for x in g:
        with torch.no_grad():
            _, _, polys = ref.newton_schulz(x, steps, torch.float64)
        y.append(ref.newton_schulz_apply(x, torch.linalg.matrix_norm(x, keepdim=True), polys))
    size = lambda ts: torch.sqrt(sum(t.pow(2).sum((-2, -1)) for t in ts) + 1e-8)[:, None, None]
    return [t * size(g) / size(y) for t in y]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes,tokens", [(((64, 128), (64, 128), (128, 64)), 20), (((300, 700), (300, 700), (700, 300)), 90), (((128, 1000), (1000, 128)), 500)])
def test_the_write_rule_and_its_derivative(shapes, tokens, dtype):
    """Several matrices with one scale between them, against the rule in 64 bits with the derivative of every norm.  u is off as the
    directions are; a gradient as the held map's result, of which the norm's share is taken away: the bound of each relative to
    what is subtracted, and 2^-8 of the cotangent's rounding to bf16 besides."""
    from dttt_b200.ttt import inner as IN
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    g = [(r(2, tokens, s[0]).mT @ r(2, tokens, s[1]) * 10.0 ** -i).to(dtype) for i, s in enumerate(shapes)]
    c = [r(*x.shape) + x.float() / x.float().std() for x in g]              # some of it along the matrices
    leaf, exact = [x.clone().requires_grad_(True) for x in g], [x.double().requires_grad_(True) for x in g]
    u, want = IN.direction(leaf, "muon5"), write_rule(exact)
    bound = math.hypot(BOUND, 2.0 ** -11 / 3 ** 0.5 * 3.4445 * 1.8)         # (the last step takes x in one half; values 0.68 to 1.21)
    assert all(off(a, b) <= bound for a, b in zip(u, want))
    got = torch.autograd.grad(sum((a * b).sum() for a, b in zip(u, c)), leaf)
    grad = torch.autograd.grad(sum((a * b.double()).sum() for a, b in zip(want, c)), exact)
    scale = [x.detach().norm(dim=(-2, -1), keepdim=True) for x in want]
    for a, b, x, k, t in zip(got, grad, exact, c, scale):
        with torch.no_grad():                                               # the held map's result, before the norms' share goes
            y, n, polys = ref.newton_schulz(x.detach(), 5, torch.float64)
            held = ref.newton_schulz_apply(k.double() * t / y.norm(dim=(-2, -1), keepdim=True), n, polys).norm()
        assert a.dtype == dtype and (a.double() - b).norm() <= (bound + 2.0 ** -7) * (b.norm() + held)
        # along the matrix by itself: what is left there is the common scale's, (c u) |g_j|^2 / |g|^2, and the gradient's own roundings
        # (half a step each, evenly spread; f32: of some products on the way; a factor of four over the mean square)
        dots = lambda p, q: (p.double() * q.double()).sum((-2, -1))
        common = sum(dots(v, w) for v, w in zip(c, want)) * dots(x, x) / sum(dots(z, z) for z in exact)
        lost = (2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -22) * 4 / 3 ** 0.5 * dots(a.double() ** 2, x * x).sqrt()
        assert torch.allclose(dots(b, x), common, rtol=1e-6) and ((dots(a, x) - common).abs() <= 2 * bound * common.abs() + lost).all()


def test_training_gradients_with_the_kernel_and_without(monkeypatch):
    """One step's outer gradients through the five-step write, with the direction and its derivative on the kernels and as statements.
    Everything between is bf16: some thirty roundings of 2^-8 on the way, independent (2e-2 together, and as much between two runs, whose
    sums differ in order); a factor of ten over that is still far below a term that is left out or counted twice."""
    from dttt_b200.engine import Engine
    from dttt_b200.ops import kernels
    from dttt_b200.schema import ModelConfig, TrainConfig
    from util import loss_and_grads, loss_config
    mc = ModelConfig(vocab_size=4096, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, suffix_len=2, chunk_size=128, window_chunks=2, qk_norm=True, mask_token_id=4095, pad_token_id=4094,
                     eos_token_id=4094)
    tc = TrainConfig(seq_len=512, batch_size=2, steps=10, warmup_steps=2, inner_lr_warmup_steps=0, inner_task="causal", outer_shift=True,
                     cart_window=64, fused_ce_block=2048, inner_update="muon5")
    eng = Engine(mc, tc, device=torch.device("cuda", 0))
    ids = torch.randint(0, 4000, (2, 512), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    n = kernels.LAUNCHES
    loss, grads, _ = loss_and_grads(eng, ids, loss_config(tc))
    assert kernels.LAUNCHES > n
    monkeypatch.setattr(kernels, "_DISABLED", kernels._DISABLED | {"newton_schulz"})
    loss2, plain, _ = loss_and_grads(eng, ids, loss_config(tc))
    assert abs(loss - loss2) <= 2.0 ** -8 * abs(loss2)
    for k in plain:
        if plain[k].norm() > 0:
            assert off(grads[k], plain[k]) <= 0.2, k


@pytest.mark.parametrize("shapes", [((2, 300, 700), (2, 300, 700)), ((128, 2000), (3, 128, 512)), ((1, 512, 1100), (40, 100, 701))])
def test_two_calls_at_once_and_two_graphs_at_once(shapes):
    """Every call and every graph has its own workspaces: side by side on two streams, on inputs that change between replays."""
    from dttt_b200.ops.newton_schulz import newton_schulz
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    data = [make(s, torch.float32, n) for n, s in enumerate(shapes)]

    def both(g, gy):
        leaf = g.detach().requires_grad_(True)
        y = newton_schulz(leaf, 8)
        return y.detach(), torch.autograd.grad(y, leaf, gy)[0]

    want = [both(*d) for d in data]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n in range(2):
            with torch.cuda.stream(sides[n]):
                got[n].append(both(*data[n]))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(a.equal(b) for out in got[n] for a, b in zip(out, want[n]))
    held = []
    for g, gy in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(g, gy)
        held.append((graph, out))
    for turn in range(3):
        for n, (g, gy) in enumerate(data):
            g2, gy2 = make(shapes[n], torch.float32, 10 + 2 * turn + n)
            g.copy_(g2); gy.copy_(gy2)
        torch.cuda.synchronize()
        for side, (graph, _) in zip(sides, held):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for (g, gy), (_, out) in zip(data, held):
            assert all(a.equal(b) for a, b in zip(out, both(g, gy)))
