"""Newton-Schulz directions on the CPU: the singular values, the derivative of the linear map, the write rule, refusals."""
import pytest
import torch

from util import loss_and_grads, loss_config, make_engine
from dttt_b200.ops import reference as ref
from dttt_b200.ops.newton_schulz import newton_schulz
from dttt_b200.ttt import inner as IN

A, B, C = ref.NEWTON_SCHULZ


@pytest.mark.parametrize("shape", [(1, 1), (5, 5), (4, 9), (9, 4), (2, 3, 6, 4), (1, 7), (7, 1)])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_singular_values_follow_the_polynomial(shape, steps):
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * 1e-4
    u, s, vt = torch.linalg.svd(g.double(), full_matrices=False)
    s = s / s.pow(2).sum(-1, keepdim=True).sqrt()
    for _ in range(steps):
        s = A * s + B * s ** 3 + C * s ** 5
    want = u @ (s[..., None] * vt)
    y = newton_schulz(g, steps)
    assert y.dtype == torch.bfloat16 and y.shape == g.shape
    # bf16 rounds by 2^-9 of a value below 2^(e+1); f32 products of at most 9 terms, amplified at most 3.4445^5 = 485 times
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 485 * 2.0 ** -21 * want.abs().max()).all()


def test_derivative_is_the_held_linear_map():
    gen = torch.Generator().manual_seed(2)
    g = torch.randn(3, 6, 4, generator=gen).requires_grad_(True)
    gy = torch.randn(3, 6, 4, generator=gen)
    _, norms, polys = ref.newton_schulz(g.detach(), 3, torch.float64)
    eye = torch.eye(4, dtype=torch.float64)
    m = torch.eye(4, dtype=torch.float64)
    for p in polys:
        m = (A * eye + p) @ m
    want = gy.double() @ m / norms
    y = newton_schulz(g, 3)
    got, = torch.autograd.grad(y, g, gy.to(torch.bfloat16), create_graph=False)
    assert got.dtype == torch.float32
    # the cotangent rounds to bf16 (2^-8) and the f32 products of four terms err far below that
    assert (got.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()
    # differences of the held map: it is linear, so a step of any size gives the derivative
    step = lambda r: ref.newton_schulz_apply(r.double(), norms, polys)
    d = torch.randn(3, 6, 4, generator=gen)
    slope = step(g.detach().double() + 0.5 * d.double()) - step(g.detach().double() - 0.5 * d.double())
    assert torch.allclose((slope * gy.double()).sum(), (want * d.double()).sum(), rtol=1e-9)


def test_derivative_twice_is_the_same_map():
    g = torch.randn(2, 3, 5).requires_grad_(True)
    gy = torch.randn(2, 3, 5).to(torch.bfloat16).requires_grad_(True)
    gx, = torch.autograd.grad(newton_schulz(g, 2), g, gy, create_graph=True)
    c = torch.randn(2, 3, 5)
    back, = torch.autograd.grad(gx, gy, c)
    _, norms, polys = ref.newton_schulz(g.detach(), 2)
    assert torch.allclose(back.float(), ref.newton_schulz_apply(c, norms, polys), rtol=2.0 ** -7, atol=1e-6)


def test_zero_scale_and_special_values():
    assert newton_schulz(torch.zeros(2, 3, 4)).eq(0).all()
    z = torch.zeros(3, 4, requires_grad=True)
    assert torch.autograd.grad(newton_schulz(z), z, torch.ones(3, 4, dtype=torch.bfloat16))[0].eq(0).all()
    g = torch.randn(3, 4)
    assert newton_schulz(g * 2.0 ** 100).equal(newton_schulz(g)) and newton_schulz(g * 2.0 ** -100).equal(newton_schulz(g))
    g[0, 0] = float("inf")
    assert newton_schulz(g).isnan().all()
    assert newton_schulz(torch.zeros(0, 3, 4)).shape == (0, 3, 4)


@pytest.mark.parametrize("g,steps,word", [(torch.zeros(4), 5, "rows, cols"), (torch.zeros(3, 0), 5, "rows, cols"),
                                          (torch.zeros(3, 3, dtype=torch.float64), 5, "float64"), (torch.zeros(3, 3), 0, "steps"),
                                          (torch.zeros(3, 3), 2.0, "steps"), (torch.zeros(3, 3), True, "steps"),
                                          (torch.zeros(3, 3), 33, "steps"), (torch.zeros(65536, 1, 1), 1, "65535")])
def test_refusals(g, steps, word):
    with pytest.raises(ValueError, match=word):
        newton_schulz(g, steps)


def test_the_write_rule_keeps_the_gradient_norm_and_trains():
    gen = torch.Generator().manual_seed(3)
    g = [torch.randn(2, 6, 9, generator=gen), torch.randn(2, 9, 6, generator=gen)]
    u = IN.direction(g, "muon5")
    assert torch.allclose(IN.seq_norm(u), IN.seq_norm(g), rtol=1e-5)
    s = torch.linalg.svdvals(u[0])
    assert (s.amax(-1) / s.amin(-1) < 2).all()                      # five iterations: all singular values within [0.68, 1.21]
    eng = make_engine(inner_update="muon5")
    loss, grads, _ = loss_and_grads(eng, torch.randint(0, 120, (2, 32), generator=gen), loss_config(eng.tc))
    assert loss == loss and all(torch.isfinite(v).all() for v in grads.values())
    assert grads["fast_weight.gate.weight"].abs().sum() > 0


def test_the_first_call_on_a_device_is_not_captured(monkeypatch):
    from dttt_b200.ops import _lib, kernels
    monkeypatch.setattr(_lib, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(_lib.KernelError, match="before the capture"):
        kernels._status_word(torch.device("cuda", 0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_write_rule_against_differences_of_itself(dtype):
    """Scaling one of several matrices leaves its polynomial as it is, so holding that constant is exact along this direction: the
    derivative has to be the slope of the rule itself.  The rule's values: the matrices' own directions y_j, which do not move,
    times |g| / |y| over all of them; checked for scales of 2 and 1/2 (exact in every type), differenced in 64 bits.
    The cotangents and, of bf16 matrices, the gradients round by 2^-8: at most that of the absolute sum of the terms each, and twice
    as much of the gradient's own, which takes their differences."""
    gen = torch.Generator().manual_seed(11)
    g = [torch.randn(2, *s, generator=gen).to(dtype) for s in ((6, 9), (9, 6), (5, 5))]
    c = [x.float() * a for x, a in zip(g, (1.0, -2.0, 0.5))]                # cotangents along the matrices: nothing cancels
    norm = lambda ts: sum(t.double().pow(2).sum((-2, -1)) for t in ts).sqrt()[:, None, None]
    y = [newton_schulz(x, 5).double() for x in g]
    for j in range(3):
        scaled = lambda t: [x.double() * t if i == j else x.double() for i, x in enumerate(g)]
        for t in (0.5, 1.0, 2.0):
            for a, b in zip(IN.direction([x.to(dtype) for x in scaled(t)], "muon5"), y):
                assert torch.allclose(a.double(), b * norm(scaled(t)) / norm(y), rtol=1e-5, atol=0)
        value = lambda t: sum((a * norm(scaled(t)) / norm(y) * b).sum() for a, b in zip(y, c))
        slope = (value(1 + 1e-4) - value(1 - 1e-4)) / 2e-4
        leaf = [x.clone().requires_grad_(True) for x in g]
        got, = torch.autograd.grad(sum((a * b).sum() for a, b in zip(IN.direction(leaf, "muon5"), c)), leaf[j:j + 1])
        terms = sum((a * norm(g) / norm(y) * b).abs().sum() for a, b in zip(y, c)) + (got.double() * g[j].double()).abs().sum()
        assert abs((got.double() * g[j].double()).sum() - slope) <= 3 * 2.0 ** -8 * terms


def test_what_the_derivative_keeps_are_saved_tensors():
    """Hooks on saved tensors see the norms and every step's matrix, and a graph that has been walked holds neither."""
    g = torch.randn(2, 4, 6, generator=torch.Generator().manual_seed(5)).requires_grad_(True)
    gy = torch.ones(2, 4, 6, dtype=torch.bfloat16)
    want, = torch.autograd.grad(newton_schulz(g, 3), g, gy)
    packed = []

    def pack(t):
        packed.append(tuple(t.shape))
        return t.clone()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = newton_schulz(g, 3)
    assert packed == [(2, 1, 1)] + 3 * [(2, 4, 4)]
    assert torch.autograd.grad(y, g, gy)[0].equal(want)
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y, g, gy)


def test_a_dual_tensor_is_refused():
    from torch.autograd import forward_ad
    g = torch.randn(3, 4)
    with forward_ad.dual_level():
        assert newton_schulz(g, 2).shape == (3, 4)
        for x in (g, g.clone().requires_grad_(True)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                newton_schulz(forward_ad.make_dual(x, torch.ones(3, 4)), 2)
    assert newton_schulz(g, 2).shape == (3, 4)


def test_the_write_rule_rounds_behind_the_projection():
    """bf16 gradients of low rank: the held map's result is large where the matrix has no singular value, and what the norm's
    derivative takes off each entry is less than half a step of that.  Rounded once, behind it, the roundings (2^-8, evenly spread)
    are independent of the matrix: a factor of four over their mean square; rounded before as well they put all of it back."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)
    dots = lambda a, b: (a.double() * b.double()).sum((-2, -1))
    g = [(r(2, 20, m).mT @ r(2, 20, n) * s).to(torch.bfloat16) for m, n, s in ((64, 128, 1.0), (64, 128, 0.1), (128, 64, 0.01))]
    c = [r(*x.shape) + x.float() / x.float().std() for x in g]
    leaf = [x.clone().requires_grad_(True) for x in g]
    u = IN.direction(leaf, "muon5")
    got = torch.autograd.grad(sum((a * b).sum() for a, b in zip(u, c)), leaf)
    for a, x in zip(got, g):
        common = sum(dots(v, w.detach()) for v, w in zip(c, u)) * dots(x, x) / sum(dots(z, z) for z in g)
        lost = 2.0 ** -8 * 4 / 3 ** 0.5 * dots(a.double() ** 2, x.double() ** 2).sqrt()
        assert a.dtype == torch.bfloat16 and ((dots(a, x) - common).abs() <= 2.0 ** -8 * common.abs() + lost).all()


def test_the_write_rule_with_and_without_recomputation():
    """Regions that are computed again in the backward pass give the meta-gradient of regions that are kept: the same statements on the
    same numbers but for the order of some f32 sums, whose 2^-24 grow up to 485-fold in the direction and by as much in its derivative:
    2^-24 485^2 = 1.4e-2 of the gradient."""
    import dataclasses as dc
    eng = make_engine(inner_update="muon5")
    ids = torch.randint(0, 120, (2, 32), generator=torch.Generator().manual_seed(3))
    lc = loss_config(eng.tc)
    l0, kept, _ = loss_and_grads(eng, ids, dc.replace(lc, remat=False))
    l1, again, _ = loss_and_grads(eng, ids, dc.replace(lc, remat=True))
    assert abs(l0 - l1) < 1e-5
    for k in kept:
        assert (kept[k] - again[k]).norm() <= 1.4e-2 * kept[k].norm() + 1e-12, k
