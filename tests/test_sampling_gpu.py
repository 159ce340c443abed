"""The sampling and commit kernels against the 64-bit statements of ``ops.reference``.

Tokens are whole numbers and have to be equal: both sides form the masses in 64 bits, and a border between two tokens lies
within the kernel's rounding of a draw with a probability of about 1e-6 per row at these sizes (fixed seeds).

Bound of the log-probability: ``x - m`` rounds once (2^-24 of at most 80: 4.8e-6), the sum of exponentials is off by at most the
probability-weighted error of the fast exponential, ``(2 + 1.2 E|d|) 2^-23`` with ``E|d| <= log V < 13`` (2.1e-6), the logarithm
and the last subtraction round once each (2^-24 of at most 80 and 13: 5.6e-6): 1.3e-5 in all.  The margin and the entropy are
weighted means with the same weights: 2.1e-6 of at most 1, and of at most 13 (2.8e-5 with the logarithm's share)."""
import math

import pytest
import torch

from dttt_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
TOL = {"logp": 1.3e-5, "margin": 4e-6, "entropy": 4e-5}


def logits(rows, V, dtype=torch.float32, seed=0, kind="zipf"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.randn(*rows, V, generator=gen, device="cuda")
    if kind == "zipf":
        x = r - 1.2 * torch.log1p(torch.randperm(V, generator=gen, device="cuda").float())
    elif kind == "flat":
        x = r * 1e-3
    elif kind == "ties":
        x = torch.round(2 * r) / 2
    elif kind == "equal":
        x = torch.zeros_like(r)
    elif kind == "wide":
        x = r * 30
    elif kind == "few":
        x = torch.where(torch.rand(*rows, V, generator=gen, device="cuda") < 3.0 / V, r, float("-inf"))
        x[..., V // 2] = 0.5
    return x.to(dtype), torch.rand(*rows, generator=gen, device="cuda")


def check(x, u, priority="logp", **kw):
    from dttt_b200.ops.sampling import sample_tokens
    bias = kw.pop("bias", None)
    out = sample_tokens(x, u, bias=bias, priority=priority, **kw)
    full = lambda v, d: (v.double() if d is torch.float64 else v.long()).expand(u.shape) if torch.is_tensor(v) else \
        torch.full(u.shape, v, dtype=d, device="cuda")
    want = ref.sample_tokens(x, u, bias, full(kw.get("temperature", 1.0), torch.float64), full(kw.get("top_k", 0), torch.int64),
                             full(kw.get("top_p", 1.0), torch.float64), full(kw.get("min_p", 0.0), torch.float64), priority)
    assert out.tokens.equal(want[0]), (out.tokens != want[0]).nonzero()[:5].tolist()
    for got, exp, tol in ((out.logp, want[1], TOL["logp"]), (out.priority, want[2], TOL[priority])):
        assert got.isnan().equal(exp.isnan())
        assert torch.nan_to_num(got - exp).abs().max().item() <= tol
    return out


PARAMS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_p=0.9), dict(temperature=1.4, top_k=40), dict(min_p=0.05),
          dict(temperature=0.8, top_k=300, top_p=0.7, min_p=0.01), dict(temperature=2.0, top_p=0.999), dict(temperature=1e-6),
          dict(temperature=1e6, top_p=0.3), dict(top_k=1), dict(top_p=1e-9), dict(min_p=1.0)]


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1023, 4096, 16384, 16385, 32001, 65537, 128256])
@pytest.mark.parametrize("kw", PARAMS)
def test_sizes_and_truncations(V, kw):
    check(*logits((2, 5), V, seed=V), **kw)


@pytest.mark.parametrize("kind", ["flat", "ties", "equal", "wide", "few"])
@pytest.mark.parametrize("kw", PARAMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_distributions_and_types(kind, kw, dtype):
    for V in (999, 40003):
        check(*logits((3, 4), V, dtype, seed=V, kind=kind), **kw)


@pytest.mark.parametrize("priority", ["logp", "margin", "entropy"])
@pytest.mark.parametrize("V", [1, 700, 20000, 128256])
def test_priorities_with_bias_and_strides(priority, V):
    x, u = logits((3, 6), V, torch.bfloat16, seed=5)
    bias = torch.where(torch.rand(3, V, device="cuda") < 0.3, -1.5, 0.0)
    if V > 1:
        bias[:, 0] = float("-inf")
    check(x, u, priority, bias=bias, top_p=0.8)
    check(x[:, :-1], u[:, :-1], priority, bias=bias, top_p=0.8)            # a view: rows of the last slot left out
    check(x[:, 1:, V // 3:], u[:, 1:], priority, top_k=7)                  # rows that start off 16 bytes
    check(x[:, ::2], u[:, ::2], priority)
    check(x[:1].expand(3, 6, V), u, priority, top_k=5)
    check(x.permute(1, 0, 2), u.t(), priority)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), u, priority)     # not contiguous along V


def test_two_and_four_dimensions_and_empty():
    from dttt_b200.ops.sampling import sample_tokens
    x, u = logits((2, 3, 4), 500)
    flat = check(x.view(24, 500), u.view(24))
    assert check(x, u).tokens.equal(flat.tokens.view(2, 3, 4))
    assert sample_tokens(x[:0], u[:0]).tokens.shape == (0, 3, 4)
    assert sample_tokens(x[:, :0].view(2, 0, 500), u[:, :0].view(2, 0)).logp.shape == (2, 0)


def test_rows_without_a_distribution_and_edge_draws():
    x, u = logits((4, 8), 50001)
    x[0, 0, 49999], x[1, 1, 3], x[2, 2], x[3, 3] = float("nan"), float("inf"), float("-inf"), -3e38
    u[0, 1], u[0, 2], u[0, 3], u[0, 4] = 0.0, 1.0, -1.0, 1 - 2 ** -24
    for kw in PARAMS:
        for pr in ("logp", "margin", "entropy"):
            out = check(x, u, pr, **kw)
            assert out.tokens[0, 0] == out.tokens[1, 1] == out.tokens[2, 2] == -1 and out.priority[0, 0].isnan()


@pytest.mark.parametrize("V", [70, 5000, 50001])
@pytest.mark.parametrize("top", [-3e38, -1e30, 1e30, 3e38, 1e12])
def test_values_whose_neighbours_are_octaves_away(V, top):
    """At 1e30 the next smaller float is far more than any temperature away: all of the mass is at the maximum."""
    x, u = logits((4, 8), V)
    x = x.abs().neg() * 1e25
    x[:] += top
    x[0], x[1, :, ::3] = top, top
    for kw in PARAMS:
        check(x, u, **kw)
    check(x.repeat(5, 9, 1), u.repeat(5, 9))                               # enough rows for the two-launch form at the largest V


@pytest.mark.parametrize("V", [3000, 20000, 128256])
@pytest.mark.parametrize("near", [100, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_p_next_to_a_border(V, near, dtype):
    """top_p so close to the part of the mass that a prefix has that 32-bit sums would not tell on which side it is: a billionth of it
    is more than the 64-bit masses are off."""
    x, u = logits((2, 8), V)
    x = x.clamp(-1, 1) * 0.5
    x[..., near:] -= 3 + math.log(V / near)                                # few candidates, or more than fit a list
    x = x[..., torch.randperm(V, device="cuda")].to(dtype)
    x[1] = x[0] = x[0, 0].clone()
    w = torch.exp((x[0, 0].double() - x[0, 0].max().double()) / 0.7).sort(descending=True).values
    part = w.cumsum(0) / w.sum()
    for j in (0, 3, near // 3, near - 10):
        for off in (-1e-5, -1e-9, 1e-9, 1e-5, 1e-3):
            check(x, u, temperature=0.7, top_p=part[j].item() * (1 + off), bias=torch.zeros(2, V, device="cuda") if j == 3 else None)


def test_parameters_per_row():
    x, u = logits((6, 8), 30000, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.rand(*s, generator=gen, device="cuda")
    t = (r(6, 1) * 2 - 0.3)
    check(x, u, temperature=t, top_k=torch.randint(-3, 200, (8,), generator=gen, device="cuda"), top_p=r(6, 8) * 1.2, min_p=r(1, 8) * 0.1)


def test_every_draw_number_of_one_row():
    """A sweep of ``u`` over one row: the tokens have to be those of the row's distribution function, in order."""
    V = 20011
    x, _ = logits((1, 1), V, seed=9)
    u = (torch.arange(4096, device="cuda").float() / 4096).view(1, -1)
    out = check(x.expand(1, 4096, V), u, temperature=1.1, top_p=0.95)
    assert (out.tokens.diff() >= 0).all()


@pytest.mark.parametrize("V", [1000, 2049, 32001, 128256, 390001])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.0), dict(temperature=0.6), dict(temperature=1e-6), dict(temperature=1e6)])
def test_untruncated_draws_over_chunks(V, kw):
    """Enough elements for the two passes over chunks: every type, priority, ragged row starts, bias, rows without a distribution."""
    rows = -(-(2 << 20) // V) + 3
    for dtype, priority in ((torch.float32, "entropy"), (torch.bfloat16, "margin"), (torch.float16, "logp")):
        for kind in ("zipf", "ties", "few"):
            x, u = logits((1, rows + 1), V + 3, dtype, seed=V, kind=kind)
            x, u = x[:, 1:, 3:], u[:, 1:].clone()
            x[0, 0] = float("-inf")
            x[0, 1, V // 2] = float("nan")
            x[0, 2, V - 1] = float("inf")
            u[0, 3], u[0, 4], u[0, 5] = 0.0, 1.0, 1 - 2 ** -24
            bias = torch.where(torch.rand(1, V, device="cuda") < 0.2, -2.0, 0.0)
            out = check(x, u, priority, bias=bias if kind == "zipf" else None, **kw)
            assert (out.tokens[0, :3] == -1).all() and (out.tokens[0, 3:] >= 0).all()
    t = torch.rand(1, rows, device="cuda") - 0.3                            # greedy rows among drawn ones
    check(*logits((1, rows), V, seed=1), temperature=t)


def test_above_the_three_cta_slices_and_refusal():
    from dttt_b200.ops.sampling import sample_tokens
    for V in (131073, 393216):
        for kw in (dict(top_p=0.9), dict(top_k=50), dict()):
            check(*logits((1, 2), V), **kw)
    with pytest.raises(ValueError, match="393216"):
        sample_tokens(torch.zeros(1, 393217, device="cuda"), torch.zeros(1, device="cuda"), top_k=5)
    with pytest.raises(ValueError, match="u "):
        sample_tokens(torch.zeros(1, 10, device="cuda"), torch.zeros(1))


def test_repeats_streams_and_graphs():
    from dttt_b200.ops.sampling import sample_tokens
    x, u = logits((2, 40), 33333)
    kw = dict(temperature=0.9, top_p=0.8, top_k=1000, priority="entropy")
    first = sample_tokens(x, u, **kw)
    for _ in range(3):
        again = sample_tokens(x, u, **kw)
        assert all(a.equal(b) for a, b in zip(first, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sample_tokens(x, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(a.equal(b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    xs, us = x.clone(), u.clone()
    with torch.cuda.graph(graph):
        held = sample_tokens(xs, us, **kw)
    x2, u2 = logits((2, 40), 33333, seed=8)
    xs.copy_(x2); us.copy_(u2)
    graph.replay()
    assert all(a.equal(b) for a, b in zip(held, sample_tokens(x2, u2, **kw)))


@pytest.mark.parametrize("kw", [dict(temperature=0.8, top_p=0.9), dict(temperature=0.9), dict(top_k=700, min_p=1e-4), dict(temperature=1.3, top_p=0.99)])
def test_two_graphs_at_once(kw):
    """Each graph has its own workspaces; replayed side by side on two streams, on inputs that change between replays."""
    from dttt_b200.ops.sampling import sample_tokens
    sides, held = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for n in range(2):
        x, u = logits((1, 70), 40001, seed=n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sample_tokens(x, u, **kw)
        held.append((graph, x, u, out))
    for turn in range(3):
        for n, (graph, x, u, out) in enumerate(held):
            x2, u2 = logits((1, 70), 40001, seed=10 * turn + n, kind=("zipf", "ties", "flat")[turn])
            x.copy_(x2); u.copy_(u2)
        torch.cuda.synchronize()
        for side, (graph, *_) in zip(sides, held):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, x, u, out in held:
            assert all(a.equal(b) for a, b in zip(out, sample_tokens(x, u, **kw)))


@pytest.mark.parametrize("V", [700, 5003, 128256, 390001])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.4), dict(top_k=650), dict(top_p=1 - 1e-7, temperature=1.3), dict(min_p=1e-30),
                                dict(temperature=0.5, top_k=699, min_p=1e-25), dict(temperature=1e-3), dict(top_k=4, top_p=0.9)])
def test_draws_below_the_unit_of_mass(V, kw):
    """Numbers near 0 draw the first tokens of a row however little mass they have: of 0 the first kept one that has any in 64
    bits, of others the one where the running mass passes.  Rows that start with masses of e^-2000 to e^-20; many rows at once,
    too, for the two-launch form.  (A border is met with the relative rounding of 64-bit sums only.)  Log-probabilities lie as low as
    -2000 here, where the three roundings to f32 (x - m, the last subtraction, the oracle's result) are 2^-24 of them each."""
    def far(x, priority, u, **kw):
        from dttt_b200.ops.sampling import sample_tokens
        got = sample_tokens(x, u, priority=priority, **kw)
        par = [torch.full(u.shape, kw.get(k, v), dtype=torch.int64 if k == "top_k" else torch.float64, device="cuda")
               for k, v in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))]
        want = ref.sample_tokens(x, u, None, *par, priority)
        assert got.tokens.equal(want[0]), (got.tokens != want[0]).nonzero()[:5].tolist()
        for a, b, tol in ((got.logp, want[1], TOL["logp"]), (got.priority, want[2], TOL[priority])):
            assert ((a - b).abs() <= tol + 3 * 2.0 ** -24 * b.abs()).all()

    gen = torch.Generator(device="cuda").manual_seed(V)
    u = torch.tensor([0.0, 1e-44, 1e-38, 3e-30, 2e-22, 1e-17, 4e-14, 1e-11, 1e-9, -1.0, 2.0 ** -24], device="cuda")[None]
    x, _ = logits((1, u.shape[1]), V, seed=V, kind="flat")
    low = V // 2
    x[..., :low] -= 20 + 100 * torch.rand(1, u.shape[1], low, generator=gen, device="cuda")
    x[..., :low // 4] = -torch.linspace(800, 60, low // 4, device="cuda")[torch.randperm(low // 4, generator=gen, device="cuda")]
    x[..., :3] = torch.tensor([-2000.0, float("-inf"), -760.0], device="cuda")
    far(x, "logp", u, **kw)
    far(x.to(torch.bfloat16), "entropy", u, **kw)
    many = -(-(9 << 20) // V) // u.shape[1] + 1
    far(x.repeat(1, many, 1)[:, :, 1:], "margin", u.repeat(1, many), **kw)


@pytest.mark.parametrize("V", [1000, 4096, 4097, 8191, 32001, 128256, 390001])
def test_one_launch_or_two(V):
    """Untruncated draws on both sides of the rule: 6.2 million elements and V above 4096 take two launches over a scratch area."""
    from dttt_b200.ops import _lib
    size = _lib.lib().dttt_sample_scratch
    edge = -(-6200000 // V)
    assert size(edge - 1, V) == 0 and (size(edge, V) > 0) == (V > 4096) and (size(4 * edge, V) > 0) == (V > 4096)
    for rows in (edge - 1, edge):
        for dtype, priority, kind, kw in ((torch.float32, "entropy", "zipf", dict()), (torch.bfloat16, "margin", "ties", dict(temperature=0.6)),
                                          (torch.float16, "logp", "few", dict(temperature=1e-6)), (torch.float32, "margin", "wide", dict(temperature=0.0)),
                                          (torch.bfloat16, "entropy", "equal", dict(temperature=1e6))):
            x, u = logits((1, rows), V + 3, dtype, seed=V, kind=kind)
            x, u = x[:, :, 3:], u.clone()
            x[0, 0] = float("-inf")
            x[0, 1, V // 2] = float("nan")
            x[0, 2, V - 1] = float("inf")
            u[0, 3], u[0, 4], u[0, 5] = 0.0, 1.0, 1 - 2 ** -24
            bias = torch.where(torch.rand(1, V, device="cuda") < 0.2, -2.0, 0.0)
            out = check(x, u, priority, bias=bias if kind == "zipf" else None, **kw)
            assert (out.tokens[0, :3] == -1).all() and (out.tokens[0, 3:] >= 0).all()


def test_two_graphs_of_the_two_launch_form():
    """Each graph has a scratch area of its own."""
    from dttt_b200.ops.sampling import sample_tokens
    sides, held = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for n in range(2):
        x, u = logits((2, 90), 40001, seed=n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sample_tokens(x, u, temperature=0.9, priority="margin")
        held.append((graph, x, u, out))
    for turn in range(3):
        for n, (graph, x, u, out) in enumerate(held):
            x2, u2 = logits((2, 90), 40001, seed=10 * turn + n, kind=("zipf", "ties", "flat")[turn])
            x.copy_(x2); u.copy_(u2)
        torch.cuda.synchronize()
        for side, (graph, *_) in zip(sides, held):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for graph, x, u, out in held:
            assert all(a.equal(b) for a, b in zip(out, sample_tokens(x, u, temperature=0.9, priority="margin")))


# ------------------------------------------------------------------------------------------------------------ commit
def commit_args(B, C, seed=0, special=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda: torch.rand(B, C, generator=gen, device="cuda")
    i = lambda: torch.randint(0, 128000, (B, C), generator=gen, device="cuda")
    priority = torch.round(-8 * r()) / 8
    if special:
        priority = torch.where(r() < 0.2, float("nan"), torch.where(r() < 0.2, float("-inf"), torch.where(r() < 0.2, -0.0, priority)))
    return [i(), r() < 0.4, r(), i(), torch.log(r()), priority, torch.randint(-1, C + 2, (B,), generator=gen, device="cuda")]


@pytest.mark.parametrize("B,C", [(1, 1), (1, 31), (7, 64), (3, 257), (300, 1024), (2, 4099), (1, 32768)])
@pytest.mark.parametrize("special", [False, True])
def test_unmask(B, C, special):
    from dttt_b200.ops.sampling import unmask
    args = commit_args(B, C, C, special)
    allowed = torch.rand(B, C, device="cuda") < 0.5
    for kw in (dict(), dict(allowed=allowed), dict(sure=-0.2), dict(allowed=allowed, sure=float("-inf"))):
        for got, want in zip(unmask(*args, **kw), ref.unmask(*args, **kw)):
            assert got.dtype == want.dtype and got.equal(want)
    for q in (0, C, C + 5, -4):
        args[6] = torch.full((B,), q, device="cuda")
        assert all(a.equal(b) for a, b in zip(unmask(*args), ref.unmask(*args)))


def test_unmask_views_empty_and_refusals():
    from dttt_b200.ops.sampling import unmask
    args = commit_args(12, 200)
    cut = [a[::2, 3:100] for a in args[:6]] + [args[6][::2]]
    assert all(a.equal(b) for a, b in zip(unmask(*cut), ref.unmask(*cut)))
    none = [a[:0] for a in args]
    assert unmask(*none).ids.shape == (0, 200)
    wide = commit_args(1, 32769)
    assert all(a.equal(b) for a, b in zip(unmask(*wide), ref.unmask(*wide)))
    with pytest.raises(ValueError, match="quota"):
        unmask(*args[:6], args[6].cpu())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = unmask(*args, sure=-0.1)
    args[5].neg_()
    graph.replay()
    assert all(a.equal(b) for a, b in zip(out, ref.unmask(*args, sure=-0.1)))
