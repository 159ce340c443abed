"""Drawing and committing on the CPU: the statements against loops over single rows, and every refusal."""
import math

import pytest
import torch

from dttt_b200.ops.sampling import sample_tokens, unmask


def one_row(x, u, t, k, p, m):
    """The definition, token by token, in Python floats."""
    V = len(x)
    top = max(x)
    if t == 0:
        return x.index(top)
    w = [math.exp((v - top) / t) for v in x]
    order = sorted(range(V), key=lambda i: (-x[i], i))[:k or V]
    mass, kept, run = math.fsum(w[i] for i in order), set(), 0.0
    for i in order:
        if p < 1 and run >= p * mass:
            break
        run += w[i]
        if w[i] >= m:
            kept.add(i)
    total, run = math.fsum(w[i] for i in kept), 0.0
    for i in range(V):
        if i in kept:
            run += w[i]
            if run > u * total:
                return i


@pytest.mark.parametrize("t,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.8, 0.0), (0.9, 0, 1.0, 0.1),
                                     (1.1, 9, 0.6, 0.05), (0.0, 3, 0.5, 0.2), (1e-3, 0, 1.0, 0.0), (0.8, 1, 1.0, 0.0), (0.8, 0, 1e-6, 0.0)])
def test_tokens_follow_the_definition(t, k, p, m):
    gen = torch.Generator().manual_seed(int(100 * t) + k)
    x = torch.randn(40, 23, generator=gen) * 2
    x[10:20] = torch.round(x[10:20])                                   # many equal values
    x[20:30, ::2] = float("-inf")
    u = torch.rand(40, generator=gen)
    out = sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert out.tokens.tolist() == [one_row(a.tolist(), b, t, k, p, m) for a, b in zip(x, u.tolist())]
    lp = torch.log_softmax(x.double(), -1)
    assert torch.allclose(out.logp.double(), lp.gather(-1, out.tokens[:, None])[:, 0], atol=1e-6) and out.priority.equal(out.logp)


def test_priorities_bias_and_rows_without_a_distribution():
    gen = torch.Generator().manual_seed(0)
    x, u = torch.randn(3, 4, 11, generator=gen), torch.rand(3, 4, generator=gen)
    bias = torch.zeros(3, 11)
    bias[:, 5] = float("-inf")
    bias[1, :] -= torch.arange(11) * 0.25
    p = torch.softmax((x + bias[:, None]).double(), -1)
    margin = sample_tokens(x, u, bias=bias, priority="margin")
    entropy = sample_tokens(x, u, bias=bias, priority="entropy")
    top = p.topk(2, -1).values
    assert (margin.tokens != 5).all() and margin.tokens.equal(entropy.tokens)
    assert torch.allclose(margin.priority.double(), top[..., 0] - top[..., 1], atol=1e-6)
    assert torch.allclose(entropy.priority.double(), torch.xlogy(p, p).sum(-1), atol=1e-6)
    x[0, 0, 3], x[1, 1, 2], x[2, 2] = float("nan"), float("inf"), float("-inf")
    out = sample_tokens(x, u)
    void = torch.zeros(3, 4, dtype=torch.bool)
    void[0, 0] = void[1, 1] = void[2, 2] = True
    assert out.tokens.eq(-1).equal(void) and out.logp.isnan().equal(void)


def test_parameters_per_row_are_the_scalars_row_by_row():
    gen = torch.Generator().manual_seed(1)
    x, u = torch.randn(4, 3, 50, generator=gen), torch.rand(4, 3, generator=gen)
    t = torch.tensor([0.0, 0.5, 1.0, 1.5])[:, None]
    k, p, m = torch.tensor([0, 4, 50]), torch.tensor([[1.0], [0.5], [0.25], [1.0]]), torch.rand(4, 3, generator=gen) * 0.1
    out = sample_tokens(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    for i in range(4):
        for j in range(3):
            one = sample_tokens(x[i, j][None], u[i, j][None], temperature=float(t[i, 0]), top_k=int(k[j]), top_p=float(p[i, 0]),
                                min_p=float(m[i, j]))
            assert int(one.tokens) == int(out.tokens[i, j])
    odd = sample_tokens(x[:1], u[:1], temperature=torch.tensor([-1.0, float("nan"), 1.0]), top_k=torch.tensor([-3, 0, 2 ** 40]),
                        top_p=torch.tensor([float("nan"), 2.0, -1.0]), min_p=torch.tensor([float("nan"), -1.0, 7.0]))
    assert odd.tokens.equal(x[:1].argmax(-1))                          # greedy, greedy, the best token alone


def test_draw_numbers_at_the_edges():
    x = torch.tensor([[float("-inf"), 0.0, 1.0, float("-inf")]]).expand(5, 4)
    u = torch.tensor([0.0, -1.0, float("nan"), 1.0, 7.0])
    assert sample_tokens(x, u).tokens.tolist() == [1, 1, 1, 2, 2]
    assert sample_tokens(x[:0], u[:0]).tokens.shape == (0,)


@pytest.mark.parametrize("change,word", [(dict(temperature=-0.1), "temperature"), (dict(temperature=float("nan")), "temperature"),
                                         (dict(temperature=float("inf")), "temperature"), (dict(top_k=-1), "top_k"),
                                         (dict(top_p=0.0), "top_p"), (dict(top_p=1.5), "top_p"), (dict(min_p=-0.1), "min_p"),
                                         (dict(min_p=1.01), "min_p"), (dict(priority="best"), "priority"),
                                         (dict(bias=torch.zeros(2, 6)), "bias"), (dict(bias=torch.zeros(3, 7, dtype=torch.float64)), "bias"),
                                         (dict(u=torch.zeros(2)), "u "), (dict(u=torch.zeros(3, dtype=torch.float64)), "u "),
                                         (dict(logits=torch.zeros(7)), "logits"), (dict(logits=torch.zeros(3, 0)), "logits"),
                                         (dict(logits=torch.zeros(3, 7, dtype=torch.int64)), "logits"),
                                         (dict(top_k=torch.tensor([0.5, 1.0, 2.0])), "top_k"), (dict(top_p=torch.ones(2)), "top_p"),
                                         (dict(temperature=torch.ones(3, dtype=torch.int64)), "temperature")])
def test_sample_refusals(change, word):
    args = dict(logits=torch.zeros(3, 7), u=torch.zeros(3))
    args.update(change)
    with pytest.raises(ValueError, match=word):
        sample_tokens(args.pop("logits"), args.pop("u"), **args)


def commit_args(B=3, C=9, seed=0):
    gen = torch.Generator().manual_seed(seed)
    known = torch.rand(B, C, generator=gen) < 0.4
    return [torch.randint(0, 50, (B, C), generator=gen), known, torch.zeros(B, C), torch.randint(50, 99, (B, C), generator=gen),
            -torch.rand(B, C, generator=gen), torch.round(torch.randn(B, C, generator=gen)), torch.randint(0, C, (B,), generator=gen)]


@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("sure", [None, -0.3])
def test_unmask_commits_the_best_open_slots(part, sure):
    args = commit_args()
    ids, known, held, tokens, logp, priority, quota = args
    allowed = torch.rand(3, 9, generator=torch.Generator().manual_seed(4)) < 0.6 if part else None
    out = unmask(*args, allowed=allowed, sure=sure)
    for b in range(3):
        open_ = [i for i in range(9) if not known[b, i] and (allowed is None or allowed[b, i])]
        want = set(sorted(open_, key=lambda i: (-float(priority[b, i]), i))[:int(quota[b])])
        if sure is not None:
            want |= {i for i in range(9) if not known[b, i] and float(logp[b, i]) >= sure}
        assert {i for i in range(9) if out.where[b, i]} == want
    assert out.ids.equal(torch.where(out.where, tokens, ids)) and out.known.equal(known | out.where)
    assert out.logp.equal(torch.where(out.where, logp, held))


@pytest.mark.parametrize("at,bad", [(0, torch.zeros(3, 8, dtype=torch.int64)), (0, torch.zeros(9, dtype=torch.int64)),
                                    (1, torch.zeros(3, 9)), (2, torch.zeros(3, 9, dtype=torch.float64)), (3, torch.zeros(3, 9)),
                                    (4, torch.zeros(3, 9, dtype=torch.bfloat16)), (5, torch.zeros(2, 9)),
                                    (6, torch.zeros(3, dtype=torch.int32)), (6, torch.zeros(2, dtype=torch.int64))])
def test_unmask_refusals(at, bad):
    args = commit_args()
    args[at] = bad
    with pytest.raises(ValueError, match="unmask"):
        unmask(*args)
    with pytest.raises(ValueError, match="sure"):
        unmask(*commit_args(), sure=float("nan"))


@pytest.mark.parametrize("k", [5.5, torch.tensor(2.25), float("inf"), float("nan")])
def test_a_part_of_a_token_is_not_a_top_k(k):
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(torch.zeros(2, 9), torch.zeros(2), top_k=k)
    assert sample_tokens(torch.zeros(2, 9), torch.zeros(2), top_k=5.0).tokens.tolist() == [0, 0]
