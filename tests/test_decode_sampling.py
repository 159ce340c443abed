"""Decoding with truncated and inverse draws and the five-step write: determinism, agreement of the options, refusals."""
import pytest
import torch

from util import make_engine, tiny_model
from dttt_b200 import generate as G
from dttt_b200.ckpt import store as CK
from dttt_b200.utils import rng

PROMPT = torch.randint(0, 120, (11,), generator=torch.Generator().manual_seed(3))


def run(net, opts, seed=5, **kw):
    return G.generate(net, PROMPT, 14, rng.key(seed), steps=4, fused_ce_block=0, opts=opts, **kw)


@pytest.mark.parametrize("opts", [G.DecodeOpts(top_k=5), G.DecodeOpts(top_p=0.8), G.DecodeOpts(min_p=0.1), G.DecodeOpts(sampler="inverse"),
                                  G.DecodeOpts(top_k=20, top_p=0.9, min_p=0.02, priority="margin", presence_penalty=0.5),
                                  G.DecodeOpts(top_p=0.7, priority="entropy", remask_loop=1, remask_k=3),
                                  G.DecodeOpts(top_p=0.9, threshold=0.05), G.DecodeOpts(top_p=0.9, order="random")])
@pytest.mark.parametrize("kw", [dict(), dict(outer_shift=True, inner_task="causal", inner_update_rule="muon5")])
def test_draws_are_deterministic_and_keep_the_prompt(opts, kw):
    net = make_engine().net(train=False)
    a, b, c = run(net, opts, temperature=1.0, **kw), run(net, opts, temperature=1.0, **kw), run(net, opts, seed=6, temperature=1.0, **kw)
    assert a.shape == (25,) and torch.equal(a, b) and torch.equal(a[:11], PROMPT) and not torch.equal(a, c)
    assert (a != 127).all() and (a >= 0).all()


def test_the_best_token_alone_is_the_greedy_choice():
    net = make_engine().net(train=False)
    for kw in (dict(), dict(outer_shift=True, inner_task="causal")):
        greedy = run(net, G.DecodeOpts(), temperature=0.0, **kw)
        assert torch.equal(greedy, run(net, G.DecodeOpts(sampler="inverse"), temperature=0.0, **kw))
        assert torch.equal(greedy, run(net, G.DecodeOpts(top_k=1), temperature=1.0, **kw))
        assert torch.equal(greedy, run(net, G.DecodeOpts(top_p=1e-6), temperature=0.7, **kw))


def test_read_block_and_cli(tmp_path, capsys):
    eng = make_engine(mc=tiny_model(read_block=4))
    out = G.generate(eng.net(train=False), PROMPT[:5], 12, rng.key(1), steps=4, temperature=1.0, fused_ce_block=0, outer_shift=True,
                     inner_task="causal", opts=G.DecodeOpts(top_p=0.9))
    assert out.shape == (17,)
    d = CK.save(str(tmp_path / "ck"), 0, make_engine(), "h")
    G.main(["--ckpt", d, "--prompt_ids", "5,6,7,8", "--max_new_tokens", "6", "--steps", "2", "--inner_task", "causal", "--temperature", "0.8",
            "--top_k", "30", "--top_p", "0.9", "--min_p", "0.01", "--sampler", "inverse", "--inner_update", "muon5"])
    printed = capsys.readouterr().out.strip().split(",")
    assert len(printed) == 6 and all(0 <= int(x) < 128 for x in printed)


@pytest.mark.parametrize("opts", [G.DecodeOpts(sampler="beam"), G.DecodeOpts(top_k=-1), G.DecodeOpts(top_p=0.0), G.DecodeOpts(top_p=1.5),
                                  G.DecodeOpts(min_p=-0.1), G.DecodeOpts(min_p=1.1)])
def test_refusals(opts):
    with pytest.raises(ValueError, match="DecodeOpts"):
        run(make_engine().net(train=False), opts)


@pytest.mark.parametrize("opts", [G.DecodeOpts(top_p=0.9), G.DecodeOpts(top_k=5, presence_penalty=0.5), G.DecodeOpts(sampler="inverse", threshold=0.1),
                                  G.DecodeOpts(min_p=0.1, remask_loop=1, remask_k=3)])
@pytest.mark.parametrize("kw", [dict(), dict(outer_shift=True, inner_task="causal")])
def test_logits_without_a_distribution_are_an_error_and_never_an_index(opts, kw, monkeypatch):
    """A model that has diverged: every row of logits is NaN, so there is no token to commit; what the embedding is asked for stays
    inside its table."""
    from dttt_b200.ops import embed as E
    net = make_engine().net(train=False)
    seen, plain = [], E.embedding
    monkeypatch.setattr(E, "embedding", lambda table, ids, *a, **k: seen.append(ids.clone()) or plain(table, ids, *a, **k))
    with torch.no_grad():
        net.p("final_norm.weight").fill_(float("nan"))
    with pytest.raises(FloatingPointError, match="distribution"):
        run(net, opts, temperature=1.0, **kw)
    assert seen and all(((ids >= 0) & (ids < 128)).all() for ids in seen)


def test_only_rows_that_are_drawn_need_a_distribution(monkeypatch):
    """A slot whose token is known is not drawn: what its logits hold does not matter.  A slot that is open does, and rounds that end by
    confidence end with the first of it."""
    net = make_engine().net(train=False)
    plain, rounds = G.block_forward, []

    def broken(where):
        def forward(net, ids, pos, state, *a, **k):
            rounds.append(1)
            out = plain(net, ids, pos, state, *a, **k)
            for slot in where:
                out[0][:, slot] = float("nan")
            return out
        return forward

    decode = lambda opts: G.decode_block(net, ids, known, pos, G.init_state(net), rng.key(3), 3, 1.0, opts=opts)
    ids = torch.tensor([[5, 6, 7, 127, 127, 127, 127, 127]])
    known, pos = ids != 127, torch.arange(8)[None]
    monkeypatch.setattr(G, "block_forward", broken([0, 2]))
    out, _ = decode(G.DecodeOpts(top_p=0.9))
    assert torch.equal(out[:, :3], ids[:, :3]) and ((out >= 0) & (out < 127)).all()
    monkeypatch.setattr(G, "block_forward", broken([4]))
    for opts in (G.DecodeOpts(top_p=0.9), G.DecodeOpts(top_p=0.9, threshold=0.999)):
        rounds.clear()
        with pytest.raises(FloatingPointError):
            decode(opts)
    assert len(rounds) == 1
