"""A few blocks decoded on the GPU with the kernels of a block together: draws, commits, the five-step write."""
import pytest
import torch

from util import tiny_train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_k=50, min_p=0.02, priority="margin", presence_penalty=0.5),
                                dict(sampler="inverse", priority="entropy", threshold=0.02)])
def test_blocks_on_the_kernels(kw):
    from dttt_b200 import generate as G
    from dttt_b200.engine import Engine
    from dttt_b200.ops import _lib, kernels
    from dttt_b200.schema import ModelConfig
    from dttt_b200.utils import rng
    mc = ModelConfig(vocab_size=4096, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, suffix_len=2, chunk_size=128, window_chunks=2, qk_norm=True, mask_token_id=4095, pad_token_id=4094,
                     eos_token_id=4094)
    eng = Engine(mc, tiny_train(compute_dtype="bfloat16", fused_ce_block=2048, seq_len=512), device=torch.device("cuda", 0))
    net = eng.net(train=False)
    prompt = torch.randint(0, 4000, (150,), generator=torch.Generator().manual_seed(1))
    seen = []
    # (the write's gradient adds up in an order that may change from run to run, so runs are compared with its step at 0)
    for seed, lr in ((1, 0.0), (1, 0.0), (2, 0.0), (2, 1.0)):
        n = kernels.LAUNCHES
        out = G.generate(net, prompt, 200, rng.key(seed), steps=4, temperature=0.9, inner_lr=lr, inner_task="causal", outer_shift=True,
                         inner_update_rule="muon5", opts=G.DecodeOpts(**kw))
        torch.cuda.synchronize()
        _lib.check_status()
        assert kernels.LAUNCHES > n and out.shape == (350,) and torch.equal(out[:150].cpu(), prompt)
        assert ((out >= 0) & (out < 4095)).all()
        seen.append(out)
    assert torch.equal(seen[0], seen[1]) and not torch.equal(seen[0], seen[2])


def test_a_training_step_with_the_five_step_write():
    """The meta-gradient runs through the direction's derivative on the kernels."""
    from dttt_b200.engine import Engine
    from dttt_b200.ops import _lib
    from dttt_b200.schema import ModelConfig, TrainConfig
    mc = ModelConfig(vocab_size=4096, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, suffix_len=2, chunk_size=128, window_chunks=2, qk_norm=True, mask_token_id=4095, pad_token_id=4094,
                     eos_token_id=4094)
    tc = TrainConfig(seq_len=512, batch_size=2, steps=10, warmup_steps=2, inner_lr_warmup_steps=0, inner_task="causal", outer_shift=True,
                     cart_window=64, fused_ce_block=2048, inner_update="muon5")
    eng = Engine(mc, tc, device=torch.device("cuda", 0))
    ids = torch.randint(0, 4000, (2, 512), device="cuda")
    for s in range(2):
        m = eng.train_step(ids, s)
    torch.cuda.synchronize()
    _lib.check_status()
    assert m["finite"] == 1.0 and m["gnorm_fast_weight"] > 0


def test_a_diverged_model_is_refused():
    """Logits without a distribution: an error at the end of the block, and token ids inside the vocabulary until then."""
    from dttt_b200 import generate as G
    from dttt_b200.engine import Engine
    from dttt_b200.ops import embed as E
    from dttt_b200.schema import ModelConfig
    from dttt_b200.utils import rng
    mc = ModelConfig(vocab_size=4096, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, suffix_len=2, chunk_size=128, window_chunks=2, qk_norm=True, mask_token_id=4095, pad_token_id=4094,
                     eos_token_id=4094)
    eng = Engine(mc, tiny_train(compute_dtype="bfloat16", fused_ce_block=2048, seq_len=512), device=torch.device("cuda", 0))
    net, plain = eng.net(train=False), E.embedding
    with torch.no_grad():
        net.p("final_norm.weight").fill_(float("nan"))

    def looked_up(table, ids, *a, **k):
        assert ((ids >= 0) & (ids < 4096)).all()                            # on the host, before the lookup is launched
        return plain(table, ids, *a, **k)

    E.embedding = looked_up
    try:
        with pytest.raises(FloatingPointError, match="distribution"):
            G.generate(net, torch.arange(20), 100, rng.key(1), steps=3, temperature=0.9, outer_shift=True, inner_task="causal",
                       opts=G.DecodeOpts(top_p=0.9, presence_penalty=0.5))
    finally:
        E.embedding = plain


def test_a_kernel_that_gave_up_is_reported(monkeypatch):
    """A block whose kernels recorded an error (here: put into the status word by the test, before the block's write) does not become
    context of the next one in silence."""
    from dttt_b200 import generate as G
    from dttt_b200.engine import Engine
    from dttt_b200.ops import _lib
    from dttt_b200.schema import ModelConfig
    from dttt_b200.utils import rng
    mc = ModelConfig(vocab_size=4096, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, suffix_len=2, chunk_size=128, window_chunks=2, qk_norm=True, mask_token_id=4095, pad_token_id=4094,
                     eos_token_id=4094)
    eng = Engine(mc, tiny_train(compute_dtype="bfloat16", fused_ce_block=2048, seq_len=512), device=torch.device("cuda", 0))
    net, blocks, plain = eng.net(train=False), [], G.commit_block

    def commit(*a, **k):
        blocks.append(1)
        if len(blocks) == 2:
            _lib.status_tensor(torch.device("cuda", 0))[0] = 3
        return plain(*a, **k)

    monkeypatch.setattr(G, "commit_block", commit)
    with pytest.raises(_lib.KernelError, match="accumulator"):
        G.generate(net, torch.arange(20), 400, rng.key(1), steps=2, outer_shift=True, inner_task="causal", inner_update_rule="muon5")
    assert len(blocks) == 2
    _lib.check_status()                                                     # the report has reset the word
