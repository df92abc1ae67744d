"""Generation against the oracle model, which computes every sequence anew from its first token in fp32 or 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout, init_flat
from cme213_final_project_b200.config import ModelConfig
from cme213_final_project_b200.generate import CacheFull, Generator, Sampling, main
from cme213_final_project_b200.models.reference import forward

PROMPTS = [[1, 2, 3, 4, 5], list(range(40)), [7], [(i * 7) % 65 for i in range(61)]]


def model(dtype, hidden=128, heads=4, layers=2, vocab=65, seq_len=96):
    cfg = ModelConfig(mode="gpt", vocab_size=vocab, seq_len=seq_len, hidden=hidden, heads=heads, ff=2 * hidden, layers=layers, batch_size=1,
                      activation="gelu", causal=True, head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg, align=64)
    flat = init_flat(layout, 3)
    flat *= 4.0                                            # (with the small weights of a fresh model all logits are nearly the same)
    return cfg, layout, flat.to(dtype).cuda()


def oracle(cfg, layout, params, tokens):
    """Logits after each token, in 64 bits."""
    P = {k: v.double().cpu() for k, v in layout.views(params).items()}
    one = ModelConfig(**{**cfg.__dict__, "seq_len": len(tokens)})
    P["pos_embed"] = P["pos_embed"][:len(tokens)]
    return forward(P, one, torch.tensor(tokens, dtype=torch.int32), None)[1]


@pytest.mark.parametrize("heads", [4, 2, 1])
@pytest.mark.parametrize("chunk", [512, 7])
def test_logits_after_prompts_and_steps(heads, chunk):
    """Logits are held to 1 % of their spread; products are exact in fp32."""
    cfg, layout, params = model(torch.float32, heads=heads)
    gen = Generator(cfg, layout, params, len(PROMPTS))
    logits = gen.prefill(PROMPTS, chunk)
    want = torch.stack([oracle(cfg, layout, params, p)[-1] for p in PROMPTS])
    assert float((logits.cpu().double() - want).abs().max()) < 0.01 * float(want.std())
    more = [3, 9, 27, 50]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    positions = i32(gen.cache.lengths)
    gen.cache.grow([1] * 4)
    logits = gen.forward(i32(more), positions, i32([0, 1, 2, 3, 4]), i32(gen.cache.lengths), i32([0, 1, 2, 3]))
    want = torch.stack([oracle(cfg, layout, params, p + [t])[-1] for p, t in zip(PROMPTS, more)])
    assert float((logits.cpu().double() - want).abs().max()) < 0.01 * float(want.std())
    assert ops.attention_check_status() == 0 and ops.gemm_check_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_run_is_what_its_steps_are(dtype):
    """With a CUDA graph or without, all prompts at once or one by one: greedy tokens of one model are close to the oracle's best."""
    cfg, layout, params = model(dtype)
    runs = [Generator(cfg, layout, params, len(PROMPTS)).generate(PROMPTS, 12, cuda_graph=g) for g in (True, False)]
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    tokens, logprobs = runs[0]
    for p, row, lp in zip(PROMPTS, tokens.tolist(), logprobs.tolist()):
        logits = oracle(cfg, layout, params, p + row)[len(p) - 1:-1]
        # a bf16 model's logits are off by some 2^-8 of their spread in each of its layers
        slack = (0.02 if dtype == torch.float32 else 0.1) * float(logits.std())
        for x, t, l in zip(logits, row, lp):
            assert float(x.max() - x[t]) <= slack
            assert abs(float(torch.log_softmax(x, 0)[t]) - l) <= 2 * slack
    assert ops.attention_check_status() == 0


def test_sampling_masks_and_seeds():
    cfg, layout, params = model(torch.bfloat16)
    only = [5, 11, 64]
    make = lambda seed, **kw: Generator(cfg, layout, params, 4).generate(PROMPTS, 20, Sampling(1.5, allowed=only, **kw), seed)[0]
    a, b, c = make(1), make(1), make(2)
    assert torch.equal(a, b) and not torch.equal(a, c) and set(a.unique().tolist()) <= set(only)
    # one token may come, and once it has come it may not again: the mask and the penalty together end nothing, a mask without tokens does
    d = Generator(cfg, layout, params, 4).generate(PROMPTS, 4, Sampling(0.0, allowed=[]))[0]
    assert bool((d == -1).all())
    # a penalty for what was generated: no token comes twice
    e = Generator(cfg, layout, params, 4).generate(PROMPTS, 20, Sampling(0.0, presence=1e4))[0]
    assert all(len(set(r)) == 20 for r in e.tolist())
    # a bias decides
    f = Generator(cfg, layout, params, 4).generate(PROMPTS, 3, Sampling(0.0, bias={17: 1e4}))[0]
    assert bool((f == 17).all())


def test_pages_run_out_and_prompts_are_too_long():
    cfg, layout, params = model(torch.bfloat16)
    with pytest.raises(CacheFull):
        Generator(cfg, layout, params, 4, pages=3).generate(PROMPTS, 4)
    with pytest.raises(ValueError):
        Generator(cfg, layout, params, 4).generate(PROMPTS, 60)
    with pytest.raises(ValueError):
        Generator(cfg, layout, params, 4).prefill(PROMPTS[:3])
    gen = Generator(cfg, layout, params, 4)
    gen.generate(PROMPTS, 96 - 61 + 1)                     # up to the last position


def test_train_then_generate(tmp_path, capsys):
    """A few steps on a text of one phrase, a checkpoint, and the phrase comes back."""
    from cme213_final_project_b200.train import main as train
    text, ck = tmp_path / "text.txt", tmp_path / "model.ck"
    text.write_text("the quick brown fox jumps over the lazy dog. " * 400)
    assert train([str(text), "--preset", "tiny-gpt", "--epochs", "8", "--lr", "3e-3", "--save-checkpoint", str(ck)]) == 0
    capsys.readouterr()
    assert main(["--checkpoint", str(ck), "--data", str(text), "--prompt", "the quick", "--prompt", "jumps over", "--max-new", "30",
                 "--temperature", "0"]) == 0
    out = capsys.readouterr().out
    assert "the quick brown fox jumps over the" in out and "jumps over the lazy dog. the" in out
