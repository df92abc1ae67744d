"""Several runs of one generator on the GPU, with its CUDA graph: each gives what a new generator gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout, init_flat
from cme213_final_project_b200.config import ModelConfig
from cme213_final_project_b200.generate import CacheFull, Generator, Sampling

PROMPTS = [[1, 2, 3, 4, 5], list(range(40)), [7], [(i * 7) % 65 for i in range(61)]]


def generator(dtype, **kw):
    cfg = ModelConfig(mode="gpt", vocab_size=65, seq_len=96, hidden=128, heads=4, ff=256, layers=2, batch_size=1, activation="gelu", causal=True,
                      head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg, align=64)
    return Generator(cfg, layout, (init_flat(layout, 3) * 4.0).to(dtype).cuda(), len(PROMPTS), **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sampling", [None, Sampling(1.0, 1.2, 0.1, 0.3)])
def test_a_run_does_not_depend_on_the_runs_before_it(dtype, sampling):
    other = [[9], [8, 8], list(range(30)), [1]]
    want = [generator(dtype).generate(p, 12, sampling) for p in (PROMPTS, other)]
    g = generator(dtype)
    logits = g.prefill(PROMPTS)
    for p, w in ((PROMPTS, want[0]), (other, want[1]), (PROMPTS, want[0])):
        got = g.generate(p, 12, sampling)
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    assert torch.equal(g.prefill(PROMPTS), logits)
    assert ops.attention_check_status() == 0 and ops.gemm_check_status() == 0


def test_a_run_after_one_that_failed():
    g = generator(torch.bfloat16, pages=9)
    with pytest.raises(CacheFull):
        g.generate(PROMPTS, 36)
    few = [[1, 2], [3], [4, 5, 6], [7]]
    got, want = g.generate(few, 10), generator(torch.bfloat16).generate(few, 10)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
