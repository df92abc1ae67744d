"""Runs of a generator on the CPU, with the operators replaced by plain torch: what a call does may not depend on the calls before it."""
import pytest
import torch

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout, init_flat
from cme213_final_project_b200.config import ModelConfig
from cme213_final_project_b200.generate import CacheFull, Generator, Sampling

PROMPTS = [[1, 2, 3, 4, 5], list(range(20)), [7], [(i * 7) % 33 for i in range(31)]]


def plain_layernorm(x, gamma, beta, eps):
    return (torch.nn.functional.layer_norm(x, x.shape[-1:], gamma, beta, eps),)


def plain_gemm(a, b, *, b_trans=False, bias=None, act=None, residual=None, allow_tf32=True):
    y = a @ (b.T if b_trans else b)
    y = y if bias is None else y + bias
    y = torch.nn.functional.gelu(y) if act else y
    return y if residual is None else y + residual


def places(n, offsets, lengths):
    """(row, sequence, position) of all new tokens."""
    offs = offsets.tolist()
    assert offs[0] == 0 and offs[-1] == n
    for b, length in enumerate(lengths.tolist()):
        for row in range(offs[b], offs[b + 1]):
            yield row, b, length - offs[b + 1] + row


def plain_append(k, v, cache_k, cache_v, pages, offsets, lengths):
    P = cache_k.shape[2]
    for row, b, pos in places(k.shape[0], offsets, lengths):
        at = pages[b, pos // P]
        assert at >= 0
        cache_k[at, :, pos % P], cache_v[at, :, pos % P] = k[row], v[row]


def plain_attention(q, cache_k, cache_v, pages, offsets, lengths):
    P, out = cache_k.shape[2], torch.empty_like(q)
    for row, b, pos in places(q.shape[0], offsets, lengths):
        at = torch.arange(pos + 1)
        page = pages[b].long()[at // P]
        k, v = cache_k[page, :, at % P], cache_v[page, :, at % P]          # [keys, heads, head_dim]
        p = torch.softmax(torch.einsum("hd,thd->ht", q[row], k) * q.shape[-1] ** -0.5, 1)
        out[row] = torch.einsum("ht,thd->hd", p, v)
    return out, None


def plain_next_token(logits, *, history, lengths, prompts, temperature, repetition, presence, frequency, noise=None, allowed=None,
                     bias_ids=None, bias_values=None):
    x = logits.clone()
    for r in range(x.shape[0]):
        told = history[r, :lengths[r]].tolist()
        assert all(0 <= t < x.shape[1] for t in told)
        for t in set(told):
            x[r, t] = x[r, t] / repetition[r] if x[r, t] > 0 else x[r, t] * repetition[r]
        for t in told[prompts[r]:]:
            x[r, t] -= frequency[r]
        for t in set(told[prompts[r]:]):
            x[r, t] -= presence[r]
        if temperature[r] > 0:
            x[r] /= temperature[r]
    token = (x if noise is None else x + noise).argmax(1)
    return token.to(torch.int32), torch.log_softmax(x, 1).gather(1, token[:, None])[:, 0], None


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    for name, f in (("add", torch.add), ("layernorm_fwd", plain_layernorm), ("gemm", plain_gemm), ("cache_append", plain_append),
                    ("paged_attention", plain_attention), ("next_token", plain_next_token)):
        monkeypatch.setattr(ops, name, f)


def generator(seqs=4, **kw):
    cfg = ModelConfig(mode="gpt", vocab_size=33, seq_len=48, hidden=64, heads=2, ff=64, layers=2, batch_size=1, activation="gelu",
                      causal=True, head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg)
    return Generator(cfg, layout, init_flat(layout, 3) * 6.0, seqs, page=8, **kw)


def run(g, prompts, new=8, **kw):
    return g.generate(prompts, new, cuda_graph=False, **kw)


def same(a, b):
    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prompts_are_taken_in_anew_each_time():
    g = generator()
    first = g.prefill(PROMPTS)
    assert torch.equal(g.prefill(PROMPTS), first) and g.cache.lengths == [len(p) for p in PROMPTS]
    assert torch.equal(g.prefill(PROMPTS[::-1], 7), generator().prefill(PROMPTS[::-1], 7))
    assert torch.equal(g.prefill(PROMPTS), first)


@pytest.mark.parametrize("sampling", [None, Sampling(0.0, 1.3, 0.2, 0.4), Sampling(1.0)])
def test_a_run_does_not_depend_on_the_runs_before_it(sampling):
    other = [[9], [8, 8], list(range(30)), [1]]
    want = [run(generator(), p, sampling=sampling) for p in (PROMPTS, other)]
    assert want[0][0].unique().numel() > 3                 # (a model that says one thing only would show nothing)
    g = generator()
    for p, w in ((PROMPTS, want[0]), (other, want[1]), (other, want[1]), (PROMPTS, want[0])):
        assert same(run(g, p, sampling=sampling), w)


def test_as_many_runs_as_one_likes():
    g = generator()
    for _ in range(6):                                     # (a cache that kept them would be full after the second)
        run(g, PROMPTS, 17)
    assert sorted([p for o in g.cache.owned for p in o] + g.cache.free) == list(range(g.cache.k.shape[1]))


def test_a_run_after_one_that_failed():
    g = generator(pages=9)
    with pytest.raises(CacheFull):
        run(g, PROMPTS, 16)
    assert same(run(g, PROMPTS, 2), run(generator(), PROMPTS, 2))


@pytest.mark.parametrize("chunk", [0, -1, -512])
def test_a_chunk_has_a_token_at_least(chunk):
    g = generator()
    first = run(g, PROMPTS, 2)
    for call in (lambda: g.prefill(PROMPTS, chunk), lambda: run(g, PROMPTS, 2, chunk=chunk)):
        with pytest.raises(ValueError, match="chunk"):
            call()
        assert g.cache.lengths == [len(p) + 1 for p in PROMPTS]            # refused before anything has changed
    assert same(run(g, PROMPTS, 2, chunk=1), run(generator(), PROMPTS, 2, chunk=1)) and first[0].shape == (4, 2)


@pytest.mark.parametrize("new", [0, -1, -40])
def test_a_run_has_a_token_at_least(new):
    g = generator()
    run(g, PROMPTS, 2)
    with pytest.raises(ValueError, match="max_new"):
        run(g, PROMPTS[::-1], new)
    assert g.cache.lengths == [len(p) + 1 for p in PROMPTS]                # refused before anything has changed


def test_what_has_no_room_is_refused_before_anything_changes():
    g = generator(pages=12)
    first = run(g, PROMPTS, 2)
    held = [list(o) for o in g.cache.owned]
    with pytest.raises(CacheFull):
        run(g, PROMPTS, 16)                                # room for the prompts, not for what follows
    with pytest.raises(CacheFull):
        g.prefill([list(range(30))] * 4, 7)                # for the first chunks only
    with pytest.raises(ValueError):
        g.prefill([[1], [2], [3], [4] * 49], 7)            # beyond the model's positions
    assert [list(o) for o in g.cache.owned] == held and g.cache.lengths == [len(p) + 1 for p in PROMPTS]
    assert same(run(g, PROMPTS, 2), first)
    logits = g.prefill([[k] * (8 * k) for k in (1, 2, 4, 5)])         # every page
    assert logits.shape == (4, 33) and not g.cache.free


@pytest.mark.parametrize("token", [-1, 33, 10 ** 6])
def test_prompts_have_tokens_of_the_vocabulary(token):
    g = generator()
    run(g, PROMPTS, 2)
    for call in (g.prefill, lambda p: run(g, p, 2)):
        with pytest.raises(ValueError, match="vocabulary"):
            call([[1], [2, 3, token], [4], [5]])
    assert g.cache.lengths == [len(p) + 1 for p in PROMPTS]                # refused before anything has changed


@pytest.mark.parametrize("token", [-1, 33, 63, 64, 10 ** 6])
def test_allowed_tokens_are_of_the_vocabulary(token):
    with pytest.raises(ValueError, match="vocabulary"):
        Sampling(allowed=[3, token]).tensors(2, 33, "cpu")


@pytest.mark.parametrize("allow,data", [("ab", False), ("abz", True), ("z", True), ("aé", True), ("", True)])
def test_the_command_takes_only_characters_that_can_come(allow, data, tmp_path, capsys):
    from cme213_final_project_b200.checkpoint import save_checkpoint
    from cme213_final_project_b200.generate import main
    text, ck = tmp_path / "text.txt", tmp_path / "model.ck"
    text.write_text("abc abc")
    cfg = ModelConfig(mode="gpt", vocab_size=4, seq_len=8, hidden=32, heads=1, ff=32, layers=1, batch_size=1, activation="gelu", causal=True,
                      head_layout="split", tied_embeddings=True, final_layernorm=True, init="normal")
    layout = ArenaLayout(cfg)
    flat = init_flat(layout, 1)
    save_checkpoint(str(ck), layout, flat, flat * 0, flat * 0, 0)
    args = ["--checkpoint", str(ck), "--allow", allow, "--prompt", "ab" if data else "0,1", "--max-new", "2"]
    assert main(args + (["--data", str(text)] if data else [])) == 1
    assert "--allow" in capsys.readouterr().err
