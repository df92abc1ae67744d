"""Bookkeeping of the paged cache, sampling's tensors and the command line, without a GPU."""
import pytest
import torch

from cme213_final_project_b200.config import preset
from cme213_final_project_b200.arena import ArenaLayout
from cme213_final_project_b200.generate import CacheFull, Generator, PagedCache, Sampling, build_parser, main


def cache(pages=10, seqs=3, max_len=64, page=8):
    return PagedCache(2, 2, 32, seqs, max_len, pages, page, torch.float32, "cpu")


def consistent(c):
    held = [p for o in c.owned for p in o] + c.free
    assert sorted(held) == list(range(c.k.shape[1]))
    for b, o in enumerate(c.owned):
        assert c.table[b, :len(o)].tolist() == o and bool((c.table[b, len(o):] == -1).all())
        assert len(o) == -(-c.lengths[b] // c.page)


def test_pages_are_taken_as_sequences_grow_and_given_back():
    c = cache()
    c.grow([1, 0, 17])
    consistent(c)
    assert c.lengths == [1, 0, 17] and len(c.free) == 10 - 1 - 3
    c.grow([7, 1, 7])
    consistent(c)
    assert len(c.free) == 10 - 1 - 1 - 3
    c.grow([1, 0, 0])
    consistent(c)
    c.release(2)
    consistent(c)
    assert c.lengths == [9, 1, 0] and len(c.free) == 7
    c.grow([0, 0, 56])
    consistent(c)
    assert not c.free


def test_nothing_changes_where_there_is_no_room():
    c = cache()
    c.grow([60, 0, 0])
    before = (list(c.lengths), [list(o) for o in c.owned], list(c.free), c.table.clone())
    with pytest.raises(CacheFull):
        c.grow([0, 8, 9])
    with pytest.raises(ValueError):
        c.grow([5, 0, 0])                                  # beyond max_len
    with pytest.raises(ValueError):
        c.grow([-1, 0, 0])
    assert (c.lengths, c.owned, c.free) == before[:3] and torch.equal(c.table, before[3])
    with pytest.raises(ValueError):
        cache(page=12)


def test_sampling_tensors():
    kw = Sampling(0.5, 1.2, 0.1, 0.2, {3: 1.5, 40: -2.0}, [0, 31, 32, 63, 64]).tensors(2, 65, "cpu")
    assert kw["bias_ids"].tolist() == [[3, 40]] * 2 and kw["bias_values"].tolist() == [[1.5, -2.0]] * 2
    words = [w % 2 ** 32 for w in kw["allowed"][0].tolist()]
    assert words == [1 | 1 << 31, 1 | 1 << 31, 1]
    assert kw["temperature"].tolist() == [0.5, 0.5] and kw["allowed"].dtype == torch.int32


def test_models_that_cannot_generate():
    cfg, _ = preset("parity-h128")
    layout = ArenaLayout(cfg)
    with pytest.raises(ValueError):
        Generator(cfg, layout, torch.zeros(layout.total), 1)
    cfg, _ = preset("tiny-gpt")
    cfg.hidden, cfg.heads = 96, 2
    layout = ArenaLayout(cfg)
    with pytest.raises(ValueError):
        Generator(cfg, layout, torch.zeros(layout.total), 1)


def test_rows_without_a_token_end():
    t, l = Generator._ended(torch.tensor([[1, -1, 2], [3, 4, 5]]), torch.zeros(2, 3))
    assert t.tolist() == [[1, -1, -1], [3, 4, 5]] and l[0, 1] == float("-inf") and l[1, 2] == 0


def test_command_line(tmp_path, capsys):
    a = build_parser().parse_args(["--checkpoint", "x", "--prompt", "a", "--prompt", "b", "--temperature", "0"])
    assert a.prompt == ["a", "b"] and a.temperature == 0.0 and a.page == 16
    assert main(["--checkpoint", str(tmp_path / "none")]) == 1
    assert "Error" in capsys.readouterr().err
