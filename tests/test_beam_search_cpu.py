"""Books of a cache whose sequences are beams, and what is refused, without a GPU."""
import ctypes

import pytest
import torch

from cme213_final_project_b200 import ops
from cme213_final_project_b200.arena import ArenaLayout
from cme213_final_project_b200.config import preset
from cme213_final_project_b200.generate import CacheFull, Generator, PagedCache, build_parser

INT, LONG, PTR = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p


def cache(pages=40, seqs=6, max_len=64, page=8, **kw):
    return PagedCache(2, 2, 32, seqs, max_len, pages, page, device="cpu", **kw)


@pytest.mark.parametrize("prompt,new", [((1, 20), 0), ((8, 16), 9), ((13, 64), 0), ((3, 30), 34)])
def test_a_fork_gives_each_beam_its_pages(prompt, new):
    c = cache()
    c.grow([prompt[0], 0, 0, prompt[1], 0, 0])
    need = c.forked(prompt, 3, new)
    spare = c.fork(3, new).tolist()
    held = [p for o in c.owned for p in o]
    assert sorted(held + c.free) == list(range(40)) and len(held) == need
    written = []                                           # pages that a beam writes: behind the full ones of the prompt
    for b in range(6):
        n = prompt[b // 3]
        row = c.table[b].tolist()
        written += row[n // 8:-(-(n + new) // 8)] + [spare[b]]
        assert all(p == -1 for p in row[-(-(n + new) // 8):])
        assert all(p >= 0 for p in row[:n // 8]) if b % 3 == 0 else all(p == -1 for p in row[:n // 8])
    assert len(set(written)) == len(written) and min(written) >= 0
    with pytest.raises(ValueError):
        c.grow([0] * 6)
    with pytest.raises(ValueError):
        c.release(0)
    c.clear()
    assert len(c.free) == 40 and bool((c.table == -1).all())
    c.grow([1] * 6)


def test_no_room_for_a_fork():
    c = cache(pages=12)
    c.grow([9, 0, 0, 9, 0, 0])
    free = list(c.free)
    with pytest.raises(CacheFull):
        c.fork(3, 8)
    with pytest.raises(ValueError):
        c.fork(3, 60)
    assert c.free == free and not c.shared


def test_forks_that_are_refused():
    c = cache()
    c.grow([9, 0, 2, 9, 0, 0])
    free, owned = list(c.free), [list(o) for o in c.owned]
    for beams in (0, 3, 4, 6):                             # none; sequence 2 or 3 holds something; not a divisor of 6
        with pytest.raises(ValueError):
            c.fork(beams, 8)
    with pytest.raises(ValueError):
        c.fork(1, -1)
    assert c.free == free and c.owned == owned and not c.shared
    c.fork(1, 8)
    with pytest.raises(ValueError):                        # beams already
        c.fork(1, 8)
    c.clear()
    c.grow([9, 0, 0, 9, 0, 0])
    c.fork(3, 8)
    assert c.shared


def test_scales_of_a_cache():
    assert cache().k_scales is None and cache().scales(0) == {} and cache().scales() == {}
    c = cache(dtype=torch.int8)
    assert c.k.dtype == torch.int8 and c.k_scales.shape == (2, 40, 2, 1) and c.scales(1)["v_scales"].shape == (40, 2, 1)
    assert cache(dtype=torch.int8, page=48).k_scales.shape[-1] == 3 and cache(dtype=torch.int8, page=48, block=24).k_scales.shape[-1] == 2
    for block in (0, 4, 12, 32, 96):
        with pytest.raises(ValueError):
            cache(dtype=torch.int8, page=48, block=block)


def test_refusals_of_a_search():
    cfg = preset("tiny-gpt")[0]
    layout = ArenaLayout(cfg, align=64)
    params = torch.zeros(layout.total)
    for seqs, beams in ((4, 0), (4, 3), (66, 33), (4, -1)):
        with pytest.raises(ValueError):
            Generator(cfg, layout, params, seqs, beams=beams)
    gen = Generator(cfg, layout, params, 4, beams=2)
    for kw in (dict(prompts=[[1]]), dict(prompts=[[1], []]), dict(prompts=[[1], [cfg.vocab_size]]), dict(max_new=0), dict(end=cfg.vocab_size), dict(end=-1),
               dict(allowed=[cfg.vocab_size]), dict(chunk=0), dict(max_new=cfg.seq_len + 1), dict(prompts=[[1], [2], [3], [4]])):
        with pytest.raises(ValueError):
            gen.beam_search(**{**dict(prompts=[[1], [2]], max_new=4), **kw})
    assert not gen.cache.shared and gen.cache.lengths == [0] * 4


def test_flags():
    a = build_parser().parse_args(["--checkpoint", "x"])
    assert a.beams == 0 and a.cache_dtype == "model" and a.temperature is None
    a = build_parser().parse_args(["--checkpoint", "x", "--beams", "4", "--end", ".", "--length-power", "0.7", "--cache-dtype", "int8"])
    assert (a.beams, a.end, a.length_power, a.cache_dtype) == (4, ".", 0.7, "int8")


# ----------------------------------------------------------------------------------------------------------------------
# What the library refuses before anything is launched
# ----------------------------------------------------------------------------------------------------------------------
class Paged(ctypes.Structure):
    _fields_ = ([(n, INT) for n in ("seqs", "heads", "kv_heads", "head_dim", "page", "width", "num_pages", "dtype", "rows", "max_len")]
                + [("scale", ctypes.c_float)]
                + [(n, LONG) for n in ("q_token", "q_head", "v_token", "v_head", "k_page_stride", "k_head_stride", "k_slot_stride",
                                       "v_page_stride", "v_head_stride", "v_slot_stride")]
                + [("q", PTR), ("nv", PTR), ("k", PTR), ("v", PTR), ("pages", PTR), ("pages_ld", LONG), ("offsets", PTR), ("lengths", PTR),
                   ("o", PTR), ("lse", PTR), ("ws", PTR), ("ws_bytes", LONG)])


class Scales(ctypes.Structure):
    _fields_ = [("k", PTR), ("v", PTR), ("block", INT), ("k_page", LONG), ("k_head", LONG), ("v_page", LONG), ("v_head", LONG)]


class Beams(ctypes.Structure):
    _fields_ = ([(n, INT) for n in ("groups", "beams", "width", "vocab", "dtype")] + [("logits", PTR), ("logits_ld", LONG), ("scores", PTR), ("finished", PTR),
                 ("allowed", PTR), ("allowed_ld", LONG), ("parents", PTR), ("tokens", PTR), ("out", PTR), ("ws", PTR), ("ws_bytes", LONG)])


class Pages(ctypes.Structure):
    _fields_ = [("base", PTR), ("heads", INT), ("row_bytes", INT), ("per", INT), ("layer", LONG), ("page", LONG), ("head", LONG), ("row", LONG)]


class Reorder(ctypes.Structure):
    _fields_ = ([(n, INT) for n in ("groups", "beams", "width", "slots", "layers", "num_pages", "tensors")] + [("t", Pages * 4), ("pages", PTR),
                 ("pages_ld", LONG), ("spare", PTR), ("parents", PTR), ("lengths", PTR), ("new_pages", PTR), ("new_spare", PTR)])


def library():
    lib = ops.host_lib()
    if lib is None:
        pytest.skip("native library not built")
    return lib


def paged(**changed):
    d = Paged(seqs=4, heads=12, kv_heads=12, head_dim=64, page=16, width=8, num_pages=32, dtype=1, rows=4, max_len=2 ** 31 - 1, scale=0.125,
              q_token=768, q_head=64, v_token=768, v_head=64)
    for x in "kv":
        setattr(d, x + "_page_stride", 12 * 16 * 64)
        setattr(d, x + "_head_stride", 16 * 64)
        setattr(d, x + "_slot_stride", 64)
    for name, value in changed.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("block,changed", [(0, {}), (4, {}), (12, {}), (32, {}), (-8, {}), (8, dict(head_dim=48)), (8, dict(page=12)), (8, dict(dtype=2)),
                                           (8, dict(k_slot_stride=72)), (8, dict(k=8)), (8, dict(q_token=4)), (8, dict(kv_heads=0)), (8, dict(scale=0.0)),
                                           (8, dict(heads=13)), (8, dict(v_page_stride=100))])
def test_refused_caches(block, changed):
    lib = library()
    s, d, out = Scales(block=block, k_page=12, v_page=12), paged(**changed), (INT * 5)()
    assert lib.cme_paged_attention8_plan(ctypes.byref(d), ctypes.byref(s), 0, 0, 148, out) != 0
    if "scale" not in changed and "heads" not in changed:
        assert lib.cme_paged_append8(ctypes.byref(d), ctypes.byref(s), None) != 0


def test_plans_of_8_bit_caches():
    lib = library()

    def plan(block=16, backend=0, splits=0, **changed):
        s, out = Scales(block=block), (INT * 5)()
        rc = lib.cme_paged_attention8_plan(ctypes.byref(paged(**changed)), ctypes.byref(s), backend, splits, 148, out)
        return None if rc else dict(zip(("kernel", "row_tile", "tiles", "parts", "keys"), out))

    one = plan(seqs=1, rows=1, width=44)
    assert one["kernel"] == 0 and one["parts"] in (2, 4, 8)                      # a cluster
    many = plan(seqs=64, rows=64, width=64, heads=16, kv_heads=16)
    assert many["kernel"] == 1                                                   # a stream
    assert plan(seqs=32, rows=16000, width=64, dtype=0, heads=4, kv_heads=4)["kernel"] == 2
    assert plan(backend=3, dtype=0) is None


@pytest.mark.parametrize("changed", [dict(beams=0), dict(beams=33), dict(width=0), dict(width=33), dict(vocab=0), dict(dtype=2), dict(groups=-1),
                                     dict(groups=1 << 20, beams=32)])
def test_refused_beams(changed):
    d = Beams(**{**dict(groups=2, beams=4, width=4, vocab=100, dtype=1), **changed})
    assert library().cme_beam_step_ws_bytes(ctypes.byref(d), ctypes.byref(LONG())) != 0
    assert library().cme_beam_step(ctypes.byref(d), None) != 0


def test_a_vocabulary_near_the_largest_integer_is_refused():
    for vocab, fine in ((1 << 30, True), ((1 << 30) + 1, False), (2 ** 31 - 1, False)):
        d = Beams(groups=1, beams=1, width=1, vocab=vocab, dtype=1, ws_bytes=0)
        library().cme_beam_step_ws_bytes(ctypes.byref(d), ctypes.byref(LONG()))
        library().cme_last_error.restype = ctypes.c_char_p
        assert (b"too many tokens" not in library().cme_last_error()) == fine


@pytest.mark.parametrize("changed", [dict(beams=0), dict(groups=-1), dict(slots=0), dict(tensors=5), dict(layers=-1), dict(heads=0), dict(row_bytes=0),
                                     dict(row_bytes=18), dict(page=24), dict(base=8), dict(per=0)])
def test_refused_reorders(changed):
    t = dict(base=256, heads=2, row_bytes=64, per=1, layer=4096, page=2048, head=1024, row=64)
    top = dict(groups=2, beams=4, width=4, slots=16, layers=2, num_pages=9, tensors=1)
    top.update({k: v for k, v in changed.items() if k in top})
    d = Reorder(**top)
    d.t[0] = Pages(**{**t, **{k: v for k, v in changed.items() if k in t}})
    assert library().cme_cache_reorder(ctypes.byref(d), None) != 0
