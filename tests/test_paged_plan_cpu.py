"""Which kernel a call of paged attention takes and how it divides the keys, through the native library without a GPU."""
import ctypes

import pytest

from cme213_final_project_b200 import ops

CLUSTER, STREAM, ROWS, TC = range(4)
F32, BF16 = 0, 1
INT, LONG, PTR = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p


class Paged(ctypes.Structure):
    _fields_ = ([(n, INT) for n in ("seqs", "heads", "kv_heads", "head_dim", "page", "width", "num_pages", "dtype", "rows", "max_len")]
                + [("scale", ctypes.c_float)]
                + [(n, LONG) for n in ("q_token", "q_head", "v_token", "v_head", "k_page_stride", "k_head_stride", "k_slot_stride",
                                       "v_page_stride", "v_head_stride", "v_slot_stride")]
                + [("q", PTR), ("nv", PTR), ("k", PTR), ("v", PTR), ("pages", PTR), ("pages_ld", LONG), ("offsets", PTR), ("lengths", PTR),
                   ("o", PTR), ("lse", PTR), ("ws", PTR), ("ws_bytes", LONG)])


def plan(seqs, rows, longest, heads=12, kv_heads=12, head_dim=64, dtype=BF16, page=16, backend=0, splits=0, sms=148, **changed):
    width = -(-longest // page)
    d = Paged(seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, width=width, num_pages=seqs * width, dtype=dtype,
              rows=rows, max_len=2 ** 31 - 1, scale=0.125, q_token=heads * head_dim, q_head=head_dim)
    for x in "kv":
        setattr(d, x + "_page_stride", kv_heads * page * head_dim)
        setattr(d, x + "_head_stride", page * head_dim)
        setattr(d, x + "_slot_stride", head_dim)
    for name, value in changed.items():
        setattr(d, name, value)
    lib = ops.host_lib()
    if lib is None:
        pytest.skip("native library not built")
    out = (INT * 5)()
    rc = lib.cme_paged_attention_plan(ctypes.byref(d), backend, splits, sms, out)
    return (rc, None) if rc else (0, dict(zip(("kernel", "row_tile", "tiles", "parts", "keys"), out)))


def made(*args, **kw):
    rc, p = plan(*args, **kw)
    assert rc == 0
    return p


def test_single_tokens_take_small_tiles():
    few = made(1, 1, 700)
    assert few["kernel"] == CLUSTER and few["row_tile"] == 16 and few["parts"] == 8
    many = made(64, 64, 1024, heads=16, kv_heads=16)
    assert many["kernel"] == STREAM and many["parts"] == 2 * 148
    assert made(16, 16, 32768, heads=32, kv_heads=8, head_dim=128, page=64)["kernel"] == STREAM
    assert made(32, 32, 2048, heads=4, kv_heads=4, head_dim=128, dtype=F32)["parts"] == 148           # one CTA an SM


def test_chunks_take_the_tensor_core_kernel():
    p = made(16, 4000, 1024)
    assert p["kernel"] == TC and p["row_tile"] == 128
    p = made(2, 3500, 8192, heads=32, kv_heads=8, head_dim=128, page=64)
    assert p["kernel"] == TC and p["row_tile"] == 256 and p["parts"] == 1
    assert made(16, 4000, 1024, heads=10, kv_heads=2)["row_tile"] == 125                                # whole tokens of 5 heads
    assert made(16, 4000, 1024, dtype=F32)["kernel"] == ROWS
    assert made(16, 40000, 1024, heads=129, kv_heads=1)["kernel"] in (STREAM, ROWS)                     # a token has too many rows


def test_long_keys_and_few_rows_are_divided():
    p = made(1, 128, 8192)
    assert p["kernel"] == TC and p["parts"] > 4


@pytest.mark.parametrize("seed", range(4))
def test_a_plan_covers_all_rows_and_keys(seed):
    import random
    r = random.Random(seed)
    for _ in range(300):
        kv, group, dtype, D = r.randint(1, 16), r.choice([1, 2, 5, 8, 200]), r.choice([F32, BF16]), r.choice([32, 64, 128])
        seqs, longest, backend, splits = r.randint(1, 200), r.randint(1, 100000), r.choice([0, 1, 2, 3]), r.choice([0, 1, 3, 8, -7, 1000])
        rows = r.randint(0, seqs * r.choice([1, 4, 600]))
        rc, p = plan(seqs, rows, longest, heads=kv * group, kv_heads=kv, head_dim=D, dtype=dtype, page=r.choice([8, 16, 48, 256]),
                     backend=backend, splits=splits)
        if backend == 3 and (dtype == F32 or group > 128):
            assert rc
            continue
        assert rc == 0 and p["parts"] >= 1 and p["row_tile"] >= 1
        # sequences of any share of the rows, each with a tile that is not full
        if p["kernel"] != STREAM:
            assert p["tiles"] * p["row_tile"] >= rows * group and (rows == 0 or p["tiles"] >= min(seqs, rows))
        if p["kernel"] in (ROWS, TC):
            assert p["parts"] * p["keys"] >= longest and p["keys"] % 64 == 0 and p["parts"] <= 128
        if p["kernel"] == CLUSTER:
            assert p["parts"] in (1, 2, 4, 8)


@pytest.mark.parametrize("changed", [dict(head_dim=48), dict(page=12), dict(page=4), dict(heads=13), dict(scale=0.0), dict(scale=float("inf")),
                                     dict(k_slot_stride=65), dict(q_token=12 * 64 + 4), dict(dtype=7), dict(k=8), dict(q=4),
                                     dict(max_len=-1)])
def test_what_the_kernels_do_not_take_is_refused(changed):
    assert plan(4, 4, 100, **changed)[0] != 0
