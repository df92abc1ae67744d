"""Offsets that are not in order: what the call returns is not defined, but it ends, and nothing outside of its buffers is touched."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from cme213_final_project_b200 import ops


@pytest.mark.parametrize("seqs,rows,key_tiles,heads", [(65536, 8192, 3000, 2), (65536, 8192, 7000, 1)])
def test_more_shared_rows_than_31_bits_of_key_tiles(seqs, rows, key_tiles, heads):
    """Every second sequence has all rows.  (Counted in 32 bits, the tiles of the stream's CTAs came out negative.)"""
    D, page = 64, 128
    q = torch.randn(rows, heads, D, device="cuda").to(torch.bfloat16)
    ck, cv = (torch.randn(4, heads, page, D, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.zeros(1, key_tiles, dtype=torch.int32, device="cuda").expand(seqs, key_tiles)
    offsets = (torch.arange(seqs + 1, device="cuda") % 2 * rows).to(torch.int32)
    lengths = torch.full((seqs,), key_tiles * page, dtype=torch.int32, device="cuda")
    ops.paged_attention(q, ck, cv, table, offsets, lengths, backend="single", splits=-1000)
    torch.cuda.synchronize()
    assert ops.attention_check_status() == 0
    # and in order again: one token over two pages
    one = torch.arange(2, dtype=torch.int32, device="cuda")
    two = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    args = (q[:1], ck, cv, two, one, torch.tensor([200], dtype=torch.int32, device="cuda"))
    a, b = ops.paged_attention(*args, backend="single", splits=-4), ops.paged_attention(*args, backend="single", splits=1)
    assert bool(((a[0].float() - b[0].float()).abs() <= 2 ** -7 * b[0].float().abs() + 1e-3).all()) and bool(((a[1] - b[1]).abs() < 1e-4).all())
