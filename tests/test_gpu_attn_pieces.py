"""Further pieces of prompts over long caches: several chunks of keys and
several blocks of rows at once, beside sequences of one row."""
import pytest
import torch

from rhizome_b200 import ops
from tests.test_gpu_attn import BF, F32, Paged, check_tree, cu_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d,H,Hkv", [(BF, 128, 8, 2), (BF, 64, 3, 1), (F32, 32, 4, 2), (BF, 96, 4, 1)])
def test_pieces_over_long_caches(dtype, d, H, Hkv):
    check_tree([20000, 7000, 12300, 0], [700, 1, 65, 300], H, Hkv, d, dtype, page=64, seed=H, chain=True)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F32, 64)])
@pytest.mark.parametrize("bound", [100, 1000, 5000])
def test_pieces_do_not_depend_on_the_batch(dtype, d, bound):
    """With the caller's own bound: alone, and in a table that is wider."""
    cached, counts = [9000, 0, 15000, 400], [90, 33, 1, 100]
    c = Paged(cached, counts, 2, d, 16, dtype, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    at, cu = cu_of(counts)
    q = torch.randn(at[-1], 8, d, generator=g, device="cuda").to(dtype)
    lens = torch.tensor(cached, dtype=torch.int32, device="cuda")
    wide = torch.full((4, 8192), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    o, lse = ops.attn_tree_fwd(q, c.kc, c.vc, wide, lens, cu, bound, with_lse=True)
    for i, (a, b) in enumerate(zip(at, at[1:])):
        alone = ops.attn_tree_fwd(q[a:b], c.kc, c.vc, c.table[i:i + 1], lens[i:i + 1], cu_of([b - a])[1], bound, with_lse=True)
        assert torch.equal(alone[0], o[a:b]) and torch.equal(alone[1], lse[a:b])


def test_scratch_of_a_piece_over_a_wide_table():
    """8,192 rows of 32 heads and a table for 131,072 positions: what the call
    allocates besides its output."""
    H, Hkv, d, page, rows = 32, 8, 128, 16, 8192
    q = torch.zeros(rows, H, d, device="cuda", dtype=BF)
    kc = torch.zeros(4, Hkv, page, d, device="cuda", dtype=BF)
    table = torch.zeros(1, 131072 // page, device="cuda", dtype=torch.int32)
    cached = torch.zeros(1, device="cuda", dtype=torch.int32)
    cu = cu_of([rows])[1]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    o = ops.attn_tree_fwd(q, kc, kc, table, cached, cu, rows)
    assert torch.cuda.max_memory_allocated() - before < 10 * o.numel() * o.element_size()
