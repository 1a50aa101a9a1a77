"""Attention over batches of very many sequences, most of them empty or short:
the kernels' ways of finding their work."""
import random

import pytest
import torch

from rhizome_b200 import ops
from tests.test_gpu_attn import BF, F32, cu_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1 << 20, 1 << 22])
def test_prompts_between_millions_of_empty_ones(n):
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = {0: 300, 5: 1, n // 2: 700, n - 1: 64}
    counts = torch.zeros(n, dtype=torch.int64)
    for i, m in lens.items():
        counts[i] = m
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).cuda()
    total = int(counts.sum())
    q = torch.randn(total, 4, 128, generator=g, device="cuda").to(BF)
    k, v = (torch.randn(total, 2, 128, generator=g, device="cuda").to(BF) for _ in range(2))
    o = ops.attn_varlen_fwd(q, k, v, cu)
    assert not ops.device_status()
    assert torch.equal(o, ops.attn_varlen_fwd(q, k, v, cu_of(list(lens.values()))[1]))


def test_f32_prompts_between_a_million_empty_ones():
    g = torch.Generator(device="cuda").manual_seed(2)
    n = 1 << 20
    lens = {0: 33, 1: 100, 77: 1, n // 2: 300, n - 2: 64, n - 1: 5}
    counts = torch.zeros(n, dtype=torch.int64)
    for i, m in lens.items():
        counts[i] = m
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).cuda()
    total = int(counts.sum())
    q = torch.randn(total, 4, 32, generator=g, device="cuda")
    k, v = (torch.randn(total, 2, 32, generator=g, device="cuda") for _ in range(2))
    o, lse = ops.attn_varlen_fwd(q, k, v, cu, with_lse=True)
    want, want_lse = ops.attn_varlen_fwd(q, k, v, cu_of(list(lens.values()))[1], with_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("paged", [False, True])
def test_f32_batches_of_very_many_short_sequences(paged):
    """Each slice of the batch by itself gives the same bits; offsets need not
    start at row 0."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, page = 150000, 8
    counts = torch.randint(0, 4, (n,), generator=torch.Generator().manual_seed(3))
    counts[500] = 130
    at = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    total = int(at[-1])
    cu = at.to(torch.int32).cuda()
    q = torch.randn(total, 2, 32, generator=g, device="cuda")
    k, v = (torch.randn(total, 1, 32, generator=g, device="cuda") for _ in range(2))
    if paged:
        width = 5000 // page  # wide enough for several chunks
        cache = [torch.randn(700, 1, page, 32, generator=g, device="cuda") for _ in range(2)]
        table = torch.randint(0, 700, (n, width), generator=g, device="cuda", dtype=torch.int32)
        cached = torch.randint(0, 40, (n,), generator=g, device="cuda", dtype=torch.int32)
        cached[::5000] = 3000
        call = lambda a, b, rows, off: ops.attn_tree_fwd(q[rows], *cache, table[a:b], cached[a:b], off, 4)  # noqa: E731
    else:
        call = lambda a, b, rows, off: ops.attn_varlen_fwd(q[rows], k[rows], v[rows], off)  # noqa: E731
    o = call(0, n, slice(0, total), cu)
    for a, b in ((0, 3), (490, 510), (74990, 75010), (n - 20, n)):
        rows = slice(int(at[a]), int(at[b]))
        part = call(a, b, rows, (cu[a:b + 1] - cu[a]).contiguous())
        assert torch.equal(part, o[rows]), (a, b)
        # the same rows of the whole buffers, found from a row that is not the first
        if not paged:
            whole = ops.attn_varlen_fwd(q, k, v, cu[a:b + 1].contiguous())
            assert torch.equal(whole[rows], o[rows]), (a, b)


@pytest.mark.parametrize("d,nodes", [(128, 1), (64, 3)])
def test_few_rows_of_more_sequences_than_one_launch_holds(d, nodes):
    """The same form whatever the number of sequences: the same bits as calls
    with fewer of them, on both sides of the launches' borders."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n, page = 9000, 16
    width = 1600 // page
    counts = torch.randint(0, nodes + 1, (n,), generator=torch.Generator().manual_seed(4))
    at = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    total = int(at[-1])
    cu = at.to(torch.int32).cuda()
    q = torch.randn(total, 8, d, generator=g, device="cuda").to(BF)
    kc, vc = (torch.randn(500, 2, page, d, generator=g, device="cuda").to(BF) for _ in range(2))
    table = torch.randint(0, 500, (n, width), generator=g, device="cuda", dtype=torch.int32)
    cached = torch.randint(0, 1500, (n,), generator=g, device="cuda", dtype=torch.int32)
    parent = None if nodes == 1 else torch.randint(-1, 1, (total,), generator=g, device="cuda", dtype=torch.int32)
    o, lse = ops.attn_tree_fwd(q, kc, vc, table, cached, cu, nodes, parent=parent, with_lse=True)
    for a, b in ((0, 4), (4090, 4100), (4096, 4200), (8190, 8195), (n - 5, n)):
        rows = slice(int(at[a]), int(at[b]))
        part = ops.attn_tree_fwd(q[rows], kc, vc, table[a:b], cached[a:b], (cu[a:b + 1] - cu[a]).contiguous(), nodes,
                                 parent=None if parent is None else parent[rows], with_lse=True)
        assert torch.equal(part[0], o[rows]) and torch.equal(part[1], lse[rows]), (a, b)
