"""Tree attention with split key axes, so with the join of the chunks, inside
captured graphs and from several threads."""
import pytest
import torch

from rhizome_b200 import ops
from tests.test_gpu_attn import BF, F32, Paged, check_tree, cu_of
from tests.test_gpu_serving_threads import at_once

pytestmark = pytest.mark.gpu

# (type, width, query heads per K/V head, nodes): the form for few rows, row tiles, fp32 arithmetic
FORMS = [(BF, 128, 4, 1), (BF, 64, 2, 5), (BF, 128, 4, 24), (F32, 32, 4, 7), (BF, 128, 2, 200)]


def case(dtype, d, group, nodes, seed, longest=20000, n=5):
    r = torch.Generator().manual_seed(seed)
    cached = [longest] + torch.randint(0, longest, (n - 1,), generator=r).tolist()
    counts = [nodes] + torch.randint(0, nodes + 1, (n - 1,), generator=r).tolist()
    c = Paged([longest] * n, [nodes] * n, 2, d, 32, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(n * nodes, 2 * group, d, generator=g, device="cuda").to(dtype)
    lens = torch.tensor(cached, dtype=torch.int32, device="cuda")
    return c, q, lens, cu_of(counts)[1], counts


@pytest.mark.parametrize("dtype,d,group,nodes", FORMS)
def test_captured_joins_replay_with_new_lengths(dtype, d, group, nodes):
    """The captured call, its workspace its own, against the same call outside."""
    c, q, lens, cu, counts = case(dtype, d, group, nodes, 1)
    need = ops.attn_tree_workspace_bytes(q.shape[0], nodes, c.table.shape[1], 32, 2 * group, 2, d, dtype)
    assert need > 0
    ws = torch.empty(need, device="cuda", dtype=torch.uint8)
    out = torch.full_like(q, 7.0)

    def step():
        return ops.attn_tree_fwd(q, c.kc, c.vc, c.table, lens, cu, nodes, out=out, with_lse=True, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step()
        total = o.float().sum(0)  # a kernel behind the join, on its results
    r = torch.Generator().manual_seed(2)
    for turn in range(12):
        cached = torch.randint(0, 20001, (5,), generator=r)
        if turn % 3 == 0:
            cached[turn % 5] = 0
        fresh = torch.randint(0, nodes + 1, (5,), generator=r)
        lens.copy_(cached)
        cu.copy_(torch.cat([torch.zeros(1, dtype=torch.int64), fresh.cumsum(0)]))
        out.fill_(7.0)
        ws.fill_(turn * 37 % 256)  # nothing is kept from one replay to the next
        graph.replay()
        rows = int(fresh.sum())
        want, want_lse = ops.attn_tree_fwd(q, c.kc, c.vc, c.table, lens, cu, nodes, out=torch.full_like(q, 7.0), with_lse=True)
        assert torch.equal(o, want) and torch.equal(lse[:rows], want_lse[:rows])
        assert torch.equal(total, want.float().sum(0))
    assert not ops.device_status()


def test_two_graphs_with_one_workspace_in_turn():
    jobs = []
    ws = torch.empty(1 << 28, device="cuda", dtype=torch.uint8)
    for i, (dtype, d, group, nodes) in enumerate(FORMS[:3]):
        c, q, lens, cu, _ = case(dtype, d, group, nodes, 10 + i)
        call = lambda c=c, q=q, lens=lens, cu=cu, nodes=nodes: ops.attn_tree_fwd(  # noqa: E731
            q, c.kc, c.vc, c.table, lens, cu, nodes, out=torch.zeros_like(q), workspace=ws)
        want = call().clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = call()
        jobs.append((graph, o, want, call))  # (the call keeps the graph's inputs alive)
    for _ in range(20):
        for graph, o, want, _ in jobs:
            graph.replay()
        for graph, o, want, _ in jobs:
            assert torch.equal(o, want)
            o.zero_()


def test_threads_with_split_trees_and_prompts():
    """Each with a workspace and a stream of its own."""
    jobs = []
    for i, (dtype, d, group, nodes) in enumerate(FORMS):
        c, q, lens, cu, _ = case(dtype, d, group, nodes, 20 + i, longest=9000, n=3)
        need = ops.attn_tree_workspace_bytes(q.shape[0], nodes, c.table.shape[1], 32, 2 * group, 2, d, dtype)
        ws = torch.empty(need, device="cuda", dtype=torch.uint8)
        jobs.append(lambda c=c, q=q, lens=lens, cu=cu, nodes=nodes, ws=ws: ops.attn_tree_fwd(
            q, c.kc, c.vc, c.table, lens, cu, nodes, out=torch.zeros_like(q), workspace=ws))
    g = torch.Generator(device="cuda").manual_seed(1)
    for d in (64, 128):
        q, k, v = (torch.randn(1500, h, d, generator=g, device="cuda").to(BF) for h in (8, 2, 2))
        cu = cu_of([700, 1, 799])[1]
        jobs.append(lambda q=q, k=k, v=v, cu=cu: ops.attn_varlen_fwd(q, k, v, cu))
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    for got, w in zip(at_once(jobs, times=60), want):
        assert torch.equal(got, w)
    assert not ops.device_status()


def test_outputs_do_not_depend_on_what_the_workspace_held():
    for dtype, d, group, nodes in FORMS:
        c, q, lens, cu, counts = case(dtype, d, group, nodes, 3, longest=12000)
        need = ops.attn_tree_workspace_bytes(q.shape[0], nodes, c.table.shape[1], 32, 2 * group, 2, d, dtype)
        ws = torch.empty(need + 256, device="cuda", dtype=torch.uint8)
        seen = []
        for fill in (0, 255, 127):
            ws.fill_(fill)
            seen.append(ops.attn_tree_fwd(q, c.kc, c.vc, c.table, lens, cu, nodes, out=torch.zeros_like(q), workspace=ws[:need]))
            assert (ws[need:] == fill).all()
        assert torch.equal(seen[0], seen[1]) and torch.equal(seen[0], seen[2])


def test_a_tree_over_a_cache_of_one_chunk_and_one_more_key():
    """Lengths around the borders of chunks, for each form."""
    for dtype, d, group, nodes in FORMS[:4]:
        for key in (255, 256, 257, 511, 512, 513, 2559, 2560, 2561, 5120, 5121):
            check_tree([max(key - nodes, 0), key], [nodes, nodes], 2 * group, 2, d, dtype, page=64, seed=key)
