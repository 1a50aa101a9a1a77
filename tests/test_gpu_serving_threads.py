"""Calls of the serving operators from several host threads at once, with sizes
that ask for different amounts of shared memory, each on its own stream."""
import threading

import pytest
import torch

from rhizome_b200 import ops

pytestmark = pytest.mark.gpu


def at_once(jobs, times=200):
    """Runs every job `times` times in a thread and stream of its own; their
    last results, or the first error."""
    results, errors = [None] * len(jobs), []
    go = threading.Barrier(len(jobs))
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()

    def run(i):
        try:
            with torch.cuda.stream(streams[i]):
                go.wait()
                for _ in range(times):
                    results[i] = jobs[i]()
        except Exception as e:  # to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]
    return results


def test_trees_of_different_bounds():
    def job(nodes, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k, v = (torch.randn(nodes, 2, 128, generator=g, device="cuda") for _ in range(3))
        k = k / k.norm(dim=-1, keepdim=True)
        a, b = (torch.rand(nodes, 2, generator=g, device="cuda") for _ in range(2))
        cu = torch.tensor([0, nodes], dtype=torch.int32, device="cuda")
        par = torch.arange(-1, nodes - 1, dtype=torch.int32, device="cuda")
        return lambda: ops.gdr_tree_step(q, k, v, a, b, cu, par, nodes)[0]

    jobs = [job(64, 1), job(1, 2), job(17, 3)]
    want = [j() for j in jobs]
    for got, w in zip(at_once(jobs), want):
        assert torch.equal(got, w)


def test_attention_of_different_widths():
    def job(d, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(90, 4, d, generator=g, device="cuda")
        k, v = (torch.randn(90, 2, d, generator=g, device="cuda") for _ in range(2))
        cu = torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
        return lambda: ops.attn_varlen_fwd(q, k, v, cu)

    jobs = [job(256, 1), job(132, 2), job(200, 3)]
    want = [j() for j in jobs]
    for got, w in zip(at_once(jobs), want):
        assert torch.equal(got, w)
