"""The delta rule over trees of drafted tokens: against the f64 oracle applied
along every node's path, against gdr_multistep on chains, and what takes no
part."""
import random

import numpy as np
import pytest
import torch

from oracle import oracle as O
from rhizome_b200 import ops
from tests.gpu_util import device_inputs, host, make_inputs, to_dev
from tests.tolerance import assert_bf16, assert_fp32

pytestmark = pytest.mark.gpu


def random_tree(r, m):
    return [-1 if t == 0 else r.randint(-1, t - 1) for t in range(m)]


def oracle_tree(parents, q, k, v, a, b, root):
    """(o [m, H, d], states [m, H, d, d]) by gated_delta_step from each node's
    parent state; zeros for nodes that take no part (states: None there)."""
    m, H, d = q.shape
    o, states = np.zeros((m, H, d)), [None] * m
    for t, p in enumerate(parents):
        if p < -1 or p >= t or (p >= 0 and states[p] is None):
            continue
        before = root if p < 0 else states[p]
        ro, rs = O.gdr_varlen(np.array([0, 1]), q[t:t + 1], k[t:t + 1], v[t:t + 1], a[t:t + 1],
                              b[t:t + 1], state_in=before[None])
        o[t], states[t] = ro[0], rs[0]
    return o, states


def run_case(dtype, d, H, counts, seed, pool=True, parents=None, most=64):
    r = random.Random(seed)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tokens, n = int(cu[-1]), len(counts)
    q, k, v, a, b = make_inputs(seed, tokens, H, d, dtype)
    parents = [random_tree(r, m) for m in counts] if parents is None else parents
    slots = np.array(r.sample(range(n + 3), n), dtype=np.int32)
    start = O.make_normal(seed, 22, (n + 3, H, d, d), 0.02).astype(np.float32).astype(np.float64)
    dpool = to_dev(start, torch.float32) if pool else None
    states = torch.full((tokens, H, d, d), 7.0, device="cuda")
    args = device_inputs(q, k, v, a, b, dtype)
    par = torch.tensor([p for seq in parents for p in seq], dtype=torch.int32, device="cuda")
    o, st = ops.gdr_tree_step(*args, to_dev(cu, torch.int32), par, most, state_pool=dpool,
                              slot_idx=to_dev(slots, torch.int32) if pool else None, states=states)
    assert st is states
    check = assert_fp32 if dtype == "f32" else assert_bf16
    for i, m in enumerate(counts):
        x = slice(int(cu[i]), int(cu[i]) + m)
        root = start[slots[i]] if pool else np.zeros((H, d, d))
        kept = [p if t < most else -2 for t, p in enumerate(parents[i])]
        ro, rs = oracle_tree(kept, q[x], k[x], v[x], a[x], b[x], root)
        if m == 0:
            continue
        check(host(o[x]), ro, f"o of tree {i}")
        for t in range(m):
            if rs[t] is None:
                assert (states[x][t] == 7.0).all(), "a node that takes no part keeps its states"
                assert (o[x][t] == 0).all()
            else:
                check(host(states[x][t]), rs[t], f"state of node {t} of tree {i}")
    if pool:
        assert np.array_equal(host(dpool), start), "the pool is not modified"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [4, 6, 32, 128, 200])
def test_trees_match_oracle(dtype, d):
    run_case(dtype, d, 2, [5, 1, 0, 13], 40 + d)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_trees_of_64_and_zero_start(dtype):
    run_case(dtype, 32, 1, [64, 3], 7, pool=False)


def test_nodes_that_take_no_part():
    trees = [[-1, 0, -2, 2, 1, 5, 7, 3], [0, -1, 1, -5]]  # padding, its children, itself, later nodes
    run_case("f32", 32, 2, [8, 4], 8, parents=trees)
    run_case("f32", 32, 2, [8, 4], 8, parents=trees, most=3)
    run_case("f32", 32, 2, [70], 9, parents=[[-1] + list(range(69))])
    run_case("f32", 32, 2, [4], 9, most=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chain_equals_multistep(dtype):
    """Without a parent array the nodes are a chain: gdr_multistep's result,
    up to the order of the row sums."""
    n, T, H, d = 3, 8, 4, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k, v = (torch.nn.functional.normalize(rnd(n, T, H, d), dim=-1).to(dtype) for _ in range(3))
    a, b = torch.sigmoid(rnd(n, T, H)), torch.sigmoid(rnd(n, T, H))
    pool = rnd(n, H, d, d)
    outs, states = ops.gdr_multistep(q, k, v, a, b, max_positions=T, state_pool=pool)
    cu = torch.arange(0, n * T + 1, T, device="cuda", dtype=torch.int32)
    flat = [x.reshape(n * T, *x.shape[2:]) for x in (q, k, v, a, b)]
    o, st = ops.gdr_tree_step(*flat, cu, None, T, state_pool=pool)
    assert_fp32(host(st), host(states.reshape(st.shape)), "states")
    (assert_fp32 if dtype == torch.float32 else assert_bf16)(host(o), host(outs.reshape(o.shape)), "o")


def test_rows_behind_the_last_sequence_and_bad_slots():
    H, d = 2, 32
    q = torch.randn(9, H, d, device="cuda")
    a = torch.full((9, H), 0.5, device="cuda")
    cu = torch.tensor([0, 3, 6], device="cuda", dtype=torch.int32)
    out, states = torch.full_like(q, 7.0), torch.full((9, H, d, d), 7.0, device="cuda")
    slots = torch.tensor([5, 0], device="cuda", dtype=torch.int32)
    pool = torch.ones(2, H, d, d, device="cuda")
    ops.gdr_tree_step(q, q, q, a, a, cu, None, 8, state_pool=pool, slot_idx=slots, out=out, states=states)
    assert torch.isnan(out[:3]).all() and torch.isfinite(out[3:6]).all()
    assert (out[6:] == 7).all() and (states[6:] == 7).all()
