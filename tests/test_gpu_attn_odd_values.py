"""Values of V (and K) that are not finite, where some rows of a tile see them
and others must not: long prompts, split key axes, both row tiles of a unit."""
import math

import pytest
import torch

from rhizome_b200 import ops
from tests.test_gpu_attn import BF, F32, check_prompt, check_tree, cu_of

pytestmark = pytest.mark.gpu


def spoil_ends(q, k, v, at):
    for a, b in zip(at, at[1:]):
        if b - a > 1000:
            v[b - 3, 0, 1] = math.inf
            v[b - 70, -1, 2] = math.nan


@pytest.mark.parametrize("H,Hkv,d", [(1, 1, 128), (4, 1, 64), (8, 2, 128)])
def test_one_value_near_the_end_of_a_long_prompt(H, Hkv, d):
    check_prompt([200, 12000, 300], H, Hkv, d, BF, seed=H, spoil=spoil_ends)


def test_the_other_prompts_of_a_spoiled_batch_keep_their_bits():
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [500, 40000, 700, 1]
    at, cu = cu_of(lens)
    q = torch.randn(at[-1], 4, 128, generator=g, device="cuda").to(BF)
    k = torch.randn(at[-1], 1, 128, generator=g, device="cuda").to(BF)
    v = torch.randn(at[-1], 1, 128, generator=g, device="cuda").to(BF)
    clean = ops.attn_varlen_fwd(q, k, v, cu)
    v[at[2] - 5, 0, 7] = math.inf
    o, lse = ops.attn_varlen_fwd(q, k, v, cu, with_lse=True)
    assert not ops.device_status()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        last = b - 5 if i == 1 else b
        assert torch.equal(o[a:last], clean[a:last]), f"rows of prompt {i}"
    seen = torch.zeros(5, 4, 128, dtype=torch.bool, device="cuda")
    seen[:, :, 7] = True
    assert torch.equal(o[at[2] - 5:at[2]] == math.inf, seen)
    assert torch.equal(o[at[2] - 5:at[2]][~seen], clean[at[2] - 5:at[2]][~seen])
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 2), (64, 1)])
@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128), (BF, 64)])
def test_values_all_along_a_prompt(dtype, d, H, Hkv):
    """Every fifth key has one value that is not finite, in a channel of its
    own for d keys; every third of those also a K that is not."""
    def spoil(q, k, v, at):
        for a, b in zip(at, at[1:]):
            for n, j in enumerate(range(a + 2, b, 5)):
                v[j, :, n % d] = (math.inf, -math.inf, math.nan)[n // d % 3]
                if n % 3 == 0:
                    k[j, :, 3] = math.inf if n % 2 else -math.inf
    check_prompt([300, 1, 60, 520], H, Hkv, d, dtype, seed=H, spoil=spoil)


def test_values_in_keys_that_only_the_second_row_tile_sees_whole():
    """One head to a K/V head: row tiles of 128 tokens; the key is below every
    row of the second tile and between rows of the first."""
    for key in (0, 1, 63, 64, 100, 127, 128, 129, 200, 255):
        def spoil(q, k, v, at):
            v[key, 0, 9] = math.inf
        check_prompt([256, 10], 1, 1, 128, BF, seed=key, spoil=spoil)


def spoil_nodes(c, q):
    for i in range(len(c.k)):
        L = c.k[i].shape[0]
        c.v[i][L - 2, :, 1] = math.nan
        c.v[i][L - 3, 0, 2] = math.inf
        c.v[i][L - 4, :, 2] = -math.inf
        c.v[i][L - 5, -1, :] = math.inf
        c.v[i][L - 10, 0, 4] = math.nan
        c.k[i][L - 3, :, 0] = math.nan
        if i % 2:
            c.v[i][L - 1, :, 5] = math.inf
            c.k[i][L - 1, :, 1] = math.inf


# Few rows: chunks of 512 keys; the last boundary of 3575 + 16 lies between the nodes.
@pytest.mark.parametrize("d,group,cached,counts", [(128, 4, [3000, 9000, 510], [4, 4, 4]), (64, 1, [3575, 1020], [16, 9]),
                                                   (128, 16, [700, 5000], [1, 1])])
@pytest.mark.parametrize("chain", [False, True])
def test_split_keys_with_few_rows(d, group, cached, counts, chain):
    check_tree(cached, counts, 2 * group, 2, d, BF, seed=group, chain=chain, most=max(counts),
               change=spoil_nodes if counts[0] > 4 else spoil_last)


def spoil_last(c, q):
    for i in range(len(c.k)):
        L, own = c.k[i].shape[0], 4
        c.v[i][L - 1, :, 5] = math.inf
        if L > 3000:
            c.v[i][max(L - own, 0), 0, 2] = math.nan


# Row tiles: chunks of 2560 keys; the last boundary of 51190 + 24 lies between the nodes.
@pytest.mark.parametrize("d,group,cached,counts,chain", [
    (128, 4, [6000, 20000, 50], [20, 64, 33], False), (64, 8, [51190], [24], False), (128, 4, [51190], [24], True),
    (128, 1, [7000, 100], [300, 200], True), (64, 24, [9000], [20], False)])
def test_split_keys_in_row_tiles(d, group, cached, counts, chain):
    check_tree(cached, counts, 2 * group, 2, d, BF, page=64, seed=group, chain=chain, change=spoil_nodes)


@pytest.mark.parametrize("dtype,d", [(F32, 32), (F32, 200), (BF, 128), (BF, 64)])
def test_rows_whose_scores_are_all_minus_infinity(dtype, d):
    """0 / 0 by the formula: they are rows that see nothing (o = 0, lse = -inf),
    whatever V holds there; the rows after them see finite scores too."""
    def spoil(q, k, v, at):
        q[:, :, 0] = q[:, :, 0].abs() + 0.5
        for a, b in zip(at, at[1:]):
            k[a:a + 3, :, 0] = -math.inf
            v[a:a + 2, :, 1] = math.inf
            v[a + 1:a + 3, :, 2] = math.nan
    check_prompt([200, 3, 70], 4, 2, d, dtype, seed=1, spoil=spoil)

    def change(c, q):
        q[:, :, 0] = q[:, :, 0].abs() + 0.5
        for k, v in zip(c.k, c.v):
            k[:-2, :, 0] = -math.inf
            v[5, :, 3] = math.inf
            v[-3, :, 1] = math.nan
    for nodes in (1, 3, 20):
        check_tree([700, 6000, 10], [nodes] * 3, 4, 2, d, dtype, page=64, seed=nodes, change=change)
        check_tree([700, 6000, 10], [nodes] * 3, 4, 2, d, dtype, page=64, seed=nodes, change=change, chain=True)
