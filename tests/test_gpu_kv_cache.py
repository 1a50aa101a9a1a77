"""The paged cache of the Global blocks on the GPU: block tables and slot maps
against a request-by-request form, bit for bit, and the append."""
import random

import pytest
import torch

from rhizome_b200 import capi, ops
from tests.attn_ref import step_tables

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_tables(cached, fresh, held, width, free, page, max_tokens, cursor=None, seed=0):
    r = random.Random(seed)
    n = len(cached)
    table = [[r.randrange(1 << 20) for _ in range(width)] for _ in range(n)]
    dev = torch.tensor(table, dtype=torch.int32, device="cuda").reshape(n, width)
    got = ops.kv_step_tables(i32(cached), i32(fresh), dev, i32(held), i32(free), page, max_tokens,
                             cursor=None if cursor is None else i32([cursor]))
    cu, slots, want, now, at, missing = step_tables(cached, fresh, table, held, free, page, max_tokens,
                                                    cursor or 0)
    assert got[0].tolist() == cu
    assert got[1].tolist() == slots
    assert dev.tolist() == want
    assert got[2].tolist() == now
    assert got[3].tolist() == [at] and got[4].tolist() == [missing]


@pytest.mark.parametrize("page", [8, 16, 1024])
@pytest.mark.parametrize("n", [1, 31, 513, 1500])
def test_tables_match_request_by_request(n, page):
    r = random.Random(n * page)
    cached = [r.choice([0, 1, page - 1, page, page + 1, r.randrange(3 * page)]) for _ in range(n)]
    fresh = [r.choice([0, 1, 1, page, r.randrange(2 * page)]) for _ in range(n)]
    width = 5
    # some requests own pages ahead of their positions (a rejected draft's)
    held = [min(width, -(-c // page) + r.choice([0, 0, 1])) for c in cached]
    free = [5000 + 3 * j for j in range(3 * n + 4)]
    check_tables(cached, fresh, held, width, free, page, sum(fresh) + 7, cursor=2)


def test_tables_when_pages_run_out():
    page, width = 8, 4
    cached, fresh, held = [3, 8, 20, 0, 31], [6, 1, 30, 9, 1], [1, 1, 3, 0, 4]
    for num_free in range(0, 8):  # the list ends inside and between requests
        check_tables(cached, fresh, held, width, list(range(100, 100 + num_free)), page, 60)
    check_tables(cached, fresh, held, width, list(range(100, 106)), page, 60, cursor=9)  # past the list
    check_tables(cached, fresh, held, width, list(range(100, 106)), page, 60, cursor=-3)
    check_tables(cached, fresh, held, width, list(range(100, 106)), page, 10)  # rows past the map


def test_tables_odd_requests():
    check_tables([], [], [], 3, [1, 2], 16, 5)
    check_tables([-5, 4], [3, -2], [0, 9], 2, [1, 2, 3], 8, 4)  # negative lengths are 0, held is at most the width
    check_tables([5, 4], [3, 2], [0, 0], 0, [1, 2, 3], 8, 5)    # a table of no columns
    check_tables([0, 70], [70, 0], [0, 0], 9, list(range(40)), 8, 70)  # fresh = 0 takes nothing
    check_tables([2 ** 31 - 10], [100], [1], 2, [7], 1024, 100)  # positions past 31 bits


def test_tables_many_rows_over_many_ctas():
    r = random.Random(5)
    n, page = 64, 16
    fresh = [r.randint(1, 3000) for _ in range(n)]
    need = sum(-(-f // page) for f in fresh)
    check_tables([0] * n, fresh, [0] * n, 188, r.sample(range(10 * need), need + 3), page, sum(fresh) + 100)


def test_tables_entries_that_the_table_lacks():
    """A held entry of -1 (no page behind it) gives slots of -1."""
    table = i32([[4, -1, 6]])
    cu, slots, held, cursor, missing = ops.kv_step_tables(i32([6]), i32([12]), table, i32([3]), i32([9]), 8, 12)
    assert slots.tolist() == [38, 39] + [-1] * 8 + [48, 49]
    assert held.tolist() == [3] and cursor.tolist() == [0] and missing.tolist() == [0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,d,page,tokens", [(1, 4, 8, 1), (3, 12, 8, 37), (2, 32, 16, 300), (8, 128, 64, 515),
                                              (5, 100, 32, 2500), (1, 256, 1024, 3)])
def test_append_places_rows(dtype, H, d, page, tokens):
    torch.manual_seed(tokens)
    blocks = -(-tokens // page) + 3
    k = torch.randn(tokens, H, d, device="cuda").to(dtype)
    v = torch.randn(tokens, H, d, device="cuda").to(dtype)
    slots = torch.randperm(blocks * page, device="cuda")[:tokens]
    slots[::5] = -1
    slots[1::7] = blocks * page + slots[1::7].clamp(min=0)  # beyond the cache: skipped (slots stay distinct)
    kc = torch.randn(blocks, H, page, d, device="cuda").to(dtype)
    vc = torch.randn(blocks, H, page, d, device="cuda").to(dtype)
    rk, rv = kc.clone(), vc.clone()
    ok = (slots >= 0) & (slots < blocks * page)
    rk[slots[ok] // page, :, slots[ok] % page] = k[ok]
    rv[slots[ok] // page, :, slots[ok] % page] = v[ok]
    ops.kv_append(k, v, slots, kc, vc)
    assert torch.equal(kc, rk) and torch.equal(vc, rv)


def test_append_takes_slices_of_a_fused_projection():
    torch.manual_seed(1)
    tokens, H, d, page = 50, 2, 64, 16
    fused = torch.randn(tokens, 4 * H + 2, d, device="cuda", dtype=torch.bfloat16)
    k, v = fused[:, 1:1 + H], fused[:, 2 * H + 1:3 * H + 1]
    kc = torch.zeros(5, H, page, d, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    slots = torch.arange(tokens, device="cuda")
    ops.kv_append(k, v, slots, kc, vc)
    assert torch.equal(kc.transpose(1, 2).reshape(-1, H, d)[:tokens], k)
    assert torch.equal(vc.transpose(1, 2).reshape(-1, H, d)[:tokens], v)
    # bf16 rows that start on 8-byte boundaries only
    flat = torch.randn(tokens, 3 * 12, device="cuda", dtype=torch.bfloat16)
    k, v = flat[:, 12:24].unflatten(1, (1, 12)), flat[:, 24:].unflatten(1, (1, 12))
    kc = torch.zeros(5, 1, page, 12, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    ops.kv_append(k, v, slots, kc, vc)
    assert torch.equal(kc.reshape(-1, 12)[:tokens], k[:, 0]) and torch.equal(vc.reshape(-1, 12)[:tokens], v[:, 0])


def test_append_refuses_rows_that_are_not_contiguous():
    k = torch.zeros(4, 8, 2, device="cuda").transpose(1, 2)
    kc = torch.zeros(2, 2, 8, 8, device="cuda")
    slots = torch.zeros(4, device="cuda", dtype=torch.int64)
    with pytest.raises(capi.InvalidArgument, match="contiguous"):
        ops.kv_append(k, k, slots, kc, kc.clone())
