"""Softmax attention of the Global blocks on the GPU against the 64-bit form:
packed prompts and trees over the paged cache."""
import math
import random

import pytest
import torch

from rhizome_b200 import ops
from tests.attn_ref import assert_close, attention, seen_causal, seen_tree

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def rounded(dtype, d):
    """Whether this width's form rounds probabilities (the tensor cores')."""
    return dtype == BF and d in (64, 128)


def cu_of(counts):
    at = [0]
    for m in counts:
        at.append(at[-1] + m)
    return at, torch.tensor(at, dtype=torch.int32, device="cuda")


def check_prompt(lens, H, Hkv, d, dtype, seed=0, scale=None, spoil=None, fused=False, behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    at, cu = cu_of(lens)
    tokens = at[-1] + behind
    x = torch.randn(tokens, H + 2 * Hkv, d, generator=g, device="cuda").to(dtype)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if spoil:
        spoil(q, k, v, at)
    out = torch.full((tokens, H, d), 7.0, device="cuda", dtype=dtype)
    o, lse = ops.attn_varlen_fwd(q, k, v, cu, scale=scale, out=out, with_lse=True)
    assert o is out and not ops.device_status()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if a == b:
            continue
        ref = attention(q[a:b], k[a:b], v[a:b], seen_causal(b - a, device="cuda"), scale, rounded(dtype, d))
        assert_close(o[a:b], ref[0], ref[2], f"o of prompt {i} of {b - a}")
        assert_close(lse[a:b], ref[1], ref[3], f"lse of prompt {i} of {b - a}")
    assert (out[at[-1]:] == 7).all(), "rows behind the last prompt"
    return o


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 1), (6, 2), (8, 8), (5, 1), (64, 1)])
@pytest.mark.parametrize("dtype,d", [(F32, 32), (F32, 128), (BF, 32), (BF, 64), (BF, 128)])
def test_prompts_of_every_length(dtype, d, H, Hkv):
    check_prompt([1, 2, 0, 63, 64, 65, 3, 127, 128, 129, 200], H, Hkv, d, dtype, seed=H)


@pytest.mark.parametrize("dtype,d", [(F32, 4), (F32, 100), (F32, 256), (BF, 8), (BF, 96), (BF, 256), (BF, 200)])
def test_prompts_of_every_width(dtype, d):
    check_prompt([70, 1, 33, 130], 4, 2, d, dtype, seed=d)


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF, 128), (BF, 64)])
def test_long_prompts(dtype, d):
    check_prompt([1500, 1, 777, 1025], 4, 2, d, dtype, seed=3, scale=0.3)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_prompt_inputs_may_be_slices_and_rows_behind_stay(dtype):
    check_prompt([40, 100, 5], 4, 2, 128, dtype, fused=True, behind=9)


def spoil_future(q, k, v, at):
    """Every kind of value that is not finite, in rows that others of their
    tile do not see, and in a whole later prompt."""
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if b - a > 40:
            v[b - 7, :, 3] = math.nan
            v[b - 20, 0, 5] = math.inf
            v[b - 30, -1, :] = -math.inf
            k[b - 3, :, 0] = math.nan
            k[b - 11, 0, 1] = math.inf


@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128), (BF, 64), (BF, 40)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(dtype, d):
    check_prompt([50, 3, 200, 300], 6, 2, d, dtype, seed=5, spoil=spoil_future)


@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128)])
def test_large_scores(dtype, d):
    """Scores in the hundreds: the running maximum moves by more than an
    exponential's range between tiles."""
    def grow(q, k, v, at):
        k *= torch.linspace(0.1, 40, k.shape[0], device="cuda")[:, None, None].to(dtype)
        q *= 4
    check_prompt([400, 150], 2, 1, d, dtype, seed=6, spoil=grow)


def test_prompt_results_do_not_depend_on_the_batch():
    g = torch.Generator(device="cuda").manual_seed(9)
    lens = [300, 17, 700, 128]
    at, cu = cu_of(lens)
    q = torch.randn(at[-1], 8, 128, generator=g, device="cuda").to(BF)
    k = torch.randn(at[-1], 2, 128, generator=g, device="cuda").to(BF)
    v = torch.randn(at[-1], 2, 128, generator=g, device="cuda").to(BF)
    o = ops.attn_varlen_fwd(q, k, v, cu)
    for a, b in zip(at, at[1:]):
        alone = ops.attn_varlen_fwd(q[a:b], k[a:b], v[a:b], cu_of([b - a])[1])
        assert torch.equal(alone, o[a:b])


@pytest.mark.parametrize("dtype,d", [(F32, 32), (F32, 200), (BF, 96)])
def test_results_do_not_depend_on_the_rows_of_a_tile(dtype, d):
    """A call of little work takes smaller row tiles: the same bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    counts = [70, 0, 333, 1] + [250] * 40
    at, cu = cu_of(counts)
    q = torch.randn(at[-1], 6, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(at[-1], 2, d, generator=g, device="cuda").to(dtype)
    v = torch.randn(at[-1], 2, d, generator=g, device="cuda").to(dtype)
    o = ops.attn_varlen_fwd(q, k, v, cu)
    for a, b in list(zip(at, at[1:]))[:6]:
        assert torch.equal(ops.attn_varlen_fwd(q[a:b], k[a:b], v[a:b], cu_of([b - a])[1]), o[a:b])


# ------------------------------------------------------------------ the paged cache

class Paged:
    """A cache in shuffled pages, unwritten rows and unused pages NaN."""

    def __init__(self, cached, counts, Hkv, d, page, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-(c + m) // page) for c, m in zip(cached, counts)]
        self.num_blocks = sum(need) + 3
        order = torch.randperm(self.num_blocks, generator=g, device="cuda").tolist()
        self.page, self.k, self.v = page, [], []
        self.kc = torch.full((self.num_blocks, Hkv, page, d), math.nan, device="cuda", dtype=dtype)
        self.vc = self.kc.clone()
        self.table = torch.full((len(cached), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for i, (c, m) in enumerate(zip(cached, counts)):
            pages = order[at:at + need[i]]
            at += need[i]
            self.table[i, :need[i]] = torch.tensor(pages, dtype=torch.int32)
            k = torch.randn(c + m, Hkv, d, generator=g, device="cuda").to(dtype)
            v = torch.randn(c + m, Hkv, d, generator=g, device="cuda").to(dtype)
            self.k.append(k)
            self.v.append(v)
        self.table = self.table.cuda()
        self.fill()

    def fill(self):
        """(Re)writes the pages from the plain rows."""
        for i, (k, v) in enumerate(zip(self.k, self.v)):
            pos = torch.arange(k.shape[0], device="cuda")
            block = self.table[i].long()[pos // self.page]
            ok = block >= 0
            self.kc[block[ok], :, (pos % self.page)[ok]] = k[ok]
            self.vc[block[ok], :, (pos % self.page)[ok]] = v[ok]


def random_tree(r, m):
    return [-1 if t == 0 else r.randint(-1, t - 1) for t in range(m)]


def check_tree(cached, counts, H, Hkv, d, dtype, page=16, seed=0, chain=False, parents=None, most=None, scale=None,
               change=None, hide=None):
    r = random.Random(seed)
    c = Paged(cached, counts, Hkv, d, page, dtype, seed)
    at, cu = cu_of(counts)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(at[-1] + 3, H, d, generator=g, device="cuda").to(dtype)
    if parents is None and not chain:
        parents = [random_tree(r, m) for m in counts]
    par = None if chain else torch.tensor([p for x in parents for p in x] + [0] * 3, dtype=torch.int32, device="cuda")
    if change:
        change(c, q)
        c.fill()
    hidden = hide(c) if hide else {}
    most = max(counts + [1]) if most is None else most
    out = torch.full((at[-1] + 3, H, d), 7.0, device="cuda", dtype=dtype)
    o, lse = ops.attn_tree_fwd(q, c.kc, c.vc, c.table, torch.tensor(cached, dtype=torch.int32, device="cuda"), cu, most,
                               parent=par, scale=scale, out=out, with_lse=True)
    assert not ops.device_status()
    for i, (a, b) in enumerate(zip(at, at[1:])):
        m = b - a
        if m == 0:
            continue
        if chain:
            seen = seen_causal(m, cached[i])
            seen[most:] = False
        else:
            seen = seen_tree([p if t < most else -2 for t, p in enumerate(parents[i])], cached[i])
        for key in hidden.get(i, ()):
            seen[:, key] = False
        ref = attention(q[a:b], c.k[i], c.v[i], seen.cuda(), scale, rounded(dtype, d))
        assert_close(o[a:b], ref[0], ref[2], f"o of tree {i} ({cached[i]} + {m})")
        assert_close(lse[a:b], ref[1], ref[3], f"lse of tree {i} ({cached[i]} + {m})")
    assert (out[at[-1]:] == 7).all(), "rows behind the last sequence"
    return o


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 1), (8, 2), (6, 2), (16, 1), (40, 1)])
@pytest.mark.parametrize("dtype,d", [(F32, 32), (F32, 128), (BF, 32), (BF, 64), (BF, 128)])
def test_single_tokens(dtype, d, H, Hkv):
    check_tree([0, 1, 5, 16, 31, 64, 127, 255, 256, 600, 1300], [1] * 11, H, Hkv, d, dtype, seed=H, chain=True)


@pytest.mark.parametrize("page", [8, 16, 64, 256, 1024])
@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 64), (BF, 128)])
def test_trees_of_every_size(dtype, d, page):
    check_tree([0, 3, 130, 700, 64, 1, 40], [1, 7, 20, 64, 0, 33, 2], 8, 2, d, dtype, page=page, seed=page)


@pytest.mark.parametrize("group", [1, 3, 8, 24, 64])
@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF, 128), (BF, 64), (BF, 72)])
def test_trees_of_every_group(dtype, d, group):
    check_tree([100, 0, 513], [9, 64, 30], group, 1, d, dtype, seed=group)


@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128), (BF, 64)])
def test_pieces_of_a_prompt(dtype, d):
    """No parent array: any number of rows, each sees the rows before it."""
    check_tree([0, 200, 37], [300, 129, 1], 4, 2, d, dtype, seed=2, chain=True)
    check_tree([0, 200, 37], [300, 129, 1], 4, 2, d, dtype, seed=2, chain=True, most=100)


@pytest.mark.parametrize("dtype,d,group", [(F32, 32, 4), (BF, 128, 4), (BF, 128, 16), (BF, 64, 1)])
def test_long_caches(dtype, d, group):
    check_tree([5000, 9000], [3, 5], group, 1, d, dtype, page=64, seed=1)
    check_tree([20000], [20], group, 1, d, dtype, page=32, seed=2)


@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128)])
def test_nodes_that_take_no_part(dtype, d):
    trees = [[-1, 0, -2, 2, 1, 5, 7, 3], [0, -1, 1, -5]]
    check_tree([30, 300], [8, 4], 4, 2, d, dtype, parents=trees)
    check_tree([30, 300], [8, 4], 4, 2, d, dtype, parents=trees, most=3)
    check_tree([30, 0], [8, 4], 4, 2, d, dtype, parents=[[-2] * 8, [-2] * 4])
    check_tree([10], [70], 4, 2, d, dtype, parents=[[-1] + list(range(69))], most=64)
    check_tree([10], [3], 4, 2, d, dtype, most=0)


@pytest.mark.parametrize("dtype,d,H", [(F32, 32, 4), (BF, 128, 4), (BF, 64, 32)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them_in_a_tree(dtype, d, H):
    def change(c, q):
        for i in range(len(c.k)):
            L = c.k[i].shape[0]
            c.v[i][L - 2, :, 1] = math.nan
            c.v[i][L - 5, 0, 2] = math.inf
            c.k[i][L - 4, :, 0] = math.nan
            c.v[i][L - 7, :, 2] = -math.inf
    check_tree([100, 3, 250], [12, 20, 9], H, 2, d, dtype, seed=4, change=change)


@pytest.mark.parametrize("dtype,d,H", [(F32, 32, 4), (BF, 128, 4), (BF, 64, 48)])
def test_pages_that_are_not_there(dtype, d, H):
    """Table entries outside the cache: their positions are seen by nobody."""
    def hide(c):
        c.table[0, 2] = -1
        c.table[1, 0] = c.num_blocks
        c.table[1, 5] = -7
        return {0: range(32, 48), 1: [*range(16), *range(80, 96)]}
    check_tree([100, 90], [5, 20], H, 2, d, dtype, seed=4, hide=hide)
    check_tree([1000, 500], [5, 20], H, 2, d, dtype, seed=4, hide=hide)


@pytest.mark.parametrize("dtype,d", [(F32, 32), (BF, 128)])
def test_positions_beyond_the_table(dtype, d):
    c = Paged([30], [6], 1, d, 8, dtype, 3)
    q = torch.randn(6, 2, d, device="cuda").to(dtype)
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    cached = torch.tensor([30], dtype=torch.int32, device="cuda")
    table = c.table[:, :4].contiguous()  # 32 positions: rows 2.. have none
    o, lse = ops.attn_tree_fwd(q, c.kc, c.vc, table, cached, cu, 6, with_lse=True)
    seen = seen_causal(6, 30)
    seen[2:] = False
    ref = attention(q, c.k[0], c.v[0], seen.cuda(), None, rounded(dtype, d))
    assert_close(o, ref[0], ref[2], "o")
    assert_close(lse, ref[1], ref[3], "lse")
    # tables of no columns and caches of no pages: nothing is seen
    for tab, kc, vc in ((c.table[:, :0].contiguous(), c.kc, c.vc), (c.table, c.kc[:0], c.vc[:0])):
        o, lse = ops.attn_tree_fwd(q, kc, vc, tab, cached, cu, 6, with_lse=True)
        assert (o == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("nodes,H", [(1, 4), (20, 8), (64, 32)])
def test_tree_results_do_not_depend_on_the_batch(nodes, H):
    d, page = 128, 16
    cached, counts = [2100, 0, 700, 5000], [nodes] * 4
    c = Paged(cached, counts, 2, d, page, BF, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(4 * nodes, H, d, generator=g, device="cuda").to(BF)
    lens = torch.tensor(cached, dtype=torch.int32, device="cuda")
    o = ops.attn_tree_fwd(q, c.kc, c.vc, c.table, lens, cu_of(counts)[1], nodes)
    for i in range(4):
        alone = ops.attn_tree_fwd(q[i * nodes:(i + 1) * nodes], c.kc, c.vc, c.table[i:i + 1], lens[i:i + 1],
                                  cu_of([nodes])[1], nodes)
        assert torch.equal(alone, o[i * nodes:(i + 1) * nodes])


def test_many_sequences():
    r = random.Random(1)
    n = 700
    check_tree([r.randrange(40) for _ in range(n)], [r.randrange(3) for _ in range(n)], 2, 1, 128, BF, seed=1)
    check_prompt([r.randrange(9) for _ in range(n)], 2, 1, 128, BF, seed=1)
    check_prompt([r.randrange(9) for _ in range(n)], 2, 1, 32, F32, seed=1)


@pytest.mark.parametrize("d,nodes,H", [(128, 24, 8), (128, 64, 8), (64, 40, 16), (128, 2, 16), (128, 20, 32)])
def test_many_trees_over_real_caches(d, nodes, H):
    """More units than CTAs, most with rows for one of a CTA's two row tiles:
    the idle half must not run ahead of the key ring."""
    r = random.Random(nodes)
    n = 60
    check_tree([r.randint(0, 5000) for _ in range(n)], [r.randint(1, nodes) for _ in range(n)], H, 2 if H < 32 else 8, d, BF,
               seed=nodes)


def test_trees_in_several_scheduling_groups():
    """Units are ordered by cost in groups of sequences: more than two groups,
    with sequences of no rows, no cache, one chunk and several."""
    r = random.Random(5)
    n = 450
    check_tree([r.choice([0, 3, 64, 500, 2559, 2560, 2561, 6000]) if r.random() < 0.3 else r.randint(0, 300) for _ in range(n)],
               [r.choice([0, 1, 5, 17, 33]) for _ in range(n)], 8, 1, 64, BF, seed=5)


def test_more_sequences_than_the_few_row_form_holds():
    r = random.Random(6)
    n = 4200
    check_tree([r.randrange(20) for _ in range(n)], [1] * n, 2, 1, 64, BF, page=8, seed=6)


@pytest.mark.parametrize("H,Hkv,nodes", [(8, 1, 6), (16, 8, 24)])
def test_caches_of_the_most_chunks(H, Hkv, nodes):
    check_tree([170000, 5], [nodes, nodes], H, Hkv, 64, BF, page=64, seed=7)


def test_many_prompts_of_mixed_lengths():
    r = random.Random(8)
    check_prompt([r.choice([1, 30, 100, 128, 200, 700]) for _ in range(60)], 16, 4, 128, BF, seed=8)
    check_prompt([r.choice([1, 30, 100, 128, 200, 700]) for _ in range(60)], 8, 8, 64, BF, seed=9)


# ------------------------------------------------------------------ a step as an engine runs it

@pytest.mark.parametrize("dtype", [BF, F32])
def test_prefill_draft_verify_and_commit_together(dtype):
    """Prompts admitted (tables, append, packed attention), a drafted tree
    verified, its accepted path appended again at its final slots, and one
    decode token, against plain attention over each sequence's whole history."""
    H, Hkv, d, page, n = 8, 2, 128, 16, 3
    r = random.Random(3)
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda m: [torch.randn(m, x, d, generator=g, device="cuda").to(dtype) for x in (H, Hkv, Hkv)]  # noqa: E731
    kc = torch.full((64, Hkv, page, d), math.nan, device="cuda", dtype=dtype)
    vc = kc.clone()
    table = torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(n, dtype=torch.int32, device="cuda")
    cursor = torch.zeros(1, dtype=torch.int32, device="cuda")
    free = torch.randperm(64, generator=g, device="cuda").to(torch.int32)
    history = [(torch.empty(0, Hkv, d, device="cuda", dtype=dtype),) * 2 for _ in range(n)]

    def admit(cached, counts):
        nonlocal held, cursor
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        cu, slots, held, cursor, missing = ops.kv_step_tables(i32(cached), i32(counts), table, held, free, page,
                                                              sum(counts), cursor=cursor)
        assert missing.item() == 0
        return cu, slots, i32(cached)

    def verify(o, q, k, v, counts, seen, what):
        a = 0
        for i, m in enumerate(counts):
            kk = torch.cat([history[i][0], k[a:a + m]])
            vv = torch.cat([history[i][1], v[a:a + m]])
            ref = attention(q[a:a + m], kk, vv, seen[i].cuda(), None, rounded(dtype, d))
            assert_close(o[a:a + m], ref[0], ref[2], what)
            a += m

    lens = [37, 100, 16]
    q, k, v = rnd(sum(lens))
    cu, slots, _ = admit([0] * n, lens)
    ops.kv_append(k, v, slots, kc, vc)
    verify(ops.attn_varlen_fwd(q, k, v, cu), q, k, v, lens, [seen_causal(m) for m in lens], "prompts")
    for i, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        history[i] = (k[a:b], v[a:b])

    counts = [9, 20, 1]
    parents = [random_tree(r, m) for m in counts]
    q, k, v = rnd(sum(counts))
    cu, slots, cached = admit(lens, counts)
    ops.kv_append(k, v, slots, kc, vc)
    par = torch.tensor([p for x in parents for p in x], dtype=torch.int32, device="cuda")
    o = ops.attn_tree_fwd(q, kc, vc, table, cached, cu, 20, parent=par)
    verify(o, q, k, v, counts, [seen_tree(p, c) for p, c in zip(parents, lens)], "trees")

    # accept the path to each tree's last node; the others' rows are overwritten
    final = torch.full((sum(counts),), -1, dtype=torch.int64)
    kept = []
    for i, (a, p) in enumerate(zip(cu.tolist(), parents)):
        path, t = [], counts[i] - 1
        while t >= 0:
            path.insert(0, t)
            t = p[t]
        rows = [a + t for t in path]
        final[rows] = slots.cpu()[a:a + len(path)]
        kept.append(len(path))
        history[i] = (torch.cat([history[i][0], k[rows]]), torch.cat([history[i][1], v[rows]]))
    ops.kv_append(k, v, final.cuda(), kc, vc)
    lens = [c + m for c, m in zip(lens, kept)]

    q, k, v = rnd(n)
    owned = held.clone()
    cu, slots, cached = admit(lens, [1] * n)
    assert (held >= owned).all() and (held - owned).max() <= 1, "the draft's pages are used first"
    ops.kv_append(k, v, slots, kc, vc)
    o = ops.attn_tree_fwd(q, kc, vc, table, cached, cu, 1)
    verify(o, q, k, v, [1] * n, [seen_causal(1, c) for c in lens], "decode")


def test_a_captured_step_replays_with_new_lengths():
    """One captured graph of tables, append and attention serves steps whose
    lengths, tables and inputs change between replays."""
    n, H, Hkv, d, page, dtype = 4, 8, 2, 128, 16, BF
    g = torch.Generator(device="cuda").manual_seed(5)
    kc = torch.zeros(200, Hkv, page, d, device="cuda", dtype=dtype)
    vc = torch.zeros_like(kc)
    table = torch.full((n, 40), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(200, generator=g, device="cuda").to(torch.int32)
    cached, fresh, held = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    cursor = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = 24  # room for the batch, padded
    q = torch.zeros(rows, H, d, device="cuda", dtype=dtype)
    k = torch.zeros(rows, Hkv, d, device="cuda", dtype=dtype)
    v = torch.zeros_like(k)
    ws = torch.empty(max(1, ops.attn_tree_workspace_bytes(rows, 8, 40, page, H, Hkv, d, dtype)), device="cuda",
                     dtype=torch.uint8)

    def step():
        cu, slots, now, at, _ = ops.kv_step_tables(cached, fresh, table, held, free, page, rows, cursor=cursor)
        ops.kv_append(k, v, slots, kc, vc)
        o = ops.attn_tree_fwd(q, kc, vc, table, cached, cu, 8, workspace=ws)
        held.copy_(now)
        cursor.copy_(at)
        cached.add_(fresh)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # nothing is fresh: leaves the state as it is
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    history = [(torch.empty(0, Hkv, d, device="cuda", dtype=dtype),) * 2 for _ in range(n)]
    r = random.Random(1)
    for _ in range(60):
        counts = [r.choice([0, 1, 5, 8]) for _ in range(n)]
        if sum(counts) > rows:
            continue
        fresh.copy_(torch.tensor(counts, dtype=torch.int32))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        a = 0
        for i, m in enumerate(counts):
            history[i] = (torch.cat([history[i][0], k[a:a + m]]), torch.cat([history[i][1], v[a:a + m]]))
            if m:
                ref = attention(q[a:a + m], *history[i], seen_causal(m, history[i][0].shape[0] - m, "cuda"), None, True)
                assert_close(o[a:a + m], ref[0], ref[2], f"replayed step, sequence {i}")
            a += m


def test_calls_on_another_stream():
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(500, 4, 128, generator=g, device="cuda").to(BF)
    k = torch.randn(500, 2, 128, generator=g, device="cuda").to(BF)
    cu = cu_of([200, 300])[1]
    want = ops.attn_varlen_fwd(q, k, k, cu)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.attn_varlen_fwd(q, k, k, cu)
        out = got.clone()
    side.synchronize()
    assert torch.equal(out, want)
