"""Refusals of the Global blocks' entry points and of the tree step, on a host
without a GPU: every bad argument is an error status before any device work,
and the wrappers check their torch arguments first."""
import math

import pytest
import torch

from rhizome_b200 import build, capi, ops
from tests.attn_ref import attention, seen_causal, seen_tree, step_tables

FAKE = 1 << 20  # an aligned non-null address; never dereferenced by validation
BF16, F32 = capi.RHZ_DTYPE_BF16, capi.RHZ_DTYPE_F32


@pytest.fixture(scope="module")
def lib():
    build.build()
    return capi.lib()


def refusals(fn, names, good, bad):
    """Each of `bad` = (status, overrides) on top of the good arguments."""
    for status, over in bad:
        assert fn(*[{**good, **over}[x] for x in names]) == status, over


def test_tree_step_refusals(lib):
    names = "o st pool slots cu par q k v al be n tokens most slots_n H d dt stream".split()
    good = dict.fromkeys(names, FAKE) | dict(slots=None, n=2, tokens=9, most=8, slots_n=4, H=2, d=32, dt=F32, stream=None)
    S, I, D = capi.RHZ_ERR_SHAPE, capi.RHZ_ERR_INVALID, capi.RHZ_ERR_DTYPE
    refusals(lib.rhz_gdr_tree_step, names, good, [
        (D, dict(dt=5)), (S, dict(d=0)), (S, dict(d=257)), (S, dict(H=0)), (S, dict(n=-1)), (S, dict(tokens=-1)),
        (S, dict(most=65)), (S, dict(most=-1)), (S, dict(n=5)), (S, dict(tokens=1 << 31)),
        (I, dict(q=None)), (I, dict(st=None)), (I, dict(cu=None)), (I, dict(par=FAKE + 2)), (I, dict(k=FAKE + 4)),
        (I, dict(pool=FAKE + 8)), (capi.RHZ_OK, dict(n=0)), (capi.RHZ_OK, dict(tokens=0))])


def test_step_tables_refusals(lib):
    names = "cu slot table held_out cur_out miss cached fresh held free cur n width free_n rows page stream".split()
    good = dict.fromkeys(names, FAKE) | dict(held_out=2 * FAKE, cur_out=2 * FAKE, n=4, width=8, free_n=9, rows=16,
                                             page=16, stream=None)
    S, I = capi.RHZ_ERR_SHAPE, capi.RHZ_ERR_INVALID
    refusals(lib.rhz_kv_step_tables, names, good, [
        (S, dict(page=0)), (S, dict(page=4)), (S, dict(page=24)), (S, dict(page=2048)), (S, dict(page=-16)),
        (S, dict(n=-1)), (S, dict(width=-1)), (S, dict(free_n=-1)), (S, dict(rows=-1)), (S, dict(width=1 << 32)),
        (I, dict(held_out=FAKE)), (I, dict(cur_out=FAKE)), (I, dict(cu=None)), (I, dict(slot=FAKE + 4)),
        (I, dict(free=None)), (I, dict(cur_out=None)), (I, dict(table=None)), (I, dict(miss=FAKE + 1))])


def test_append_refusals(lib):
    names = "kc vc k v slot tokens ks vs blocks page H d dt stream".split()
    good = dict.fromkeys(names, FAKE) | dict(tokens=4, ks=64, vs=64, blocks=3, page=16, H=2, d=32, dt=BF16, stream=None)
    S, I, D = capi.RHZ_ERR_SHAPE, capi.RHZ_ERR_INVALID, capi.RHZ_ERR_DTYPE
    refusals(lib.rhz_kv_append, names, good, [
        (D, dict(dt=2)), (S, dict(page=17)), (S, dict(d=30)), (S, dict(ks=60)), (S, dict(vs=66)), (S, dict(tokens=-1)),
        (S, dict(blocks=-1)), (S, dict(H=0)), (I, dict(k=FAKE + 4)), (I, dict(kc=FAKE + 8)), (I, dict(v=None)),
        (I, dict(slot=None)), (capi.RHZ_OK, dict(tokens=0)), (capi.RHZ_OK, dict(blocks=0))])


ATTN_BAD = [(capi.RHZ_ERR_DTYPE, dict(dt=3)), (capi.RHZ_ERR_SHAPE, dict(H=6)), (capi.RHZ_ERR_SHAPE, dict(Hkv=0)),
            (capi.RHZ_ERR_SHAPE, dict(H=65, Hkv=1, qs=65 * 32)), (capi.RHZ_ERR_SHAPE, dict(d=36)),
            (capi.RHZ_ERR_SHAPE, dict(d=264)), (capi.RHZ_ERR_SHAPE, dict(d=0)),
            (capi.RHZ_ERR_INVALID, dict(scale=0.0)), (capi.RHZ_ERR_INVALID, dict(scale=-1.0)),
            (capi.RHZ_ERR_INVALID, dict(scale=math.nan)), (capi.RHZ_ERR_INVALID, dict(scale=math.inf)),
            (capi.RHZ_ERR_SHAPE, dict(n=-1)), (capi.RHZ_ERR_SHAPE, dict(tokens=-1)),
            (capi.RHZ_ERR_SHAPE, dict(tokens=1 << 31)), (capi.RHZ_ERR_SHAPE, dict(qs=8 * 32 - 8)),
            (capi.RHZ_ERR_SHAPE, dict(qs=8 * 32 + 4)), (capi.RHZ_ERR_INVALID, dict(q=None)),
            (capi.RHZ_ERR_INVALID, dict(q=FAKE + 8)), (capi.RHZ_ERR_INVALID, dict(o=None)),
            (capi.RHZ_ERR_INVALID, dict(k=FAKE + 2)), (capi.RHZ_ERR_INVALID, dict(cu=None)),
            (capi.RHZ_ERR_INVALID, dict(lse=FAKE + 2)), (capi.RHZ_OK, dict(n=0)), (capi.RHZ_OK, dict(tokens=0))]


def test_varlen_attention_refusals(lib):
    names = "o lse q k v cu n tokens qs ks vs H Hkv d scale dt stream".split()
    good = dict.fromkeys(names, FAKE) | dict(n=2, tokens=9, qs=256, ks=128, vs=128, H=8, Hkv=4, d=32, scale=0.5,
                                             dt=BF16, stream=None)
    refusals(lib.rhz_attn_varlen_fwd, names, good, ATTN_BAD + [(capi.RHZ_ERR_SHAPE, dict(ks=120)),
                                                              (capi.RHZ_ERR_SHAPE, dict(vs=132))])


def test_tree_attention_refusals(lib):
    names = "o lse q k v table cached cu par n tokens most qs width blocks page H Hkv d scale dt ws wsb stream".split()
    good = dict.fromkeys(names, FAKE) | dict(n=2, tokens=9, most=8, qs=256, width=4, blocks=10, page=16, H=8, Hkv=4,
                                             d=32, scale=0.5, dt=BF16, ws=None, wsb=0, stream=None)
    S, I = capi.RHZ_ERR_SHAPE, capi.RHZ_ERR_INVALID
    refusals(lib.rhz_attn_tree_fwd, names, good, ATTN_BAD + [
        (S, dict(most=65)), (S, dict(most=-1)), (S, dict(page=12)), (S, dict(width=-1)), (S, dict(blocks=-1)),
        (S, dict(width=1 << 28)), (S, dict(blocks=1 << 27)), (I, dict(table=None)), (I, dict(cached=None)),
        (I, dict(par=FAKE + 1)), (I, dict(width=1 << 12))])  # the last: long tables need a workspace
    assert b"workspace too small" in lib.rhz_last_error()
    need = lib.rhz_attn_tree_workspace_bytes(9, 8, 1 << 12, 16, 8, 4, 32, BF16)
    assert need > 9 * 8 * 32 * 4
    refusals(lib.rhz_attn_tree_fwd, names, good, [(I, dict(width=1 << 12, ws=FAKE, wsb=need - 1)),
                                                  (I, dict(width=1 << 12, ws=FAKE + 16, wsb=need))])
    assert b"aligned" in lib.rhz_last_error()
    w = lib.rhz_attn_tree_workspace_bytes
    assert w(9, 8, 4, 16, 8, 4, 32, BF16) == 0  # short tables need none
    assert w(-1, 8, 4, 16, 8, 4, 32, BF16) == 0 and w(9, 8, 4, 15, 8, 4, 32, BF16) == 0 and w(9, 8, 4, 16, 8, 3, 32, 9) == 0


def test_tree_attention_refuses_sizes_whose_products_overflow(lib):
    names = "o lse q k v table cached cu par n tokens most qs width blocks page H Hkv d scale dt ws wsb stream".split()
    good = dict.fromkeys(names, FAKE) | dict(n=2, tokens=9, most=8, qs=256, width=4, blocks=10, page=16, H=8, Hkv=4,
                                             d=32, scale=0.5, dt=BF16, ws=None, wsb=0, stream=None)
    S = capi.RHZ_ERR_SHAPE
    refusals(lib.rhz_attn_tree_fwd, names, good, [(S, dict(width=1 << 60)), (S, dict(blocks=1 << 62)),
                                                  (S, dict(blocks=(1 << 62) + 1))])


def test_valid_calls_without_gpu_report_a_device_error(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert lib.rhz_attn_varlen_fwd(*[FAKE] * 6, 2, 9, 256, 128, 128, 8, 4, 32, 0.5, BF16, None) == capi.RHZ_ERR_DEVICE
    assert lib.rhz_kv_append(*[FAKE] * 5, 4, 64, 64, 3, 16, 2, 32, F32, None) == capi.RHZ_ERR_DEVICE


def test_wrappers_check_their_arguments_first():
    q, k = torch.zeros(9, 8, 32), torch.zeros(9, 4, 32)
    cu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(capi.InvalidArgument, match="CUDA tensor"):
        ops.attn_varlen_fwd(q, k, k, cu)
    with pytest.raises(capi.ShapeError, match="k has shape"):
        ops._rows(k[:8], "k", k.dtype, 9, 4, 32)
    with pytest.raises(capi.DtypeError):
        ops._rows(k.bfloat16(), "k", k.dtype, 9, 4, 32)
    with pytest.raises(capi.ShapeError):
        ops.attn_varlen_fwd(q[0], k, k, cu)
    with pytest.raises(capi.InvalidArgument, match="contiguous"):
        ops.attn_varlen_fwd(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, cu)
    cache, table = torch.zeros(5, 4, 16, 32), torch.zeros(2, 6, dtype=torch.int32)
    with pytest.raises(capi.ShapeError, match="k_cache"):
        ops.attn_tree_fwd(q, cache[0], cache, table, cu[:2], cu, 4)
    with pytest.raises(capi.InvalidArgument, match="CUDA tensor"):
        ops.attn_tree_fwd(q, cache, cache, table, cu[:2], cu, 4)
    with pytest.raises(capi.ShapeError, match="k has"):
        ops._rows(k[:, :3], "k", k.dtype, 9, 4, 32)
    with pytest.raises(capi.InvalidArgument, match="CUDA tensor"):
        ops.kv_step_tables(cu, cu, torch.zeros(3, 4, dtype=torch.int32), cu, cu, 16, 4)
    with pytest.raises(capi.ShapeError, match="one dimension"):
        ops._index(table, "cached")
    with pytest.raises(capi.ShapeError, match="expected \\[tokens, H, d\\]"):
        ops.gdr_tree_step(q[0], q, q, q, q, cu, None, 4)


# ------------------------------------------------------------------ the plain forms themselves

def test_plain_attention_is_softmax():
    torch.manual_seed(0)
    q, k, v = torch.randn(5, 4, 8), torch.randn(9, 2, 8), torch.randn(9, 2, 8)
    for seen in (seen_causal(5, 4), seen_tree([-1, 0, 0, 1, -1], 4)):
        o, lse, _, _ = attention(q, k, v, seen)
        x = torch.einsum("mhd,lhd->hml", q.double(), k.double().repeat_interleave(2, 1)) / math.sqrt(8)
        x = x.masked_fill(~seen, -math.inf)
        want = torch.einsum("hml,lhd->mhd", torch.softmax(x, -1), v.double().repeat_interleave(2, 1))
        assert torch.allclose(o, want, atol=1e-12) and torch.allclose(lse, torch.logsumexp(x, -1).T, atol=1e-12)


def test_plain_attention_keeps_masked_values_out():
    q, k, v = torch.randn(4, 1, 4), torch.randn(4, 1, 4), torch.randn(4, 1, 4)
    v[3], k[2] = math.nan, math.nan
    o, lse, _, _ = attention(q, k, v, seen_causal(4))
    assert torch.isfinite(o[:2]).all() and torch.isnan(o[2:]).all() and torch.isfinite(lse[:2]).all()
    o, lse, _, _ = attention(q, k, v, torch.zeros(4, 4, dtype=torch.bool))
    assert (o == 0).all() and (lse == -math.inf).all()


def test_plain_trees_and_tables():
    assert seen_tree([-1, 0, -2, 2, 1, 5, 4], 1).int().tolist() == [
        [1, 1, 0, 0, 0, 0, 0, 0], [1, 1, 1, 0, 0, 0, 0, 0], [0] * 8, [0] * 8, [1, 1, 1, 0, 0, 1, 0, 0], [0] * 8,
        [1, 1, 1, 0, 0, 1, 0, 1]]
    got = step_tables([3, 8], [6, 1], [[50, 0], [51, 0]], [1, 1], [7], 8, 8)
    assert got == ([0, 6, 7], [403, 404, 405, 406, 407, 56, -1, -1], [[50, 7], [51, 0]], [2, 1], 1, 1)


def test_attention_refuses_more_sequences_than_its_walk_over_them_allows(lib):
    for n, want in ((1 << 22, capi.RHZ_OK), ((1 << 22) + 1, capi.RHZ_ERR_SHAPE)):
        assert lib.rhz_attn_varlen_fwd(*[FAKE] * 6, n, 0, 256, 128, 128, 8, 4, 32, 0.5, BF16, None) == want
        assert lib.rhz_attn_tree_fwd(*[FAKE] * 9, n, 0, 8, 256, 4, 10, 16, 8, 4, 32, 0.5, BF16, None, 0, None) == want


def test_scratch_of_prompt_pieces_is_bounded_by_their_outputs(lib):
    """A bound of rows beyond a tree's fills the card by itself: four chunks of
    keys at most, whatever the table's width, once the row blocks do."""
    w = lib.rhz_attn_tree_workspace_bytes
    for tokens, width, page, H, Hkv, d, dt in ((8192, 8192, 16, 32, 8, 128, BF16), (65536, 10240, 16, 32, 4, 128, BF16),
                                               (8192, 1 << 20, 16, 32, 8, 128, F32), (4096, 4096, 64, 64, 64, 96, BF16),
                                               (8192, 1 << 17, 1024, 16, 1, 64, BF16)):
        chunk = tokens * H * (d + 1) * 4
        assert chunk < w(tokens, tokens, width, page, H, Hkv, d, dt) <= 4 * chunk + (1 << 20), (tokens, H, d)
    # trees (up to 64 nodes) keep theirs, and a bound just above comes down from it in steps
    tree = w(512, 64, 8192, 16, 32, 8, 128, BF16)
    assert tree > 30 * 512 * 32 * 129 * 4
    sizes = [w(512, most, 8192, 16, 32, 8, 128, BF16) for most in (64, 65, 128, 129, 256, 512, 4096)]
    assert sizes == sorted(sizes, reverse=True) and sizes[-1] <= 4 * 512 * 32 * 129 * 4 + (1 << 20)
    assert w(512, 4096, 8192, 16, 300, 300, 128, BF16) == 0  # (150 K/V heads and more: one chunk as ever)


def test_attention_refuses_a_scale_whose_product_with_log2_e_overflows(lib):
    for scale, want in ((3e38, capi.RHZ_ERR_INVALID), (2.0 ** 127, capi.RHZ_ERR_INVALID), (2.0 ** 126, capi.RHZ_OK), (1e-40, capi.RHZ_OK)):
        assert lib.rhz_attn_varlen_fwd(*[FAKE] * 6, 0, 0, 256, 128, 128, 8, 4, 32, scale, BF16, None) == want
        assert lib.rhz_attn_tree_fwd(*[FAKE] * 9, 0, 0, 8, 256, 4, 10, 16, 8, 4, 32, scale, BF16, None, 0, None) == want


def test_a_tensor_on_another_device_is_named():
    dev = torch.device("cpu")
    ops._same_device(dev, k=torch.zeros(1), parent=None)
    with pytest.raises(capi.InvalidArgument, match="v_cache is on meta, expected cpu"):
        ops._same_device(dev, k_cache=torch.zeros(1), v_cache=torch.zeros(1, device="meta"))
