"""The operators for drafted tokens and shared pages against their definitions
(branches_ref.py): attention of a tree of drafted tokens, the move of accepted
ones, sequences that continue others, and the pages that lengths need."""
import ctypes
import math
import os
import random

import pytest
import torch

import rocm_attn_b200
from branches_ref import (compact_ref, fork_ref, random_pool, random_tree, resize_ref, tree_bound, tree_ref)
from paged_ref import make_cache
from test_paged_cpu import LL3, PagedCache

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _q(B, Hq, S, D, dtype, seed=1):
    return torch.randn(B, Hq, S, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _trees(B, S, seed=0):
    rng = random.Random(seed)
    return ints([random_tree(S, rng) for _ in range(B)]).reshape(B, S)


def _close(out, ref, n, dtype, vmax=8.0):
    o, absum, smax = ref
    assert out.dtype == dtype and out.shape == o.shape
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    err, tol = (out - o).abs(), tree_bound(o, absum, smax, n, o.shape[3], dtype, vmax)
    assert (err <= tol).all(), f"error {(err / tol).max():.2f} of the bound"


def _tree(attn, lens, S, Hq, Hkv, D, ps, dtype, chain=False, new=None, seed=0, layout="hnd", width=None, scale=None):
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=seed, layout=layout, width=width)
    q = _q(len(lens), Hq, S, D, dtype, seed + 1)
    par = None if chain else _trees(len(lens), S, seed)
    nl = None if new is None else ints(new)
    out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), None if chain else par.cuda(),
                         None if new is None else nl.cuda(), scale)
    _close(out, tree_ref(q, k, v, table, ln, par, nl, scale), max(lens), dtype)
    assert attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# attn_tree
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,new", [
    ([1], None), ([5, 2, 0, 9], [5, 3, 0, 0]), ([7, 130, 64, 63, 65, 129], [3, 5, 4, 5, 1, 2]),
    ([700, 3, 0, 1300], [5, 1, 2, 4]), ([0, 0], None), ([256, 128], None)], ids=str)
def test_tree_lengths(attn, lens, new, D, dtype):
    _tree(attn, lens, 5, 8, 2, D, 16, dtype, new=new)
    _tree(attn, lens, 5, 8, 2, D, 16, dtype, new=new, chain=True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("S", [1, 2, 3, 16, 31, 33, 64, 65, 127, 129, 200])
def test_tree_sizes(attn, S, dtype):
    _tree(attn, [S + 40, S, 300], S, 4, 2, 64, 16, dtype, seed=S)
    _tree(attn, [S + 70, S + 1], S, 2, 1, 128, 16, dtype, seed=S, new=[S, max(1, S - 1)])


def test_tree_of_the_largest_size(attn):
    _tree(attn, [1500], 1024, 2, 1, 64, 64, BF16)
    _tree(attn, [1100], 1024, 1, 1, 128, 64, F16, chain=True)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [1, 5, 8, 16, 24, 33, 40, 72, 80, 96, 100, 136, 192, 250, 256])
def test_tree_head_dims(attn, D, dtype):
    _tree(attn, [200, 41], 6, 6, 2, D, 16, dtype, seed=D)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (9, 3), (7, 1), (16, 1), (17, 1), (80, 2), (64, 1)])
def test_tree_groups(attn, Hq, Hkv, dtype):
    _tree(attn, [150, 333], 7, Hq, Hkv, 64, 16, dtype, seed=Hq)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ps", [1, 2, 3, 7, 8, 24, 32, 48, 100, 128, 256, 300, 1024])
def test_tree_page_sizes(attn, ps, dtype):
    _tree(attn, [257, 9, 130], 9, 4, 2, 128, ps, dtype, seed=ps, layout="nhd" if ps % 2 else "hnd")
    _tree(attn, [333], 4, 4, 4, 64, ps, dtype, seed=ps)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tree_many_sequences(attn, dtype):
    lens = [(i * 7) % 23 for i in range(700)]
    lens[211] = 1500
    _tree(attn, lens, 3, 2, 1, 64, 8, dtype, new=[i % 4 for i in range(700)])


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (256, BF16), (64, F32)])
@pytest.mark.parametrize("S,Hq", [(3, 4), (40, 8)])
def test_tree_one_sequence_over_the_grid(attn, D, dtype, S, Hq):
    _tree(attn, [40001], S, Hq, 1, D, 16, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tree_drafts_across_tiles(attn, dtype):
    # the drafted tokens begin at every place of a tile
    for n in range(100, 260, 7):
        _tree(attn, [n], 20, 2, 1, 64, 32, dtype, seed=n, width=300)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tree_strides(attn, dtype):
    # rows that are not 16-byte aligned, K and V of different strides, strided q, table and tree, one tree for all
    k, v, table, ln = make_cache([77, 200], 2, 64, 16, dtype)
    q = _q(2, 4, 6, 64, dtype)
    tree = _trees(1, 6).expand(2, 6)
    ref = tree_ref(q, k, v, table, ln, tree)
    kx = torch.zeros(*k.shape[:3], 67, dtype=dtype, device="cuda")[..., 1:65]
    kx.copy_(k)
    vx = torch.zeros(k.shape[2], k.shape[0], k.shape[1], 64, dtype=dtype, device="cuda").permute(1, 2, 0, 3)
    vx.copy_(v)
    qx = torch.zeros(2, 6, 4, 64, dtype=dtype, device="cuda").transpose(1, 2)
    qx.copy_(q)
    tx = torch.zeros(2, 2 * table.shape[1], dtype=torch.int32, device="cuda")[:, ::2]
    tx.copy_(table)
    px = torch.zeros(1, 12, dtype=torch.int32, device="cuda")[:, ::2]
    px.copy_(tree[:1])
    for kk in (kx, k.cuda()):
        for pp in (tree.cuda(), tree[:1].cuda().expand(2, 6), px.expand(2, 6)):
            _close(attn.attn_tree(qx, kk, vx, tx, ln.cuda(), pp), ref, 200, dtype)
    # a head dim that is not the innermost is copied for q; one that starts off 16 bytes
    qt = q.cuda().transpose(1, 3).contiguous().transpose(1, 3)
    _close(attn.attn_tree(qt, kx, vx, tx, ln.cuda(), px.expand(2, 6)), ref, 200, dtype)
    qo = torch.zeros(2, 4, 6, 67, dtype=dtype, device="cuda")[..., 1:65]
    qo.copy_(q)
    _close(attn.attn_tree(qo, k.cuda(), v.cuda(), table.cuda(), ln.cuda(), px.expand(2, 6)), ref, 200, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_takes_nothing_from_tokens_it_does_not_follow(attn, dtype, D):
    # two branches, one of which has NaN and infinite keys and values; the tokens before them too
    S, n = 8, 150
    par = ints([[-1, 0, 0, 1, 2, 3, 4, 5]])  # 0 -> 1 -> 3 -> 5 -> 7 and 0 -> 2 -> 4 -> 6
    k, v, table, ln = make_cache([n], 1, D, 16, dtype)
    q = _q(1, 2, S, D, dtype)
    base = n - S
    for s, (kk, vv) in {2: (math.nan, math.inf), 4: (math.inf, math.nan), 6: (-math.inf, -math.inf)}.items():
        p, r = int(table[0, (base + s) // 16]), (base + s) % 16
        k[p, 0, r, 3], v[p, 0, r, 5] = kk, vv
    out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), par.cuda()).cpu()
    ref = tree_ref(q, k, v, table, ln, par)
    good = [0, 1, 3, 5, 7]
    _close(out[:, :, good], tuple(x[:, :, good] for x in ref), n, dtype)
    assert out[:, :, 2].isnan().all() and out[:, :, 4].isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_infinite_values_of_tokens_that_are_followed(attn, dtype, D):
    n, S = 140, 6
    par = ints([[-1, 0, 1, -1, 3, 4]])
    k, v, table, ln = make_cache([n], 2, D, 16, dtype)
    q = _q(1, 4, S, D, dtype)
    base = n - S
    v[int(table[0, (base + 1) // 16]), 0, (base + 1) % 16, 7] = math.inf
    v[int(table[0, (base + 4) // 16]), 1, (base + 4) % 16, 9] = math.nan
    v[int(table[0, 2]), 1, 3, 11] = -math.inf  # of the context: everybody sees it
    out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), par.cuda()).cpu().double()
    o, absum, smax = tree_ref(q, k, v, table, ln, par)
    assert torch.equal(out.isnan(), o.isnan()) and torch.equal(out.isinf(), o.isinf())
    assert o.isinf().any() and o.isnan().any()
    fine = o.isfinite()
    tol = tree_bound(o, absum, smax, n, D, dtype)
    assert ((out - o).abs()[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_tree_infinite_scores(attn, dtype):
    # rows whose every score is -inf are NaN, those that also see others are not
    k, v, table, ln = make_cache([4, 150], 1, 64, 16, dtype)
    k[int(table[0, 0]), 0, :2] = -math.inf
    k[int(table[1, 3]), 0, 5] = -math.inf
    q = _q(2, 2, 4, 64, dtype).abs() + 0.1
    par = ints([[-1, -1, 0, 1]] * 2)
    par[0] = ints([-1, 0, -1, 2])
    out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), par.cuda()).cpu()
    assert out[0, :, :2].isnan().all() and not out[0, :, 2:].isnan().any() and not out[1].isnan().any()
    k2 = k.clone()
    k2[int(table[1, 3]), 0, 5] = 0
    k2[int(table[0, 0]), 0, :2] = 0
    ref = tree_ref(q, k2, v, table, ln, par, drop=lambda b, t: b == 1 and t == 53)
    _close(out[:, :, 2:], tuple(x[:, :, 2:] for x in ref), 150, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_growing_scores(attn, dtype, D):
    # the maximum grows by small and by large steps from tile to tile
    for step in (0.5, 4.0, 40.0):
        k, v, table, ln = make_cache([900], 1, D, 16, dtype, seed=3)
        q = _q(1, 2, 3, D, dtype, 5)
        lift = torch.arange(57)[:, None] * 16 + torch.arange(16)[None]
        for j in range(57):
            p = int(table[0, j])
            k[p, 0] = (k[p, 0].double() + q[0, 0, 1].double() / q[0, 0, 1].double().norm() ** 2 * D ** 0.5 *
                       step * (lift[j] / 64.0)[:, None]).to(dtype)
        par = _trees(1, 3)
        out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), par.cuda())
        _close(out, tree_ref(q, k, v, table, ln, par), 900, dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_tree_scale(attn, dtype):
    _tree(attn, [100, 50], 4, 4, 4, 64, 16, dtype, scale=0.7)
    _tree(attn, [100, 50], 4, 4, 4, 128, 16, dtype, scale=1e-30)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_bad_pages_lengths_and_parents(attn, dtype, D):
    k, v, table, ln = make_cache([100, 90, 60], 2, D, 16, dtype)
    q = _q(3, 4, 5, D, dtype)
    par = _trees(3, 5, 3)
    drop = lambda b, t: (b, t // 16) in ((0, 2), (1, 5))  # noqa: E731
    ref = tree_ref(q, k, v, table, ln, par, drop=drop)
    bad = table.clone()
    bad[0, 2], bad[1, 5] = 10 ** 9, -5
    k, v, q, ln = k.cuda(), v.cuda(), q.cuda(), ln.cuda()
    _close(attn.attn_tree(q, k, v, bad.cuda(), ln, par.cuda()), ref, 100, dtype)
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0
    # parents that are no earlier token count as -1
    wrong, right = par.clone(), par.clone()
    wrong[0, 2], wrong[1, 4], wrong[2, 3] = 2, 900, -2
    right[0, 2] = right[1, 4] = right[2, 3] = -1
    good = attn.attn_tree(q, k, v, table.cuda(), ln, right.cuda())
    assert attn.check_status(0) == 0
    assert torch.equal(attn.attn_tree(q, k, v, table.cuda(), ln, wrong.cuda()), good)
    assert attn.check_status(0) == 8
    # behind the drafted ones parents do not matter
    n = ints([2, 3, 0]).cuda()
    wrong[0, 2:], wrong[1, 3:], wrong[2] = 77, -9, 1000
    attn.attn_tree(q, k, v, table.cuda(), ln, wrong.cuda(), n)
    assert attn.check_status(0) == 0
    # lengths behind the table, more drafted tokens than S
    long = ln + ints([200, 0, 0]).cuda()
    out = attn.attn_tree(q, k, v, table.cuda(), long, par.cuda())
    assert attn.check_status(0) == 8 and torch.isfinite(out[1:]).all()
    many = attn.attn_tree(q, k, v, table.cuda(), ln, par.cuda(), ints([6, 9, 5]).cuda())
    assert attn.check_status(0) == 8
    assert torch.equal(many, attn.attn_tree(q, k, v, table.cuda(), ln, par.cuda()))


def test_tree_of_one_token_is_attn_decode(attn):
    for dtype in (F16, BF16, F32):
        k, v, table, ln = (x.cuda() for x in make_cache([300, 77, 1, 0], 2, 128, 16, dtype))
        q = _q(4, 8, 1, 128, dtype).cuda()
        a, b = attn.attn_tree(q, k, v, table, ln), attn.attn_decode(q, k, v, table, ln)
        # both are within the bound of the exact result
        ref = tree_ref(q.cpu(), k.cpu(), v.cpu(), table.cpu(), ln.cpu())
        tol = 2 * tree_bound(*ref, 300, 128, dtype).cuda()
        assert ((a.double() - b.double()).abs() <= tol).all()


def test_tree_empty_calls_and_refusals(attn):
    k, v, table, ln = (x.cuda() for x in make_cache([40, 20], 2, 64, 16, F16))
    q = _q(2, 4, 3, 64, F16).cuda()
    for shape in ((2, 4, 0, 64), (2, 0, 3, 64)):
        assert attn.attn_tree(torch.empty(shape, dtype=F16, device="cuda"), k, v, table, ln).shape == shape
    none = attn.attn_tree(q[:0], k, v, table[:0], ln[:0])
    assert none.shape == (0, 4, 3, 64)
    tree = _trees(2, 3).cuda()
    for bad in (lambda: attn.attn_tree(q[:1], k, v, table, ln), lambda: attn.attn_tree(q[..., :32], k, v, table, ln),
                lambda: attn.attn_tree(q[:, :3], k, v, table, ln), lambda: attn.attn_tree(q.float(), k, v, table, ln),
                lambda: attn.attn_tree(q, k, v[:, :1], table, ln), lambda: attn.attn_tree(q, k, v, table, ln.long()),
                lambda: attn.attn_tree(q, k, v, table, ln, tree[:, :2]),
                lambda: attn.attn_tree(q, k, v, table, ln, tree.long()),
                lambda: attn.attn_tree(q, k, v, table, ln, tree[:1]), lambda: attn.attn_tree(q[0], k, v, table, ln),
                lambda: attn.attn_tree(q, k, v, table, ln, tree, ln[:1]),
                lambda: attn.attn_tree(q, k, v, table, ln, tree.cpu()),
                lambda: attn.attn_tree(q.repeat(1, 1, 400, 1), k, v, table, ln)):
        with pytest.raises(RuntimeError):
            bad()
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (64, F32)])
def test_tree_results_repeat_bit_for_bit(attn, D, dtype):
    k, v, table, ln = (x.cuda() for x in make_cache([3000, 10, 700], 2, D, 16, dtype))
    q, par = _q(3, 8, 9, D, dtype).cuda(), _trees(3, 9).cuda()
    first = attn.attn_tree(q, k, v, table, ln, par)
    for _ in range(5):
        assert torch.equal(attn.attn_tree(q, k, v, table, ln, par), first)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (64, F32)])
def test_tree_captured_and_on_two_streams(attn, D, dtype):
    # two captured calls, replayed with other lengths, trees and queries, and at once on two streams
    lens = [[500, 60, 0], [90, 700, 33]]
    data = []
    for i in range(2):
        k, v, table, ln = make_cache([800, 800, 800], 2, D, 16, dtype, seed=i)
        data.append([x.cuda() for x in (k, v, table)] + [ints(lens[i]).cuda(), _q(3, 4, 6, D, dtype, i).cuda(),
                                                         _trees(3, 6, i).cuda(), ints([6, 4, 5]).cuda()])
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for k, v, table, ln, q, par, new in data:
        attn.attn_tree(q, k, v, table, ln, par, new)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attn.attn_tree(q, k, v, table, ln, par, new))
        graphs.append(g)
    for turn in range(2):
        for (k, v, table, ln, q, par, new), other in zip(data, lens[::-1]):
            if turn:
                ln.copy_(ints(other))
                q.neg_()
                par.copy_(_trees(3, 6, 9))
                new.copy_(ints([1, 6, 0]))
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for (k, v, table, ln, q, par, new), out in zip(data, outs):
            assert torch.equal(out, attn.attn_tree(q, k, v, table, ln, par, new))
            _close(out, tree_ref(*(x.cpu() for x in (q, k, v, table, ln, par, new))), 800, dtype)


@pytest.mark.parametrize("dtype,Hq,S", [(BF16, 4, 2), (BF16, 4, 5), (F16, 8, 30), (F32, 4, 5)])
def test_offsets_past_32_bits(attn, dtype, Hq, S):
    # the last pages of a cache of more than 2^32 bytes and 2^31 elements
    ps, D = 256, 128
    P = 2 ** 31 // (ps * D) + 64
    cache = torch.zeros(P, 1, ps, D, dtype=dtype, device="cuda")
    k, v, table, ln = make_cache([700], 1, D, ps, dtype, spare=0)
    cache[P - 3:] = k.cuda()
    far = (table + P - 3).cuda()
    q, par = _q(1, Hq, S, D, dtype), _trees(1, S)
    out = attn.attn_tree(q.cuda(), cache, cache, far, ln.cuda(), par.cuda())
    _close(out, tree_ref(q, k, k, table, ln, par), 700, dtype)
    if S != 5:
        return
    kept, new = ints([[1, 4]]), ints([5])
    attn.kv_compact(cache, cache.clone(), far, ln.cuda(), kept.cuda(), new.cuda())
    was = k.clone()
    for i, a in enumerate((1, 4)):
        k[int(table[0, (695 + i) // ps]), 0, (695 + i) % ps] = was[int(table[0, (695 + a) // ps]), 0, (695 + a) % ps]
    assert torch.equal(cache[P - 3:].cpu().nan_to_num(7.0), k.nan_to_num(7.0))
    # a fork whose source and copy lie there
    refs = torch.ones(P, dtype=torch.int32, device="cuda")
    refs[P - 5] = 0
    t, h, n, m = attn.kv_fork(cache, cache.clone(), far, ints([3]).cuda(), ln.cuda(), refs, ints([0, 0]).cuda())
    assert m.tolist() == [0] and t[1].tolist() == far[0, :2].tolist() + [P - 5] and n.tolist() == [700, 700]
    assert torch.equal(cache[P - 5, :, :188], cache[int(far[0, 2]), :, :188]) and not cache[P - 5, :, 188:].any()
    assert attn.check_status(0) == 0


def test_more_sequences_than_a_grid_dimension(attn):
    # 70000 sequences of one or two tokens
    B, ps, D = 70000, 2, 64
    lens = torch.tensor([1 + i % 2 for i in range(B)], dtype=torch.int32).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(B + 50000, 1, ps, D, generator=g, device="cuda", dtype=F16) for _ in range(2))
    table, held = torch.full((B, 1), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    refs = torch.zeros(B + 50000, dtype=torch.int32, device="cuda")
    refs[5] = 3
    assert not attn.kv_resize(table, held, lens, refs, ps).any()
    assert torch.equal(table[:, 0], torch.tensor([i for i in range(B + 1) if i != 5], dtype=torch.int32).cuda())
    for S in (1, 9):
        q = torch.randn(B, 1, S, D, generator=g, device="cuda", dtype=F16)
        one = torch.ones(B, dtype=torch.int32, device="cuda")
        out = attn.attn_tree(q, k, v, table, lens, new_lens=one).double()
        kk, vv = k[table[:, 0].long(), 0].double(), v[table[:, 0].long(), 0].double()
        x = (q[:, 0, 0].double()[:, None] * kk).sum(2) / 8
        x[lens == 1, 1] = -math.inf
        want = (torch.softmax(x, 1)[..., None] * vv).sum(1)
        assert ((out[:, 0, 0] - want).abs() <= 2.0 ** -9 * (1 + want.abs())).all() and not out[:, :, 1:].any()
    moved = attn.kv_compact(k, v, table, lens, torch.zeros(B, 1, dtype=torch.int32, device="cuda"), one)
    assert torch.equal(moved, lens)
    parents = torch.arange(B, dtype=torch.int32, device="cuda") // 2 * 2
    t, h, n, m = attn.kv_fork(k, v, table, held, lens, refs, parents)
    assert m.tolist() == [0] and torch.equal(n, lens[parents.long()])
    assert torch.equal(t[::2], table[::2]) and int(refs.clamp(0, 1).sum()) == B + 1 and t.unique().numel() == B
    assert torch.equal(k[t[1::2, 0].long(), :, 0], k[t[::2, 0].long(), :, 0])
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,S", [(BF16, 1), (BF16, 40), (F16, 9), (F32, 3)])
def test_cache_without_pages(attn, dtype, S):
    k = torch.empty(0, 2, 16, 64, dtype=dtype, device="cuda")
    q = torch.randn(2, 4, S, 64, device="cuda").to(dtype)
    table, ln = ints([[0], [0]]).cuda(), ints([0, 0]).cuda()
    assert not attn.attn_tree(q, k, k, table, ln).any() and attn.check_status(0) == 0
    attn.attn_tree(q, k, k, table, ints([3, 0]).cuda())
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0
    refs = torch.zeros(0, dtype=torch.int32, device="cuda")
    held = ints([0, 0]).cuda()
    assert attn.kv_resize(table, held, ints([5, 0]).cuda(), refs, 16).tolist() == [1, 0]
    t, h, n, m = attn.kv_fork(k, k, table, held, ln, refs, ints([1, 0, -1]).cuda())
    assert n.tolist() == [0, 0, 0] and m.tolist() == [0] and attn.check_status(0) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_that_are_not_there_may_hold_anything(attn, D):
    # queries behind the drafted tokens, in rows that share a warp with others
    k, v, table, ln = make_cache([90, 200], 2, D, 16, BF16)
    for S, Hq in ((2, 4), (7, 8), (40, 16)):
        q, new = _q(2, Hq, S, D, BF16), ints([S - 1, 1])
        q[0, :, S - 1:] = math.nan
        q[1, :, 1:] = math.inf
        out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), new_lens=new.cuda())
        _close(out, tree_ref(q, k, v, table, ln, new_lens=new), 200, BF16)
        assert not out[0, :, S - 1:].any() and not out[1, :, 1:].any()


# ---------------------------------------------------------------------------
# the watchdog (tests/test_watchdog_gpu.py says how the test build works)
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("lens,D,Hq,S,ps", [([300, 40], 128, 8, 9, 16), ([2000, 700], 64, 4, 30, 24), ([900], 256, 4, 12, 64),
                                            ([3000, 50], 128, 8, 50, 32), ([700], 64, 16, 40, 16), ([300, 90], 128, 4, 3, 16)])
def test_watchdog_fires_and_recovers(lens, D, Hq, S, ps):
    # CTA 0's first wait is for 16 bytes more than come: it ends by the limit, the kernel reports it and
    # returns, and the next launch is clean
    lib = ctypes.CDLL(os.path.join(os.path.dirname(rocm_attn_b200.KERNEL_LIB_PATH), "librocm_attn_wdtest.so"))
    p, i = ctypes.c_void_p, ctypes.c_int
    lib.attn_set_wait_limit_ns.argtypes = [ctypes.c_ulonglong]
    lib.launch_attn_tree.argtypes = [p, p, p, p, i, i, ctypes.c_float, p, ctypes.c_longlong, p, p, ctypes.c_size_t, p]
    k, v, table, ln = make_cache(lens, 2, D, ps, BF16)
    q, par = _q(len(lens), Hq, S, D, BF16), _trees(len(lens), S)
    dk, dv, dt, dl, dq, dp = (t.cuda() for t in (k, v, table, ln, q, par))
    out = torch.zeros_like(dq)
    st = LL3(*dk.stride()[:3])
    c = PagedCache(dk.data_ptr(), dv.data_ptr(), k.shape[0], 2, ps, D, 1, st, st, dt.data_ptr(), dt.shape[1], dt.shape[1],
                   dl.data_ptr(), len(lens))
    size = ctypes.c_size_t()
    assert lib.attn_tree_workspace_bytes(ctypes.byref(c), Hq, S, ctypes.byref(size)) == 0
    space = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def run():
        assert lib.launch_attn_tree(ctypes.byref(c), dq.data_ptr(), None, out.data_ptr(), Hq, S, -1.0, dp.data_ptr(), S,
                                    None, space.data_ptr(), size.value, stream) == 0
        status = ctypes.c_int(-1)
        assert lib.attn_get_status(stream, ctypes.byref(status)) == 0
        return status.value

    assert run() == 0
    lib.attn_set_wait_limit_ns(1_000_000)
    lib.attn_test_drop_arrival(1)
    try:
        assert run() == 7
    finally:
        lib.attn_test_drop_arrival(0)
        lib.attn_set_wait_limit_ns(0)
    assert run() == 0
    _close(out, tree_ref(q, k, v, table, ln, par), max(lens), BF16)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128), (F32, 64)])
def test_layers_as_heads_of_one_cache(attn, dtype, D):
    # three layers of two kv heads in one cache: each layer reads a view, one fork and one compaction move them all
    S, Hq, ps = 6, 8, 16
    k, v, table, ln = make_cache([150, 90], 6, D, ps, dtype)
    dk, dv = k.cuda(), v.cuda()
    P = k.shape[0]
    refs = torch.zeros(P, dtype=torch.int32)
    held = (ln + ps - 1) // ps
    for b in range(2):
        refs[table[b, :held[b]].long()] += 1
    table, held, lens, missing = attn.kv_fork(dk, dv, table.cuda(), held.cuda(), ln.cuda(), refs.cuda(), ints([0, 1, 1]).cuda())
    assert missing.tolist() == [0]
    q, par = _q(3, Hq, S, D, dtype), _trees(3, S)
    for layer in range(3):
        heads = slice(2 * layer, 2 * layer + 2)
        out = attn.attn_tree(q.cuda(), dk[:, heads], dv[:, heads], table, lens, par.cuda())
        _close(out, tree_ref(q, dk[:, heads].cpu(), dv[:, heads].cpu(), table.cpu().clamp(min=0), lens.cpu(), par), 150, dtype)
    for x, was in ((dk, k), (dv, v)):
        # the copy of sequence 1's last page, all layers
        new, old = int(table[2, 5]), int(table[1, 5])
        assert new != old and torch.equal(x[new, :, :10], x[old, :, :10]) and torch.equal(x[old, :, :10].cpu(), was[old, :, :10])


# ---------------------------------------------------------------------------
# kv_compact
# ---------------------------------------------------------------------------


def _paths(new, width, rng):
    out = []
    for n in new:
        m = rng.randint(0, min(n, width)) if n > 0 else 0
        out.append(sorted(rng.sample(range(n), m)) + [-1] * (width - m))
    return ints(out).reshape(len(new), width)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,layout", [(64, 16, "hnd"), (128, 7, "nhd"), (5, 3, "hnd"), (256, 64, "hnd"), (80, 1, "nhd"),
                                         (33, 24, "hnd")])
@pytest.mark.parametrize("S", [1, 8, 40, 130])
def test_compact(attn, S, D, ps, layout, dtype):
    rng = random.Random(S * D)
    lens = [S, S + 37, S + 200, 0, S + 1]
    new = [S, max(1, S - 3), S, 0, S]
    k, v, table, ln = make_cache(lens, 3, D, ps, dtype, layout=layout, seed=S, poison=False)
    kept = _paths(new, S, rng)
    kg, vg = k.cuda(), v.cuda()
    if layout == "nhd":
        kg, vg = (x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    got = attn.kv_compact(kg, vg, table.cuda(), ln.cuda(), kept.cuda(), ints(new).cuda())
    want = compact_ref(k, v, table, ln, kept, ints(new))
    assert torch.equal(got.cpu(), want) and got.dtype == torch.int32
    assert torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)
    assert attn.check_status(0) == 0


def test_compact_edges_of_lists(attn):
    # nothing kept, all kept, the last alone, lists that go wrong, tokens before the sequence's start, strided lists
    S = 6
    lists = [[-1, 3, 4], [0, 1, 2], [5, -1, -1], [1, 1, 2], [2, 6, -1], [3, -7, 1], [0, 4, 5], [2, 4, 5]]
    lens = [50, 50, 50, 50, 50, 50, 4, 3]
    k, v, table, ln = make_cache(lens, 2, 64, 16, F16, poison=False)
    kg, vg = k.cuda(), v.cuda()
    kept = torch.zeros(8, 6, dtype=torch.int32, device="cuda")[:, ::2]
    kept.copy_(ints(lists))
    new = ints([S] * 8)
    got = attn.kv_compact(kg, vg, table.cuda(), ln.cuda(), kept, new.cuda())
    want = compact_ref(k, v, table, ln, ints(lists), new)
    assert want.tolist() == [44, 47, 45, 45, 45, 45, 1, 0]
    assert torch.equal(got.cpu(), want) and torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)
    assert attn.check_status(0) == 8
    # bad pages are neither read nor written
    bad = table.clone()
    bad[0] = 2 ** 30
    attn.kv_compact(kg, vg, bad[:1].cuda(), ints([50]).cuda(), ints([[2, 5]]).cuda(), ints([S]).cuda())
    assert attn.check_status(0) == 8 and torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)
    assert attn.kv_compact(kg, vg, table.cuda(), ln.cuda(), kept[:, :0], new.cuda()).tolist() == [44] * 6 + [0, 0]
    assert attn.kv_compact(kg, vg, table[:0].cuda(), ln[:0].cuda(), kept[:0], new[:0].cuda()).shape == (0,)


# ---------------------------------------------------------------------------
# kv_resize
# ---------------------------------------------------------------------------


def _resize(attn, table, held, lens, refs, ps):
    """The operator against the definition, on lists that are changed."""
    t, h, r = ints(table).reshape(len(table), len(table[0]) if table else 3).cuda(), ints(held).cuda(), ints(refs).cuda()
    missing = attn.kv_resize(t, h, ints(lens).cuda(), r, ps)
    want = resize_ref(table, held, lens, refs, ps)
    assert missing.tolist() == want and h.tolist() == held and r.tolist() == refs and t.tolist() == table
    return want


@pytest.mark.parametrize("B,W,P,ps", [(1, 1, 1, 16), (1, 700, 900, 1), (3, 9, 40, 16), (64, 20, 1500, 16), (300, 5, 1000, 7),
                                      (1500, 3, 9000, 4), (16, 64, 70000, 16)])
def test_resize(attn, B, W, P, ps):
    rng = random.Random(B)
    table, held, lens, refs = random_pool(rng, B, W, P, ps, shared=0.2)
    for turn in range(6):
        most = W * ps
        lens = [rng.choice([0, most, rng.randint(0, most), min(most, max(0, held[b] * ps + rng.randint(-ps, ps)))])
                for b in range(B)]
        if turn == 4:
            lens = [-3] * B
        _resize(attn, table, held, lens, refs, ps)
        assert attn.check_status(0) == 0


def test_resize_without_enough_pages(attn):
    table, held, refs = [[-1] * 4 for _ in range(5)], [0] * 5, [0, 1, 0, 0, 2, 0, 0]
    assert _resize(attn, table, held, [20, 33, 16, 16, 0], refs, 16) == [0, 0, 1, 1, 0]
    assert held == [2, 3, 0, 0, 0] and refs == [1, 1, 1, 1, 2, 1, 1]
    # pages given back in a call are there for the next one
    assert _resize(attn, table, held, [0, 33, 16, 16, 0], refs, 16) == [0, 0, 1, 1, 0]
    assert _resize(attn, table, held, [0, 33, 16, 16, 0], refs, 16) == [0, 0, 0, 0, 0]
    assert attn.check_status(0) == 0
    # more than the pool has
    table, held, refs = [[-1] * 64], [0], [0] * 8
    assert _resize(attn, table, held, [1000], refs, 16) == [63]
    assert _resize(attn, [], [], [], [0] * 8, 16) == []
    assert _resize(attn, [[-1, -1]], [0], [5], [], 16) == [1]


def test_resize_reports_what_is_out_of_range(attn):
    t, h, r = ints([[0, 1], [2, 3], [4, 99], [5, 5]]).cuda(), ints([2, -1, 2, 2]).cuda(), ints([1, 1, 1, 1, 1, 1, 0, 0]).cuda()
    missing = attn.kv_resize(t, h, ints([80, 0, 0, 0]).cuda(), r, 16)  # too long, bad count, bad page, page given back twice
    assert attn.check_status(0) == 8
    assert h.tolist() == [2, 0, 0, 0] and missing.tolist() == [0] * 4
    assert r.tolist() == [1, 1, 1, 1, 0, -1, 0, 0] and t[0].tolist() == [0, 1]
    # the page whose count is negative is not given out
    attn.kv_resize(t, h, ints([32, 32, 32, 0]).cuda(), r, 16)
    assert attn.check_status(0) == 0 and t.tolist()[1:3] == [[4, 6], [4, 99]] and h.tolist() == [2, 2, 0, 0]


def test_resize_refusals(attn):
    t, h, n, r = ints([[-1, -1]] * 2).cuda(), ints([0, 0]).cuda(), ints([5, 5]).cuda(), ints([0] * 8).cuda()
    wide = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for bad in (lambda: attn.kv_resize(wide[:, ::2], h, n, r, 16), lambda: attn.kv_resize(t[:1].expand(2, 2), h, n, r, 16),
                lambda: attn.kv_resize(t, h[:1], n, r, 16), lambda: attn.kv_resize(t, h, n[:1], r, 16),
                lambda: attn.kv_resize(t, h.long(), n, r, 16), lambda: attn.kv_resize(t, h, n, r[::2], 16),
                lambda: attn.kv_resize(t, h, n, r, 0), lambda: attn.kv_resize(t, wide[:, 0], n, r, 16),
                lambda: attn.kv_resize(t, h, n, r.cpu(), 16), lambda: attn.kv_resize(t, h, n, r, 1 << 31)):
        with pytest.raises(RuntimeError):
            bad()
    attn.kv_resize(wide[:, :2], h, n, r, 16)  # rows apart
    assert wide.tolist() == [[0, 0, 0, 0], [1, 0, 0, 0]] and attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# kv_fork
# ---------------------------------------------------------------------------


def _fork(attn, table, held, lens, refs, parents, Hkv, D, ps, dtype, layout="hnd", seed=0):
    """The operator against the definition; the new lists."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(len(refs), Hkv, ps, D, generator=g).to(dtype) for _ in range(2))
    kg, vg = k.cuda(), v.cuda()
    if layout == "nhd":
        kg, vg = (x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    r, W = ints(refs).cuda(), len(table[0])
    t, h, n, missing = attn.kv_fork(kg, vg, ints(table).reshape(-1, W).cuda(), ints(held).cuda(), ints(lens).cuda(), r,
                                    ints(parents).cuda())
    want = fork_ref(k, v, table, held, lens, refs, parents, ps)
    assert t.shape == (len(parents), W) and t.tolist() == want[0] and h.tolist() == want[1] and n.tolist() == want[2]
    assert missing.tolist() == [want[3]] and r.tolist() == refs
    assert torch.equal(kg.cpu(), k) and torch.equal(vg.cpu(), v)
    return want


@pytest.mark.parametrize("dtype,D,layout", [(F16, 64, "hnd"), (BF16, 128, "nhd"), (F32, 80, "hnd"), (BF16, 33, "hnd"),
                                            (F32, 256, "nhd")])
@pytest.mark.parametrize("B,n,W,P,ps", [(1, 1, 1, 3, 16), (1, 7, 4, 60, 16), (6, 6, 5, 90, 24), (20, 33, 3, 200, 3),
                                        (9, 2, 6, 70, 64), (3, 4, 5, 40, 1), (4, 1200, 2, 1300, 4), (1100, 40, 2, 1500, 2)])
def test_fork(attn, B, n, W, P, ps, dtype, D, layout):
    rng = random.Random(B * 31 + n)
    for turn in range(2):
        table, held, lens, refs = random_pool(rng, B, W, P, ps)
        parents = [rng.randrange(-1, B) for _ in range(n)]
        if turn:
            parents = sorted(parents)
        _fork(attn, table, held, lens, refs, parents, 3, D, ps, dtype, layout, seed=turn)
        assert attn.check_status(0) == 0


def test_pools_of_more_pages_than_are_noted(attn):
    # more counts than a warp keeps the bits of; the free pages few and at the end, and then many
    rng, P = random.Random(5), 700_003
    for free in ([P - 1 - 7 * i for i in range(40)], sorted(rng.sample(range(P), 300_000))):
        refs = [1] * P
        for p in free:
            refs[p] = 0
        table, held = [[-1] * 9 for _ in range(6)], [0] * 6
        lens = [18, 1, 0, 11, 17, 16]
        assert _resize(attn, table, held, lens, refs, 2) == [0] * 6
        parents = [rng.randrange(6) for _ in range(9)]
        _fork(attn, table, held, lens, refs, parents, 1, 8, 2, F16)
        assert attn.check_status(0) == 0


def test_fork_edges(attn):
    # a page that others hold is copied for the first child too; released pages are not given out by the call
    table, held, lens = [[0, 1], [0, 1], [2, -1]], [2, 2, 1], [20, 20, 16]
    refs = [2, 2, 1, 0, 0, 0]
    new = _fork(attn, table, held, lens, refs, [0, 1, 1, 2, -1], 2, 64, 16, F16)
    assert new[0][:4] == [[0, 3], [0, 4], [0, 5], [2, -1]] and refs == [3, 0, 1, 1, 1, 1]
    # too few free pages: nothing changes
    table, held, lens, refs = [[0, 1]], [2], [17], [1, 1, 0]
    new = _fork(attn, table, held, lens, refs, [0, 0, 0, 0], 2, 64, 16, BF16)
    assert new[3] == 2 and new[1] == [0] * 4 and refs == [1, 1, 0]
    # no new sequence: all is given back
    _fork(attn, [[0, 1], [0, 2]], [2, 2], [20, 20], [2, 1, 1, 0], [], 2, 64, 16, F16)
    # pages held ahead of the tokens go back
    new = _fork(attn, [[3, 1, 2]], [3], [5], [0, 1, 1, 1], [0, 0], 1, 64, 16, F32)
    assert new[0] == [[3, -1, -1], [0, -1, -1]]
    assert attn.check_status(0) == 0
    # lengths behind the pages that are held, parents that are none, counts out of range
    k = torch.zeros(6, 1, 16, 64, dtype=F16, device="cuda")
    r = ints([1, 1, 1, 0, 0, 0]).cuda()
    t, h, n, m = attn.kv_fork(k, k.clone(), ints([[0, 1], [2, 7]]).cuda(), ints([1, 5]).cuda(), ints([30, 16]).cuda(), r,
                              ints([0, 2, -4, 1]).cuda())
    assert attn.check_status(0) == 8
    assert t.tolist() == [[0, -1], [-1, -1], [-1, -1], [2, -1]] and n.tolist() == [16, 0, 0, 16] and m.tolist() == [0]
    assert r.tolist() == [1, 1, 1, 0, 0, 0]


def test_fork_refusals(attn):
    k, t, h, n, r = torch.zeros(6, 1, 16, 64, dtype=F16, device="cuda"), *(ints(x).cuda() for x in (
        [[0, 1], [2, 3]], [2, 2], [20, 20], [1, 1, 1, 1, 0, 0]))
    p = ints([0, 1]).cuda()
    for bad in (lambda: attn.kv_fork(k, k, t, h[:1], n, r, p), lambda: attn.kv_fork(k, k, t, h, n, r[:5], p),
                lambda: attn.kv_fork(k, k, t, h, n, r, p.long()), lambda: attn.kv_fork(k, k, t, h, n, r, p[None]),
                lambda: attn.kv_fork(k, k[..., :32], t, h, n, r, p), lambda: attn.kv_fork(k, k, t, h, n, r.cpu(), p),
                lambda: attn.kv_fork(k[:1].expand(6, 1, 16, 64), k, t, h, n, r, p)):
        with pytest.raises(RuntimeError):
            bad()


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------


def test_captured_pages(attn):
    # one captured step of taking pages, forking and giving back, replayed over changing data
    ps, P, W = 16, 64, 6
    k, v = (torch.randn(P, 2, ps, 64, device="cuda", dtype=F16) for _ in range(2))
    table, held, refs = torch.full((4, W), -1, dtype=torch.int32, device="cuda"), ints([0] * 4).cuda(), ints([0] * P).cuda()
    lens, parents = ints([0] * 4).cuda(), ints([0, 0, 1, 2]).cuda()
    kept, new = ints([[1, 3, -1]] * 4).cuda(), ints([4] * 4).cuda()

    def step():
        missing = attn.kv_resize(table, held, lens, refs, ps)
        after = attn.kv_compact(k, v, table, lens, kept, new)
        t, h, n, m = attn.kv_fork(k, v, table, held, after, refs, parents)
        table.copy_(t), held.copy_(h), lens.copy_(n)
        return missing, m

    saved = [x.clone() for x in (k, v, table, held, refs, lens)]
    step()
    for x, y in zip((k, v, table, held, refs, lens), saved):
        x.copy_(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    rng = random.Random(4)
    lists = [table.tolist(), held.tolist(), refs.tolist(), lens.tolist()]
    kr, vr = k.cpu(), v.cpu()
    for _ in range(12):
        now = [min(W * ps, n + rng.randint(4, 25)) for n in lists[3]]
        par = [rng.randrange(4) for _ in range(4)]
        path = [sorted(rng.sample(range(4), 2)) + [-1] for _ in range(4)]
        lens.copy_(ints(now)), parents.copy_(ints(par)), kept.copy_(ints(path))
        g.replay()
        t, h, r = lists[:3]
        m0 = resize_ref(t, h, now, r, ps)
        after = compact_ref(kr, vr, ints(t), ints(now), ints(path), ints([4] * 4))
        t, h, n, m1 = fork_ref(kr, vr, t, h, after.tolist(), r, par, ps)
        lists = [t, h, r, n]
        assert got[0].tolist() == m0 and got[1].tolist() == [m1]
        assert [table.tolist(), held.tolist(), refs.tolist(), lens.tolist()] == lists
        assert torch.equal(k.cpu(), kr) and torch.equal(v.cpu(), vr)
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_speculative_steps(attn, dtype, D):
    # prompts, then steps that draft trees, check them, keep a path and give back what the others held; each
    # sequence's tokens are also kept apart, in order
    B, Hq, Hkv, ps, S, P = 3, 4, 2, 16, 7, 64
    rng, g = random.Random(1), torch.Generator().manual_seed(2)
    kc, vc = (torch.full((P, Hkv, ps, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    table, held = torch.full((B, 12), -1, dtype=torch.int32, device="cuda"), ints([0] * B).cuda()
    refs = ints([0] * P).cuda()
    prompt = [20, 47, 33]
    lens = ints(prompt).cuda()
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    assert attn.kv_resize(table, held, lens, refs, ps).tolist() == [0] * B
    k, v = rand(B, Hkv, max(prompt), D), rand(B, Hkv, max(prompt), D)
    attn.kv_append(k.cuda(), v.cuda(), kc, vc, table, lens, new_lens=lens)
    dense = [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate(prompt)]
    for _ in range(6):
        new = [S, rng.randint(1, S), rng.randint(0, S)]
        n, tree = ints(new).cuda(), ints([random_tree(S, rng) for _ in range(B)])
        lens = lens + n
        assert attn.kv_resize(table, held, lens, refs, ps).tolist() == [0] * B
        k, v, q = rand(B, Hkv, S, D), rand(B, Hkv, S, D), rand(B, Hq, S, D)
        attn.kv_append(k.cuda(), v.cuda(), kc, vc, table, lens, new_lens=n)
        out = attn.attn_tree(q.cuda(), kc, vc, table, lens, tree.cuda(), n).cpu()
        kept = []
        for b in range(B):
            # the definition over the sequence's own tokens, as one page each
            kk, vv = (torch.cat([d, x[b, :, :new[b]]], 1) for d, x in zip(dense[b], (k, v)))
            row = torch.arange(1, dtype=torch.int32).reshape(1, 1)
            ref = tree_ref(q[b:b + 1], kk[None], vv[None], row, ints([kk.shape[1]]), tree[b:b + 1], ints(new[b:b + 1]))
            _close(out[b:b + 1], ref, kk.shape[1], dtype)
            path, s = [], rng.randrange(new[b]) if new[b] else -1
            while s >= 0:
                path.append(s)
                s = int(tree[b, s])
            path = path[::-1]
            at = dense[b][0].shape[1]
            dense[b] = tuple(x[:, list(range(at)) + [at + s for s in path]] for x in (kk, vv))
            kept.append(path + [-1] * (S - len(path)))
        lens = attn.kv_compact(kc, vc, table, lens, ints(kept).cuda(), n)
        attn.kv_resize(table, held, lens, refs, ps)
        assert lens.tolist() == [d[0].shape[1] for d in dense]
        assert int(refs.sum()) == sum(-(-x // ps) for x in lens.tolist())
    attn.kv_resize(table, held, lens * 0, refs, ps)
    assert int(refs.abs().sum()) == 0 and attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F32, 64)])
def test_beam_steps(attn, dtype, D):
    # two prompts, three beams each, attended to by attn_decode after each fork
    from paged_ref import decode_ref, decode_tolerance

    ps, P, W, Hq, Hkv = 16, 80, 8, 4, 2
    rng, g = random.Random(7), torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    kc, vc = (torch.full((P, Hkv, ps, D), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    table, held = torch.full((2, W), -1, dtype=torch.int32, device="cuda"), ints([0, 0]).cuda()
    refs, lens = ints([0] * P).cuda(), ints([37, 16]).cuda()
    attn.kv_resize(table, held, lens, refs, ps)
    k, v = rand(2, Hkv, 37, D), rand(2, Hkv, 37, D)
    attn.kv_append(k.cuda(), v.cuda(), kc, vc, table, lens, new_lens=lens)
    dense = [(k[b, :, :n], v[b, :, :n]) for b, n in enumerate((37, 16))]
    parents = [0, 0, 0, 1, 1, 1]
    for _ in range(20):
        table, held, lens, missing = attn.kv_fork(kc, vc, table, held, lens, refs, ints(parents).cuda())
        assert missing.tolist() == [0]
        dense = [dense[p] for p in parents]
        lens = lens + 1
        assert attn.kv_resize(table, held, lens, refs, ps).tolist() == [0] * 6
        k, v, q = rand(6, Hkv, 1, D), rand(6, Hkv, 1, D), rand(6, Hq, 1, D)
        attn.kv_append(k.cuda(), v.cuda(), kc, vc, table, lens)
        dense = [tuple(torch.cat([d, x[b]], 1) for d, x in zip(dense[b], (k, v))) for b in range(6)]
        out = attn.attn_decode(q.cuda(), kc, vc, table, lens).cpu()
        for b in range(6):
            kk, vv = dense[b]
            ref = decode_ref(q[b:b + 1], kk[None], vv[None], torch.zeros(1, 1, dtype=torch.int32), ints([kk.shape[1]]))
            tol = decode_tolerance(*ref[:3], kk.shape[1], D, dtype)
            assert ((out[b:b + 1].double() - ref[0]).abs() <= tol).all()
        parents = [rng.randrange(3) for _ in range(3)] + [3 + rng.randrange(3) for _ in range(3)]
    attn.kv_resize(table, held, lens * 0, refs, ps)
    assert int(refs.abs().sum()) == 0 and attn.check_status(0) == 0
