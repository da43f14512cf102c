"""Edges of the operators for drafted tokens and shared pages that the tests of
their forms (test_branches_gpu.py) leave out, against the definitions
(branches_ref.py)."""
import math
import random

import pytest
import torch

import test_branches_gpu
from branches_ref import compact_ref, tree_ref
from paged_ref import make_cache
from test_branches_gpu import BF16, F16, F32, _close, _q, _trees, ints

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# attn_tree
# ---------------------------------------------------------------------------

# Rows per kv head and type: the kernels up to 8, up to 128 and above, the plain one.
FORMS = [(BF16, 4, 2, 3), (F16, 8, 1, 1), (BF16, 8, 2, 9), (F16, 32, 2, 8), (BF16, 16, 1, 20), (F16, 4, 1, 70), (F32, 8, 2, 9)]


@pytest.mark.parametrize("dtype,Hq,Hkv,S", FORMS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps,W", [(16, 7), (24, 5), (8, 27), (7, 17), (100, 3)])
def test_tree_lengths_behind_the_table(attn, ps, W, D, dtype, Hq, Hkv, S):
    # tokens behind the table's last are left out: the first sequences' lengths pass it by much, by fewer tokens than
    # are drafted, by as many and by one, the last ones' do not
    cap = W * ps
    lens = [cap + 300, 2 ** 31 - 1, cap + S // 2 + 1, cap + S, cap + 1, cap, max(S, cap // 2)]
    B = len(lens)
    k, v, table, _ = make_cache([cap] * B, Hkv, D, ps, dtype, poison=False)
    q, par, ln = _q(B, Hq, S, D, dtype), _trees(B, S), ints(lens)
    # what an earlier call leaves in shared memory may not count
    bad = torch.full_like(v, math.nan).cuda()
    attn.attn_tree(q.cuda(), (100 * k).cuda(), bad, table.cuda(), ints([cap] * B).cuda(), par.cuda())
    assert attn.check_status(0) == 0
    for tree in (par, None):
        out = attn.attn_tree(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), None if tree is None else tree.cuda())
        assert attn.check_status(0) == 8
        _close(out, tree_ref(q, k, v, table, ln, tree), cap, dtype)


@pytest.mark.parametrize("lens,D,Hq,S,ps", [([300, 40], 128, 8, 9, 7), ([2000, 700], 64, 4, 30, 100), ([900], 256, 4, 12, 1),
                                            ([3000, 50], 128, 8, 50, 7), ([700], 64, 16, 40, 100), ([2500], 64, 8, 9, 7)])
def test_watchdog_where_copies_are_of_16_bytes(attn, lens, D, Hq, S, ps):
    # pages that no box of 8 rows divides: the first copy's arrival is not told
    test_branches_gpu.test_watchdog_fires_and_recovers(lens, D, Hq, S, ps)


# ---------------------------------------------------------------------------
# Page bounds after drafted tokens
# ---------------------------------------------------------------------------


def _check_bounds(bounds, k, table, lens):
    """Whether every key of every sequence lies within the bounds of its page."""
    ps = k.shape[2]
    bounds, k = bounds.cpu().float(), k.cpu().float()
    for b, n in enumerate(lens.tolist()):
        for t in range(n):
            p = int(table[b, t // ps])
            assert (bounds[p, :, 0] <= k[p, :, t % ps]).all() and (k[p, :, t % ps] <= bounds[p, :, 1]).all()


def _bounds_in(D, heads, pages, dtype, off):
    """Storage for bounds, 16-byte aligned or not."""
    x = torch.full((pages, heads, 2, D + off), math.nan, dtype=dtype, device="cuda")
    return x[..., off:]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,layout,off", [(64, 16, "hnd", 0), (128, 3, "nhd", 0), (256, 8, "hnd", 0), (80, 1, "hnd", 0),
                                             (33, 4, "hnd", 0), (64, 5, "hnd", 1)])
@pytest.mark.parametrize("S", [4, 40])
def test_compact_keeps_page_bounds(attn, S, D, ps, layout, off, dtype):
    # contexts that end anywhere in a page, drafted keys larger than those before, paths that end late in them
    H, rng = 2, random.Random(S + D)
    ctx = [15, 16, 0, 1, 31, 2 * ps, 3 * ps - 1]
    B, new = len(ctx), [S, S, S, max(1, S - 1), 2, S, S]
    lens = [c + n for c, n in zip(ctx, new)]
    k, v, table, _ = make_cache(lens, H, D, ps, dtype, layout=layout, poison=False)
    at, n = ints(ctx), ints(new)
    kc, vc, t = k.cuda(), v.cuda(), table.cuda()
    if layout == "nhd":
        kc, vc = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
    bounds = _bounds_in(D, H, k.shape[0], dtype, off)
    attn.kv_page_bounds(kc, t, at.cuda(), bounds=bounds)
    x = (_q(B, H, S, D, dtype, 5).float() * torch.arange(1, S + 1)[:, None]).to(dtype).cuda()
    attn.kv_append(x, x, kc, vc, t, ints(lens).cuda(), n.cuda(), bounds=bounds)
    paths = [[S - 1]] + [sorted(rng.sample(range(m), rng.randint(0, m))) for m in new[1:]]
    kept = ints([p + [-1] * (S - len(p)) for p in paths])
    want, k, v = bounds.cpu().clone(), kc.cpu().clone(), vc.cpu().clone()
    after = attn.kv_compact(kc, vc, t, ints(lens).cuda(), kept.cuda(), n.cuda(), bounds=bounds)
    # the definition: a page that a key comes to takes it in
    assert torch.equal(after.cpu(), compact_ref(k, v, table, ints(lens), kept, n))
    assert torch.equal(kc.cpu(), k) and torch.equal(vc.cpu(), v)
    for b in range(B):
        for i, a in enumerate(kept[b].tolist()):
            if a < 0:
                break
            p, r = int(table[b, (ctx[b] + i) // ps]), (ctx[b] + i) % ps
            want[p, :, 0] = torch.minimum(want[p, :, 0], k[p, :, r])
            want[p, :, 1] = torch.maximum(want[p, :, 1], k[p, :, r])
    assert torch.equal(bounds.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    _check_bounds(bounds, kc, table, after)
    assert attn.check_status(0) == 0


def test_selection_after_compaction_finds_the_moved_key(attn):
    # 15 tokens, four drafted across the page's end, the last of them accepted: it comes to page 0, whose keys are
    # small.  Selection of the pages that the next tokens read has to see it there.
    ps, D = 16, 64
    for dtype in (F16, BF16, F32):
        kc, vc = (torch.zeros(8, 1, ps, D, dtype=dtype, device="cuda") for _ in range(2))
        table = ints([[5, 2, 7, 0]]).cuda()
        bounds = torch.zeros(8, 1, 2, D, dtype=dtype, device="cuda")
        small = (_q(1, 1, 15, D, dtype) / 16).cuda()
        attn.kv_append(small, small, kc, vc, table, ints([15]).cuda(), bounds=bounds)
        drafts = (_q(1, 1, 4, D, dtype, 2) / 16).cuda()
        drafts[0, 0, 3] = 4
        attn.kv_append(drafts, drafts, kc, vc, table, ints([19]).cuda(), bounds=bounds)
        lens = attn.kv_compact(kc, vc, table, ints([19]).cuda(), ints([[3]]).cuda(), ints([4]).cuda(), bounds=bounds)
        assert lens.tolist() == [16] and bool((kc[5, 0, 15] == 4).all())
        more = (_q(1, 1, 40, D, dtype, 3) / 8).cuda()
        attn.kv_append(more, more, kc, vc, table, ints([56]).cuda(), bounds=bounds)
        q = torch.ones(1, 1, 1, D, dtype=dtype, device="cuda")
        assert attn.kv_select_pages(q, bounds, table, ints([56]).cuda(), ps, 2).tolist() == [[[0, 3]]]
        assert bool((bounds[5, 0, 1] == 4).all())


def test_compact_refuses_bounds_that_do_not_fit(attn):
    k = torch.zeros(6, 2, 16, 64, dtype=F16, device="cuda")
    t, n, kept, new = (ints(x).cuda() for x in ([[0, 1]], [20], [[1]], [4]))
    good = torch.zeros(6, 2, 2, 64, dtype=F16, device="cuda")
    for bad in (good[:5], good[:, :1], good[:, :, :1], good[..., :32], good.float(), good.cpu(), good[0],
                good[:1].expand(6, 2, 2, 64), good.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(RuntimeError, match="bounds"):
            attn.kv_compact(k, k.clone(), t, n, kept, new, bounds=bad)
    attn.kv_compact(k, k.clone(), t, n, kept, new, bounds=good)
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,layout,off", [(64, 16, "hnd", 0), (128, 3, "nhd", 0), (256, 64, "hnd", 0), (80, 2, "hnd", 0),
                                             (33, 4, "hnd", 0), (64, 5, "hnd", 1), (255, 7, "hnd", 0)])
def test_fork_keeps_page_bounds(attn, D, ps, layout, off, dtype):
    # beams of two prompts fork, append with bounds and fork again; free pages had other tokens before
    H, P = 3, 60
    rng = random.Random(D)
    kc, vc = (torch.zeros(P, H, ps, D, dtype=dtype, device="cuda") for _ in range(2))
    if layout == "nhd":
        kc, vc = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
    bounds = _bounds_in(D, H, P, dtype, off)
    bounds.zero_()  # too narrow for what will come
    lens, refs = ints([4 * ps - 1, ps + 1]).cuda(), ints([0] * P).cuda()
    table, held = torch.full((2, 9), -1, dtype=torch.int32, device="cuda"), ints([0, 0]).cuda()
    assert not attn.kv_resize(table, held, lens, refs, ps).any()
    x = _q(2, H, 4 * ps, D, dtype, 3).cuda()
    attn.kv_append(x, x, kc, vc, table, lens, new_lens=lens, bounds=bounds)
    parents = [0, 0, 1, 1, 0]
    for turn in range(2 * ps if ps < 8 else 4):
        was, free = bounds.clone(), refs == 0
        old, old_lens, src = table.cpu(), lens.tolist(), list(parents)
        table, held, lens, missing = attn.kv_fork(kc, vc, table, held, lens, refs, ints(parents).cuda(), bounds=bounds)
        assert missing.tolist() == [0]
        for i, a in enumerate(src):
            last = old_lens[a] // ps
            if old_lens[a] % ps and int(table[i, last]) != int(old[a, last]):
                p = int(table[i, last])
                assert bool(free[p]) and torch.equal(bounds[p], was[int(old[a, last])])
                was[p] = bounds[p]
        assert torch.equal(bounds.nan_to_num(7.0), was.nan_to_num(7.0))  # others stay as they are
        _check_bounds(bounds, kc, table, lens)
        lens = lens + 1
        assert not attn.kv_resize(table, held, lens, refs, ps).any()
        x = (turn + 2) * _q(5, H, 1, D, dtype, turn).cuda()
        attn.kv_append(x, x, kc, vc, table, lens, bounds=bounds)
        _check_bounds(bounds, kc, table, lens)
        parents = [rng.randrange(5) for _ in range(5)]
    # too few free pages: bounds stay as they are, too
    refs.clamp_(min=1)
    was = bounds.clone()
    if (lens % ps).any():
        *_, missing = attn.kv_fork(kc, vc, table, held, lens, refs, ints([0, 1, 2, 3, 4] * 2).cuda(), bounds=bounds)
        assert missing.item() > 0 and torch.equal(bounds.nan_to_num(7.0), was.nan_to_num(7.0))
    assert attn.check_status(0) == 0


def test_fork_refuses_bounds_that_do_not_fit(attn):
    k = torch.zeros(6, 2, 16, 64, dtype=F16, device="cuda")
    t, h, n, r, p = (ints(x).cuda() for x in ([[0, 1]], [2], [20], [1, 1, 0, 0, 0, 0], [0, 0]))
    good = torch.zeros(6, 2, 2, 64, dtype=F16, device="cuda")
    for bad in (good[:5], good[:, :1], good[:, :, :1], good[..., :32], good.float(), good.cpu(), good[0],
                good[:1].expand(6, 2, 2, 64)):
        with pytest.raises(RuntimeError, match="bounds"):
            attn.kv_fork(k, k.clone(), t, h, n, r, p, bounds=bad)
    assert r.tolist() == [1, 1, 0, 0, 0, 0] and attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 100), (F32, 128)])
def test_captured_steps_keep_page_bounds(attn, dtype, D):
    # one captured step (drafts, compaction, fork) over two layers kept as heads of one cache, replayed over changing
    # data on another stream; each layer's compaction is given its heads of cache and bounds
    ps, P, W, B, S, H = 8, 120, 9, 4, 6, 2
    kc, vc = (torch.zeros(P, 2 * H, ps, D, dtype=dtype, device="cuda") for _ in range(2))
    bounds = torch.zeros(P, 2 * H, 2, D, dtype=dtype, device="cuda")
    table, held, refs = torch.full((B, W), -1, dtype=torch.int32, device="cuda"), ints([0] * B).cuda(), ints([0] * P).cuda()
    lens, parents, kept = ints([0] * B).cuda(), ints([0] * B).cuda(), ints([[-1] * S] * B).cuda()
    x = torch.zeros(B, 2 * H, S, D, dtype=dtype, device="cuda")
    layers = [slice(0, H), slice(H, 2 * H)]

    def step():
        attn.kv_resize(table, held, lens + S, refs, ps)
        drafted = (held * ps - lens).clamp(0, S)
        lens.add_(drafted)
        after = None
        for h in layers:
            attn.kv_append(x[:, h], x[:, h], kc[:, h], vc[:, h], table, lens, drafted, bounds=bounds[:, h])
        for h in layers:
            after = attn.kv_compact(kc[:, h], vc[:, h], table, lens, kept, drafted, bounds=bounds[:, h])
        attn.kv_resize(table, held, after, refs, ps)
        t, n, l, missing = attn.kv_fork(kc, vc, table, held, after, refs, parents, bounds=bounds)
        table.copy_(t), held.copy_(n), lens.copy_(l)
        return missing

    side = torch.cuda.Stream()
    step()  # from nothing to nothing: no token is kept
    assert lens.tolist() == [0] * B and int(refs.sum()) == 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        missing = step()
    rng, want = random.Random(D), [0] * B
    for turn in range(10):
        par = [rng.randrange(B) for _ in range(B)]
        paths = [sorted(rng.sample(range(S), rng.randint(0, S - 1))) for _ in range(B)]
        want = [want[p] + len(paths[p]) for p in par]
        x.copy_((turn + 1) * _q(B, 2 * H, S, D, dtype, turn))
        parents.copy_(ints(par)), kept.copy_(ints([p + [-1] * (S - len(p)) for p in paths]))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert missing.tolist() == [0] and lens.tolist() == want
        _check_bounds(bounds, kc, table, lens)
    assert max(want) > ps and attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# Steps when pages run out
# ---------------------------------------------------------------------------


def _alone(cache, table, n):
    """The tokens of a sequence, in order: [Hkv, n, D]."""
    ps = cache.shape[2]
    t = torch.arange(n)
    return cache.cpu()[table.cpu()[t // ps].long(), :, t % ps].transpose(0, 1)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("Hq", [2, 8, 32])
def test_drafts_without_pages_leave_other_sequences_alone(attn, Hq, dtype):
    # sequence 0 has given a page back that sequence 1 holds by now, the pool is empty, and 0 drafts across its
    # page's end, 2 within its page: the documented step writes to what they hold, and nowhere else
    Hkv, ps, S, D = 2, 16, 7, 64
    kc, vc = (torch.zeros(5, Hkv, ps, D, dtype=dtype, device="cuda") for _ in range(2))
    table, held, refs = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), ints([0] * 3).cuda(), ints([0] * 5).cuda()
    assert not attn.kv_resize(table, held, ints([30, 0, 0]).cuda(), refs, ps).any()
    assert not attn.kv_resize(table, held, ints([13, 0, 0]).cuda(), refs, ps).any()
    lens = ints([13, 48, 3]).cuda()
    assert not attn.kv_resize(table, held, lens, refs, ps).any()
    assert int(table[0, 1]) == int(table[1, 0]) and held.tolist() == [1, 3, 1] and refs.tolist() == [1] * 5
    x = _q(3, Hkv, 48, D, dtype, 4)
    attn.kv_append(x.cuda(), x.neg().cuda(), kc, vc, table, lens, new_lens=lens)
    dense = [x[b, :, :n] for b, n in enumerate(lens.tolist())]

    lacks = attn.kv_resize(table, held, lens + S, refs, ps)
    drafted = (held * ps - lens).clamp(0, S)
    lens += drafted
    assert lacks.tolist() == [1, 1, 0] and drafted.tolist() == [3, 0, 7] and drafted.dtype == torch.int32
    x, q, par = _q(3, Hkv, S, D, dtype, 5), _q(3, Hq, S, D, dtype, 6), _trees(3, S)
    attn.kv_append(x.cuda(), x.neg().cuda(), kc, vc, table, lens, drafted)
    out = attn.attn_tree(q.cuda(), kc, vc, table, lens, par.cuda(), drafted)
    k = torch.zeros(3, Hkv, 48, D, dtype=dtype)
    for b, n in enumerate(drafted.tolist()):
        dense[b] = torch.cat([dense[b], x[b, :, :n]], 1)
        assert torch.equal(_alone(kc, table[b], int(lens[b])), dense[b])
        assert torch.equal(_alone(vc, table[b], int(lens[b])), dense[b].neg())
        k[b, :, :dense[b].shape[1]] = dense[b]
    _close(out, tree_ref(q, k, k.neg(), ints([[0], [1], [2]]), lens.cpu(), par, drafted.cpu()), 48, dtype)

    lens = attn.kv_compact(kc, vc, table, lens, ints([[1, -1], [-1, -1], [2, 5]]).cuda(), drafted)
    attn.kv_resize(table, held, lens, refs, ps)
    assert lens.tolist() == [14, 48, 5] and refs.tolist() == [1] * 5
    for b, at in ((0, list(range(13)) + [14]), (1, list(range(48))), (2, [0, 1, 2, 5, 8])):
        assert torch.equal(_alone(kc, table[b], int(lens[b])), dense[b][:, at])
    assert attn.check_status(0) == 0


def test_beams_without_pages_leave_other_sequences_alone(attn):
    # five pages, all held in the end: a beam at its page's end stays as it is while others go on
    Hkv, ps, D = 2, 4, 64
    kc, vc = (torch.zeros(5, Hkv, ps, D, dtype=BF16, device="cuda") for _ in range(2))
    table, held, refs = torch.full((1, 4), -1, dtype=torch.int32, device="cuda"), ints([0]).cuda(), ints([0] * 5).cuda()
    lens = ints([6]).cuda()
    assert not attn.kv_resize(table, held, lens, refs, ps).any()
    x = _q(1, Hkv, 6, D, BF16)
    attn.kv_append(x.cuda(), x.cuda(), kc, vc, table, lens)
    dense = [x[0]] * 3
    table, held, lens, missing = attn.kv_fork(kc, vc, table, held, lens, refs, ints([0, 0, 0]).cuda())
    assert missing.tolist() == [0]  # four pages are held now
    for turn in range(5):
        attn.kv_resize(table, held, lens + 1, refs, ps)
        grown = (held * ps - lens).clamp(0, 1)
        lens += grown
        assert grown.tolist() == ([1, 1, 1] if turn < 2 else [1, 0, 0])
        x, q = _q(3, Hkv, 1, D, BF16, turn), _q(3, 4, 1, D, BF16, turn + 9)
        attn.kv_append(x.cuda(), x.cuda(), kc, vc, table, lens, grown)
        out = attn.attn_decode(q.cuda(), kc, vc, table, lens)
        dense = [torch.cat([d, x[b]], 1) if g else d for b, (d, g) in enumerate(zip(dense, grown.tolist()))]
        for b in range(3):
            n = dense[b].shape[1]
            assert torch.equal(_alone(kc, table[b], int(lens[b])), dense[b])
            one = dense[b][None]
            _close(out[b:b + 1], tree_ref(q[b:b + 1], one, one, ints([[0]]), ints([n])), n, BF16)
    # a fork that lacks pages: the given tensors go on
    assert lens.tolist() == [11, 8, 8]
    new = attn.kv_fork(kc, vc, table, held, lens, refs, ints([0, 0, 0]).cuda())
    assert new[3].item() == 2 and not new[1].any() and not new[2].any()
    for b in range(3):
        assert torch.equal(_alone(kc, table[b], int(lens[b])), dense[b])
    assert attn.check_status(0) == 0
