"""The paged key-value cache operators at the ends of what their documentation
allows: the largest tables, scores and weights at the ends of their types'
ranges, work on several streams, captured runs."""
import math

import pytest
import torch

from paged_ref import bounds_ref, decode_bound, decode_ref, decode_tolerance, make_cache, select_ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

MAX_CAPACITY = 2 ** 31 - 65537  # tokens a block table may name


def _wide_table():
    """A block table of one sequence, pages of one token, as wide as allowed (8.6 GB): page 0 throughout."""
    return torch.zeros(1, MAX_CAPACITY, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D", [8, 5])
def test_append_at_the_end_of_the_widest_table(attn, D):
    # one new token where 131072 are offered: the pages of the others would lie behind position 2^31
    S = 131072
    table = _wide_table()
    table[0, -S:] = torch.arange(1, S + 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([MAX_CAPACITY], dtype=torch.int32, device="cuda")
    new = torch.ones(1, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, 1, S, D, device="cuda").to(F16) for _ in range(2))
    kc, vc = (torch.zeros(S + 2, 1, 1, D, dtype=F16, device="cuda") for _ in range(2))
    attn.kv_append(k, v, kc, vc, table, lens, new_lens=new)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[S, 0, 0], x[0, 0, 0])
        assert (c[:S] == 0).all() and (c[S + 1] == 0).all()
    attn.kv_append(k, v, kc, vc, table, lens)  # all of them new
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[1:S + 1, 0, 0], x[0, 0])
        assert (c[0] == 0).all() and (c[S + 1] == 0).all()
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("width", [4, 5000])
def test_select_of_the_longest_list(attn, width):
    # the list's length is the largest int: the pages there are, and -1 to its end
    top = 2 ** 31 - 1
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    lens = torch.tensor([3 * 16], dtype=torch.int32, device="cuda")
    bounds = torch.zeros(1, 1, 2, 8, dtype=F16, device="cuda")
    q = torch.ones(1, 1, 1, 8, dtype=F16, device="cuda")
    pages = attn.kv_select_pages(q, bounds, table, lens, 16, top)
    assert pages.shape == (1, 1, top)
    assert pages[0, 0, :4].tolist() == [0, 1, 2, -1]
    assert int(pages[0, 0, 3:].max()) == -1 and int(pages[0, 0, 3:].min()) == -1
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("lens", [[5000], [MAX_CAPACITY], [MAX_CAPACITY, 40, MAX_CAPACITY - 3]], ids=str)
def test_select_from_the_widest_table(attn, lens):
    # pages of one token; scores 0 but for a few pages up to the end (8 bytes of scratch memory a table entry)
    B, D = len(lens), 8
    table = _wide_table().expand(B, -1)
    places = [3, 17, 4990, 10 ** 9, MAX_CAPACITY - 40, MAX_CAPACITY - 5]
    table[0, places] = torch.arange(1, len(places) + 1, dtype=torch.int32, device="cuda")
    bounds = torch.zeros(len(places) + 1, 1, 2, D, dtype=F16, device="cuda")
    bounds[1:, 0, 1] = 1
    q = torch.ones(B, 1, 1, D, dtype=F16, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pages = attn.kv_select_pages(q, bounds, table, n, 1, 8)
    for b, length in enumerate(lens):
        best = [p for p in places if p < length - 1]
        rest = [p for p in range(20) if p not in best][:7 - len(best)]  # ties to the lower page
        assert pages[b, 0].tolist() == sorted(best + rest) + [length - 1]
    assert attn.check_status(0) == 0


def _q(B, Hq, D, dtype, seed=1):
    return torch.randn(B, Hq, 1, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 33])
@pytest.mark.parametrize("width", [None, 900])  # one launch, and runs over the whole grid
@pytest.mark.parametrize("lens", [[1, 16, 70, 0, 150], [3000, 5, 700, 0, 40]], ids=str)
def test_every_score_minus_infinity(attn, lens, width, D, dtype):
    # The formula's 0 / 0 where all of a sequence's scores are -inf, zeros only where there is no token; a part
    # of them weighs nothing.  Of five sequences: all -inf, the first 5 finite, all but the last -inf, empty,
    # all -inf for kv head 0 alone.
    k, v, table, ln = make_cache(lens, 2, D, 16, dtype, width=width)
    q = _q(5, 6, D, dtype).abs() + 0.1
    ps = 16
    for b, heads, gone in ((0, (0, 1), range(lens[0])), (1, (0, 1), range(5, lens[1])), (2, (0, 1), range(lens[2] - 1)),
                           (4, (0,), range(lens[4]))):
        for t in gone:
            k[int(table[b, t // ps]), list(heads), t % ps, D // 2] = -math.inf
    args = tuple(t.cuda() for t in (q, k, v, table, ln))
    o, absum, smax, w = decode_ref(q, k, v, table, ln)
    assert o[0].isnan().all() and o[4, :3].isnan().all() and not o[1:4].isnan().any() and not o[4, 3:].isnan().any()
    # the bound from the finite scores: what weighs nothing adds nothing
    k0 = k.masked_fill(k == -math.inf, 0.0)
    smax = decode_ref(q, k0, v, table, ln)[2]
    tol = decode_tolerance(o, absum, smax, max(lens), D, dtype)
    cap = table.shape[1] * ps
    weights = torch.zeros(5, 2, cap, device="cuda")
    pages = torch.arange(table.shape[1], dtype=torch.int32).expand(5, 2, -1).contiguous().cuda()
    for out in (attn.attn_decode(*args), attn.attn_decode(*args, pages=pages), attn.attn_decode(*args, weights=weights)):
        out = out.cpu().double()
        assert torch.equal(out.isnan(), o.isnan())
        ok = ~o.isnan()
        assert ((out - o).abs() <= tol)[ok].all()
        assert (out[3] == 0).all()
    got = weights.cpu()
    assert torch.equal(got.isnan(), w.isnan())
    # a weight's bound, as in the tests of the weights: a score's exponential and the denominator, summed over 3 heads
    rel = 2 * ((D + 4) * 2.0 ** -23 * float(smax.max()) + 2.0 ** -21 + max(lens) * 2.0 ** -23) + 4 * 2.0 ** -24
    ok = ~w.isnan()
    assert ((got.double() - w).abs() <= rel * w)[ok].all()
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128), (BF16, 256), (F32, 64), (F16, 33)])
@pytest.mark.parametrize("width", [None, 900])
def test_weights_of_absent_tokens_beside_nan(attn, dtype, D, width):
    # a sequence whose softmax is NaN: its tokens' weights are NaN, those of tokens in a page outside the cache stay
    k, v, table, ln = make_cache([100, 100], 2, D, 16, dtype, width=width)
    q = _q(2, 6, D, dtype)
    k[int(table[0, 1]), 0, 7, 3] = math.nan
    table[0, 3], table[1, 3] = -1, 2 ** 30
    start = torch.rand(2, 2, table.shape[1] * 16, generator=torch.Generator().manual_seed(4))
    w = start.cuda()
    attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), weights=w)
    w = w.cpu()
    live = torch.ones(100, dtype=torch.bool)
    live[48:64] = False
    assert w[0, 0, :100][live].isnan().all()
    assert torch.equal(w[0, 0, 48:64], start[0, 0, 48:64])
    assert (w[0, 1, :100][live] > start[0, 1, :100][live]).any() and not w[0, 1].isnan().any()
    assert torch.equal(w[1, :, 48:64], start[1, :, 48:64]) and torch.equal(w[:, :, 100:], start[:, :, 100:])
    assert attn.check_status(0) == 8


@pytest.mark.parametrize("octaves", [12.0, 20.5, 24.625, 25.125, 28.0])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256, 33])
@pytest.mark.parametrize("L,width", [(150, None), (150, 900), (3000, None)])
def test_small_weights_beside_a_large_one(attn, L, width, D, dtype, octaves):
    # Every eighth token takes all the weight and has a zero V row; the others, `octaves` powers of two below,
    # make up the whole output.  Scores are exact: q is one column of K.
    k, v, table, ln = make_cache([L, L - 9], 2, D, 16, dtype, width=width)
    ps = 16
    for b in range(2):
        t = torch.arange(int(ln[b]))
        page, row = table[b, t // ps].long(), t % ps
        sink = t % 8 == (3 if b else 0)
        k[page, :, row, 0] = torch.where(sink, 0.0, -octaves).to(dtype)[:, None]
        x = (v[page, :, row].abs().clamp(max=3) + 1) * 2.0 ** 12
        v[page, :, row] = torch.where(sink[:, None, None], 0.0, x).to(dtype)
    q = torch.zeros(2, 6, 1, D).to(dtype)
    q[..., 0] = 1
    scale = math.log(2.0)
    o, absum, _, w = decode_ref(q, k, v, table, ln, scale)
    smax = torch.full((2, 6, 1, 1), octaves * scale, dtype=torch.float64)
    tol = decode_bound(o, absum, smax, L, D, dtype)
    assert (tol < 0.02 * o.abs()).all()  # the outputs are of such weights alone
    args = tuple(t.cuda() for t in (q, k, v, table, ln))
    weights = torch.zeros(2, 2, table.shape[1] * ps, device="cuda")
    for out in (attn.attn_decode(*args, scale=scale), attn.attn_decode(*args, scale=scale, weights=weights)):
        err = (out.cpu().double() - o).abs()
        assert (err <= tol).all(), f"error {(err / tol).max():.2f} of the bound"
    rel = 2 * ((D + 4) * 2.0 ** -23 * octaves * scale + 2.0 ** -21 + L * 2.0 ** -23) + 4 * 2.0 ** -24
    assert ((weights.cpu().double() - w).abs() <= rel * w).all()
    assert attn.check_status(0) == 0


def test_status_covers_every_stream(attn):
    # a bad page met late on another stream is reported by the check that follows the call
    k, v, table, ln = make_cache([100], 2, 64, 16, BF16)
    table[0, 3] = -7
    args = tuple(t.cuda() for t in (_q(1, 4, 64, BF16), k, v, table, ln))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # kernels loaded and memory at hand, which may synchronise
        attn.attn_decode(*args)
        torch.cuda._sleep(1000)
    side.synchronize()
    assert attn.check_status(0) == 8
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s of work before it
        attn.attn_decode(*args)
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0


def _marked_case(D, n, dtype, trend):
    """One sequence whose every 64 tokens add the same amount to one column of the output, at scores whose
    maximum rises (or falls) along the sequence: q picks column 0 of K, the score in powers of two."""
    k, v, table, ln = make_cache([n], 1, D, 16, dtype)
    t = torch.arange(n)
    tile = t // 64
    level = ((tile * 5) % 4 + 12 * (tile if trend > 0 else int(tile[-1]) - tile) // int(tile[-1])).double() - 8
    page, row = table[0, t // 16].long(), t % 16
    k[page, 0, row] = 0
    k[page, 0, row, 0] = level.to(dtype)
    v[page, 0, row] = 0
    v[page, 0, row, tile % D] = (2.0 ** -level).to(dtype)
    q = torch.zeros(1, 4, 1, D).to(dtype)
    q[..., 0] = 1
    return (q, k, v, table, ln), tile, level


@pytest.mark.parametrize("trend", [1, -1])
@pytest.mark.parametrize("D,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16), (256, BF16), (64, F32), (100, F16)])
def test_every_part_of_a_long_sequence_counts(attn, D, dtype, trend):
    # one sequence over every CTA of the grid, more parts than the join takes in one turn: a tile of 64 tokens that
    # is missing, counted twice or scaled by a power of two would be beyond the bound
    n, scale = 40001, math.log(2.0)
    case, tile, level = _marked_case(D, n, dtype, trend)
    o, absum, _, w = decode_ref(*case, scale)
    tol = decode_bound(o, absum, torch.full((1, 4, 1, 1), 8 * scale, dtype=torch.float64), n, D, dtype)
    part = torch.zeros(int(tile[-1]) + 1, dtype=torch.float64).index_add_(0, tile, torch.exp2(level) * torch.exp2(-level))
    part = part / torch.exp2(level).sum()  # what a tile adds to its column
    column = torch.arange(len(part)) % D
    full = tile.bincount() == 64
    assert (part[full] > 2 * tol[0, 0, 0, column[full]]).all()
    args = tuple(t.cuda() for t in case)
    weights = torch.zeros(1, 1, case[3].shape[1] * 16, device="cuda")
    out = attn.attn_decode(*args, scale=scale)
    for got in (out, attn.attn_decode(*args, scale=scale, weights=weights)):
        err = (got.cpu().double() - o).abs()
        assert (err <= tol).all(), f"error {(err / tol).max():.2f} of the bound"
    rel = 2 * ((D + 4) * 2.0 ** -23 * 8 * scale + 2.0 ** -21 + n * 2.0 ** -23) + 5 * 2.0 ** -24
    assert ((weights.cpu().double() - w).abs() <= rel * w).all()
    assert torch.equal(out, attn.attn_decode(*args, scale=scale))
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype,D,ps", [(BF16, 128, 16), (F16, 64, 24), (F32, 33, 8)])
def test_captured_bounds_and_selection_follow_lengths_and_pages(attn, dtype, D, ps):
    # bounds, selection and the attention over it, captured and replayed on other keys, lengths and pages
    W, top = 60, 5
    k, v, table, ln = make_cache([50, 0, 300, 3], 2, D, ps, dtype, width=W, poison=False, spare=240)
    dk, dv, dt, dl = (t.cuda() for t in (k, v, table, ln))
    q = _q(4, 8, D, dtype)
    dq = q.cuda()
    kept_bounds = torch.zeros(k.shape[0], 2, 2, D, dtype=dtype, device="cuda")

    def step():
        fresh = attn.kv_page_bounds(dk, dt, dl)
        attn.kv_page_bounds(dk, dt, dl, bounds=kept_bounds)
        pages = attn.kv_select_pages(dq, fresh, dt, dl, ps, top)
        return fresh, pages, attn.attn_decode(dq, dk, dv, dt, dl, pages=pages)

    dt.copy_(torch.arange(4 * W, dtype=torch.int32).reshape(4, W))
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fresh, pages, out = step()
    kept = torch.zeros(kept_bounds.shape, dtype=dtype)
    for i, new in enumerate(([50, 0, 300, 3], [1, W * ps, 5, 0], [300, 301, 302, 303])):
        gen = torch.Generator().manual_seed(i)
        k = torch.randn(k.shape, generator=gen).to(dtype)
        q = torch.randn(q.shape, generator=gen).to(dtype)
        ln = torch.tensor(new, dtype=torch.int32)
        table = torch.randperm(k.shape[0], generator=gen)[:4 * W].reshape(4, W).to(torch.int32)
        kept = torch.randn(kept.shape, generator=gen).to(dtype)
        for d, t in ((dk, k), (dq, q), (dl, ln), (dt, table), (kept_bounds, kept)):
            d.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        want = bounds_ref(k, table, ln, torch.zeros(kept.shape, dtype=dtype))
        assert torch.equal(fresh.cpu(), want)
        assert torch.equal(kept_bounds.cpu(), bounds_ref(k, table, ln, kept.clone()))
        chosen = select_ref(q, want, table, ln, ps, top)
        assert torch.equal(pages.cpu(), chosen)
        o, absum, smax, _ = decode_ref(q, k, v, table, ln, pages=chosen)
        assert ((out.cpu().double() - o).abs() <= decode_bound(o, absum, smax, top * ps, D, dtype, vmax=8.0)).all()
    assert attn.check_status(0) == 0


def test_table_without_pages(attn):
    # a block table of no entries names no token: weights of no elements go with it
    k = torch.zeros(4, 2, 16, 64, dtype=F16, device="cuda")
    t, n = torch.zeros(3, 0, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 2, 0, device="cuda")
    q = torch.ones(3, 4, 1, 64, dtype=F16, device="cuda")
    assert (attn.attn_decode(q, k, k, t, n, weights=w) == 0).all()
    new = torch.arange(3, dtype=torch.int32, device="cuda")[:, None]
    lens, new_w, kept = attn.kv_evict(k, k.clone(), t, n, w, new, 5, recent=2)
    assert lens.tolist() == [0, 0, 0] and (new_w == 0).all() and (kept == -1).all()
    assert new_w.shape == (3, 2, 16) and kept.shape == (3, 2, 5)
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_decode_and_evict_over_the_widest_table(attn, dtype):
    # 2^31 - 65537 tokens in pages of one, the same page but for the last, whose score makes it weigh as much
    # as 2^31 others.  All sums are of equal powers of two and exact up to the join of at most 600 parts.
    n, D = MAX_CAPACITY, 8
    table = _wide_table()
    table[0, -1] = 1
    k, v = torch.zeros(8, 1, 1, D, dtype=dtype), torch.zeros(8, 1, 1, D, dtype=dtype)
    k[1, 0, 0, 0] = 31
    v[0], v[1] = 1, 3
    q = torch.zeros(1, 1, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 1
    k, v = k.cuda(), v.cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    total = n - 1 + 2.0 ** 31
    rel = 600 * 2.0 ** -24 + 2.0 ** -20
    want = (n - 1 + 3 * 2.0 ** 31) / total
    out = attn.attn_decode(q, k, v, table, lens, scale=math.log(2.0))
    assert ((out.double() - want).abs() <= want * (rel + torch.finfo(dtype).eps / 2)).all()
    w = torch.zeros(1, 1, n, device="cuda")
    assert torch.equal(attn.attn_decode(q, k, v, table, lens, scale=math.log(2.0), weights=w), out)
    # log2 of the sum, 32, is off by half a step of 2^-18
    rel = rel + 2.0 ** -18
    assert abs(float(w[0, 0, -1]) * total / 2.0 ** 31 - 1) <= rel
    lo, hi = float(w[0, 0, :-1].min()), float(w[0, 0, :-1].max())
    assert lo == hi and abs(lo * total - 1) <= rel
    w[0, 0, n - 100] = 2
    w[0, 0, 5] = 1
    new = torch.arange(2, 7, dtype=torch.int32, device="cuda")[None]
    new_lens, new_w, kept = attn.kv_evict(k, v, table, lens, w, new, 5, recent=2)
    # the two largest, of the others, all equal, the lowest, and the last two
    assert kept[0, 0].tolist() == [0, 5, n - 100, n - 2, n - 1] and new_lens.tolist() == [5]
    assert torch.equal(new_w[0, 0], w[0, 0, kept[0, 0].long()])
    assert (k[2:6] == k[0]).all() and torch.equal(k[6], k[1]) and torch.equal(v[6], v[1]) and (k[7] == 0).all()
    bounds = attn.kv_page_bounds(k, table, lens)
    assert torch.equal(bounds[:2, :, 0], k[:2, :, 0]) and torch.equal(bounds[:2, :, 1], k[:2, :, 0])
    assert attn.check_status(0) == 0
