"""The paged key-value cache operators against their definitions in 64 bits
(paged_ref.py): attention of one new token, the cache's writer, page bounds,
page selection and eviction."""
import ctypes
import math
import os

import pytest
import torch

import rocm_attn_b200
from paged_ref import (bounds_ref, decode_ref, decode_tolerance, evict_ref, make_cache, rows, select_ref)

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _q(B, Hq, D, dtype, seed=1):
    return torch.randn(B, Hq, 1, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _close(out, ref, n, dtype):
    o, absum, smax, _ = ref
    assert out.dtype == dtype
    err = (out.cpu().double() - o).abs()
    tol = decode_tolerance(o, absum, smax, n, o.shape[3], dtype)
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"error {(err / tol).max():.2f} of the bound"


def _decode(attn, lens, Hq, Hkv, D, ps, dtype, layout="hnd", seed=0, scale=None, width=None):
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=seed, layout=layout, width=width)
    q = _q(len(lens), Hq, D, dtype, seed + 1)
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), scale=scale)
    assert out.shape == q.shape
    _close(out, decode_ref(q, k, v, table, ln, scale), max(lens), dtype)
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2, 15, 16, 17, 0], [63, 64, 65, 127, 128, 129], [700, 3, 0, 1300],
                                  [0, 0]], ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_decode_lengths(attn, lens, D, dtype):
    _decode(attn, lens, 8, 2, D, 16, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [1, 5, 8, 16, 24, 33, 40, 72, 80, 96, 100, 136, 192, 250, 256])
def test_decode_head_dims(attn, D, dtype):
    _decode(attn, [200, 41], 6, 2, D, 16, dtype, seed=D)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (2, 1), (9, 3), (7, 1), (16, 2), (16, 1), (17, 1), (80, 2), (64, 1)])
def test_decode_groups(attn, Hq, Hkv, dtype):
    _decode(attn, [150, 333], Hq, Hkv, 64, 16, dtype, seed=Hq)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("ps", [1, 2, 3, 7, 8, 24, 32, 100, 128, 300, 1024])
def test_decode_page_sizes(attn, ps, dtype):
    _decode(attn, [257, 5, 130], 4, 2, 128, ps, dtype, seed=ps, layout="nhd" if ps % 2 else "hnd")


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_decode_many_sequences(attn, dtype):
    # more sequences than threads of a CTA, most short, some empty, one long
    lens = [(i * 7) % 23 for i in range(300)]
    lens[211] = 1500
    _decode(attn, lens, 2, 1, 64, 8, dtype)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (256, BF16), (64, F32)])
def test_decode_long_split(attn, D, dtype):
    # one sequence over every CTA of the grid
    _decode(attn, [40001], 4, 1, D, 16, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,Hkv,L", [(1, 1, 64), (1, 2, 128), (2, 1, 300), (1, 8, 517), (5, 8, 1000), (32, 8, 100),
                                     (40, 16, 64)])
@pytest.mark.parametrize("width", [None, 700])
def test_decode_short_caches_and_wide_tables(attn, B, Hkv, L, width, dtype):
    # few tiles by the table's width (one launch, clusters of each size) and many, by the same lengths
    lens = [max(0, L - 37 * b) for b in range(B)]
    _decode(attn, lens, 4 * Hkv, Hkv, 128, 16, dtype, seed=B, width=width)


def test_decode_masked_tail_of_nan(attn):
    # a chunk whose later 16 tokens are absent, in every position of the tile, with NaN behind them
    for n in range(1, 140, 3):
        _decode(attn, [n], 2, 1, 64, 32, BF16, seed=n)
        _decode(attn, [n], 2, 1, 64, 48, F16, seed=n, width=300)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_decode_unaligned_and_mixed_strides(attn, dtype):
    # rows that are not 16-byte aligned, K and V of different strides, strided q
    k, v, table, ln = make_cache([77, 200], 2, 64, 16, dtype)
    q = _q(2, 4, 64, dtype)
    ref = decode_ref(q, k, v, table, ln)
    kx = torch.zeros(*k.shape[:3], 67, dtype=dtype, device="cuda")[..., 1:65]
    kx.copy_(k)
    vx = torch.zeros(k.shape[2], k.shape[0], k.shape[1], 64, dtype=dtype, device="cuda").permute(1, 2, 0, 3)
    vx.copy_(v)
    qx = torch.zeros(2, 1, 4, 64, dtype=dtype, device="cuda").transpose(1, 2)
    qx.copy_(q)
    tx = torch.zeros(2, 2 * table.shape[1], dtype=torch.int32, device="cuda")[:, ::2]
    tx.copy_(table)
    for kk in (kx, k.cuda()):
        _close(attn.attn_decode(qx, kk, vx, tx, ln.cuda()), ref, 200, dtype)
    wide = torch.zeros(2, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    _close(attn.attn_decode(qx, kx, vx, wide[:, :table.shape[1]], ln.cuda()), ref, 200, dtype)
    # a head dim that is not the innermost is copied for q
    qt = q.cuda().transpose(1, 3).contiguous().transpose(1, 3)
    _close(attn.attn_decode(qt, kx, vx, wide[:, :table.shape[1]], ln.cuda()), ref, 200, dtype)


def test_decode_scale_and_extreme_scores(attn):
    _decode(attn, [100, 50], 4, 4, 64, 16, F16, scale=0.7)
    k, v, table, ln = make_cache([90], 1, 64, 16, F16)
    k[k.isfinite()] *= 200  # scores of tens of thousands: one token takes all
    q = _q(1, 4, 64, F16) * 100
    o = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda()).cpu().double()
    best = (q[0, :, 0].double() @ rows(k, table[0], 0, range(90)).double().t()).argmax(1)
    assert torch.equal(o[0, :, 0], rows(v, table[0], 0, best).double())


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_decode_nan_and_inf_in_tokens(attn, dtype):
    # a NaN key makes its head's rows NaN, as the formula does, and no other; -inf scores weigh nothing
    k, v, table, ln = make_cache([70, 70, 70], 2, 64, 16, dtype)
    q = _q(3, 4, 64, dtype).abs() + 0.1
    k[int(table[0, 2]), 1, 3, 5] = math.nan
    k[int(table[1, 4]), 0, 2] = -math.inf
    k[int(table[2, 0]), 0, 0] = math.inf
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda()).cpu()
    ref = decode_ref(q, k, v, table, ln)
    assert torch.equal(out.isnan(), ref[0].isnan())
    assert ref[0][0, 2:].isnan().all() and ref[0][2, :2].isnan().all() and not ref[0][1].isnan().any()
    k2 = k.clone()
    k2[int(table[0, 2]), 1, 3, 5] = 0
    k2[int(table[2, 0]), 0, 0] = 0
    k2[int(table[1, 4]), 0, 2] = 0
    r2 = decode_ref(q, k2, v, table, ln, drop=lambda b, t: b == 1 and t == 66)
    # head 0 of sequence 1 without its token 66
    err = (out[1, :2].double() - r2[0][1, :2]).abs()
    assert (err <= decode_tolerance(*(x[1, :2] for x in r2[:3]), 70, 64, dtype)).all()


def test_decode_bad_pages_and_lengths(attn):
    # entries outside the cache count as absent and are reported once
    k, v, table, ln = make_cache([100, 60, 40], 2, 64, 16, BF16)
    q = _q(3, 4, 64, BF16)
    table[0, 3], table[2, 0], table[2, 1], table[2, 2] = -7, k.shape[0], 2 ** 31 - 1, -2 ** 31
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda())
    ref = decode_ref(q, k, v, table.clamp(0, k.shape[0] - 1), ln,
                     drop=lambda b, t: (b == 0 and t // 16 == 3) or b == 2)
    _close(out, ref, 100, BF16)
    assert (out[2] == 0).all()
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0
    # a length beyond the table ends with the table
    k, v, table, ln = make_cache([96, 30], 2, 64, 16, F32)
    q = _q(2, 4, 64, F32)
    far = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32)
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), far.cuda())
    _close(out, decode_ref(q, k, v, table, torch.tensor([96, 0])), 96, F32)
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0


def test_decode_empty_calls(attn):
    for B, W, P in ((0, 4, 4), (2, 0, 4), (2, 3, 0)):
        k = torch.zeros(P, 2, 16, 64, dtype=F16, device="cuda")
        table = torch.zeros(B, W, dtype=torch.int32, device="cuda")
        out = attn.attn_decode(torch.ones(B, 4, 1, 64, dtype=F16, device="cuda"), k, k, table,
                               torch.zeros(B, dtype=torch.int32, device="cuda"))
        assert out.shape == (B, 4, 1, 64) and (out == 0).all()
    assert attn.check_status(0) == 0


def test_decode_offsets_past_32_bits(attn):
    # the last pages of a cache of more than 2^32 bytes and 2^31 elements
    P = 2 ** 31 // (256 * 128) + 64
    cache = torch.zeros(P, 1, 256, 128, dtype=BF16, device="cuda")
    k, v, table, ln = make_cache([700], 1, 128, 256, BF16, spare=0)
    cache[P - 3:] = k.cuda()
    table[:, :3] += P - 3
    q = _q(1, 4, 128, BF16)
    out = attn.attn_decode(q.cuda(), cache, cache, table.cuda(), ln.cuda())
    _close(out, decode_ref(q, k, k, table - (P - 3), ln), 700, BF16)
    new = torch.randn(1, 1, 1, 128).to(BF16)
    before = cache[P - 3:].clone()
    attn.kv_append(new.cuda(), new.cuda(), cache, cache, table.cuda(), ln.cuda())
    changed = (cache[P - 3:] != before) & ~(cache[P - 3:].isnan() & before.isnan())
    where = changed.nonzero()[:, :3].unique(dim=0)
    page = int(table[0, 699 // 256]) - (P - 3)
    assert where.tolist() == [[page, 0, 699 % 256]]
    assert torch.equal(cache[P - 3 + page, 0, 699 % 256], new[0, 0, 0].cuda())


# ---------------------------------------------------------------------------
# attention weights
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lens,Hq,Hkv,D,ps", [([1, 0, 33, 500], 8, 2, 64, 16), ([4000], 4, 1, 128, 32),
                                              ([130, 257], 34, 1, 40, 7), ([65, 300], 6, 2, 33, 16),
                                              ([200, 100], 8, 8, 256, 16)])
def test_decode_weights(attn, lens, Hq, Hkv, D, ps, dtype):
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=3)
    B, cap = len(lens), table.shape[1] * ps
    q = _q(B, Hq, D, dtype)
    start = torch.rand(B, Hkv, cap + 9, generator=torch.Generator().manual_seed(5))
    w = torch.zeros(Hkv, B, cap + 9, device="cuda").transpose(0, 1)
    w.copy_(start)
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), weights=w)
    o, absum, smax, ref = decode_ref(q, k, v, table, ln)
    _close(out, (o, absum, smax, None), max(lens), dtype)
    assert torch.equal(out, attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda()))
    # each weight is off as a score's exponential and the denominator are (see decode_tolerance); the sum
    # over g heads and the addition round g + 1 times
    rel = 2 * ((D + 4) * 2.0 ** -23 * float(smax.max()) + 2.0 ** -21 + max(lens) * 2.0 ** -23)
    g = Hq // Hkv
    want = start.double()
    want[:, :, :cap] += ref
    tol = torch.zeros_like(want)
    tol[:, :, :cap] = rel * ref
    tol += (g + 1) * 2.0 ** -24 * want
    got = w.cpu().double()
    assert ((got - want).abs() <= tol).all()
    for b, n in enumerate(lens):  # behind the tokens nothing changes
        assert torch.equal(w[b, :, n:].cpu(), start[b, :, n:])
    assert attn.check_status(0) == 0


def test_decode_weights_of_absent_tokens(attn):
    k, v, table, ln = make_cache([100, 20], 1, 64, 16, F16)
    table[0, 2], table[1, 0], table[1, 1] = -1, -1, -1
    w = torch.ones(2, 1, table.shape[1] * 16, device="cuda")
    q = _q(2, 2, 64, F16)
    attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), weights=w)
    assert (w[0, 0, 32:48] == 1).all() and (w[1] == 1).all() and (w[0, 0, :32] > 1).all()
    assert abs(float(w[0].sum()) - table.shape[1] * 16 - 2) < 1e-3
    assert attn.check_status(0) == 8


# ---------------------------------------------------------------------------
# attention over listed pages
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps", [(64, 16), (128, 24), (40, 5), (33, 16), (256, 32)])
def test_decode_listed_pages(attn, D, ps, dtype):
    lens = [ps * 9 + 3, 1, 0, ps * 4, ps * 20 - 1]
    k, v, table, ln = make_cache(lens, 2, D, ps, dtype, seed=D)
    g = torch.Generator().manual_seed(D)
    pages = torch.randint(-2, table.shape[1] + 2, (5, 2, 7), generator=g).to(torch.int32)
    pages[0, 0] = torch.tensor([3, 3, 0, 9, -1, 2 ** 31 - 1, -2 ** 31])  # one twice
    pages[4, 1] = -1                                       # none at all
    q = _q(5, 8, D, dtype)
    out = attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), pages=pages.cuda())
    _close(out, decode_ref(q, k, v, table, ln, pages=pages), 7 * ps, dtype)
    assert (out[4, 4:] == 0).all()
    none = torch.zeros(5, 2, 0, dtype=torch.int32, device="cuda")
    assert (attn.attn_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), ln.cuda(), pages=none) == 0).all()
    assert attn.check_status(0) == 0


def test_listing_every_page_is_the_whole(attn):
    lens = [300, 17, 1000]
    k, v, table, ln = make_cache(lens, 2, 128, 16, BF16)
    q = _q(3, 8, 128, BF16).cuda()
    args = (q, k.cuda(), v.cuda(), table.cuda(), ln.cuda())
    pages = torch.arange(table.shape[1], dtype=torch.int32, device="cuda").expand(3, 2, -1)
    _close(attn.attn_decode(*args, pages=pages), decode_ref(q.cpu(), k, v, table, ln), 1000, BF16)


# ---------------------------------------------------------------------------
# append and bounds
# ---------------------------------------------------------------------------


def _same(a, b):
    a, b = a.cpu(), b.cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,Hkv", [(128, 16, 8), (64, 24, 3), (40, 1, 2), (33, 7, 2), (256, 128, 1), (250, 16, 2),
                                      (8, 64, 33)])
@pytest.mark.parametrize("S", [1, 5, 90])
def test_append(attn, S, D, ps, Hkv, dtype):
    new = [S, min(S, 3), 0, S, 1, S]
    lens = [S, S + 2 * ps + 1, 40, S + ps // 2, 0, S + ps]
    layout = "nhd" if S == 5 else "hnd"
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=S, layout=layout)
    g = torch.Generator().manual_seed(D)
    x, y = (torch.randn(6, S, Hkv, D, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    bounds = torch.randn(k.shape[0], Hkv, 2, D, generator=g).to(dtype)
    want_k, want_v, want_b = k.clone(), v.clone(), bounds.clone()
    for with_new in (True, False):
        got_k, got_v, got_b = k.cuda(), v.cuda(), bounds.cuda()
        for b in range(6):
            n = new[b] if with_new else S
            for s in range(n):
                t = lens[b] - n + s
                if t < 0:
                    continue
                p, r = int(table[b, t // ps]), t % ps
                want_k[p, :, r], want_v[p, :, r] = x[b, :, s], y[b, :, s]
                lo, hi = (x[b, :, s], x[b, :, s]) if r == 0 else (torch.minimum(want_b[p, :, 0], x[b, :, s]),
                                                                  torch.maximum(want_b[p, :, 1], x[b, :, s]))
                want_b[p, :, 0], want_b[p, :, 1] = lo, hi
        nl = torch.tensor(new, dtype=torch.int32, device="cuda") if with_new else None
        args = (x.cuda(), y.cuda(), got_k, got_v, table.cuda(), ln.cuda())
        attn.kv_append(*args, new_lens=nl, bounds=got_b)
        assert _same(got_k, want_k) and _same(got_v, want_v) and _same(got_b, want_b)
        got_k, got_v = k.cuda(), v.cuda()
        attn.kv_append(args[0], args[1], got_k, got_v, args[4], args[5], new_lens=nl)
        assert _same(got_k, want_k) and _same(got_v, want_v)
        want_k, want_v, want_b = k.clone(), v.clone(), bounds.clone()
    assert attn.check_status(0) == 0


def test_append_out_of_range(attn):
    k, v, table, ln = make_cache([40, 33, 20, 16], 2, 64, 16, F16)
    x = torch.randn(4, 2, 4, 64).to(F16)
    table[1, 2] = 10 ** 6  # position 32 of sequence 1 has no page
    far = torch.tensor([40, 33, 20, 50], dtype=torch.int32)  # sequence 3: 48.. lies beyond the table (3 pages)
    table[3, 1:] = table[0, 1:]  # pages 1 and 2 of sequence 3 are shared, so only position 46, 47 would be written
    gk, gv = k.cuda(), v.cuda()
    attn.kv_append(x.cuda(), x.cuda(), gk, gv, table.cuda(), far.cuda())
    for b, n in enumerate([40, 33, 20, 50]):
        for s in range(4):
            t = n - 4 + s
            if t < 48 and not (b == 1 and t == 32):
                k[int(table[b, t // 16]), :, t % 16] = x[b, :, s]
    assert _same(gk, k)
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0
    # more new tokens than there are
    nl = torch.tensor([9, -3, 4, 0], dtype=torch.int32, device="cuda")
    gk = k.cuda()
    attn.kv_append(x.cuda(), x.cuda(), gk, gv, table.cuda(), torch.tensor([40, 33, 20, 16], dtype=torch.int32, device="cuda"),
                   new_lens=nl)
    assert _same(gk[int(table[0, 2]), :, 4:8], x[0])
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,Hkv", [(128, 16, 8), (64, 24, 3), (40, 1, 2), (33, 7, 2), (256, 128, 1), (250, 300, 2)])
def test_page_bounds(attn, D, ps, Hkv, dtype):
    lens = [3 * ps, 1, 0, 2 * ps - 1, 5 * ps + 2]
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=D, layout="nhd" if ps == 24 else "hnd")
    k[int(table[0, 0]), 0, 0, 0] = math.nan          # a NaN key shows in its bound
    k[int(table[4, 1]), 0, 0, 0] = math.inf
    got = attn.kv_page_bounds(k.cuda(), table.cuda(), ln.cuda())
    assert _same(got, bounds_ref(k, table, ln, torch.zeros(k.shape[0], Hkv, 2, D, dtype=dtype)))
    start = torch.randn(k.shape[0], 2, Hkv, D).to(dtype).transpose(1, 2)
    got = start.cuda()
    assert attn.kv_page_bounds(k.cuda(), table.cuda(), ln.cuda(), bounds=got).data_ptr() == got.data_ptr()
    assert _same(got, bounds_ref(k, table, ln, start.clone()))
    assert attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# page selection
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 3, 3), (256, 16, 1), (96, 4, 2), (33, 6, 2), (250, 2, 1), (1, 2, 2)])
@pytest.mark.parametrize("top", [1, 2, 9, 64, 400])
def test_select(attn, top, D, Hq, Hkv, dtype):
    ps = 4
    lens = [1200, 1, 0, 256, 257, 37]
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=D)
    bounds = bounds_ref(k, table, ln, torch.full((k.shape[0], Hkv, 2, D), math.nan, dtype=dtype))
    q = _q(6, Hq, D, dtype, seed=top)
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), ps, top)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), select_ref(q, bounds, table, ln, ps, top))
    assert attn.check_status(0) == 0


def test_select_ties_nan_and_bad_pages(attn):
    # equal scores go to the lower page, NaN before all, a page outside the cache last
    ps, n = 16, 3000
    k, v, table, ln = make_cache([n * ps], 1, 64, ps, F16, poison=False)
    q = _q(1, 2, 64, F16)
    bounds = torch.zeros(k.shape[0], 1, 2, 64, dtype=F16)
    bounds[:, 0, 1] = 1
    for top in (1, 5, 700, 2999, 3000):
        got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), ps, top)
        assert got[0, 0].tolist() == list(range(top - 1)) + [n - 1]
    bounds[int(table[0, 77]), 0, 1, 3] = math.nan
    bounds[int(table[0, 1234]), 0, 0, 9] = math.nan
    bounds[int(table[0, 2000]), 0, 1] = 2
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), ps, 6)
    assert got[0, 0].tolist() == [0, 1, 77, 1234, 2000, n - 1]
    assert torch.equal(got.cpu(), select_ref(q, bounds, table, ln, ps, 6))
    assert attn.check_status(0) == 0
    bounds.zero_()
    bounds[:, 0, 0] = -1
    table[0, 0], table[0, 5] = -1, 10 ** 7
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), ps, 4)
    assert got[0, 0].tolist() == [1, 2, 3, n - 1]
    assert attn.check_status(0) == 8
    # zeros of either sign tie
    q = torch.ones(1, 1, 1, 2, dtype=F32)
    bounds = torch.zeros(8, 1, 2, 2)
    bounds[3, 0, 0] = -0.0
    bounds[3, 0, 1] = -0.0
    table = torch.arange(8, dtype=torch.int32)[None]
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), torch.tensor([8], dtype=torch.int32).cuda(), 1, 5)
    assert got[0, 0].tolist() == [0, 1, 2, 3, 7]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_select_infinite_bounds(attn, dtype):
    # +inf and -inf in bounds, largest and smallest finite values and subnormals of the type; no q is zero
    k, v, table, ln = make_cache([900], 2, 64, 4, dtype, poison=False)
    bounds = bounds_ref(k, table, ln, torch.zeros(k.shape[0], 2, 2, 64, dtype=dtype))
    fi = torch.finfo(dtype)
    for i, (page, what, x) in enumerate([(3, 1, math.inf), (50, 0, -math.inf), (100, 1, fi.max), (130, 0, -fi.max),
                                         (150, 1, fi.smallest_normal / 4), (160, 0, -math.inf), (160, 1, math.inf)]):
        bounds[int(table[0, page]), 0, what, i] = x
    q = _q(1, 4, 64, dtype, seed=8)
    q[q == 0] = 1
    for top in (2, 4, 6, 20):
        got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), 4, top)
        assert torch.equal(got.cpu(), select_ref(q, bounds, table, ln, 4, top))


def test_select_decides_by_less_than_32_bits(attn):
    # two pages whose scores differ by less than half a step of 32 bits
    bounds = torch.zeros(3, 1, 2, 2)
    bounds[0, 0, 1] = torch.tensor([2.0 ** 20, 0.0])
    bounds[1, 0, 1] = torch.tensor([2.0 ** 20, 2.0 ** -10])
    q = torch.ones(1, 1, 1, 2)
    table = torch.arange(3, dtype=torch.int32)[None].cuda()
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table, torch.tensor([3], dtype=torch.int32).cuda(), 1, 2)
    assert got[0, 0].tolist() == [1, 2]


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------


def _evict_case(lens, Hkv, D, ps, dtype, budget, layout="hnd", seed=0):
    width = -(-budget // ps)
    k, v, table, ln = make_cache(lens, Hkv, D, ps, dtype, seed=seed, layout=layout, spare=len(lens) * width + 2)
    used = set(int(p) for b, n in enumerate(lens) for p in table[b, :-(-max(0, n) // ps)])
    free = [p for p in range(k.shape[0]) if p not in used]
    new = torch.tensor(free[:len(lens) * width], dtype=torch.int32).reshape(len(lens), width)
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(len(lens), Hkv, table.shape[1] * ps + 3, generator=g)
    return k, v, table, ln, new, w


def _check_evict(attn, k, v, table, ln, new, w, budget, recent):
    ps, H = k.shape[2], k.shape[1]
    kept, new_lens = evict_ref(w, ln, budget, recent)
    gk, gv = k.cuda(), v.cuda()
    got_lens, got_w, got_kept = attn.kv_evict(gk, gv, table.cuda(), ln.cuda(), w.cuda(), new.cuda(), budget,
                                              recent=recent)
    assert torch.equal(got_kept.cpu(), kept) and torch.equal(got_lens.cpu(), new_lens.to(torch.int32))
    want_w = torch.zeros(len(ln), H, new.shape[1] * ps)
    for b in range(len(ln)):
        m = int(new_lens[b])
        for h in range(H):
            t = kept[b, h, :m].long()
            want_w[b, h, :m] = w[b, h][t]
            to, at = new[b, torch.arange(m) // ps].long(), torch.arange(m) % ps
            kk, vv = rows(k, table[b], h, t), rows(v, table[b], h, t)
            k[to, h, at], v[to, h, at] = kk, vv
    assert _same(got_w, want_w) and _same(gk, k) and _same(gv, v)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D,ps,Hkv", [(128, 16, 4), (64, 24, 3), (33, 7, 2), (256, 128, 1)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (30, 0), (100, 16), (64, 64), (700, 5)])
def test_evict(attn, budget, recent, D, ps, Hkv, dtype):
    c = _evict_case([200, 0, 1, 99, 100, 101, 650], Hkv, D, ps, dtype, budget, seed=budget,
                    layout="nhd" if ps == 24 else "hnd")
    _check_evict(attn, *c, budget, recent)
    assert attn.check_status(0) == 0


def test_evict_ties_and_nan(attn):
    budget, n = 1000, 9000
    k, v, table, ln, new, w = _evict_case([n, n, n], 2, 16, 16, F16, budget)
    w[0] = 0.0
    w[0, 0, 1::2] = -0.0                 # zeros of either sign tie
    w[1] = (w[1] * 5).floor()            # five values
    w[2, 0, 17::1000] = math.nan
    w[2, 1] = math.nan
    w[2, 1, 5] = 1e30
    w[2, 0, 33] = math.inf
    w[2, 0, 34] = -math.inf
    _check_evict(attn, k, v, table, ln, new, w, budget, 10)


@pytest.mark.parametrize("n", [4000, 7930, 8190, 12000, 41500])
def test_evict_sizes_of_the_key_store(attn, n):
    # capacities about the limits of shared memory without and with opting in, and beyond what it holds
    c = _evict_case([n, n - 1], 1, 8, 16, F16, 600, seed=n)
    _check_evict(attn, *c, 600, 7)


@pytest.mark.parametrize("n", [3900, 4090, 21000])
def test_select_sizes_of_the_key_store(attn, n):
    k, v, table, ln = make_cache([n], 1, 8, 1, F16, poison=False)
    bounds = bounds_ref(k, table, ln, torch.zeros(k.shape[0], 1, 2, 8, dtype=F16))
    q = _q(1, 2, 8, F16)
    got = attn.kv_select_pages(q.cuda(), bounds.cuda(), table.cuda(), ln.cuda(), 1, 333)
    assert torch.equal(got.cpu(), select_ref(q, bounds, table, ln, 1, 333))


def test_evict_bad_pages(attn):
    k, v, table, ln, new, w = _evict_case([64], 1, 64, 16, F16, 32)
    w[:] = torch.arange(w.shape[2]).float()[None, None]  # keeps the last 32: pages 2 and 3
    table[0, 2], new[0, 1] = -1, 10 ** 8
    gk, gv = k.cuda(), v.cuda()
    _, _, kept = attn.kv_evict(gk, gv, table.cuda(), ln.cuda(), w.cuda(), new.cuda(), 32)
    assert kept[0, 0].tolist() == list(range(32, 64))
    assert _same(gk, k) and _same(gv, v)  # nothing could be moved
    assert attn.check_status(0) == 8 and attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# streams, graphs, a run of them together
# ---------------------------------------------------------------------------


def test_capture_follows_lengths_and_pages(attn):
    lens = [50, 0, 700, 3]
    # no page in two sequences: bounds of a page that two of them fill differently would be either's
    k, v, table, ln = make_cache(lens, 2, 128, 16, BF16, width=60, poison=False, spare=240)
    table = torch.randperm(k.shape[0])[:240].reshape(4, 60).to(torch.int32)
    q = _q(4, 8, 128, BF16)
    dk, dv, dt, dl, dq = (t.cuda() for t in (k, v, table, ln, q))
    w = torch.zeros(4, 2, 960, device="cuda")
    attn.attn_decode(dq, dk, dv, dt, dl)
    attn.attn_decode(dq, dk, dv, dt, dl, weights=w)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attn.attn_decode(dq, dk, dv, dt, dl)
            b = attn.kv_page_bounds(dk, dt, dl)
            pages = attn.kv_select_pages(dq, b, dt, dl, 16, 5)
            part = attn.attn_decode(dq, dk, dv, dt, dl, pages=pages)
        graphs.append((g, out, pages, part))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for new in ([50, 0, 700, 3], [1, 960, 5, 0], [300, 301, 302, 303]):
        dl.copy_(torch.tensor(new, dtype=torch.int32))
        table = torch.randperm(k.shape[0])[:240].reshape(4, 60).to(torch.int32)
        dt.copy_(table)
        torch.cuda.synchronize()
        for _ in range(5):
            for (g, *_), s in zip(graphs, streams):  # both at the same time
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        ln = torch.tensor(new, dtype=torch.int32)
        for g, out, pages, part in graphs:
            _close(out, decode_ref(q, k, v, table, ln), 960, BF16)
            bounds = bounds_ref(k, table, torch.where(ln > 0, ln, 0), torch.zeros(k.shape[0], 2, 2, 128, dtype=BF16))
            _close(part, decode_ref(q, k, v, table, ln, pages=pages.cpu()), 960, BF16)
            assert torch.equal(out, graphs[0][1]) and torch.equal(pages, graphs[0][2])
    assert attn.check_status(0) == 0


def test_two_streams_at_once_and_repeatable(attn):
    k, v, table, ln = make_cache([3000, 1200], 2, 64, 16, F16)
    args = [t.cuda() for t in (_q(2, 8, 64, F16), k, v, table, ln)]
    want = attn.attn_decode(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(60):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(attn.attn_decode(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_generation_run(attn):
    """Prompts, decoding steps, eviction, decoding on, sparse steps: each step against the plain attention over
    the tokens the step should see."""
    B, Hq, Hkv, D, ps, dtype = 3, 8, 2, 64, 16, F16
    g = torch.Generator().manual_seed(0)
    prompt = [70, 33, 120]
    P, W = 64, 16
    kc = torch.full((P, Hkv, ps, D), math.nan, dtype=dtype, device="cuda")
    vc = kc.clone()
    bounds = torch.zeros(P, Hkv, 2, D, dtype=dtype, device="cuda")
    table = torch.randperm(P, generator=g)[:B * W].reshape(B, W).to(torch.int32).cuda()
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    weights = torch.zeros(B, Hkv, W * ps, device="cuda")
    history = [[(torch.randn(Hkv, D, generator=g).to(dtype), torch.randn(Hkv, D, generator=g).to(dtype))
                for _ in range(n)] for n in prompt]
    S = max(prompt)
    k0, v0 = torch.zeros(B, Hkv, S, D, dtype=dtype), torch.zeros(B, Hkv, S, D, dtype=dtype)
    for b in range(B):
        for s, (x, y) in enumerate(history[b]):
            k0[b, :, s], v0[b, :, s] = x, y
    attn.kv_append(k0.cuda(), v0.cuda(), kc, vc, table, lens, new_lens=lens, bounds=bounds)
    seen = [[list(range(n)) for _ in range(Hkv)] for n in prompt]  # tokens each head still has

    def step(sparse):
        q = torch.randn(B, Hq, 1, D, generator=g).to(dtype)
        k, v = torch.randn(B, Hkv, 1, D, generator=g).to(dtype), torch.randn(B, Hkv, 1, D, generator=g).to(dtype)
        lens.add_(1)
        attn.kv_append(k.cuda(), v.cuda(), kc, vc, table, lens, bounds=bounds)
        for b in range(B):
            history[b].append((k[b, :, 0], v[b, :, 0]))
            for h in range(Hkv):
                seen[b][h].append(len(history[b]) - 1)
        if sparse:
            pages = attn.kv_select_pages(q.cuda(), bounds, table, lens, ps, 4)
            out = attn.attn_decode(q.cuda(), kc, vc, table, lens, pages=pages)
            pages = pages.cpu().tolist()
        else:
            out = attn.attn_decode(q.cuda(), kc, vc, table, lens, weights=weights)
        for b in range(B):
            for h in range(Hkv):
                tok = seen[b][h]
                if sparse:
                    tok = [t for i, t in enumerate(tok) if i // ps in pages[b][h]]
                kk = torch.stack([history[b][t][0][h] for t in tok]).double()
                vv = torch.stack([history[b][t][1][h] for t in tok]).double()
                qq = q[b, h * 4:h * 4 + 4, 0].double()
                p = torch.softmax(qq @ kk.t() / 8, 1)
                smax = (qq.abs() @ kk.abs().t()).max(1).values[:, None] / 8
                err = (out[b, h * 4:h * 4 + 4, 0].cpu().double() - p @ vv).abs()
                assert (err <= decode_tolerance(p @ vv, p @ vv.abs(), smax, len(tok), D, dtype)).all()

    for i in range(20):
        step(False)
    free = sorted(set(range(P)) - set(table.flatten().tolist()))
    new_table = torch.tensor(free[:B * 5], dtype=torch.int32).reshape(B, 5).cuda()
    w0 = weights.cpu()
    new_lens, weights2, kept = attn.kv_evict(kc, vc, table, lens, weights, new_table, 48, recent=8)
    want, _ = evict_ref(w0, lens.cpu(), 48, 8)
    assert torch.equal(kept.cpu(), want)
    for b in range(B):
        for h in range(Hkv):
            seen[b][h] = [seen[b][h][t] for t in kept[b, h].tolist() if t >= 0]
    table, lens, weights = new_table, new_lens, weights2
    attn.kv_page_bounds(kc, table, lens, bounds=bounds)
    for i in range(20):
        step(i % 2 == 1)
    assert attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# views, empty calls, large batches, captured runs
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_unaligned_views(attn, dtype):
    # every tensor a view whose rows are not 16-byte aligned, or with gaps between them
    def odd(t):
        x = torch.full((*t.shape[:-1], t.shape[-1] + 3), math.nan, dtype=t.dtype, device="cuda")[..., 1:1 + t.shape[-1]]
        return x.copy_(t)

    lens, D, ps = [70, 33], 64, 16
    k, v, table, ln = make_cache(lens, 2, D, ps, dtype, spare=9)
    x, y = torch.randn(2, 2, 5, D).to(dtype), torch.randn(2, 2, 5, D).to(dtype)
    gk, gv = odd(k), odd(v)
    bounds = odd(torch.zeros(k.shape[0], 2, 2, D, dtype=dtype))
    long = torch.tensor([75, 38], dtype=torch.int32)
    attn.kv_append(odd(x), odd(y), gk, gv, table.cuda(), long.cuda(), bounds=bounds)
    for b, n in enumerate(lens):
        for s in range(5):
            t = n + s
            k[int(table[b, t // ps]), :, t % ps], v[int(table[b, t // ps]), :, t % ps] = x[b, :, s], y[b, :, s]
    assert _same(gk, k) and _same(gv, v)
    attn.kv_page_bounds(gk, table.cuda(), long.cuda(), bounds=bounds)
    want = bounds_ref(k, table, long, torch.zeros(k.shape[0], 2, 2, D, dtype=dtype))
    used = torch.cat([table[0, :5], table[1, :3]]).long()
    assert _same(bounds.cpu()[used], want[used])
    q = _q(2, 4, D, dtype)
    pages = attn.kv_select_pages(odd(q), bounds, table.cuda(), long.cuda(), ps, 3)
    assert torch.equal(pages.cpu(), select_ref(q, want, table, long, ps, 3))
    _close(attn.attn_decode(odd(q), gk, gv, table.cuda(), long.cuda(), pages=pages),
           decode_ref(q, k, v, table, long, pages=pages.cpu()), 48, dtype)
    free = [p for p in range(k.shape[0]) if p not in used.tolist()]
    new = torch.tensor(free[:4], dtype=torch.int32).reshape(2, 2)
    w = torch.rand(2, 2, table.shape[1] * ps)
    kept, _ = evict_ref(w, long, 20, 3)
    _, _, got = attn.kv_evict(gk, gv, table.cuda(), long.cuda(), odd(w), new.cuda(), 20, recent=3)
    assert torch.equal(got.cpu(), kept)
    for b in range(2):
        for h in range(2):
            t = kept[b, h].long()
            assert torch.equal(rows(gk.cpu(), new[b], h, range(20)), rows(k, table[b], h, t))
            assert torch.equal(rows(gv.cpu(), new[b], h, range(20)), rows(v, table[b], h, t))
    assert attn.check_status(0) == 0


def test_empty_calls(attn):
    k = torch.zeros(4, 2, 16, 64, dtype=F16, device="cuda")
    t, n = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, 2, 1, 64, dtype=F16, device="cuda")
    attn.kv_append(none, none, k, k, t, n)
    assert (attn.kv_page_bounds(k, t, n) == 0).all()
    assert attn.kv_select_pages(none, torch.zeros(4, 2, 2, 64, dtype=F16, device="cuda"), t, n, 16, 3).shape == (0, 2, 3)
    a, b, c = attn.kv_evict(k, k, t, n, torch.zeros(0, 2, 48, device="cuda"), t, 5)
    assert a.shape == (0,) and b.shape == (0, 2, 48) and c.shape == (0, 2, 5)
    # no new tokens, and tables without pages
    t1, n1 = torch.zeros(1, 0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    attn.kv_append(none.new_zeros(1, 2, 0, 64), none.new_zeros(1, 2, 0, 64), k, k, t1, n1)
    assert (attn.kv_page_bounds(k, t1, n1) == 0).all()
    got = attn.kv_select_pages(none.new_zeros(1, 2, 1, 64), torch.zeros(4, 2, 2, 64, dtype=F16, device="cuda"), t1, n1, 16, 3)
    assert (got == -1).all()
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_sequences_than_a_grid_dimension(attn, dtype):
    B, D, ps = 70001, 8, 4
    k, v = (torch.randn(B, 1, ps, D, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(B, device="cuda").to(torch.int32)[:, None]
    lens = torch.ones(B, dtype=torch.int32, device="cuda")
    lens[5::7] = 0
    x, y = (torch.randn(B, 1, 1, D, device="cuda").to(dtype) for _ in range(2))
    bounds = torch.zeros(B, 1, 2, D, dtype=dtype, device="cuda")
    attn.kv_append(x, y, k, v, table, lens, bounds=bounds)
    page, live = table[:, 0].long(), lens > 0
    assert torch.equal(k[page[live], 0, 0], x[live, 0, 0]) and torch.equal(bounds[page[live], 0, 1], x[live, 0, 0])
    assert torch.equal(attn.kv_page_bounds(k, table, lens), bounds)
    out = attn.attn_decode(torch.randn(B, 2, 1, D, device="cuda").to(dtype), k, v, table, lens)
    assert torch.equal(out[live], y[live].expand(-1, 2, 1, D)) and (out[~live] == 0).all()  # one token has all the weight
    pages = attn.kv_select_pages(out, bounds, table, lens, ps, 1)
    assert torch.equal(pages[:, 0, 0] == 0, live)
    new = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    k2, v2 = torch.cat([k, k * 0]), torch.cat([v, v * 0])
    n, w, kept = attn.kv_evict(k2, v2, table, lens, torch.ones(B, 1, ps, device="cuda"), new + B, 2)
    assert torch.equal(n, lens) and torch.equal(kept[:, 0, 0] == 0, live) and (kept[:, 0, 1] == -1).all()
    assert torch.equal(k2[B:][live, 0, 0], x[live, 0, 0]) and torch.equal(v2[B:][live, 0, 0], y[live, 0, 0])
    assert attn.check_status(0) == 0


def test_captured_steps(attn):
    # append, weights and eviction captured together and replayed on new values, lengths and pages
    lens, D, ps, budget = [90, 41], 64, 16, 40
    k, v, table, ln = make_cache(lens, 2, D, ps, F16, spare=20, poison=False)
    free = [p for p in range(k.shape[0]) if p not in table.flatten().tolist()]
    new = torch.tensor(free[:6], dtype=torch.int32).reshape(2, 3)
    gk, gv, gt, gl, gn = k.cuda(), v.cuda(), table.cuda(), ln.cuda(), new.cuda()
    x, y = torch.randn(2, 2, 1, D).to(F16), torch.randn(2, 2, 1, D).to(F16)
    q = _q(2, 4, D, F16)
    gx, gy, gq = x.cuda(), y.cuda(), q.cuda()
    w = torch.zeros(2, 2, table.shape[1] * ps, device="cuda")

    def step():
        attn.kv_append(gx, gy, gk, gv, gt, gl)
        out = attn.attn_decode(gq, gk, gv, gt, gl, weights=w)
        return out, attn.kv_evict(gk, gv, gt, gl, w, gn, budget, recent=4)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, (n2, w2, kept) = step()
    for i, n in enumerate(([90, 41], [17, 90], [64, 1])):
        x, y, q = torch.randn(2, 2, 1, D).to(F16), torch.randn(2, 2, 1, D).to(F16), _q(2, 4, D, F16, seed=i)
        now = torch.tensor(n, dtype=torch.int32)
        full = torch.tensor([p for p in range(k.shape[0]) if p not in new.flatten().tolist()])
        table = full[torch.randperm(len(full))[:2 * table.shape[1]]].reshape(2, -1).to(torch.int32)
        gk.copy_(k), gv.copy_(v), gx.copy_(x), gy.copy_(y), gq.copy_(q), gl.copy_(now), gt.copy_(table)
        start = torch.rand(w.shape)
        w.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        kk, vv = k.clone(), v.clone()
        for b in range(2):
            t = n[b] - 1
            kk[int(table[b, t // ps]), :, t % ps], vv[int(table[b, t // ps]), :, t % ps] = x[b, :, 0], y[b, :, 0]
        ref = decode_ref(q, kk, vv, table, now)
        _close(out, ref, 90, F16)
        # the bound of test_decode_weights: 2 (68 2^-23 5 + 2^-21 + 90 2^-23) of a weight of at most 1
        assert torch.allclose(w.cpu().double(), start.double() + ref[3], rtol=0, atol=1e-4 * 2)
        want, lens2 = evict_ref(w.cpu(), now, budget, 4)
        assert torch.equal(kept.cpu(), want) and torch.equal(n2.cpu(), lens2.int())
        for b in range(2):
            for h in range(2):
                m = int(lens2[b])
                assert torch.equal(rows(gk.cpu(), new[b], h, range(m)), rows(kk, table[b], h, want[b, h, :m].long()))
                assert torch.equal(w2[b, h, :m].cpu(), w.cpu()[b, h][want[b, h, :m].long()])
    assert attn.check_status(0) == 0


# ---------------------------------------------------------------------------
# the watchdog (tests/test_watchdog_gpu.py says how the test build works)
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("lens,D,width", [([300, 40], 128, None), ([2000, 700], 64, None), ([5000], 128, 400),
                                          ([900], 256, 200)])
def test_watchdog_fires_and_recovers(lens, D, width):
    # CTA 0's first wait is for 16 bytes more than come: it ends by the limit, the kernel reports it and
    # returns, and the next launch is clean
    from test_paged_cpu import LL3, PagedCache

    lib = ctypes.CDLL(os.path.join(os.path.dirname(rocm_attn_b200.KERNEL_LIB_PATH), "librocm_attn_wdtest.so"))
    lib.attn_set_wait_limit_ns.argtypes = [ctypes.c_ulonglong]
    lib.launch_attn_decode.argtypes = [ctypes.c_void_p] * 4 + [ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_int,
                                                                ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                                                ctypes.c_size_t, ctypes.c_void_p]
    k, v, table, ln = make_cache(lens, 2, D, 16, BF16, width=width)
    q = _q(len(lens), 4, D, BF16)
    dk, dv, dt, dl, dq = (t.cuda() for t in (k, v, table, ln, q))
    out = torch.zeros_like(dq)
    st = LL3(*dk.stride()[:3])
    c = PagedCache(dk.data_ptr(), dv.data_ptr(), k.shape[0], 2, 16, D, 1, st, st, dt.data_ptr(), dt.shape[1], dt.shape[1],
                   dl.data_ptr(), len(lens))
    size = ctypes.c_size_t()
    assert lib.attn_decode_workspace_bytes(ctypes.byref(c), 4, False, 0, False, ctypes.byref(size)) == 0
    space = torch.empty(max(16, size.value), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def run():
        assert lib.launch_attn_decode(ctypes.byref(c), dq.data_ptr(), None, out.data_ptr(), 4, -1.0, None, 0, None, None,
                                      space.data_ptr(), size.value, stream) == 0
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
    _close(out, decode_ref(q, k, v, table, ln), max(lens), BF16)


# ---------------------------------------------------------------------------
# refusals of the binding
# ---------------------------------------------------------------------------


def test_refusals(attn):
    k = torch.zeros(4, 2, 16, 64, dtype=F16, device="cuda")
    q = torch.zeros(1, 4, 1, 64, dtype=F16, device="cuda")
    t = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    w = torch.zeros(1, 2, 64, device="cuda")
    pages = torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")

    def no(match, f, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **kw)

    d = attn.attn_decode
    no("same dtype", d, q.float(), k, k, t, n)
    no("float32, float16", d, q.double(), k.double(), k.double(), t, n)
    no("one token", d, q.expand(1, 4, 2, 64), k, k, t, n)
    no("batch size", d, q.expand(2, 4, 1, 64), k, k, t, n)
    no("head dim", d, q[..., :32], k, k, t, n)
    no("multiple", d, q[:, :3], k, k, t, n)
    no("same shape", d, q, k, k[:3], t, n)
    no("contiguous", d, q, k.transpose(2, 3), k.transpose(2, 3), t, n)
    no("int32", d, q, k, k, t.long(), n)
    no("int32", d, q, k, k, t, n.long())
    no("2D", d, q, k, k, t[0], n)
    no("same batch size", d, q, k, k, t, n.expand(2))
    no("CUDA", d, q, k, k, t.cpu(), n)
    no("together", d, q, k, k, t, n, pages=pages, weights=w)
    no("room", d, q, k, k, t, n, weights=w[:, :, :63])
    no("float32", d, q, k, k, t, n, weights=w.half())
    no("expanded", d, q, k, k, t, n, weights=w[:, :1].expand(1, 2, 64))
    no("pages must be", d, q, k, k, t, n, pages=pages[:, :1])
    big = torch.zeros(1, 1, 1, 300, dtype=F16, device="cuda")
    no("unsupported", d, big, big, big, t, n)
    x = torch.zeros(1, 2, 1, 64, dtype=F16, device="cuda")
    b = torch.zeros(4, 2, 2, 64, dtype=F16, device="cuda")
    a = attn.kv_append
    no("same dtype", a, x.float(), x, k, k, t, n)
    no("number of tokens", a, x, x.expand(1, 2, 3, 64), k, k, t, n)
    no("heads", a, x[:, :1], x, k, k, t, n)
    no("expanded", a, x, x, k[:1].expand(4, 2, 16, 64), k, t, n)
    no("bounds", a, x, x, k, k, t, n, bounds=b[:3])
    no("dtype", a, x, x, k, k, t, n, bounds=b.float())
    no("new_lens", a, x, x, k, k, t, n, new_lens=n.expand(2))
    s = attn.kv_select_pages
    no("top", s, q, b, t, n, 16, 0)
    no("page size", s, q, b, t, n, 0, 1)
    no("bounds must be", s, q, b[:, :, :1], t, n, 16, 1)
    e = attn.kv_evict
    no("budget", e, k, k, t, n, w, t, 0)
    no("budget", e, k, k, t, n, w, t, 65)
    no("recent", e, k, k, t, n, w, t, 3, recent=4)
    no("batch size", e, k, k, t, n, w, t.expand(2, 4), 3)
    assert attn.check_status(0) == 0
