"""Paged key-value caches for the tests, and the operators' definitions on the
CPU in 64 bits, one sequence and head after another."""
import math

import torch


def make_cache(B_lens, Hkv, D, ps, dtype, seed=0, width=None, layout="hnd", poison=True, spare=3):
    """(k_cache, v_cache, table, lens) on the CPU: pages in random order, every row that belongs to no
    token and every page of no sequence NaN, unused table entries far outside the cache."""
    g = torch.Generator().manual_seed(seed)
    counts = [max(0, -(-n // ps)) for n in B_lens]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g)
    width = max([1] + counts) if width is None else width
    table = torch.full((len(B_lens), width), 2 ** 30, dtype=torch.int32)
    k = torch.randn(total, Hkv, ps, D, generator=g).to(dtype)
    v = torch.randn(total, Hkv, ps, D, generator=g).to(dtype)
    used = torch.zeros(total, ps, dtype=torch.bool)
    at = 0
    for b, n in enumerate(B_lens):
        for j in range(counts[b]):
            p = int(order[at])
            at += 1
            table[b, j] = p
            used[p, :min(ps, n - j * ps)] = True
    if poison:
        bad = ~used[:, None, :, None]
        k, v = k.masked_fill(bad, math.nan), v.masked_fill(bad, math.nan)
    lens = torch.tensor(B_lens, dtype=torch.int32)
    if layout == "nhd":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    return k, v, table, lens


def rows(cache, table_row, h, tokens):
    ps = cache.shape[2]
    t = torch.as_tensor(tokens, dtype=torch.long)
    return cache[table_row[t // ps].long(), h, t % ps]


def decode_ref(q, k, v, table, lens, scale=None, pages=None, drop=None):
    """o [B, Hq, 1, D] in 64 bits, per-element bound parts (sum p |v|, max |score|, tokens), and weights
    [B, Hkv, capacity].  drop(b, token) -> True for tokens that count as absent."""
    B, Hq, _, D = q.shape
    H, ps = k.shape[1], k.shape[2]
    g = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    cap = table.shape[1] * ps
    o = torch.zeros(B, Hq, 1, D, dtype=torch.float64)
    absum = torch.zeros_like(o)
    smax = torch.zeros(B, Hq, 1, 1, dtype=torch.float64)
    w = torch.zeros(B, H, cap, dtype=torch.float64)
    for b in range(B):
        n = min(max(0, int(lens[b])), cap)
        for h in range(H):
            if pages is None:
                tok = list(range(n))
            else:
                tok = [t for p in pages[b, h].tolist() if 0 <= p < table.shape[1]
                       for t in range(p * ps, min(n, p * ps + ps))]
            if drop is not None:
                tok = [t for t in tok if not drop(b, t)]
            if not tok:
                continue
            kk, vv = rows(k, table[b], h, tok).double(), rows(v, table[b], h, tok).double()
            qq = q[b, h * g:(h + 1) * g, 0].double()
            x = scale * (qq @ kk.t())
            p = torch.softmax(x, 1)
            o[b, h * g:(h + 1) * g, 0] = p @ vv
            absum[b, h * g:(h + 1) * g, 0] = p @ vv.abs()
            smax[b, h * g:(h + 1) * g, 0, 0] = scale * (qq.abs() @ kk.abs().t()).max(1).values
            w[b, h].index_add_(0, torch.tensor(tok), p.sum(0))
    return o, absum, smax, w


def decode_tolerance(o, absum, smax, n, D, dtype):
    """Elementwise bound of |kernel - o|.

    A score is a sum of D exact products in 32 bits (each partial sum off by at most 2^-23 of sum |q k|,
    which truncating adders need), times the scale: off by (D + 4) 2^-23 smax, and its exponential by as
    much relatively, plus 2^-21 for the exponentials of the value and of the two rescalings.  Numerator and denominator
    each have it, and sums of n terms n 2^-23.  16-bit inputs round P (half a step of each weight: of sum p |v|; fp16 below 2^-14 is off by at most 2^-25
    against a largest P of 1, so by n 2^-25 max |v|) and all round the output."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * ((D + 4) * 2.0 ** -23 * smax + 2.0 ** -21 + n * 2.0 ** -23)
    tol = rel * absum + half * o.abs() + 1e-30
    if dtype != torch.float32:
        tol = tol + half * absum * (1 + rel)
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -25 * 8 + 2.0 ** -25  # |v| < 8 for these draws; subnormal outputs
    return tol


def decode_bound(o, absum, smax, n, D, dtype, vmax=0.0):
    """Elementwise bound of |kernel - o| that holds for small weights too: decode_tolerance with the fp16
    kernel's own ends of P.

    It keeps P times 2^15, so that weights from 2^-29 of the largest of their warp on are normal numbers and
    off by half a step; smaller ones are off by at most 2^-25 2^-15 = 2^-40 of the largest, each times its |v| <=
    vmax (0: there are none).  O is rounded to the output type, subnormals of fp16 by 2^-25."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * ((D + 4) * 2.0 ** -23 * smax + 2.0 ** -21 + n * 2.0 ** -23)
    tol = rel * absum + half * o.abs() + 1e-30
    if dtype != torch.float32:
        tol = tol + half * absum * (1 + rel)
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -40 * vmax + 2.0 ** -25
    return tol


def bounds_ref(k, table, lens, out):
    ps = k.shape[2]
    for b in range(table.shape[0]):
        for j in range(-(-max(0, int(lens[b])) // ps)):
            x = k[int(table[b, j]), :, :min(ps, int(lens[b]) - j * ps)]
            out[int(table[b, j])] = torch.stack([x.amin(1), x.amax(1)], 1)
    return out


def select_ref(q, bounds, table, lens, ps, top):
    B, Hq, _, D = q.shape
    H = bounds.shape[1]
    out = torch.full((B, H, top), -1, dtype=torch.int32)
    for b in range(B):
        n = -(-max(0, int(lens[b])) // ps)
        if n == 0:
            continue
        for h in range(H):
            qq = q[b, h * (Hq // H):(h + 1) * (Hq // H), 0].double()
            lo, hi = bounds[table[b, :n].long(), h].double().unbind(1)
            s = torch.maximum(qq[:, None] * lo, qq[:, None] * hi).sum((0, 2)).tolist()
            rank = sorted(range(n - 1), key=lambda i: (0 if math.isnan(s[i]) else 1, -s[i] if not math.isnan(s[i]) else 0, i))
            pick = sorted(rank[:top - 1] + [n - 1])[:top]
            out[b, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return out


def evict_ref(w, lens, budget, recent):
    """kept [B, H, budget] and new lens."""
    B, H, _ = w.shape
    kept = torch.full((B, H, budget), -1, dtype=torch.int32)
    for b in range(B):
        n = max(0, int(lens[b]))
        m = min(n, budget)
        for h in range(H):
            x = w[b, h].tolist()
            r = min(recent, n)
            rank = sorted(range(n - r), key=lambda i: (0 if math.isnan(x[i]) else 1, -x[i] if not math.isnan(x[i]) else 0, i))
            keep = sorted(rank[:m - r] + list(range(n - r, n)))
            kept[b, h, :m] = torch.tensor(keep, dtype=torch.int32)
    return kept, lens.clamp(min=0, max=budget)
