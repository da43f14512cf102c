"""Definitions of the operators for drafted tokens and shared pages, on the CPU, the attention in 64 bits, one
sequence and head after another."""
import math
import random

import torch


def random_tree(S, rng, bushy=0.4):
    """Parents of S drafted tokens: -1 or a token before."""
    return [s - 1 if s == 0 or rng.random() > bushy else rng.randrange(-1, s) for s in range(S)]


def ancestors(parents, s):
    out = []
    while s >= 0:
        out.append(s)
        p = parents[s]
        s = p if -1 <= p < s else -1
    return out


def tree_ref(q, k, v, table, lens, parents=None, new_lens=None, scale=None, drop=None):
    """o [B, Hq, S, D] in 64 bits, and the parts of its bound: sum p |v|, max |score|, both over the tokens that a
    row sees.  Only tokens that it sees are looked at, so others may hold anything.  drop(b, token): absent ones."""
    B, Hq, S, D = q.shape
    H, ps = k.shape[1], k.shape[2]
    g = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o = torch.zeros(B, Hq, S, D, dtype=torch.float64)
    absum, smax = torch.zeros_like(o), torch.zeros(B, Hq, S, 1, dtype=torch.float64)
    for b in range(B):
        n = S if new_lens is None else max(0, min(S, int(new_lens[b])))
        length = max(0, int(lens[b]))
        base = length - n
        cap = min(length, table.shape[1] * ps)
        par = list(range(-1, S - 1)) if parents is None else parents[b].tolist()
        at = torch.arange(cap)
        page = table[b, at // ps].long()
        there = torch.ones(cap, dtype=torch.bool)
        if drop is not None:
            there = torch.tensor([not drop(b, t) for t in range(cap)], dtype=torch.bool)
        page = torch.where(there, page, 0)
        for h in range(H):
            kk, vv = k[page, h, at % ps].double(), v[page, h, at % ps].double()
            for s in range(n):
                see = torch.zeros(cap, dtype=torch.bool)
                see[:max(0, min(base, cap))] = True
                for a in ancestors(par, s):
                    if 0 <= base + a < cap:
                        see[base + a] = True
                see &= there
                if not see.any():
                    continue
                qq = q[b, h * g:(h + 1) * g, s].double()
                x = scale * (qq @ kk[see].t())
                p = torch.softmax(x, 1)
                o[b, h * g:(h + 1) * g, s] = p @ vv[see]
                absum[b, h * g:(h + 1) * g, s] = p @ vv[see].abs()
                smax[b, h * g:(h + 1) * g, s, 0] = scale * (qq.abs() @ kk[see].abs().t()).max(1).values
    return o, absum, smax


def tree_bound(o, absum, smax, n, D, dtype, vmax=8.0):
    """Elementwise bound of |kernel - o|.

    A score is a sum of D exact products in 32 bits (each partial sum off by at most 2^-23 of sum |q k|,
    which truncating adders need), times the scale: off by (D + 4) 2^-23 smax, and its exponential by as much
    relatively, plus 2^-21 for the exponentials of the value and of the rescalings.  Numerator and denominator each
    have it, and sums of n terms n 2^-23.  16-bit inputs round P, by half a step of each weight at most: of sum p
    |v|.  fp16 keeps P times 2^7, relative to a maximum that the largest weight is never below, so weights below 2^-21
    of it are off by at most 2^-25 2^-7 of it, each times its |v| <= vmax.  O is rounded to its type, subnormals
    of fp16 by 2^-25."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * ((D + 4) * 2.0 ** -23 * smax + 2.0 ** -21 + n * 2.0 ** -23)
    tol = rel * absum + half * o.abs() + 1e-30
    if dtype != torch.float32:
        tol = tol + half * absum * (1 + rel)
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -32 * vmax + 2.0 ** -25
    return tol


def compact_ref(k, v, table, lens, kept, new_lens):
    """Changes k and v; the new lengths."""
    ps = k.shape[2]
    out = []
    for b in range(len(lens)):
        n = max(0, int(new_lens[b]))
        base = int(lens[b]) - n
        path, last = [], -1
        for a in kept[b].tolist():
            if not last < a < n:
                break
            path.append(a)
            last = a
        for c in (k, v):
            was = c.clone()
            for i, a in enumerate(path):
                if i != a and base + i >= 0:
                    c[int(table[b, (base + i) // ps]), :, (base + i) % ps] = \
                        was[int(table[b, (base + a) // ps]), :, (base + a) % ps]
        out.append(max(0, base + len(path)))
    return torch.tensor(out, dtype=torch.int32)


def resize_ref(table, held, lens, refs, ps):
    """Changes the lists table, held and refs; what each sequence lacks."""
    free = [p for p, r in enumerate(refs) if r == 0]
    asked = used = 0
    missing = []
    for b, n in enumerate(lens):
        want = -(-max(0, n) // ps)
        need = max(0, want - held[b])
        asked += need
        if need and asked > len(free):
            missing.append(need)
            continue
        missing.append(0)
        for j in range(want, held[b]):
            refs[table[b][j]] -= 1
        for j in range(held[b], want):
            table[b][j] = free[used]
            refs[free[used]] += 1
            used += 1
        held[b] = want
    return missing


def fork_ref(k, v, table, held, lens, refs, parents, ps):
    """Changes k, v and the list refs; the new (table, held, lens, missing) as lists."""
    W = len(table[0]) if table else 0
    free = [p for p, r in enumerate(refs) if r == 0]
    before, seen = list(refs), set()
    plan = []  # (row of pages, length, page to copy)
    for a in parents:
        if a < 0:
            plan.append(([], 0, None))
            continue
        n = min(max(0, lens[a]), held[a] * ps)
        row = table[a][:-(-n // ps)]
        copies = n % ps and (a in seen or before[row[-1]] != 1)
        plan.append((list(row), n, row[-1] if copies else None))
        seen.add(a)
    need = sum(c is not None for _, _, c in plan)
    if need > len(free):
        m = len(parents)
        return [[-1] * W for _ in range(m)], [0] * m, [0] * m, need - len(free)
    for b, h in enumerate(held):
        for p in table[b][:h]:
            refs[p] -= 1
    for row, n, copy in plan:
        if copy is not None:
            row[-1] = free.pop(0)
            for c in (k, v):
                c[row[-1], :, :n % ps] = c[copy, :, :n % ps]
        for p in row:
            refs[p] += 1
    return ([r + [-1] * (W - len(r)) for r, _, _ in plan], [len(r) for r, _, _ in plan], [n for _, n, _ in plan], 0)


def random_pool(rng, rows, W, num_pages, ps, shared=0.3):
    """(table, held, lens, refs) as lists: rows of the table that hold random pages, some in common with the row before."""
    free = list(range(num_pages))
    rng.shuffle(free)
    refs = [0] * num_pages
    table, held, lens = [], [], []
    for b in range(rows):
        n = rng.randint(0, min(W, len(free)))
        row = []
        if b and rng.random() < shared:
            row = table[-1][:rng.randint(0, min(held[-1], n))]
        while len(row) < n:
            row.append(free.pop())
        for p in row:
            refs[p] += 1
        table.append(row + [-1] * (W - len(row)))
        held.append(len(row))
        lens.append(rng.randint(max(0, (n - 1) * ps - ps), n * ps) if n else 0)
    return table, held, lens, refs
