"""Drafted tokens and shared pages on the paged key-value cache, as a generating program calls them, with plain
forms of each.

A case is one call (for the pages a sequence holds: a call that takes pages and one that gives them back) of a
generating loop at stated sizes: attention of a tree of drafted tokens (``attn_tree``), the move of the accepted
ones to their places (``kv_compact``), a step of a beam search on the cache (``kv_fork``) and the pages that the
lengths of the next step need (``kv_resize``).  ``own`` chooses between the plain forms (elementary torch operations, 32 bits for the attention) and the
package's operators.

Cache layout: k_cache and v_cache [num_pages, Hkv, page_size, D]; token t of sequence b lies in page
block_table[b, t // page_size], row t % page_size; seq_lens counts the tokens of each sequence, the drafted ones
included; held[b] entries of row b of the table name pages that the sequence holds, refs[page] counts the holders.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ELEM = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # One user, a small tree of drafts, a few hundred tokens of context: launch latency.
        dict(name="tree one bf16", op="tree", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, ps=16, L=517, S=8, chain=False),
        # A serving batch of mixed lengths, trees of up to 16 drafted tokens.
        dict(name="tree batch bf16", op="tree", dtype="bf16", B=24, Hq=32, Hkv=8, D=128, ps=16, L=4096, S=16, chain=False),
        # Long contexts, 16 drafted tokens and eight query heads to a kv head.
        dict(name="tree long fp16", op="tree", dtype="fp16", B=32, Hq=64, Hkv=8, D=128, ps=64, L=16384, S=16, chain=False),
        # Wide trees of 64 tokens over long contexts.
        dict(name="tree wide bf16", op="tree", dtype="bf16", B=8, Hq=32, Hkv=8, D=128, ps=32, L=8192, S=64, chain=False),
        # A chain of five drafts, one kv head per query head at D = 64, odd lengths, a page size that is no power of two.
        dict(name="chain d64 fp16", op="tree", dtype="fp16", B=17, Hq=16, Hkv=16, D=64, ps=24, L=2047, S=5, chain=True),
        # An fp32 cache.
        dict(name="tree fp32", op="tree", dtype="fp32", B=3, Hq=16, Hkv=4, D=64, ps=16, L=1500, S=7, chain=False),
        # What one user's drafts leave behind.
        dict(name="compact one bf16", op="compact", dtype="bf16", B=1, Hkv=8, D=128, ps=16, L=517, S=8),
        # The accepted paths of a large batch of wide trees.
        dict(name="compact batch fp16", op="compact", dtype="fp16", B=128, Hkv=8, D=128, ps=64, L=1024, S=64),
        # A step of beam search: four prompts, four beams each.
        dict(name="fork beams bf16", op="fork", dtype="bf16", B=16, width=4, Hkv=8, D=128, ps=16, L=2048),
        # A large batch of beams on large pages.
        dict(name="fork batch fp16", op="fork", dtype="fp16", B=384, width=8, Hkv=8, D=128, ps=64, L=1000),
        # A step of drafts: room for eight tokens per sequence, and what the rejected ones held goes back.
        dict(name="resize step", op="resize", B=64, ps=16, L=4096, S=8, pool=65536),
        # A batch of prompts comes and goes.
        dict(name="resize prompts", op="resize", B=64, ps=16, L=16384, S=0, pool=262144),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "compact", "fork", "resize"])
    ps = rng.choice([16, 16, 32, 64, rng.choice([8, 24, 128])])
    if op == "resize":
        B = _log_int(rng, 1, 256)
        L = _log_int(rng, 16, max(32, min(16384, (1 << 20) // B)))
        S = 0 if rng.random() < 0.4 else _log_int(rng, 1, 64)
        need = B * ((L + S + ps - 1) // ps)
        return dict(op=op, B=B, ps=ps, L=L, S=S, pool=need + _log_int(rng, 1, 131072))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    D = rng.choice([64, 128, 128, rng.choice([32, 80, 96, 256])])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    row = Hkv * D * ELEM[dtype] * 2
    if op == "tree":
        B = _log_int(rng, 1, 64)
        S = _log_int(rng, 1, 128)
        g = rng.choice([1, 2, 4, 7, 8, 16])
        # no more cache, products or scores than half of the largest listed cases have; products in fp32 cost more
        ops = (1 << 41) if dtype != "fp32" else 1 << 37
        top = min(32768, (1 << 30) // (row * B), ops // (4 * B * Hkv * g * D * S), (1 << 31) // (B * Hkv * g * S))
        L = _log_int(rng, S, max(S + 16, top))
        return dict(op=op, dtype=dtype, B=B, Hq=Hkv * g, Hkv=Hkv, D=D, ps=ps, L=L, S=S, chain=rng.random() < 0.3)
    if op == "compact":
        B, S = _log_int(rng, 1, 128), _log_int(rng, 1, 64)
        L = _log_int(rng, S, max(S + 16, min(4096, (1 << 30) // (row * B))))
        return dict(op=op, dtype=dtype, B=B, Hkv=Hkv, D=D, ps=ps, L=L, S=S)
    width = rng.choice([2, 3, 4, 5, 8])
    B = width * _log_int(rng, 1, 48)
    L = _log_int(rng, 1, max(16, min(4096, (1 << 30) // (row * B))))
    return dict(op=op, dtype=dtype, B=B, width=width, Hkv=Hkv, D=D, ps=ps, L=L)


def _lens(case):
    """The lengths of the case's sequences: between a quarter of L and L, the first L itself; the beams of one
    prompt are equally long."""
    r = random.Random("%d.%d.%d" % (case["B"], case["L"], case["ps"]))
    L, w = case["L"], case.get("width", 1)
    each = [L] + [r.randint(max(1, L // 4), L) for _ in range(case["B"] // w - 1)]
    return [n for n in each for _ in range(w)]


def _drafted(case):
    """How many tokens of each sequence are drafted: between half of S and S, the first S."""
    r = random.Random("drafted %d.%d" % (case["B"], case["S"]))
    return [min(n, case["S"] if i == 0 else r.randint(max(1, case["S"] // 2), case["S"]))
            for i, n in enumerate(_lens(case))]


def _trees(case, seed):
    """[B][S] parents: a token follows the context, or one of the last few drafted before it."""
    r = random.Random("tree %d.%d.%d" % (case["B"], case["S"], seed))
    return [[s - 1 if s == 0 or r.random() < 0.05 else max(-1, s - 1 - int(r.expovariate(0.4))) for s in range(case["S"])]
            for _ in range(case["B"])]


def _path(parents, s):
    path = []
    while s >= 0:
        path.append(s)
        s = parents[s]
    return path[::-1]


def _beams(case, seed):
    """Which beam each new one continues: the beams of one prompt that live on stay, the others' places go to copies."""
    r = random.Random("beams %d.%d.%d" % (case["B"], case["width"], seed))
    w, out = case["width"], []
    for p in range(case["B"] // w):
        live = sorted(r.sample(range(w), r.randint(1, w)))
        out += [p * w + (i if i in live else r.choice(live)) for i in range(w)]
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    B, ps, op = case["B"], case["ps"], case["op"]
    lens = _lens(case)
    counts = [(n + ps - 1) // ps for n in lens]
    ints = lambda x: torch.tensor(x, device=dev, dtype=torch.int32)  # noqa: E731
    if op == "resize":
        # pages that other sequences hold lie among the free ones
        most = [n + case["S"] for n in lens]
        width, total = (max(most) + ps - 1) // ps, case["pool"]
        order = torch.randperm(total, generator=g, device=dev, dtype=torch.int32)
        need = sum((n + ps - 1) // ps for n in most)
        refs = torch.zeros(total, device=dev, dtype=torch.int32)
        refs[order[need:need + (total - need) // 2].long()] = 1
        table = torch.full((B, width), -1, device=dev, dtype=torch.int32)
        now = counts if case["S"] else [0] * B
        taken = [sum(now[:b]) for b in range(B)]
        for b in range(B):
            table[b, :now[b]] = order[taken[b]:taken[b] + now[b]]
        refs[order[:sum(now)].long()] = 1
        s = dict(case=case, table=table, held=ints(now), refs=refs, more=ints(most), less=ints(lens if case["S"] else [0] * B))
        torch.cuda.synchronize()
        return s
    dtype, Hkv, D = DTYPES[case["dtype"]], case["Hkv"], case["D"]
    width = max(counts)
    w = case.get("width", 1)
    # the beams of one prompt share half of their pages; the rest, and all of other sequences', are their own
    shared = [c // 2 if w > 1 else 0 for c in counts]
    spare = B + 3 if op == "fork" else 0
    total = sum(c - s for c, s in zip(counts, shared)) + sum(shared[::w]) + spare
    # pages are handed out in random order, as after many sequences have come and gone
    order = torch.randperm(total, generator=g, device=dev, dtype=torch.int32)
    table = torch.full((B, width), -1, device=dev, dtype=torch.int32)
    at = 0
    for b in range(B):
        if b % w == 0:
            common = order[at:at + shared[b]]
            at += shared[b]
        table[b, :shared[b]] = common
        table[b, shared[b]:counts[b]] = order[at:at + counts[b] - shared[b]]
        at += counts[b] - shared[b]
    kc = torch.randn(total, Hkv, ps, D, generator=g, device=dev, dtype=dtype)
    vc = torch.randn(total, Hkv, ps, D, generator=g, device=dev, dtype=dtype)
    s = dict(case=case, kc=kc, vc=vc, table=table, lens=ints(lens))
    if op in ("tree", "compact"):
        new = _drafted(case)
        s["new_lens"] = ints(new)
    if op == "tree":
        s["q"] = torch.randn(B, case["Hq"], case["S"], D, generator=g, device=dev, dtype=dtype)
        s["parents"] = None if case["chain"] else ints(_trees(case, seed))
    if op == "compact":
        # the accepted path ends in a random token of the tree
        r = random.Random("path %d" % seed)
        paths = [_path(t, r.randrange(n)) for t, n in zip(_trees(case, seed), new)]
        s["kept"] = ints([p + [-1] * (case["S"] - len(p)) for p in paths])
    if op == "fork":
        s["held"] = ints(counts)
        s["parents"] = ints(_beams(case, seed))
        s["refs"] = torch.zeros(total, device=dev, dtype=torch.int32)
        named = table[table >= 0].long()
        s["refs"].index_add_(0, named, torch.ones_like(named, dtype=torch.int32))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _gather(cache, table):
    """[B, Hkv, W * page_size, D] in 32 bits: the pages of each sequence in order."""
    x = cache[table.clamp(min=0).long()]
    B, W, H, ps, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, W * ps, D).float()


def _follows(parents, B, S, device):
    """[B, S, S]: whether drafted token s is, or comes after, drafted token a."""
    at = torch.arange(S, device=device)
    if parents is None:
        return (at[None, :] <= at[:, None]).expand(B, S, S)
    # one step to the parent as a matrix, (1 + step) squared until every chain is covered
    reach = ((parents[:, :, None] == at) | (at[:, None] == at)).float()
    n = 1
    while n < S:
        reach = (torch.matmul(reach, reach) > 0).float()
        n *= 2
    return reach > 0


def _plain_tree(s):
    q, table, lens, new = s["q"], s["table"], s["lens"].long(), s["new_lens"].long()
    B, Hq, S, D = q.shape
    k, v = _gather(s["kc"], table), _gather(s["vc"], table)
    H, n = k.shape[1], k.shape[2]
    draft = torch.arange(n, device=q.device) - (lens - new)[:, None]  # [B, n], negative in the context
    follows = _follows(s["parents"], B, S, q.device)
    among = follows.gather(2, draft.clamp(0, S - 1)[:, None, :].expand(B, S, n))
    live = ((draft < 0)[:, None] | among) & (draft < new[:, None])[:, None]
    live = live & (torch.arange(S, device=q.device) < new[:, None])[:, :, None]  # rows behind the last drafted token
    x = torch.matmul(q.float().reshape(B, H, Hq // H * S, D), k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    x = x.reshape(B, H, Hq // H, S, n).masked_fill(~live[:, None, None], -math.inf)
    top = x.amax(4, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(4, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return torch.matmul(p.reshape(B, H, Hq // H * S, n), v).reshape(B, Hq, S, D).to(q.dtype)


def _plain_compact(s):
    kc, vc, kept, lens, new = s["kc"], s["vc"], s["kept"].long(), s["lens"].long(), s["new_lens"].long()
    ps = kc.shape[2]
    count = (kept >= 0).sum(1)
    base = lens - new
    i = torch.arange(kept.shape[1], device=lens.device)[None]
    # places behind the last kept token repeat that one
    i = torch.minimum(i, (count - 1).clamp(min=0)[:, None])
    src, to = base[:, None] + kept.gather(1, i), base[:, None] + i
    page, to_page = s["table"].long().gather(1, src // ps), s["table"].long().gather(1, to // ps)
    for c in (kc, vc):
        c[to_page, :, to % ps] = c[page, :, src % ps]
    return kc, vc, (base + count).int()


def _free_pages(refs):
    """Pages that nobody holds, lowest first, and how many."""
    free = refs == 0
    return torch.sort((~free).int(), stable=True).indices, free.sum()


def _plain_fork(s):
    kc, vc, table, held, lens, refs = s["kc"], s["vc"], s["table"], s["held"].long(), s["lens"].long(), s["refs"]
    src = s["parents"].long()
    ps, (B, W) = kc.shape[2], table.shape
    dev = table.device
    order, n_free = _free_pages(refs)
    n = torch.minimum(lens[src], held[src] * ps)
    full, rest = n // ps, n % ps
    count = (n + ps - 1) // ps
    b = torch.arange(len(src), device=dev)
    first = torch.full((B,), len(src), device=dev).index_reduce_(0, src, b, "amin")
    last = table[src].long().gather(1, full.clamp(max=W - 1)[:, None])[:, 0]
    copies = (rest > 0) & ~((first[src] == b) & (refs[last.clamp(min=0)] == 1))
    fresh = order[(copies.long().cumsum(0) - 1).clamp(min=0)]
    missing = (copies.sum() - n_free).clamp(min=0)
    fits = missing == 0
    # rows that copy nothing write what is there to a page that somebody holds
    to = torch.where(copies, fresh, refs.argmax())
    take = (copies & fits)[:, None, None, None] & (torch.arange(ps, device=dev) < rest[:, None])[:, None, :, None]
    for c in (kc, vc):
        c[to] = torch.where(take, c[last.clamp(min=0)], c[to])
    at = torch.arange(W, device=dev)
    pages = torch.where(copies[:, None] & (at == full[:, None]), fresh[:, None], table[src].long())
    inside = (at < count[:, None]) & fits
    was = at < held[:, None]
    refs.index_add_(0, table.clamp(min=0).reshape(-1).long(), -(was & fits).int().reshape(-1))
    refs.index_add_(0, pages.clamp(min=0).reshape(-1), inside.int().reshape(-1))
    new_table = torch.where(inside, pages, -1).int()
    return (kc, vc, refs, new_table, torch.where(fits, count, 0).int(), torch.where(fits, n, 0).int(),
            missing.int().reshape(1))


def _resize_once(table, held, lens, refs, ps):
    W = table.shape[1]
    order, n_free = _free_pages(refs)
    have = held.long()
    want = (lens.long().clamp(0, W * ps) + ps - 1) // ps
    need = (want - have).clamp(min=0)
    upto = need.cumsum(0)
    granted = (upto <= n_free) | (need == 0)
    at = torch.arange(W, device=table.device)
    gone = (at >= want[:, None]) & (at < have[:, None])
    come = granted[:, None] & (at >= have[:, None]) & (at < want[:, None])
    fresh = order[((upto - need - have)[:, None] + at).clamp(0, len(order) - 1)]
    refs.index_add_(0, table.clamp(min=0).reshape(-1).long(), -gone.int().reshape(-1))
    table.copy_(torch.where(come, fresh, table.long()))
    refs.index_add_(0, table.clamp(min=0).reshape(-1).long(), come.int().reshape(-1))
    held.copy_(torch.where(granted, want, have))
    return torch.where(granted, 0, need).int()


def _plain_resize(s):
    table, held, refs, ps = s["table"], s["held"], s["refs"], s["case"]["ps"]
    lacked = _resize_once(table, held, s["more"], refs, ps)
    lacks = _resize_once(table, held, s["less"], refs, ps)
    return table, held, refs, lacked, lacks


PLAIN = {"tree": _plain_tree, "compact": _plain_compact, "fork": _plain_fork, "resize": _plain_resize}


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _own(s):
    import rocm_attn_b200 as ra

    op = s["case"]["op"]
    if op == "tree":
        return ra.attn_tree(s["q"], s["kc"], s["vc"], s["table"], s["lens"], parents=s["parents"],
                            new_lens=s["new_lens"])
    if op == "compact":
        lens = ra.kv_compact(s["kc"], s["vc"], s["table"], s["lens"], s["kept"], s["new_lens"])
        return s["kc"], s["vc"], lens
    if op == "fork":
        return ra.kv_fork(s["kc"], s["vc"], s["table"], s["held"], s["lens"], s["refs"], s["parents"])
    ps = s["case"]["ps"]
    lacked = ra.kv_resize(s["table"], s["held"], s["more"], s["refs"], ps)
    lacks = ra.kv_resize(s["table"], s["held"], s["less"], s["refs"], ps)
    return s["table"], s["held"], s["refs"], lacked, lacks


def run(state):
    if state["case"]["op"] != "fork":
        return _own(state) if own else PLAIN[state["case"]["op"]](state)
    # a beam search goes on with the table that the step before gave it
    if own:
        table, held, lens, missing = _own(state)
    else:
        _, _, _, table, held, lens, missing = _plain_fork(state)
    state["table"], state["held"], state["lens"] = table, held, lens
    return state["kc"], state["vc"], state["refs"], table, held, lens, missing


def work(case):
    B, ps, op = case["B"], case["ps"], case["op"]
    lens = _lens(case)
    pages = sum((n + ps - 1) // ps for n in lens)
    if op == "resize":
        most = sum((n + case["S"] + ps - 1) // ps for n in lens)
        moved = most - (pages if case["S"] else 0)
        # a page's table entry and count are written, its count read, as it comes; as it goes, its count again
        return {"bytes": 24.0 * moved + 32 * B + 4, "flops": float(2 * moved + B)}
    e, H, D = ELEM[case["dtype"]], case["Hkv"], case["D"]
    if op == "tree":
        n = sum(lens)
        b = n * H * 2 * D * e + 2 * B * case["Hq"] * case["S"] * D * e + 4 * pages + 8 * B
        b += 0 if case["chain"] else 4 * B * case["S"]
        return {"bytes": b, "flops": 4.0 * case["Hq"] * D * sum(a * c for a, c in zip(lens, _drafted(case)))}
    if op == "compact":
        # paths differ by seed; about the depth of a random token, less those that stay
        moved = sum(0.6 * math.sqrt(n) for n in _drafted(case))
        return {"bytes": moved * H * 4 * D * e + 4 * B * (case["S"] + 3) + 8 * moved, "flops": moved * H * D}
    # about two of five beams are copies
    rest = sum(n % ps for n in lens) * 0.4
    return {"bytes": rest * H * 4 * D * e + 12 * pages + 16 * B, "flops": float(pages)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence after another
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    B, ps, op = case["B"], case["ps"], case["op"]
    if op == "resize":
        table, held, refs = (s[k].tolist() for k in ("table", "held", "refs"))
        answers = []
        for lens in (s["more"].tolist(), s["less"].tolist()):
            free = [p for p, r in enumerate(refs) if r == 0]
            answers.append([])
            used = asked = 0
            for b in range(B):
                want = -(-lens[b] // ps)
                asked += max(0, want - held[b])
                lack = want - held[b] if want > held[b] and asked > len(free) else 0
                for j in range(want, held[b]):
                    refs[table[b][j]] -= 1
                for j in range(held[b], 0 if lack else want):
                    table[b][j] = free[used]
                    refs[free[used]] += 1
                    used += 1
                answers[-1].append(lack)
                held[b] = held[b] if lack else want
        return tuple(torch.tensor(x, dtype=torch.int32) for x in (table, held, refs, *answers))
    kc, vc, table, lens = s["kc"], s["vc"], s["table"].tolist(), s["lens"].tolist()
    dev = kc.device
    if op == "compact":
        out = []
        for b, (n, new) in enumerate(zip(lens, _drafted(case))):
            path = [a for a in s["kept"][b].tolist() if a >= 0]
            for i, a in enumerate(path):
                (p, r), (x, y) = (divmod(n - new + t, ps) for t in (i, a))
                for c in (kc, vc):
                    c[table[b][p], :, r] = c[table[b][x], :, y]
            out.append(n - new + len(path))
        return kc, vc, torch.tensor(out, dtype=torch.int32)
    if op == "fork":
        refs, src = s["refs"].tolist(), s["parents"].tolist()
        before = list(refs)
        free = [p for p, r in enumerate(refs) if r == 0]
        new_table, taken, used = [], set(), 0
        for b in range(B):
            for p in table[b]:
                if p >= 0:
                    refs[p] -= 1
        for b, a in enumerate(src):
            row = [p for p in table[a] if p >= 0]
            rest = lens[a] % ps
            if rest and (a in taken or before[row[-1]] != 1):
                for c in (kc, vc):
                    c[free[used], :, :rest] = c[row[-1], :, :rest]
                row[-1] = free[used]
                used += 1
            taken.add(a)
            for p in row:
                refs[p] += 1
            new_table.append(row + [-1] * (len(table[0]) - len(row)))
        n = [lens[a] for a in src]
        ints = (refs, new_table, [-(-x // ps) for x in n], n, [0])
        return (kc, vc, *(torch.tensor(x, dtype=torch.int32) for x in ints))
    H, D, S, g = case["Hkv"], case["D"], case["S"], case["Hq"] // case["Hkv"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    trees = [list(range(-1, S - 1))] * B if case["chain"] else _trees(case, seed)
    for b, (n, new) in enumerate(zip(lens, _drafted(case))):
        hidden = torch.ones(new, n, dtype=torch.bool)
        hidden[:, :n - new] = False
        for t in range(new):
            hidden[t, [n - new + a for a in _path(trees[b], t)]] = False
        hidden = hidden.to(dev)
        at = torch.arange(n, device=dev)
        page = torch.tensor(table[b], device=dev)[at // ps]
        for h in range(H):
            k, v = kc[page, h, at % ps].double(), vc[page, h, at % ps].double()
            x = (s["q"][b, h * g:(h + 1) * g, :new].double() @ k.t()) / D ** 0.5
            o[b, h * g:(h + 1) * g, :new] = torch.softmax(x.masked_fill(hidden, -math.inf), 2) @ v
    return o
