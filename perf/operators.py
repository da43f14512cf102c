"""The paged key-value cache operators as a generating program calls them, with plain forms of each.

A case is one call (for the sparse form: the selection and the attention over what it selected) of a decoding
loop at stated sizes.  ``own`` chooses between the plain forms (elementary torch operations in 32 bits, 64 for
the page scores) and the package's operators.

Cache layout: k_cache and v_cache [num_pages, Hkv, page_size, D]; token t of sequence b lies in page
block_table[b, t // page_size], row t % page_size; seq_lens counts the tokens of each sequence, the newest
included.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ELEM = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # One user, one new token, a few hundred tokens of context: launch latency.
        dict(name="decode one bf16", op="decode", dtype="bf16", B=1, Hq=32, Hkv=8, D=128, ps=16, L=517, weights=False),
        # A serving batch of mixed lengths whose accumulated attention weights are kept for eviction.
        dict(name="decode weights bf16", op="decode", dtype="bf16", B=24, Hq=32, Hkv=8, D=128, ps=16, L=4096, weights=True),
        # A large batch of long contexts, eight query heads to a kv head.
        dict(name="decode long fp16", op="decode", dtype="fp16", B=64, Hq=64, Hkv=8, D=128, ps=64, L=16384, weights=False),
        # One kv head per query head at D = 64, odd lengths, a page size that is no power of two.
        dict(name="decode d64 fp16", op="decode", dtype="fp16", B=17, Hq=16, Hkv=16, D=64, ps=24, L=2047, weights=False),
        # A few long contexts, each kv head reading 64 pages of 16 tokens out of up to 1024.
        dict(name="sparse few bf16", op="sparse", dtype="bf16", B=3, Hq=32, Hkv=8, D=128, ps=16, L=16384, top=64),
        # A batch of long contexts, 128 pages of 32 tokens out of up to 1024.
        dict(name="sparse batch fp16", op="sparse", dtype="fp16", B=32, Hq=32, Hkv=8, D=128, ps=32, L=32768, top=128),
        # The write of one decoding step: one new token per sequence, page bounds kept.
        dict(name="append step bf16", op="append", dtype="bf16", B=64, Hkv=8, D=128, ps=16, L=4096, S=1),
        # The write of a batch of prompts of mixed lengths.
        dict(name="append prompts fp16", op="append", dtype="fp16", B=8, Hkv=8, D=128, ps=64, L=8192, S=8192),
        # Page bounds of one context, fp32 cache; and of a batch of long ones.
        dict(name="bounds one fp32", op="bounds", dtype="fp32", B=1, Hkv=4, D=64, ps=16, L=5001),
        dict(name="bounds batch bf16", op="bounds", dtype="bf16", B=16, Hkv=8, D=128, ps=32, L=16384),
        # Eviction: one context down to half; a batch of long contexts down to an eighth.
        dict(name="evict one bf16", op="evict", dtype="bf16", B=1, Hkv=8, D=128, ps=16, L=4099, budget=2048, recent=64),
        dict(name="evict batch fp16", op="evict", dtype="fp16", B=16, Hkv=8, D=128, ps=64, L=32768, budget=4096, recent=256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "sparse", "append", "bounds", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    D = rng.choice([64, 128, 128, rng.choice([32, 80, 96, 256])])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    B = _log_int(rng, 1, 64)
    ps = rng.choice([16, 16, 32, 64, rng.choice([8, 24, 128])])
    row = Hkv * D * ELEM[dtype] * 2
    # at most 1 GiB of cache per case, so that no drawn case costs more than the largest listed one
    top_len = max(128, min(32768, (1 << 30) // (row * B)))
    L = _log_int(rng, 64, top_len)
    c = dict(op=op, dtype=dtype, B=B, Hkv=Hkv, D=D, ps=ps, L=L)
    if op in ("decode", "sparse"):
        c["Hq"] = Hkv * rng.choice([1, 2, 4, 7, 8, 16])
    if op == "decode":
        c["weights"] = rng.random() < 0.3
    if op == "sparse":
        c["top"] = rng.randint(1, max(1, (L + ps - 1) // ps))
    if op == "append":
        c["S"] = 1 if rng.random() < 0.5 else rng.randint(1, L)
    if op == "evict":
        c["budget"] = rng.randint(max(1, L // 8), L)
        c["recent"] = rng.randint(0, c["budget"] // 4)
    return c


def _lens(case):
    """The lengths of the case's sequences: between a quarter of L and L, the first L itself."""
    r = random.Random("%d.%d.%d" % (case["B"], case["L"], case["ps"]))
    L = case["L"]
    return [L] + [r.randint(max(1, L // 4), L) for _ in range(case["B"] - 1)]


def _new_lens(case):
    """How many of each sequence's tokens are new."""
    r = random.Random("new %d.%d" % (case["B"], case["S"]))
    return [min(n, case["S"]) if case["S"] == 1 or i == 0 else r.randint(1, min(n, case["S"]))
            for i, n in enumerate(_lens(case))]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    B, Hkv, D, ps = case["B"], case["Hkv"], case["D"], case["ps"]
    lens = _lens(case)
    counts = [(n + ps - 1) // ps for n in lens]
    width = max(counts)
    budget = case.get("budget", 0)
    new_width = (budget + ps - 1) // ps
    total = sum(counts) + B * new_width
    # pages are handed out in random order, as after many sequences have come and gone
    order = torch.randperm(total, generator=g, device=dev, dtype=torch.int32)
    at = torch.arange(width, device=dev)[None, :]
    n_pages = torch.tensor(counts, device=dev)[:, None]
    first = torch.tensor([sum(counts[:b]) for b in range(B)], device=dev)[:, None]
    table = torch.where(at < n_pages, order[(first + at).clamp(max=total - 1)], -1).to(torch.int32).contiguous()
    kc = torch.randn(total, Hkv, ps, D, generator=g, device=dev, dtype=dtype)
    vc = torch.randn(total, Hkv, ps, D, generator=g, device=dev, dtype=dtype)
    s = dict(case=case, kc=kc, vc=vc, table=table, lens=torch.tensor(lens, device=dev, dtype=torch.int32))
    op = case["op"]
    if op in ("decode", "sparse"):
        s["q"] = torch.randn(B, case["Hq"], 1, D, generator=g, device=dev, dtype=dtype)
    if op == "decode" and case["weights"]:
        s["weights"] = torch.rand(B, Hkv, width * ps, generator=g, device=dev)
    if op == "sparse":
        # keys of one page are about one matter: a common part per page, so that pages differ in score
        kc += torch.randn(total, Hkv, 1, D, generator=g, device=dev, dtype=dtype) * 0.5
    if op == "append":
        S = case["S"]
        new = _new_lens(case)
        s["k"] = torch.randn(B, Hkv, S, D, generator=g, device=dev, dtype=dtype)
        s["v"] = torch.randn(B, Hkv, S, D, generator=g, device=dev, dtype=dtype)
        s["new_lens"] = None if S == 1 else torch.tensor(new, device=dev, dtype=torch.int32)
    if op in ("sparse", "append", "bounds"):
        rows = torch.full((total,), ps, device=dev)
        last = torch.tensor([n - (c - 1) * ps for n, c in zip(lens, counts)], device=dev)
        rows[table.gather(1, n_pages - 1)[:, 0].long()] = last
        if op == "append" and case["S"] == 1:
            rows[table.gather(1, n_pages - 1)[:, 0].long()] = (last - 1).clamp(min=1)
        gone = torch.arange(ps, device=dev)[None, None, :, None] >= rows[:, None, None, None]
        s["bounds"] = torch.stack([kc.masked_fill(gone, math.inf).amin(2), kc.masked_fill(gone, -math.inf).amax(2)], 2)
        if op == "bounds":
            s["bounds"].zero_()
    if op == "evict":
        # accumulated softmax weights: a few tokens hold most, many nearly nothing, some exactly nothing
        w = torch.exp(torch.randn(B, Hkv, width * ps, generator=g, device=dev) * 3 - 4)
        w = w * (torch.rand(B, Hkv, width * ps, generator=g, device=dev) > 0.02)
        pos = torch.arange(width * ps, device=dev)
        s["weights"] = torch.where(pos < s["lens"][:, None, None], w, 0.0)
        s["new_table"] = order[sum(counts):].reshape(B, new_width).contiguous()
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


def _plain_attention(q, k, v, live):
    """q [B, Hq, 1, D], k and v [B, Hkv, n, D] in 32 bits, live [B, 1 or Hkv, n] -> weights [B, Hkv, g, n], O."""
    B, Hq, _, D = q.shape
    H = k.shape[1]
    qf = q.float().reshape(B, H, Hq // H, D)
    s = torch.matmul(qf, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    s = s.masked_fill(~live[:, :, None, :], -math.inf)
    p = torch.exp(s - s.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    return p, torch.matmul(p, v).reshape(B, Hq, 1, D).to(q.dtype)


def _plain_decode(s):
    table, lens = s["table"], s["lens"]
    ps = s["kc"].shape[2]
    live = torch.arange(table.shape[1] * ps, device=lens.device) < lens[:, None]
    p, o = _plain_attention(s["q"], _gather(s["kc"], table), _gather(s["vc"], table), live[:, None])
    if "weights" not in s:
        return o
    s["weights"] += p.sum(2)
    return o, s["weights"]


def _plain_select(q, bounds, table, lens, ps, top):
    B, Hq, _, D = q.shape
    H = bounds.shape[1]
    W = table.shape[1]
    qd = q.double().reshape(B, H, Hq // H, D)
    up, down = qd.clamp(min=0).sum(2), qd.clamp(max=0).sum(2)
    b = bounds[table.clamp(min=0).long()].double()  # [B, W, H, 2, D]
    score = (b[:, :, :, 1] * up[:, None] + b[:, :, :, 0] * down[:, None]).sum(3).transpose(1, 2)
    n_pages = ((lens + ps - 1) // ps)[:, None, None]
    page = torch.arange(W, device=q.device)
    score = torch.where(page == n_pages - 1, math.inf, score)
    score = torch.where(page < n_pages, score, -math.inf)
    picked = torch.sort(score, dim=2, descending=True, stable=True).indices[:, :, :top]
    picked = torch.sort(torch.where(picked < n_pages, picked, W), dim=2).values
    picked = torch.where(picked < W, picked, -1).to(torch.int32)
    return torch.nn.functional.pad(picked, (0, top - picked.shape[2]), value=-1)


def _plain_sparse(s):
    case = s["case"]
    ps, top = case["ps"], case["top"]
    table, lens = s["table"], s["lens"]
    pages = _plain_select(s["q"], s["bounds"], table, lens, ps, top)
    B, H, n = pages.shape
    physical = table.long().gather(1, pages.clamp(min=0).long().reshape(B, H * n)).reshape(B, H, n)
    heads = torch.arange(H, device=table.device)[None, :, None]
    k, v = (c[physical.clamp(min=0), heads].reshape(B, H, n * ps, -1).float() for c in (s["kc"], s["vc"]))
    pos = pages[..., None] * ps + torch.arange(ps, device=table.device)
    live = (pages[..., None] >= 0) & (pos < lens[:, None, None, None])
    _, o = _plain_attention(s["q"], k, v, live.reshape(B, H, n * ps))
    return o, pages


def _plain_append(s):
    k, v, kc, vc, bounds = s["k"], s["v"], s["kc"], s["vc"], s["bounds"]
    B, H, S, D = k.shape
    P, _, ps, _ = kc.shape
    lens = s["lens"].long()
    new = s["new_lens"].long() if s["new_lens"] is not None else torch.full_like(lens, S)
    # tokens behind a sequence's last new one repeat that one
    t = torch.minimum(torch.arange(S, device=lens.device)[None], new[:, None] - 1)
    pos = (lens - new)[:, None] + t
    page, row = s["table"].long().gather(1, pos // ps).reshape(-1), (pos % ps).reshape(-1)
    kn, vn = (x.transpose(1, 2).gather(1, t[:, :, None, None].expand(B, S, H, D)).reshape(B * S, H, D) for x in (k, v))
    kc[page, :, row] = kn
    vc[page, :, row] = vn
    begun = torch.zeros(P, dtype=torch.int32, device=lens.device).index_reduce_(0, page, (row == 0).int(), "amax") > 0
    lo = bounds[:, :, 0].float().masked_fill(begun[:, None, None], math.inf).index_reduce_(0, page, kn.float(), "amin")
    hi = bounds[:, :, 1].float().masked_fill(begun[:, None, None], -math.inf).index_reduce_(0, page, kn.float(), "amax")
    bounds.copy_(torch.stack([lo, hi], 2))
    return kc, vc, bounds


def _plain_bounds(s):
    kc, table, bounds = s["kc"], s["table"], s["bounds"]
    ps = kc.shape[2]
    k = kc[table.clamp(min=0).long()].float()  # [B, W, H, ps, D]
    B, W = table.shape
    pos = torch.arange(W * ps, device=table.device).reshape(1, W, 1, ps, 1)
    gone = pos >= s["lens"][:, None, None, None, None]
    new = torch.stack([k.masked_fill(gone, math.inf).amin(3), k.masked_fill(gone, -math.inf).amax(3)], 3).to(kc.dtype)
    # pages behind a sequence's last one repeat its first
    page = torch.arange(W, device=table.device)[None]
    use = torch.where(page < (s["lens"][:, None] + ps - 1) // ps, page, 0).long()
    bounds[table.long().gather(1, use)] = new.gather(1, use[:, :, None, None, None].expand_as(new))
    return bounds


def _plain_evict(s):
    case = s["case"]
    budget, recent = case["budget"], case["recent"]
    kc, vc, w, lens, new_table = s["kc"], s["vc"], s["weights"], s["lens"], s["new_table"]
    ps = kc.shape[2]
    B, H, n = w.shape
    pos = torch.arange(n, device=w.device)
    ln = lens[:, None, None]
    key = torch.where(pos >= ln - recent, math.inf, w)
    key = torch.where(pos < ln, key, -math.inf)
    kept = torch.sort(key, dim=2, descending=True, stable=True).indices[:, :, :budget]
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=n)
    kept = torch.sort(torch.where(kept < ln, kept, n), dim=2).values
    new_lens = lens.clamp(max=budget)
    # places behind the last kept token repeat the first one
    place = torch.arange(budget, device=w.device)[None, None]
    place = torch.where(place < new_lens[:, None, None], place, 0).expand(B, H, budget)
    src = kept.gather(2, place)
    heads = torch.arange(H, device=w.device)[None, :, None]
    page = s["table"].long().gather(1, (src // ps).reshape(B, -1)).reshape(src.shape)
    to = new_table.long().gather(1, (place // ps).reshape(B, -1)).reshape(src.shape)
    kc[to, heads, place % ps] = kc[page, heads, src % ps]
    vc[to, heads, place % ps] = vc[page, heads, src % ps]
    live = kept < n
    new_w = torch.where(live, w.gather(2, kept.clamp(max=n - 1)), 0.0)
    new_w = torch.nn.functional.pad(new_w, (0, new_table.shape[1] * ps - budget))
    return kc, vc, new_w, torch.where(live, kept, -1).to(torch.int32), new_lens


PLAIN = {"decode": _plain_decode, "sparse": _plain_sparse, "append": _plain_append, "bounds": _plain_bounds,
         "evict": _plain_evict}


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _own(s):
    import rocm_attn_b200 as ra

    op = s["case"]["op"]
    kc, vc, table, lens = s["kc"], s["vc"], s["table"], s["lens"]
    if op == "decode":
        if "weights" in s:
            return ra.attn_decode(s["q"], kc, vc, table, lens, weights=s["weights"]), s["weights"]
        return ra.attn_decode(s["q"], kc, vc, table, lens)
    if op == "sparse":
        pages = ra.kv_select_pages(s["q"], s["bounds"], table, lens, s["case"]["ps"], s["case"]["top"])
        return ra.attn_decode(s["q"], kc, vc, table, lens, pages=pages), pages
    if op == "append":
        ra.kv_append(s["k"], s["v"], kc, vc, table, lens, new_lens=s["new_lens"], bounds=s["bounds"])
        return kc, vc, s["bounds"]
    if op == "bounds":
        return ra.kv_page_bounds(kc, table, lens, bounds=s["bounds"])
    new_lens, new_w, kept = ra.kv_evict(kc, vc, table, lens, s["weights"], s["new_table"], s["case"]["budget"],
                                        recent=s["case"]["recent"])
    return kc, vc, new_w, kept, new_lens


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    e, H, D, ps, B = ELEM[case["dtype"]], case["Hkv"], case["D"], case["ps"], case["B"]
    lens = _lens(case)
    pages = sum((n + ps - 1) // ps for n in lens)
    op = case["op"]
    if op == "decode":
        n = sum(lens)
        b = n * H * 2 * D * e + 2 * B * case["Hq"] * D * e + 4 * pages + 4 * B
        return {"bytes": b + (8 * n * H if case["weights"] else 0), "flops": 4.0 * case["Hq"] * D * n}
    if op == "sparse":
        # the selected pages are taken as full; the newest is short by less than a page
        n = sum(min(n, case["top"] * ps) for n in lens)
        b = pages * H * 2 * D * e + n * H * 2 * D * e + 2 * B * case["Hq"] * D * e + 4 * pages + 4 * B * H * case["top"]
        return {"bytes": b, "flops": 4.0 * case["Hq"] * D * n + 4.0 * pages * H * D}
    if op == "append":
        new = _new_lens(case)
        touched = sum((n - 1) // ps - (n - m) // ps + 1 for n, m in zip(lens, new))
        begun = sum((n - 1) // ps - (n - m - 1) // ps for n, m in zip(lens, new))
        # K and V rows in and out; bounds written, and read where a page was begun before
        b = sum(new) * H * 4 * D * e + (2 * touched - begun) * H * 2 * D * e + 4 * touched
        return {"bytes": b, "flops": 2.0 * sum(new) * H * D}
    if op == "bounds":
        return {"bytes": sum(lens) * H * D * e + pages * H * 2 * D * e + 4 * pages, "flops": 2.0 * sum(lens) * H * D}
    kept = sum(min(n, case["budget"]) for n in lens)
    width = (case["budget"] + ps - 1) // ps * ps
    b = kept * H * 4 * D * e + 4 * H * (sum(lens) + B * (width + case["budget"])) + 4 * pages
    return {"bytes": b, "flops": float(H * sum(lens))}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence (and kv head) after another
# ---------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op, B, H, ps = case["op"], case["B"], case["Hkv"], case["ps"]
    lens, table, kc, vc = s["lens"].tolist(), s["table"].tolist(), s["kc"], s["vc"]

    def rows(cache, b, h, tokens):
        """The rows of these tokens of (sequence b, kv head h), in 64 bits."""
        t = torch.as_tensor(tokens, device=cache.device)
        page = torch.tensor(table[b], device=cache.device)[t // ps]
        return cache[page, h, t % ps].double()

    def softmax(q, k, D):
        x = (k @ q.t()).t() / D ** 0.5
        e = torch.exp(x - x.max(dim=1, keepdim=True).values)
        return e / e.sum(dim=1, keepdim=True)

    if op in ("decode", "sparse"):
        D, g = case["D"], case["Hq"] // H
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device=kc.device)
        w = s["weights"].double() if "weights" in s else None
        picks = torch.full((B, H, case.get("top", 0)), -1, dtype=torch.int32, device=kc.device)
        for b in range(B):
            for h in range(H):
                q = s["q"][b, h * g:(h + 1) * g, 0].double()
                tokens = torch.arange(lens[b], device=kc.device)
                if op == "sparse":
                    n = (lens[b] + ps - 1) // ps
                    lo, hi = s["bounds"][torch.tensor(table[b][:n], device=kc.device), h].double().unbind(1)
                    score = torch.maximum(q[:, None] * lo, q[:, None] * hi).sum((0, 2)).tolist()
                    best = sorted(range(n - 1), key=lambda i: (-score[i], i))[:case["top"] - 1]
                    chosen = sorted(best + [n - 1])
                    picks[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
                    is_in = torch.zeros(n, dtype=torch.bool, device=kc.device)
                    is_in[torch.tensor(chosen, device=kc.device)] = True
                    tokens = tokens[is_in[tokens // ps]]
                p = softmax(q, rows(kc, b, h, tokens), D)
                o[b, h * g:(h + 1) * g, 0] = p @ rows(vc, b, h, tokens)
                if w is not None:
                    w[b, h, :lens[b]] += p.sum(0)
        return (o, picks) if op == "sparse" else o if w is None else (o, w)
    if op == "append":
        bounds = s["bounds"]
        for b, (n, m) in enumerate(zip(lens, _new_lens(case))):
            t = n - m
            while t < n:
                page, end = table[b][t // ps], min(n, (t // ps + 1) * ps)
                x = s["k"][b, :, t - (n - m):end - (n - m)]
                kc[page, :, t % ps:t % ps + end - t] = x
                vc[page, :, t % ps:t % ps + end - t] = s["v"][b, :, t - (n - m):end - (n - m)]
                lo, hi = x.amin(1), x.amax(1)
                if t % ps:
                    lo, hi = torch.minimum(lo, bounds[page, :, 0]), torch.maximum(hi, bounds[page, :, 1])
                bounds[page, :, 0], bounds[page, :, 1] = lo, hi
                t = end
        return kc, vc, bounds
    if op == "bounds":
        bounds = s["bounds"]
        for b, n in enumerate(lens):
            full = n // ps
            if full:
                x = kc[torch.tensor(table[b][:full], device=kc.device)]
                bounds[torch.tensor(table[b][:full], device=kc.device)] = torch.stack([x.amin(2), x.amax(2)], 2)
            if n % ps:
                x = kc[table[b][full], :, :n % ps]
                bounds[table[b][full]] = torch.stack([x.amin(1), x.amax(1)], 1)
        return bounds
    budget, recent = case["budget"], case["recent"]
    new_table = s["new_table"].tolist()
    new_w = torch.zeros(B, H, len(new_table[0]) * ps, device=kc.device)
    kept = torch.full((B, H, budget), -1, dtype=torch.int32, device=kc.device)
    for b, n in enumerate(lens):
        m = min(n, budget)
        to = torch.tensor(new_table[b], device=kc.device)[torch.arange(m, device=kc.device) // ps]
        for h in range(H):
            w = s["weights"][b, h, :n].cpu().numpy()
            order = (-w[:max(0, n - recent)].astype("f8")).argsort(kind="stable")[:m - min(recent, n)]
            t = torch.cat([torch.from_numpy(order).sort().values, torch.arange(n - min(recent, n), n)]).to(kc.device)
            kept[b, h, :m] = t.int()
            new_w[b, h, :m] = s["weights"][b, h][t]
            for c in (kc, vc):
                page = torch.tensor(table[b], device=kc.device)[t // ps]
                c[to, h, torch.arange(m, device=kc.device) % ps] = c[page, h, t % ps]
    return kc, vc, new_w, kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=kc.device)
