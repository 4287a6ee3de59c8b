"""Cases for the paged key / value cache and the filtered sampler: what a program that serves many sequences at once calls
between two layers, between two steps and between two requests.

  attend     queries of every sequence's newest tokens against its pages of the cache (one token each, or a chunk)
  write      new key / value rows into the pages (`admit`: with the pages reserved before and released afterwards)
  resample   sequences released and others forked into their rows; compact: live pages moved together; copy: page contents
  sample     one token a row after temperature, top-k, top-p and min-p, from given uniform numbers

A sequence is a row of `table` (page numbers, -1 where there is none) and an entry of `lens`; `ref` counts, per page, the
rows that name it (0: free).  `own` chooses between the plain torch form of each operator and the framework's.
"""
import math
import random

import torch

own = False

DENSE, BLOCK, TRANSPOSE, PREV = 0, 1, 2, 3
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def attend(name, dtype, n_seq, heads, kv_heads, d_head, page, min_len, max_len, min_q=1, max_q=1, func=DENSE, block_ctx=0, window=0):
    return {"name": name, "kind": "attend", "dtype": dtype, "n_seq": n_seq, "heads": heads, "kv_heads": kv_heads, "d_head": d_head,
            "page": page, "min_len": min_len, "max_len": max_len, "min_q": min_q, "max_q": max_q, "func": func,
            "block_ctx": block_ctx, "window": window}


def listed():
    return [
        # one stream of a two-head prior in single precision, early in its song: nothing but latency
        attend("one_token_small_f32", "f32", 1, 2, 2, 256, 16, 300, 300),
        # 16 samples of an upsampler (one head of 480 channels), positions all over the second half of the context
        attend("one_token_480_f16", "f16", 16, 1, 1, 480, 64, 4096, 8192),
        # a full serving batch with shared key / value heads, short and long sequences together: the cache is the work
        attend("one_token_grouped_bf16", "bf16", 64, 32, 8, 128, 16, 511, 8192),
        # prompts taken in chunks behind a long context
        attend("chunk_grouped_bf16", "bf16", 4, 32, 8, 128, 64, 4097, 8192, 257, 2048),
        # the 5b prior's heads (150 channels, no multiple of a vector), primed in odd chunks
        attend("chunk_150_f16", "f16", 3, 8, 8, 150, 32, 1000, 5000, 100, 1000),
        # the rows of one decode step into one layer's pages
        {"name": "write_step_bf16", "kind": "write", "dtype": "bf16", "n_seq": 64, "kv_heads": 8, "d_head": 128, "page": 16, "min_new": 1, "max_new": 1,
         "pages": 4096},
        # sixteen prompts admitted, written and let go
        {"name": "admit_prompts_f16", "kind": "admit", "dtype": "f16", "n_seq": 16, "kv_heads": 2, "d_head": 256, "page": 64, "min_new": 1, "max_new": 6144,
         "pages": 4096},
        # sixteen of 32 samples dropped and the rows given to forks of the others: an upsampler's 72 layers
        {"name": "resample_f16", "kind": "resample", "dtype": "f16", "rows": 32, "forks": 16, "pools": 144, "width": 480, "page": 64, "min_len": 1, "max_len": 250,
         "pages": 128},
        # a pool left full of holes, pushed together
        {"name": "compact_f16", "kind": "compact", "dtype": "f16", "rows": 64, "pools": 32, "width": 512, "page": 16, "pages": 2048, "live": 0.6},
        # written-to pages of a shared prefix taken apart: 1200 channels, ten rows a page
        {"name": "copy_pages_bf16", "kind": "copy", "dtype": "bf16", "pools": 16, "width": 1200, "page": 10, "pages": 512, "pairs": 61},
        # a decode step's draw over the codebook
        {"name": "sample_codes_f32", "kind": "sample", "dtype": "f32", "rows": 16, "bins": 2048, "filters": "p"},
        # a serving batch over a text vocabulary, every row with settings of its own
        {"name": "sample_text_bf16", "kind": "sample", "dtype": "bf16", "rows": 256, "bins": 128000, "filters": "mixed"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "write", "admit", "resample", "compact", "copy", "sample", "sample", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "attend":
        heads, kv_heads, d = rng.choice([(1, 1, 480), (2, 2, 256), (8, 8, 150), (32, 8, 128), (16, 16, 64), (8, 1, 128), (6, 2, 80), (5, 5, 33), (4, 4, 512)])
        page = rng.choice([1, 8, 16, 20, 48, 64, 128])
        one = rng.random() < 0.5
        n_seq = _log(rng, 1, 64 if one else 8)
        # no more bytes of cache than the largest listed case of one token has, no more products than the largest of chunks
        max_len = _log(rng, 1, min(16384, (64 * 4352 * 8 * 128 * 2) // (n_seq * kv_heads * d * SIZE[dtype])))
        max_q = 1 if one else _log(rng, 2, max(2, min(max_len, 118_000_000_000 // (n_seq * heads * d * max_len))))
        max_len = max(max_len, max_q)
        c = attend("", dtype, n_seq, heads, kv_heads, d, page, rng.randint(1, max_len), max_len, 1 if one else rng.randint(0, max_q), max_q)
        form = rng.random()
        if form < 0.25:
            c["window"] = _log(rng, 1, max_len)
        elif form < 0.5:
            c["func"], c["block_ctx"] = rng.choice([BLOCK, TRANSPOSE, PREV]), _log(rng, 1, 256)
        del c["name"]
        return c
    if kind in ("write", "admit"):
        heads, d = rng.choice([(1, 480), (2, 256), (8, 150), (8, 128), (5, 33)])
        n_seq, page = _log(rng, 1, 64), rng.choice([1, 8, 16, 20, 64])
        most = _log(rng, 1, min(6144, 16 * 6144 * 1024 // (n_seq * heads * d * SIZE[dtype])))
        need = n_seq * -(-most // page)
        return {"kind": kind, "dtype": dtype, "n_seq": n_seq, "kv_heads": heads, "d_head": d, "page": page, "min_new": rng.randint(0, most), "max_new": most,
                "pages": need + _log(rng, 1, 2048)}
    if kind == "resample":
        rows = _log(rng, 2, 64)
        pools, width, page = _log(rng, 2, 144), rng.choice([480, 512, 1200, 99]), rng.choice([4, 16, 40, 64])
        most = _log(rng, 1, 5 * page)
        pages = rows * -(-most // page) + rows
        if pools * pages * page * width * SIZE[dtype] > 144 * 64 * 64 * 480 * 2:
            pools = max(1, (144 * 64 * 64 * 480 * 2) // (pages * page * width * SIZE[dtype]))
        return {"kind": kind, "dtype": dtype, "rows": rows, "forks": rng.randint(1, rows // 2), "pools": pools, "width": width, "page": page,
                "min_len": rng.randint(0, most), "max_len": most, "pages": pages}
    if kind in ("compact", "copy"):
        width, page = rng.choice([480, 512, 1200, 99]), rng.choice([1, 10, 16, 64])
        pages = _log(rng, 8, 4096)
        pools = _log(rng, 1, max(1, min(64, (32 * 2048 * 16 * 512 * 2) // (pages * page * width * SIZE[dtype]))))
        if pools * pages * page * width * SIZE[dtype] > 32 * 2048 * 16 * 512 * 2:
            pages = max(8, (32 * 2048 * 16 * 512 * 2) // (pools * page * width * SIZE[dtype]))
        c = {"kind": kind, "dtype": dtype, "pools": pools, "width": width, "page": page, "pages": pages}
        return {**c, "pairs": rng.randint(1, pages // 2)} if kind == "copy" else {**c, "rows": _log(rng, 1, 64), "live": rng.uniform(0.05, 1.0)}
    rows = _log(rng, 1, 512)
    bins = _log(rng, 2, min(262144, 256 * 128000 * 2 // (rows * SIZE[dtype])))
    return {"kind": "sample", "dtype": dtype, "rows": rows, "bins": bins, "filters": rng.choice(["none", "k", "p", "m", "mixed", "mixed"])}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi at even distances: a batch's lengths are a matter of the case, their order of the seed."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(case):
    lens = _spread(case["min_len"], case["max_len"], case["n_seq"])
    return lens, [min(a, b) for a, b in zip(_spread(case["min_q"], case["max_q"], case["n_seq"]), lens)]


def _news(case):
    return _spread(case["min_new"], case["max_new"], case["n_seq"])


def _table(rng, lens, page, pages, width):
    """Random pages for sequences of these lengths: (rows of page numbers, references per page)."""
    free = list(range(pages))
    rng.shuffle(free)
    rows, ref = [], [0] * pages
    for n in lens:
        mine = [free.pop() for _ in range(-(-n // page))]
        for p in mine:
            ref[p] += 1
        rows.append(mine + [-1] * (width - len(mine)))
    return rows, ref


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    dev, dt = "cuda", TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    def ints(v, kind=torch.int32):
        return torch.tensor(v, dtype=kind, device=dev)

    kind, s = case["kind"], {"kind": case["kind"], "status": torch.zeros(1, dtype=torch.int32, device=dev)}
    if kind == "attend":
        lens, qs = _lens(case)
        both = list(zip(lens, qs))
        rng.shuffle(both)
        lens, qs = [b[0] for b in both], [b[1] for b in both]
        H, KV, D, page = case["heads"], case["kv_heads"], case["d_head"], case["page"]
        width = -(-case["max_len"] // page)
        pages = sum(-(-n // page) for n in lens) + 3
        rows, _ = _table(rng, lens, page, pages, width)
        cu = [sum(qs[:i]) for i in range(len(qs) + 1)]
        kp, vp = normal(pages, page, KV, D), normal(pages, page, KV, D)
        return {**s, "q": normal(cu[-1], H, D), "k": kp, "v": vp, "table": ints(rows), "lens": ints(lens), "cu": ints(cu),
                "max_q": case["max_q"], "max_len": case["max_len"], "func": case["func"], "block_ctx": case["block_ctx"], "window": case["window"]}
    if kind in ("write", "admit"):
        news = _news(case)
        rng.shuffle(news)
        H, D, page, pages = case["kv_heads"], case["d_head"], case["page"], case["pages"]
        cu = [sum(news[:i]) for i in range(len(news) + 1)]
        s.update(k=normal(cu[-1], H, D), v=normal(cu[-1], H, D), kp=normal(pages, page, H, D), vp=normal(pages, page, H, D), page=page, tokens=cu[-1])
        width = -(-case["max_new"] // page) + 1
        rows, ref = _table(rng, news, page, pages, width)
        if kind == "write":
            at = [rows[i][j // page] * page + j % page for i, n in enumerate(news) for j in range(n)]
            return {**s, "slots": ints(at, torch.int64)}
        # some pages are other sequences', so that the free ones lie between them
        need = sum(-(-n // page) for n in news)
        ref = [1] * (pages - need) + [0] * need
        rng.shuffle(ref)
        return {**s, "table": ints([[-1] * width] * len(news)), "lens": ints([0] * len(news)), "ref": ints(ref), "cu": ints(cu),
                "rows": ints(list(range(len(news))))}
    if kind == "resample":
        lens = _spread(case["min_len"], case["max_len"], case["rows"])
        rng.shuffle(lens)
        rows, ref = _table(rng, lens, case["page"], case["pages"], -(-case["max_len"] // case["page"]) + 1)
        order = list(range(case["rows"]))
        rng.shuffle(order)
        drop, keep = order[:case["forks"]], order[case["forks"]:]
        pools = normal(case["pools"], case["pages"], case["page"], case["width"])
        return {**s, "pools": pools, "each": list(pools.unbind(0)), "table": ints(rows), "lens": ints(lens), "ref": ints(ref), "page": case["page"],
                "src": ints([rng.choice(keep) for _ in drop]), "dst": ints(drop)}
    if kind in ("compact", "copy"):
        pools = normal(case["pools"], case["pages"], case["page"], case["width"])
        s.update(pools=pools, each=list(pools.unbind(0)))
        order = list(range(case["pages"]))
        rng.shuffle(order)
        if kind == "copy":
            return {**s, "src": ints(order[:case["pairs"]]), "dst": ints(order[case["pairs"]:2 * case["pairs"]])}
        live = order[:max(1, int(case["live"] * case["pages"]))]
        width = -(-len(live) // case["rows"]) + 2
        rows, ref = [], [0] * case["pages"]
        for i in range(case["rows"]):
            mine = live[i::case["rows"]] + ([live[0]] if i else [])      # everyone shares the first page
            for p in mine:
                ref[p] += 1
            rows.append((mine + [-1] * width)[:width])
        return {**s, "table": ints(rows), "ref": ints(ref)}
    R, V, f = case["rows"], case["bins"], case["filters"]
    x = torch.randn((R, V), generator=g, device=dev) * 2.5
    x += 6.0 * (torch.rand((R, V), generator=g, device=dev) < 20.0 / V)       # a handful of likely tokens
    x[torch.rand((R, V), generator=g, device=dev) < 0.02] = -math.inf          # forbidden ones
    x = x.to(dt)
    x[R // 2, :] = torch.finfo(dt).min                                        # a row that a mask has filled
    x[R // 2, V // 3:] = 0.5
    if R >= 8:
        x[R // 4] = -math.inf                                                 # and one that it leaves nothing

    def each(*choices):
        return torch.tensor([rng.choice(choices) for _ in range(R)], device=dev)

    off_i, off_f = torch.zeros(R, dtype=torch.int32, device=dev), torch.zeros(R, device=dev)
    temp = each(0.7, 0.99, 1.0, 1.3) if f != "mixed" else each(0.0, 0.5, 0.99, 1.0, 1.3)
    top_k = {"k": each(1, 5, 40, 200), "mixed": each(0, 0, 1, 40, 1000, V + 5)}.get(f, off_i).to(torch.int32)
    top_p = {"p": each(0.5, 0.9, 0.95, 0.999), "mixed": each(0.0, 0.3, 0.9, 0.95, 1.0)}.get(f, off_f).to(torch.float32)
    min_p = {"m": each(0.01, 0.05, 0.3), "mixed": each(0.0, 0.0, 0.02, 0.1)}.get(f, off_f).to(torch.float32)
    return {**s, "logits": x, "u": torch.rand(R, generator=g, device=dev), "temp": temp.to(torch.float32), "top_k": top_k, "top_p": top_p, "min_p": min_p}


# ---- plain forms -------------------------------------------------------------------------------------------------------------


def _visible(func, block, window, qpos, kpos):
    """Whether the query at qpos sees the key at kpos (arrays that broadcast)."""
    if func == BLOCK:
        return (kpos <= qpos) & (kpos // block == qpos // block)
    if func == TRANSPOSE:
        return (kpos <= qpos) & ((qpos - kpos) % block == 0)
    if func == PREV:
        return kpos // block == qpos // block - 1
    return (kpos <= qpos) & (kpos > qpos - window) if window else kpos <= qpos


def _plain_attend(s):
    q, table, lens, cu = s["q"], s["table"].long(), s["lens"].long(), s["cu"].long()
    n, (T, H, D), (_, page, KV, _) = table.shape[0], q.shape, s["k"].shape
    G, Q = H // KV, s["max_q"]
    at = table.clamp(min=0)
    k = s["k"][at].reshape(n, -1, KV, D).float().permute(0, 2, 1, 3)                    # [n, KV, L, D]
    v = s["v"][at].reshape(n, -1, KV, D).float().permute(0, 2, 1, 3)
    j = torch.arange(Q, device=q.device)
    nq = cu[1:] - cu[:-1]
    valid = j < nq[:, None]                                                             # [n, Q]
    row = torch.where(valid, cu[:-1, None] + j, T)
    qf = torch.cat([q, q.new_zeros(1, H, D)])[row].float().reshape(n, Q, KV, G, D).permute(0, 2, 3, 1, 4).reshape(n, KV, G * Q, D)
    sc = torch.matmul(qf, k.transpose(-1, -2).contiguous()).reshape(n, KV, G, Q, -1) * (1.0 / math.sqrt(D))
    qpos, kpos = (lens - nq)[:, None, None] + j[:, None], torch.arange(k.shape[2], device=q.device)
    see = _visible(s["func"], s["block_ctx"], s["window"], qpos, kpos) & (kpos < lens[:, None, None])
    sc = sc.masked_fill(~see[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, KV, G * Q, -1), v.contiguous()).reshape(n, KV, G, Q, D) / torch.where(z == 0, 1.0, z)
    out = q.new_zeros(T + 1, H, D)
    out[row.reshape(-1)] = o.permute(0, 3, 1, 2, 4).reshape(n * Q, H, D).to(q.dtype)
    return out[:T]


def _plain_write(s, slots):
    page = s["kp"].shape[1]
    s["kp"][slots // page, slots % page] = s["k"]
    s["vp"][slots // page, slots % page] = s["v"]


def _free_pages(ref):
    """Free pages from the lowest on (garbage behind the last), and their number."""
    free = ref == 0
    rank = torch.where(free, torch.cumsum(free, 0) - 1, ref.numel())
    found = torch.zeros(ref.numel() + 1, dtype=torch.int64, device=ref.device)
    found[rank] = torch.arange(ref.numel(), device=ref.device)
    return found[:-1], free.sum()


def _plain_extend(s):
    table, lens, ref, page, cu = s["table"], s["lens"].long(), s["ref"], s["page"], s["cu"].long()
    new = lens + cu[1:] - cu[:-1]
    had, has = (lens + page - 1) // page, (new + page - 1) // page
    first = torch.cumsum(has - had, 0) - (has - had)
    found, n_free = _free_pages(ref)
    col = torch.arange(table.shape[1], device=table.device)
    fresh = (col >= had[:, None]) & (col < has[:, None])
    fits = ((has - had).sum() <= n_free) & (has <= table.shape[1]).all()
    s["status"].copy_(torch.where(fits, s["status"], 1))
    fresh &= fits
    mine = found[(first[:, None] + col - had[:, None]).clamp(0, ref.numel() - 1)]
    table.copy_(torch.where(fresh, mine, table.long()))
    more = torch.zeros(ref.numel() + 1, dtype=ref.dtype, device=ref.device)
    more.index_add_(0, torch.where(fresh, mine, ref.numel()).reshape(-1), torch.ones(fresh.numel(), dtype=ref.dtype, device=ref.device))
    ref += more[:-1]
    t = torch.arange(s["tokens"], device=table.device)
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=lens.numel() - 1)
    pos = lens[seq] + t - cu[seq]
    slots = table.long()[seq, (pos // page).clamp(max=table.shape[1] - 1)] * page + pos % page
    s["lens"].copy_(torch.where(fits, new, lens))
    return torch.where((t < cu[-1]) & fits, slots, -1)


def _plain_free(s, rows):
    table, lens, ref = s["table"], s["lens"], s["ref"]
    rows = rows.long()
    pages = table[rows].long()
    less = torch.zeros(ref.numel() + 1, dtype=ref.dtype, device=ref.device)
    less.index_add_(0, torch.where(pages < 0, ref.numel(), pages).reshape(-1), torch.ones(pages.numel(), dtype=ref.dtype, device=ref.device))
    ref -= less[:-1]
    table[rows] = -1
    lens[rows] = 0


def _plain_fork(s):
    table, lens, ref, page, pools = s["table"], s["lens"], s["ref"], s["page"], s["pools"]
    src, dst = s["src"].long(), s["dst"].long()
    n = lens[src].long()
    full, part = n // page, (n % page > 0)
    found, n_free = _free_pages(ref)
    fits = part.sum() <= n_free
    s["status"].copy_(torch.where(fits, s["status"], 1))
    mine = found[(torch.cumsum(part, 0) - 1).clamp(0, ref.numel() - 1)]
    col = torch.arange(table.shape[1], device=table.device)
    pages = torch.where(col < full[:, None], table[src].long(), torch.where((col == full[:, None]) & part[:, None], mine[:, None], -1))
    pages = torch.where(fits, pages, table[dst].long())
    more = torch.zeros(ref.numel() + 1, dtype=ref.dtype, device=ref.device)
    more.index_add_(0, torch.where((pages < 0) | ~fits, ref.numel(), pages).reshape(-1), torch.ones(pages.numel(), dtype=ref.dtype, device=ref.device))
    ref += more[:-1]
    old = table.long()[src, full.clamp(max=table.shape[1] - 1)].clamp(min=0)
    table[dst] = pages.to(table.dtype)
    lens[dst] = torch.where(fits, n, lens[dst].long()).to(lens.dtype)
    # a row without a part-filled page copies a page onto itself
    pools[:, torch.where(part & fits, mine, old)] = pools[:, old]


def _plain_compact(s):
    table, ref, pools = s["table"].long(), s["ref"], s["pools"]
    live, at = ref > 0, torch.arange(ref.numel(), device=ref.device)
    n = live.sum()
    src, dst = torch.nonzero(live & (at >= n))[:, 0], torch.nonzero(~live & (at < n))[:, 0]
    to = at.clone()
    to[src] = dst
    moved = torch.zeros_like(ref)
    moved[dst] = ref[src]
    pools[:, dst] = pools[:, src]
    return torch.where(table < 0, -1, to[table.clamp(min=0)]).to(s["table"].dtype), torch.where(at < n, torch.where(live, ref, moved), 0)


def _plain_sample(s):
    x, u, k = s["logits"].double(), s["u"].double(), s["top_k"].long()[:, None]
    T, top_p, min_p = s["temp"].double()[:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    x = torch.where(torch.isnan(x), -math.inf, x)
    at = torch.arange(x.shape[1], device=x.device)
    m = x.amax(1, keepdim=True)
    w = torch.where(x == m, 1.0, torch.exp((x - m) / torch.where(T > 0, T, 1.0)))
    ws, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    ws = torch.where((k <= 0) | (at < k), ws, 0.0)
    cum = torch.cumsum(ws, 1)
    keep = (cum - ws <= top_p * cum[:, -1:]) | (top_p <= 0) | (top_p >= 1)
    ws = torch.where(keep & ((ws >= min_p.clamp(max=1.0)) | (min_p <= 0)), ws, 0.0)
    wk = torch.zeros_like(w).scatter_(1, order, ws)
    cum = torch.cumsum(wk, 1)
    last = torch.where(wk > 0, at, -1).amax(1)
    tok = torch.minimum((cum <= u[:, None] * cum[:, -1:]).sum(1), last)
    first = torch.where(x == m, at, x.shape[1]).amin(1)
    tok = torch.where(T[:, 0] > 0, tok, first)
    return torch.where(m[:, 0] == -math.inf, -1, tok)


def run(s):
    kind = s["kind"]
    if own:
        from jukebox_amd import hip_ops as H
    if kind == "attend":
        if own:
            return H.attn_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], s["max_q"], s["max_len"], func=s["func"],
                                block_ctx=s["block_ctx"], window=s["window"])
        return _plain_attend(s)
    if kind == "write":
        if own:
            H.kv_write(s["k"], s["v"], s["kp"], s["vp"], s["slots"])
        else:
            _plain_write(s, s["slots"])
        return [s["kp"], s["vp"]]
    if kind == "admit":
        if own:
            slots = H.pages_extend(s["table"], s["lens"], s["ref"], s["cu"], s["page"], s["tokens"], s["status"])
            H.kv_write(s["k"], s["v"], s["kp"], s["vp"], slots)
            H.pages_free(s["table"], s["lens"], s["ref"], s["rows"], s["status"])
        else:
            slots = _plain_extend(s)
            _plain_write(s, slots)
            _plain_free(s, s["rows"])
        return [slots, s["kp"], s["vp"], s["table"], s["lens"], s["ref"], s["status"]]
    if kind == "resample":
        if own:
            H.pages_free(s["table"], s["lens"], s["ref"], s["dst"], s["status"])
            H.pages_fork(s["each"], s["table"], s["lens"], s["ref"], s["src"], s["dst"], s["page"], s["status"])
        else:
            _plain_free(s, s["dst"])
            _plain_fork(s)
        return [s["table"], s["lens"], s["ref"], s["status"], s["pools"]]
    if kind == "compact":
        table, ref = H.pages_compact(s["each"], s["table"], s["ref"]) if own else _plain_compact(s)
        return [table, ref, s["pools"]]
    if kind == "copy":
        if own:
            H.pages_copy(s["each"], s["src"], s["dst"])
        else:
            s["pools"][:, s["dst"].long()] = s["pools"][:, s["src"].long()]
        return s["pools"]
    if own:
        return H.sample_filtered(s["logits"], s["u"], s["temp"], s["top_k"], s["top_p"], s["min_p"])
    return _plain_sample(s)


# ---- what one pass cannot do without -----------------------------------------------------------------------------------------


def _seen(case, n, nq):
    """(query, key) pairs of a sequence of n tokens whose last nq are queries, and the keys that any of them sees."""
    func, b, w = case["func"], case["block_ctx"], case["window"]
    pairs, keys = 0, 0
    first = n - nq
    for p in range(first, n):
        pairs += (p % b + 1 if func == BLOCK else p // b + 1 if func == TRANSPOSE else (b if p >= b else 0) if func == PREV
                  else min(p + 1, w) if w else p + 1)
    if nq:
        if func == BLOCK:
            keys = n - first // b * b
        elif func == TRANSPOSE:
            keys = n if nq >= b else sum(p // b + 1 for p in range(first, n))
        elif func == PREV:
            keys = max(0, ((n - 1) // b) * b - max(0, first // b - 1) * b)
        else:
            keys = min(n, nq + w - 1) if w else n
    return pairs, keys


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "attend":
        lens, qs = _lens(case)
        seen = [_seen(case, n, nq) for n, nq in zip(lens, qs)]
        return {"bytes": e * case["d_head"] * (2 * sum(qs) * case["heads"] + 2 * case["kv_heads"] * sum(k for _, k in seen)),
                "flops": 4.0 * case["d_head"] * case["heads"] * sum(p for p, _ in seen)}
    if kind in ("write", "admit"):
        n = sum(_news(case))
        moved = 2 * 2 * n * case["kv_heads"] * case["d_head"] * e + 8 * n
        if kind == "admit":
            moved += 4 * case["pages"] + 8 * n + 3 * 4 * sum(-(-k // case["page"]) for k in _news(case))
        return {"bytes": moved, "flops": 0}
    if kind == "sample":
        return {"bytes": case["rows"] * (case["bins"] * e + 28), "flops": 0}
    page = case["pools"] * case["page"] * case["width"] * e
    if kind == "copy":
        return {"bytes": 2 * case["pairs"] * page, "flops": 0}
    if kind == "compact":
        n = max(1, int(case["live"] * case["pages"]))
        return {"bytes": 2 * page * n * (case["pages"] - n) / case["pages"] + 8 * case["pages"] + 8 * (n + 3 * case["rows"]), "flops": 0}
    lens = _spread(case["min_len"], case["max_len"], case["rows"])
    share = case["forks"] / case["rows"]                     # which rows are dropped is the seed's matter
    return {"bytes": share * (2 * page * sum(n % case["page"] > 0 for n in lens) + 24 * sum(-(-n // case["page"]) for n in lens)) + 4 * case["pages"],
            "flops": 0}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "attend":
        k, v, q, page = s["k"], s["v"], s["q"], s["k"].shape[1]
        H, KV, D = q.shape[1], k.shape[2], q.shape[2]
        lens, cu, out = s["lens"].tolist(), s["cu"].tolist(), []
        for i, n in enumerate(lens):
            nq = cu[i + 1] - cu[i]
            if not nq:
                continue
            at = s["table"][i, :-(-n // page)].long()
            kk, vv = k[at].reshape(-1, KV, D)[:n].double(), v[at].reshape(-1, KV, D)[:n].double()
            pos = torch.arange(n, device=q.device)
            see = _visible(s["func"], s["block_ctx"], s["window"], pos[n - nq:, None], pos[None, :])
            o = torch.zeros(nq, H, D, dtype=torch.float64, device=q.device)
            for h in range(H):
                a = torch.where(see, q[cu[i]:cu[i + 1], h].double() @ kk[:, h * KV // H].T / math.sqrt(D), -math.inf)
                a = torch.softmax(a, 1)
                o[:, h] = torch.where(see.any(1, keepdim=True), a, 0.0) @ vv[:, h * KV // H]
            out.append(o)
        return torch.cat(out) if out else torch.zeros(0, H, D, dtype=torch.float64, device=q.device)
    if kind == "sample":
        x = s["logits"].double().cpu().numpy()
        u, T, K, P, M = (s[name].double().tolist() for name in ("u", "temp", "top_k", "top_p", "min_p"))
        import numpy as np
        got = []
        for i in range(x.shape[0]):
            r = np.where(np.isnan(x[i]), -np.inf, x[i])
            top = r.max()
            if top == -np.inf or T[i] <= 0:
                got.append(-1 if top == -np.inf else int(np.argmax(r)))
                continue
            order = np.argsort(-r, kind="stable")
            order = order[:int(K[i])] if K[i] > 0 else order
            w = np.exp((r[order] - top) / T[i])
            if 0 < P[i] < 1:
                before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
                order, w = order[before <= P[i] * w.sum()], w[before <= P[i] * w.sum()]
            if M[i] > 0:
                order, w = order[w >= min(M[i], 1.0)], w[w >= min(M[i], 1.0)]
            by = np.argsort(order)
            cum = np.cumsum(w[by])
            got.append(int(order[by][min(np.searchsorted(cum, u[i] * cum[-1], side="right"), np.flatnonzero(w[by])[-1])]))
        return torch.tensor(got)
    if kind == "write":
        at = s["slots"].cpu()
        kp, vp = s["kp"].cpu(), s["vp"].cpu()
        kp.reshape(-1, *kp.shape[2:])[at], vp.reshape(-1, *vp.shape[2:])[at] = s["k"].cpu(), s["v"].cpu()
        return [kp, vp]
    if kind == "copy":
        pools = s["pools"].cpu()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pools[:, b] = pools[:, a]
        return pools
    table, ref = s["table"].tolist(), s["ref"].tolist()
    if kind == "compact":
        n, pools = sum(c > 0 for c in ref), s["pools"].cpu()
        holes, to = [p for p in range(n) if ref[p] == 0], {}
        for p in range(n, len(ref)):
            if ref[p]:
                to[p] = holes.pop(0)
                pools[:, to[p]] = pools[:, p]
                ref[to[p]], ref[p] = ref[p], 0
        return [torch.tensor([[to.get(p, p) for p in r] for r in table], dtype=torch.int32), torch.tensor(ref, dtype=torch.int32), pools]
    page, lens = s["page"], s["lens"].tolist()
    if kind == "admit":
        kp, vp = s["kp"].cpu(), s["vp"].cpu()
        free, slots, cu, was = [p for p, c in enumerate(ref) if c == 0], [], s["cu"].tolist(), list(ref)
        for i in range(len(lens)):
            n = cu[i + 1] - cu[i]
            mine = [free.pop(0) for _ in range(-(-n // page))]
            slots += [mine[j // page] * page + j % page for j in range(n)]
        kp.reshape(-1, *kp.shape[2:])[slots], vp.reshape(-1, *vp.shape[2:])[slots] = s["k"].cpu(), s["v"].cpu()
        return [torch.tensor(slots, dtype=torch.int64), kp, vp, s["table"], s["lens"], torch.tensor(was, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
    pools = s["pools"].cpu()
    dst = s["dst"].tolist()
    for r in dst:
        for p in table[r]:
            if p >= 0:
                ref[p] -= 1
        table[r], lens[r] = [-1] * len(table[r]), 0
    free = [p for p, c in enumerate(ref) if c == 0]
    for a, b in zip(s["src"].tolist(), dst):
        lens[b] = lens[a]
        for c in range(-(-lens[a] // page)):
            table[b][c] = table[a][c]
            if (c + 1) * page > lens[a]:
                table[b][c] = free.pop(0)
                pools[:, table[b][c]] = pools[:, table[a][c]]
            ref[table[b][c]] += 1
    return [torch.tensor(table, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), torch.tensor(ref, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), pools]
