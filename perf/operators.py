"""The operators of the 16-bit paged key-value cache, as work to be measured: appending rows to the pages, attention of one
new token over them (split over the cache's length, optionally with a sliding window and sink tokens, optionally adding the
attention weights that each cached token received to a running sum), attention of many new tokens over them (causal, the same
window and sinks), and eviction of the tokens with the smallest sums.

A pool is [pages, kv heads, 2, page, head dim] (keys, then values, of `page` tokens); a block table row lists a sequence's
pages.  `run` computes an operator in its plain form with torch operations in 32 bits, or, where `own` is true, by the calls
of flagrot_releaser_b200.kv16."""
import math
import random

import torch

own = False

LOG2E = 1.4426950408889634
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one request that has just begun to answer: 77 cached tokens; the time is launch and latency
        dict(name="decode_1x77", op="decode", type="bf16", B=1, L=77, spread=0, Hq=32, Hkv=8, D=128, page=16, window=0, sinks=0,
             weights=False),
        # the serving batch of this repository's default benchmark: 64 requests of up to 4096 cached tokens
        dict(name="decode_64x4096", op="decode", type="bf16", B=64, L=4096, spread=1024, Hq=32, Hkv=8, D=128, page=16, window=0,
             sinks=0, weights=False),
        # one long document (the single-sequence workload of the benchmark): all of the card works on one row
        dict(name="decode_1x131072", op="decode", type="fp16", B=1, L=131072, spread=0, Hq=32, Hkv=8, D=128, page=32, window=0,
             sinks=0, weights=False),
        # a sliding-window layer of a 64-head model: 32 long requests that see 4 sinks and the last 1024 tokens
        dict(name="decode_window_32x16384", op="decode", type="bf16", B=32, L=16384, spread=9000, Hq=64, Hkv=8, D=128, page=16,
             window=1024, sinks=4, weights=False),
        # a serving step that keeps the score of every cached token for the eviction that follows
        dict(name="decode_weights_32x8192", op="decode", type="bf16", B=32, L=8192, spread=3000, Hq=32, Hkv=8, D=128, page=16,
             window=0, sinks=0, weights=True),
        # a short question after a short cached prompt
        dict(name="prefill_1x33", op="prefill", type="fp16", B=1, n=33, nspread=0, L=133, spread=0, Hq=8, Hkv=2, D=64, page=16,
             window=0, sinks=0),
        # four requests with 512 new tokens each over a cached document of 32 768 tokens (this repository's prefill workload)
        dict(name="prefill_4x512_32768", op="prefill", type="bf16", B=4, n=512, nspread=0, L=33280, spread=0, Hq=32, Hkv=8, D=128,
             page=16, window=0, sinks=0),
        # whole prompts of uneven lengths through a sliding-window layer with sinks
        dict(name="prefill_window_3x8000", op="prefill", type="bf16", B=3, n=8000, nspread=3001, L=8000, spread=-1, Hq=32, Hkv=8,
             D=128, page=16, window=1024, sinks=4),
        # a batch at its budget: uneven rows go to the pages of a 2048-token cache
        dict(name="evict_32x4096", op="evict", type="bf16", B=32, L=4096, spread=1500, Hkv=8, D=128, page=16, budget=2048, sinks=4,
             recent=128),
        # one long document cut to an eighth
        dict(name="evict_1x60000", op="evict", type="fp16", B=1, L=60000, spread=0, Hkv=8, D=128, page=32, budget=7500, sinks=4,
             recent=512),
        # one decode step's rows, some of them padding
        dict(name="write_64", op="write", type="bf16", T=64, Hkv=8, D=128, page=16, pages=4096, holes=True),
        # a prompt's rows
        dict(name="write_65536", op="write", type="bf16", T=65536, Hkv=8, D=128, page=16, pages=4200, holes=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "evict", "write"])
    kind = rng.choice(["bf16", "fp16"])
    D, page, Hkv = rng.choice([64, 128, 128]), rng.choice([16, 16, 32, 64]), rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 4, 4, 7, 8, 8, 16])
    if op == "decode":
        L = _log(rng, 40, 65536)
        B = min(_log(rng, 1, 256), max(1, 4_000_000 // (L * Hkv)))
        w = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op=op, type=kind, B=B, L=L, spread=rng.randrange(L), Hq=G * Hkv, Hkv=Hkv, D=D, page=page, window=w,
                    sinks=rng.choice([0, 1, 4]) if w else 0, weights=rng.random() < 0.4)
    if op == "prefill":
        L = _log(rng, 40, 12000)
        n = min(L, _log(rng, 2, 6000))
        B = min(_log(rng, 1, 16), max(1, 1_500_000_000 // (n * L * G * Hkv)))
        w = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op=op, type=kind, B=B, n=n, nspread=rng.randrange(n), L=L, spread=-1, Hq=G * Hkv, Hkv=Hkv, D=D, page=page,
                    window=w, sinks=rng.choice([0, 1, 4]) if w else 0)
    if op == "evict":
        L = _log(rng, 64, 60000)
        B = min(_log(rng, 1, 64), max(1, 1_000_000 // (L * Hkv)))
        budget = max(24, int(L * rng.uniform(0.1, 0.9)))
        return dict(op=op, type=kind, B=B, L=L, spread=rng.randrange(L), Hkv=Hkv, D=D, page=page, budget=budget,
                    sinks=rng.choice([0, 4]), recent=rng.randrange(1, budget - 8))
    T = _log(rng, 1, 40000)
    return dict(op=op, type=kind, T=T, Hkv=Hkv, D=D, page=page, pages=(T + 2000) // page + 7, holes=rng.random() < 0.5)


def _lens(case):
    """(cached tokens, new tokens) of every row: a case's own, the same for every seed"""
    r = random.Random("%d %d %d" % (case["B"], case["L"], case["spread"]))
    n = [case.get("n", 1) - (r.randrange(case["nspread"] + 1) if case.get("nspread") else 0) for _ in range(case["B"])]
    if case["spread"] < 0:          # every row keeps the case's distance between its length and its new tokens
        return [case["L"] - case["n"] + k for k in n], n
    return [case["L"] - (r.randrange(case["spread"] + 1) if case["spread"] else 0) for _ in range(case["B"])], n


def _visible(pos, window, sinks):
    """keys that the query at position pos sees"""
    if window <= 0 or pos + 1 <= window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    D, Hkv = case["D"], case["Hkv"]
    if case["op"] == "write":
        t = case["T"] * 2 * Hkv * D * 2
        return {"bytes": 2 * t + 8 * case["T"], "flops": 0}
    lens, new = _lens(case)
    if case["op"] == "evict":
        kept = [min(x, case["budget"]) for x in lens]
        moved = sum(kept) * Hkv * 2 * D * 2 * 2
        return {"bytes": moved + sum(4 * x for x in lens) * Hkv + sum(8 * x for x in kept) * Hkv, "flops": 0}
    Hq, w, s = case["Hq"], case["window"], case["sinks"]
    if case["op"] == "decode":
        vis = sum(_visible(x - 1, w, s) for x in lens)
        byt = vis * Hkv * 2 * D * 2 + 2 * case["B"] * Hq * D * 2 + (vis * Hkv * 8 if case["weights"] else 0)
        return {"bytes": byt, "flops": 4 * D * Hq * vis}
    pairs, keys = 0, 0
    for x, n in zip(lens, new):
        pairs += sum(_visible(p, w, s) for p in range(x - n, x))
        first = max(0, x - n - w + 1) if w > 0 else 0
        keys += x - first + min(s, first)
    return {"bytes": keys * Hkv * 2 * D * 2 + 2 * sum(new) * Hq * D * 2, "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _pages(lens, page, g, spare=3):
    """a block table [B, widest] over shuffled pages, and the number of pages"""
    need = [-(-x // page) for x in lens]
    total = sum(need) + spare
    ids = torch.randperm(total, generator=g, device="cuda")[:sum(need)].int()
    width = max(max(need), 1)
    at = torch.arange(width, device="cuda")[None, :]
    cnt = torch.tensor(need, device="cuda")[:, None]
    start = torch.cumsum(cnt, 0) - cnt
    table = torch.where(at < cnt, ids[(start + at).clamp(max=max(sum(need) - 1, 0))], torch.zeros((), dtype=torch.int32, device="cuda"))
    return table.contiguous(), total


def _rows(shape, kind, g):
    """activations: normal, a few channels of each head larger than the rest"""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x[..., :4] *= 3
    return x.to(TYPES[kind])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    D, Hkv, page, kind = case["D"], case["Hkv"], case["page"], case["type"]
    st = dict(case=case)
    if case["op"] == "write":
        T = case["T"]
        qkv = _rows((T, 2 * Hkv + 4, D), kind, g)                   # keys and values as a slice of a fused projection's output
        st["kv"] = qkv[:, 4:]
        st["pool"] = _rows((case["pages"], Hkv, 2, page, D), kind, g)
        if case["holes"]:
            slots = torch.randperm(case["pages"] * page, generator=g, device="cuda")[:T]
            st["slots"] = torch.where(torch.rand(T, generator=g, device="cuda") < 0.1, -torch.ones_like(slots), slots)
        else:
            ids = torch.randperm(case["pages"], generator=g, device="cuda")
            t = torch.arange(T, device="cuda")
            st["slots"] = ids[t // page] * page + t % page
        return st
    lens, new = _lens(case)
    st["table"], pages = _pages(lens, page, g)
    st["pool"] = _rows((pages, Hkv, 2, page, D), kind, g)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    B, width = st["table"].shape
    if case["op"] == "evict":
        budget = case["budget"]
        e = torch.rand(B, Hkv, width * page, generator=g, device="cuda")
        st["weights"] = e.pow(8) * 30                               # few tokens hold most of the weight
        st["dst_table"], dst_pages = _pages([budget] * B, page, g)
        st["dst_pool"] = torch.zeros(dst_pages, Hkv, 2, page, D, dtype=TYPES[kind], device="cuda")
        st["kept"] = torch.empty(B, Hkv, budget, dtype=torch.int32, device="cuda")
        st["new_lens"] = torch.empty(B, dtype=torch.int32, device="cuda")
        st["new_weights"] = torch.empty(B, Hkv, st["dst_table"].shape[1] * page, device="cuda")
        return st
    Hq = case["Hq"]
    st["qscale"] = LOG2E / math.sqrt(D)
    T = sum(new)
    st["q"] = (torch.randn(T, Hq, D, generator=g, device="cuda") * 1.5).to(TYPES[kind])
    st["out"] = torch.zeros(T, Hq * D, dtype=TYPES[kind], device="cuda")
    if case["op"] == "prefill":
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        st["nmax"] = max(new)
    elif case["weights"]:
        st["weights"] = torch.rand(B, Hkv, width * page, generator=g, device="cuda")
    if own:
        from flagrot_releaser_b200 import kv16
        st["ws"] = kv16.Workspace(B, Hkv, Hq // Hkv, D, width * page, "cuda", weights=bool(case.get("weights")),
                                  new_tokens=T if case["op"] == "prefill" else 0)
    return st


# ---------------------------------------------------------------------------------------------------------------- the pass
def run(st):
    c = st["case"]
    if own:
        from flagrot_releaser_b200 import kv16
        if c["op"] == "write":
            kv16.write(st["kv"], st["slots"], st["pool"])
            return st["pool"]
        if c["op"] == "evict":
            kv16.evict(st["pool"], st["table"], st["lens"], st["weights"], c["budget"], c["sinks"], c["recent"], st["kept"],
                       st["new_lens"], st["new_weights"], dst_pool=st["dst_pool"], dst_table=st["dst_table"])
            return st["dst_pool"], st["kept"], st["new_lens"], st["new_weights"]
        if c["op"] == "prefill":
            kv16.prefill(st["q"], st["cu"], st["pool"], st["table"], st["lens"], st["out"], st["qscale"], window=c["window"],
                         sinks=c["sinks"], ws=st["ws"])
            return st["out"]
        kv16.attn(st["q"], st["pool"], st["table"], st["lens"], st["out"], st["ws"], st["qscale"], window=c["window"],
                  sinks=c["sinks"], weights=st.get("weights"))
        return (st["out"], st["weights"]) if c["weights"] else st["out"]
    return {"write": _write, "evict": _evict, "prefill": _prefill, "decode": _decode}[c["op"]](st)


def _write(st):
    pool, slots, kv = st["pool"], st["slots"], st["kv"]
    page, Hkv = pool.shape[3], pool.shape[1]
    keep = slots >= 0
    s = slots[keep]
    pool.transpose(1, 3)[s // page, s % page] = kv[keep].unflatten(1, (2, Hkv))
    return pool


def _gather(pool, table):
    """keys and values of the rows' pages in position order, [B, kv heads, tokens, head dim] in 32 bits"""
    x = pool[table.long()]                                         # B, width, Hkv, 2, page, D
    x = x.permute(3, 0, 2, 1, 4, 5).flatten(3, 4).float()
    return x[0], x[1]


def _softmax(s, see):
    """rows of 2^(s - max) / sum over the visible keys; zeros for a row that sees none"""
    s = torch.where(see, s, s.new_full((), -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp2(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _decode(st):
    c = st["case"]
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    k, v = _gather(st["pool"], st["table"])
    j = torch.arange(k.shape[2], device="cuda")[None, :]
    ln = st["lens"].long()[:, None]
    see = j < ln
    if c["window"] > 0:
        see = see & ((j >= ln - c["window"]) | (j < c["sinks"]))
    see = see[:, None, None, :]
    q = st["q"].float().view(B, Hkv, c["Hq"] // Hkv, D)
    p = _softmax(torch.matmul(q, k.transpose(2, 3)) * st["qscale"], see)
    v = torch.where(see.transpose(2, 3), v, torch.zeros((), device="cuda"))
    st["out"].copy_(torch.matmul(p, v).reshape(B, -1))
    if not c["weights"]:
        return st["out"]
    st["weights"] += p.sum(2)
    return st["out"], st["weights"]


def _prefill(st):
    c = st["case"]
    B, Hkv, D, G = c["B"], c["Hkv"], c["D"], c["Hq"] // c["Hkv"]
    k, v = _gather(st["pool"], st["table"])
    cu, ln = st["cu"].long(), st["lens"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(st["nmax"], device="cuda")[None, :]
    row = (cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"].float()[row]                                       # B, nmax, Hq, D
    q = q.view(B, -1, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    pos = (ln - n)[:, None] + i                                    # B, nmax
    j = torch.arange(k.shape[2], device="cuda")
    see = (j <= pos[..., None]) & (i < n[:, None])[..., None]
    if c["window"] > 0:
        see = see & ((j > pos[..., None] - c["window"]) | (j < c["sinks"]))
    s = (torch.matmul(q, k.transpose(2, 3)) * st["qscale"]).view(B, Hkv, G, -1, k.shape[2])
    p = _softmax(s, see[:, None, None])
    del s
    o = torch.matmul(p.flatten(2, 3), v).view(B, Hkv, G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, st["nmax"], -1)
    t = torch.arange(st["q"].shape[0], device="cuda")
    b = torch.bucketize(t, cu[1:], right=True)
    st["out"].copy_(o[b, t - cu[b]])
    return st["out"]


def _evict(st):
    c = st["case"]
    w, ln = st["weights"], st["lens"].long()
    B, Hkv, W = w.shape
    j = torch.arange(W, device="cuda")[None, :]
    new = ln.clamp(max=c["budget"])
    # 0 the largest: forced tokens, then by weight (ties: the lower position first), then what is beyond the row's length
    forced = (j < c["sinks"]) | (j >= ln[:, None] - c["recent"])
    rank = torch.where(forced[:, None], w.new_full((), math.inf), w)
    rank = torch.where((j < ln[:, None])[:, None], rank, w.new_full((), -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    slot = torch.arange(order.shape[-1], device="cuda")
    live = slot < new[:, None, None]
    order = torch.where(live, order, order.new_full((), 1 << 30)).sort(-1).values
    kept = st["kept"].fill_(-1)
    kept[..., :order.shape[-1]] = torch.where(live, order, order.new_full((), -1)).int()
    src = torch.where(live, order, torch.zeros_like(order))
    st["new_weights"].zero_()
    st["new_weights"][..., :order.shape[-1]] = torch.where(live, w.gather(-1, src), torch.zeros((), device="cuda"))
    st["new_lens"].copy_(new)
    page = c["page"]
    h = torch.arange(Hkv, device="cuda")[None, :, None]
    pg = st["table"].long().gather(1, (src // page).flatten(1)).view_as(src)
    rows = st["pool"].transpose(2, 3)[pg, h, src % page]
    dpg = st["dst_table"].long()[:, slot // page][:, None].expand_as(src)
    dst = st["dst_pool"].transpose(2, 3)
    old = dst[dpg, h, (slot % page).expand_as(src)]
    dst[dpg, h, (slot % page).expand_as(src)] = torch.where(live[..., None, None], rows, old)
    return st["dst_pool"], st["kept"], st["new_lens"], st["new_weights"]


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    c, pool = case, st["pool"]
    if c["op"] == "write":
        out = pool.double()
        for t, s in enumerate(st["slots"].tolist()):
            if s >= 0:
                out[s // c["page"], :, :, s % c["page"]] = st["kv"][t].double().view(2, c["Hkv"], -1).transpose(0, 1)
        return out
    lens, new = _lens(c)
    Hkv, D, page = c["Hkv"], c["D"], c["page"]

    def row(b):
        pg = st["table"][b, :-(-lens[b] // page)].long()
        x = pool[pg].double().permute(2, 1, 0, 3, 4).reshape(2, Hkv, -1, D)
        return x[:, :, :lens[b]]

    if c["op"] == "evict":
        dst, w2 = st["dst_pool"].double(), torch.zeros_like(st["new_weights"], dtype=torch.float64)
        for b in range(c["B"]):
            n = lens[b]
            kv = row(b)
            m = min(n, c["budget"])
            pgs = st["dst_table"][b].long()
            for h in range(Hkv):
                w = st["weights"][b, h, :n].double()
                if n <= c["budget"]:
                    keep = torch.arange(n, device="cuda")
                else:
                    head, tail = torch.arange(c["sinks"], device="cuda"), torch.arange(n - c["recent"], n, device="cuda")
                    body = w[c["sinks"]:n - c["recent"]]
                    best = torch.sort(-body, stable=True).indices[:c["budget"] - c["sinks"] - c["recent"]] + c["sinks"]
                    keep = torch.cat([head, best.sort().values, tail])
                w2[b, h, :m] = w[keep]
                at = torch.arange(m, device="cuda")
                dst[pgs[at // page], h, :, at % page] = kv[:, h][:, keep].transpose(0, 1)
        return dst, None, None, w2
    G = c["Hq"] // Hkv
    out = torch.zeros(st["q"].shape[0], c["Hq"], D, dtype=torch.float64, device="cuda")
    acc = st["weights"].double() if c.get("weights") else None
    at = 0
    for b in range(c["B"]):
        kv, n = row(b), new[b]
        pos = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        j = torch.arange(lens[b], device="cuda")[None, :]
        hide = j > pos
        if c["window"] > 0:
            hide = hide | ((j <= pos - c["window"]) & (j >= c["sinks"]))
        for h in range(c["Hq"]):
            s = (st["q"][at:at + n, h].double() @ kv[0, h // G].T) * (st["qscale"] / LOG2E)
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            out[at:at + n, h] = p @ kv[1, h // G]
            if acc is not None:
                acc[b, h // G, :lens[b]] += p[0]
        at += n
    out = out.view(out.shape[0], -1)
    return (out, acc) if acc is not None else out
