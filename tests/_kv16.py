"""Plain 64-bit forms of the 16-bit cache's operators and the caches the tests build, shared by the kv16 tests.  Everything
here is torch on whatever device the tensors are on."""
import math

import torch

LOG2E = 1.4426950408889634


def make_cache(lens, Hkv, D, page, dtype, g, device="cuda", spare=3, poison=True, outlier=3.0):
    """(pool, block table, seq_lens) of rows with the given lengths over shuffled pages.  With poison every slot that no row
    owns (the rest of a row's last page and the spare pages) is NaN, and unused table entries name a spare page."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    ids = torch.randperm(total, generator=g)
    table = ids[-1].int() * torch.ones(len(lens), max(max(need), 1), dtype=torch.int32)
    pool = torch.full((total, Hkv, 2, page, D), float("nan") if poison else 0.25, dtype=dtype)
    o = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = ids[o:o + need[b]].int()
        for i in range(need[b]):
            m = min(page, n - i * page)
            x = torch.randn(Hkv, 2, m, D, generator=g)
            x[..., :3] *= outlier
            pool[ids[o + i], :, :, :m] = x.to(dtype)
        o += need[b]
    return pool.to(device), table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)


def rows_of(pool, table_row, n):
    """keys, values [Hkv, n, D] fp64 of the first n positions of a row"""
    page, Hkv, D = pool.shape[3], pool.shape[1], pool.shape[4]
    x = pool[table_row[:-(-n // page)].long()].double()
    x = x.permute(2, 1, 0, 3, 4).reshape(2, Hkv, -1, D)[:, :, :n]
    return x[0], x[1]


def attend(q, k, v, pos, qscale, window, sinks):
    """q [n, Hq, D] fp64 at positions pos [n] over k, v [Hkv, L, D]: (out [n, Hq, D], p [n, Hq, L], A [n, Hq, D] = sum p |v|,
    S [n, Hq] = max over the visible keys of sum_d |q k| * qscale).  Values that a token does not see take no part in it."""
    Hkv, L, D = k.shape
    G = q.shape[1] // Hkv
    j = torch.arange(L, device=q.device)[None, :]
    pos = torch.as_tensor(pos, device=q.device)[:, None]
    see = j <= pos
    if window > 0:
        see = see & ((j > pos - window) | (j < sinks))
    qq = q.view(-1, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)                       # Hkv, G n, D
    see = see.repeat(G, 1)[None]
    nan0 = lambda x: torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    s = (qq @ k.transpose(1, 2)) * qscale
    s = torch.where(see, s, s.new_full((), -math.inf))
    m = s.amax(-1, keepdim=True) if L else s.new_full((Hkv, qq.shape[1], 1), -math.inf)
    p = torch.where(see, torch.exp2(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros_like(s))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    vv = v if bool(torch.isfinite(v).all()) else nan0(v)
    out, A = p @ vv, p @ vv.abs()
    S = torch.where(see, (qq.abs() @ nan0(k).abs().transpose(1, 2)) * abs(qscale), torch.zeros_like(s))
    S = S.amax(-1) if L else S.new_zeros(Hkv, qq.shape[1])
    back = lambda x: x.view(Hkv, G, -1, *x.shape[2:]).permute(2, 0, 1, *range(3, x.dim() + 1)).flatten(1, 2)  # noqa: E731
    return back(out), back(p), back(A), back(S)


def p_error(S, D, L):
    """Bound of the relative error of a softmax weight computed in 32 bits.  The score is a sum of D exact products of
    16-bit values (D roundings of at most 2^-24 of sum |q k|, two more for the scaling), so 2^s is off by ln 2 * (D + 2) *
    2^-24 * S, for the weight and for its reference alike; exp2 itself 2^-22 (twice: against a reference that moves, a
    weight is a product of at most a few of them, counted as four); the sum of L weights L * 2^-24, in pieces of a tree or
    a running sum at most that."""
    return 2 * math.log(2) * (D + 2) * 2.0 ** -24 * S + 4 * 2.0 ** -22 + L * 2.0 ** -24


def evict_ref(weights, n, budget, sinks, recent):
    """kept positions [Hkv][...] of one row (weights [Hkv, >= n]) by the definition"""
    out = []
    for w in weights[:, :n].double().cpu():
        if n <= budget:
            out.append(list(range(n)))
            continue
        mid = list(range(sinks, n - recent))
        key = [float("-inf") if math.isnan(x) else x for x in w.tolist()]
        nan = [math.isnan(x) for x in w.tolist()]
        best = sorted(mid, key=lambda j: (nan[j], -key[j], j))[:budget - sinks - recent]
        out.append(list(range(sinks)) + sorted(best) + list(range(n - recent, n)))
    return out
