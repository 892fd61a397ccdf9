"""The 16-bit paged cache on a GPU against its plain 64-bit forms: writer, decode attention (window, sinks, weights), prefill
attention, eviction, and a run of them together.

Tolerances count roundings: an output is rounded once to its type (eps / 2 relative); a softmax weight is off by
tests._kv16.p_error in 32 bits, twice (its numerator and the row's sum); weights that meet the values in 16 bits add eps / 2
(prefill) or 2^-16 (decode, where a weight is the sum of two 16-bit numbers); the sum over L values in 32 bits L * 2^-24,
part of p_error already.  Each of these multiplies A = sum p |v|."""
import math

import pytest
import torch

from tests import _kv16 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    from flagrot_releaser_b200 import kv16
    kv16.lib()
    yield kv16
    assert kv16.device_status() == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def queries(n, Hq, D, dtype, g, scale=1.5, pad=0):
    """[n, Hq, D] as a slice of wider rows, so that strides and rows differ"""
    x = (torch.randn(n, Hq + pad, D, generator=g) * scale).to(dtype).to(DEV)
    return x[:, pad:] if pad else x


def bound(o, A, S, D, L, dtype, prefill):
    eps = torch.finfo(dtype).eps
    d = 2 * R.p_error(S, D, L)[..., None] + (eps / 2 if prefill else 2.0 ** -16)
    return (eps / 2) * (o.abs() + d * A) + d * A + 1e-30 + (2.0 ** -25 if dtype == FP else 0.0)


# ------------------------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("dtype,D,page,Hkv,T", [(BF, 128, 16, 8, 1), (FP, 64, 16, 1, 3), (BF, 64, 32, 2, 77), (FP, 128, 64, 3, 500),
                                                (BF, 128, 128, 5, 1025), (BF, 128, 16, 8, 20000)])
def test_write(K, dtype, D, page, Hkv, T):
    g = gen(T + D)
    npg = T // page + 9
    pool = torch.randn(npg, Hkv, 2, page, D, generator=g).to(dtype).to(DEV)
    buf = torch.randn(T, 2 * Hkv + 3, D + 8, generator=g).to(dtype).to(DEV)
    kv = buf[:, 2:2 + 2 * Hkv, 8:]
    slots = torch.randperm(npg * page, generator=g)[:T]
    bad = torch.rand(T, generator=g)
    slots[bad < 0.1] = -1
    slots[(bad >= 0.1) & (bad < 0.13)] = npg * page              # past the pool: skipped
    slots[(bad >= 0.13) & (bad < 0.15)] = 1 << 62
    exp = pool.clone()
    ok = (slots >= 0) & (slots < npg * page)
    s = slots[ok].to(DEV)
    exp.transpose(1, 3)[s // page, s % page] = kv[ok.to(DEV)].unflatten(1, (2, Hkv))
    K.write(kv, slots.to(DEV), pool)
    assert torch.equal(pool, exp)


# ----------------------------------------------------------------------------------------------------------------- decode
def run_attn(K, q, pool, bt, lens, qscale, window=0, sinks=0, weights=None, ws=None, pad=0):
    B, Hq, D = q.shape
    Hkv, page = pool.shape[1], pool.shape[3]
    if ws is None:
        ws = K.Workspace(B, Hkv, Hq // Hkv, D, bt.shape[1] * page, DEV, weights=weights is not None)
    out = torch.full((B, Hq * D + pad), 7.0, dtype=q.dtype, device=DEV)
    K.attn(q, pool, bt, lens, out[:, :Hq * D], ws, qscale, window=window, sinks=sinks, weights=weights)
    assert int(ws.tickets.abs().max()) == 0
    assert bool((out[:, Hq * D:] == 7.0).all())
    return out[:, :Hq * D].view(B, Hq, D) if pad == 0 else out[:, :Hq * D].reshape(B, Hq, D)


def check_attn(out, q, pool, bt, lens, qscale, window, sinks, w0=None, w1=None):
    B, Hq, D = q.shape
    Hkv, page = pool.shape[1], pool.shape[3]
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            assert bool((out[b] == 0).all())
            if w0 is not None:
                assert torch.equal(w0[b], w1[b])
            continue
        k, v = R.rows_of(pool, bt[b], n)
        o, p, A, S = R.attend(q[b:b + 1].double(), k, v, [n - 1], qscale, window, sinks)
        err = (out[b:b + 1].double() - o).abs()
        tol = bound(o, A, S, D, n, q.dtype, False)
        assert bool((err <= tol).all()), (b, n, float((err / tol).max()), float(err.max()))
        if w0 is None:
            continue
        G = Hq // Hkv
        add = p[0].view(Hkv, G, n).sum(1)
        exp = w0[b, :, :n].double() + add
        wt = (2 * R.p_error(S[0].view(Hkv, G).amax(1), D, n)[:, None] + G * 2.0 ** -24) * add + 2.0 ** -24 * exp.abs()
        werr = (w1[b, :, :n].double() - exp).abs()
        assert bool((werr <= wt).all()), (b, n, float((werr / wt.clamp(min=1e-300)).max()))
        assert torch.equal(w0[b, :, n:], w1[b, :, n:])
        hid = torch.arange(n, device=DEV)
        hid = (hid >= sinks) & (hid < n - window) if window > 0 else hid < 0
        assert torch.equal(w0[b, :, :n][:, hid], w1[b, :, :n][:, hid])


LENS = [0, 1, 2, 7, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 255, 256, 257, 300, 511, 513, 1000, 1025]


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 17, 32, 40])
@pytest.mark.parametrize("D,page,dtype", [(128, 16, BF), (64, 16, FP), (128, 64, FP), (64, 128, BF), (128, 32, BF)])
def test_attn_lengths_and_groups(K, G, D, page, dtype):
    g = gen(G * 1000 + D + page)
    Hkv = 2
    pool, bt, lens = R.make_cache(LENS, Hkv, D, page, dtype, g)
    q = queries(len(LENS), G * Hkv, D, dtype, g, pad=1)
    w0 = torch.rand(len(LENS), Hkv, bt.shape[1] * page + 5, generator=g).to(DEV)
    w1 = w0.clone()
    out = run_attn(K, q, pool, bt, lens, R.LOG2E / math.sqrt(D), weights=w1, pad=16)
    check_attn(out, q, pool, bt, lens, R.LOG2E / math.sqrt(D), 0, 0, w0, w1)
    plain = run_attn(K, q, pool, bt, lens, R.LOG2E / math.sqrt(D))
    check_attn(plain, q, pool, bt, lens, R.LOG2E / math.sqrt(D), 0, 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 4), (16, 0), (17, 4), (64, 1), (100, 33), (128, 200), (500, 4), (2000, 4),
                                          (1 << 30, 7)])
@pytest.mark.parametrize("dtype,D,page,G", [(BF, 128, 16, 4), (FP, 64, 64, 8)])
def test_attn_window_and_sinks(K, window, sinks, dtype, D, page, G):
    """hidden keys inside the sequence hold NaN and infinities: they must not reach the output"""
    g = gen(window * 31 + sinks)
    Hkv = 3
    pool, bt, lens = R.make_cache(LENS, Hkv, D, page, dtype, g)
    pc = pool.cpu()
    for b, n in enumerate(LENS):
        for j in range(sinks, max(n - window, 0)):
            pc[int(bt[b, j // page]), :, :, j % page] = float("nan") if j % 3 else float("inf")
    pool = pc.to(DEV)
    q = queries(len(LENS), G * Hkv, D, dtype, g)
    w0 = torch.rand(len(LENS), Hkv, bt.shape[1] * page, generator=g).to(DEV)
    w1 = w0.clone()
    out = run_attn(K, q, pool, bt, lens, R.LOG2E / math.sqrt(D), window, sinks, weights=w1)
    check_attn(out, q, pool, bt, lens, R.LOG2E / math.sqrt(D), window, sinks, w0, w1)
    out = run_attn(K, q, pool, bt, lens, R.LOG2E / math.sqrt(D), window, sinks)
    check_attn(out, q, pool, bt, lens, R.LOG2E / math.sqrt(D), window, sinks)


@pytest.mark.parametrize("lens,Hkv,G,dtype", [([33000], 1, 4, BF), ([70001], 2, 8, FP), ([20000, 3, 0, 9000, 1], 4, 1, BF),
                                              ([513] * 150, 4, 4, BF), (list(range(300)), 1, 2, FP)])
def test_attn_long_and_wide(K, lens, Hkv, G, dtype):
    g = gen(len(lens))
    pool, bt, ln = R.make_cache(lens, Hkv, 128, 16, dtype, g)
    q = queries(len(lens), G * Hkv, 128, dtype, g)
    w0 = torch.zeros(len(lens), Hkv, bt.shape[1] * 16, device=DEV)
    w1 = w0.clone()
    qs = R.LOG2E / math.sqrt(128)
    out = run_attn(K, q, pool, bt, ln, qs, weights=w1)
    check_attn(out, q, pool, bt, ln, qs, 0, 0, w0, w1)
    again = run_attn(K, q, pool, bt, ln, qs)
    check_attn(again, q, pool, bt, ln, qs, 0, 0)
    assert torch.equal(again, run_attn(K, q, pool, bt, ln, qs)), "two calls on the same inputs differ"


@pytest.mark.parametrize("lens,Hkv,G,D,dtype", [([4096] * 64, 8, 4, 128, BF), ([3000, 5000, 7] * 20, 4, 12, 64, FP), ([60000], 8, 32, 128, BF)])
def test_attn_repeated_calls_agree_bit_for_bit(K, lens, Hkv, G, D, dtype):
    """copies that land in another order must not change what a warp reads, nor CTAs that finish in another order the join"""
    g = gen(8)
    pool, bt, ln = R.make_cache(lens, Hkv, D, 16, dtype, g)
    q = queries(len(lens), G * Hkv, D, dtype, g)
    ws = K.Workspace(len(lens), Hkv, G, D, bt.shape[1] * 16, DEV)
    out = [torch.empty(len(lens), G * Hkv * D, dtype=dtype, device=DEV) for _ in range(60)]
    for o in out:
        K.attn(q, pool, bt, ln, o, ws, 0.12)
    assert all(torch.equal(out[0], o) for o in out[1:])


def test_attn_extreme_scores(K):
    """scores of some thousands, of both signs; a negative scale"""
    g = gen(5)
    lens = [40, 700, 1]
    pool, bt, ln = R.make_cache(lens, 2, 128, 16, BF, g)
    q = queries(3, 8, 128, BF, g, scale=60)
    for qs in (3.0, -3.0, 0.0):
        out = run_attn(K, q, pool, bt, ln, qs)
        check_attn(out, q, pool, bt, ln, qs, 0, 0)


def test_attn_shared_table_and_clamped_inputs(K):
    """a stride-0 table; lengths past the table are taken as its end, negative ones as 0; a table entry outside the pool
    reads as a page of zeros"""
    g = gen(6)
    pool, bt, _ = R.make_cache([320], 2, 64, 16, FP, g)
    q = queries(4, 8, 64, FP, g)
    ln = torch.tensor([320, 100000, -5, 37], dtype=torch.int32, device=DEV)
    out = run_attn(K, q, pool, bt.expand(4, -1), ln, 0.2)
    check_attn(out, q, pool, bt.expand(4, -1), torch.tensor([320, 320, 0, 37]), 0.2, 0, 0)
    bad = bt.repeat(2, 1)
    bad[0, 3], bad[1, 5] = -1, pool.shape[0]
    zeros = torch.cat([pool, torch.zeros_like(pool[:1])])
    ref = torch.where((bad < 0) | (bad >= pool.shape[0]), torch.full_like(bad, pool.shape[0]), bad)
    ln = torch.tensor([300, 320], dtype=torch.int32, device=DEV)
    out = run_attn(K, q[:2], pool, bad, ln, 0.2)
    check_attn(out, q[:2], zeros, ref, ln, 0.2, 0, 0)


def test_attn_offsets_past_32_bits(K):
    """a pool of more than 2^32 bytes, its last pages in use"""
    Hkv, page, D = 8, 16, 128
    npg = (1 << 32) // K.chunk_bytes(page, D) // Hkv + 700
    pool = torch.zeros(npg, Hkv, 2, page, D, dtype=BF, device=DEV)
    g = gen(9)
    ids = torch.tensor([npg - 1, 0, npg - 2, npg // 2 + 1], dtype=torch.int32)
    pool[ids.long()] = torch.randn(4, Hkv, 2, page, D, generator=g).to(BF).to(DEV)
    bt, ln = ids[None].to(DEV), torch.tensor([61], dtype=torch.int32, device=DEV)
    q = queries(1, 32, D, BF, g)
    out = run_attn(K, q, pool, bt, ln, 0.1)
    check_attn(out, q, pool, bt, ln, 0.1, 0, 0)
    kv = torch.randn(2, 2 * Hkv, D, generator=g).to(BF).to(DEV)
    K.write(kv, torch.tensor([npg * page - 1, npg * page - 17], device=DEV), pool)
    assert torch.equal(pool[npg - 1, :, 0, 15], kv[0, :Hkv]) and torch.equal(pool[npg - 2, :, 1, 15], kv[1, Hkv:])


@pytest.mark.parametrize("G,Hkv", [(130, 1), (71, 2), (256, 1)])
def test_attn_many_heads_per_group(K, G, Hkv):
    g = gen(G)
    lens = [1, 40, 700]
    pool, bt, ln = R.make_cache(lens, Hkv, 64, 16, BF, g)
    q = queries(3, G * Hkv, 64, BF, g)
    w0 = torch.rand(3, Hkv, bt.shape[1] * 16, generator=g).to(DEV)
    w1 = w0.clone()
    out = run_attn(K, q, pool, bt, ln, 0.17, weights=w1)
    check_attn(out, q, pool, bt, ln, 0.17, 0, 0, w0, w1)


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 40, 2 ** 35), (-7, 5), (5, 2 ** 31 - 1), (0, 3)])
def test_window_and_sinks_of_any_size(K, window, sinks):
    """a window or sinks beyond every position act as no window; a negative window is none"""
    g = gen(13)
    pool, bt, ln = R.make_cache([300, 17], 1, 64, 16, BF, g)
    q = queries(2, 4, 64, BF, g)
    out = run_attn(K, q, pool, bt, ln, 0.2, window, sinks)
    check_attn(out, q, pool, bt, ln, 0.2, min(window, 1 << 30), min(sinks, 1 << 30))
    check_prefill(K, [300, 17], [300, 9], 1, 4, 64, 16, BF, window, sinks, 17)


def test_attn_workspace_of_a_larger_call_and_refusal(K):
    """one workspace serves smaller calls too, in any order; a call it is too small for is refused"""
    g = gen(7)
    pool, bt, ln = R.make_cache([500, 40, 900], 2, 128, 16, BF, g)
    ws = K.Workspace(3, 2, 8, 128, bt.shape[1] * 16, DEV, weights=True)
    for G, B in ((8, 3), (2, 1), (4, 3), (1, 2)):
        q = queries(B, 2 * G, 128, BF, g)
        out = run_attn(K, q, pool, bt[:B], ln[:B], 0.1, ws=ws)
        check_attn(out, q, pool, bt[:B], ln[:B], 0.1, 0, 0)
    small = K.Workspace(1, 2, 1, 128, 16, DEV)
    q, w = queries(3, 16, 128, BF, g), torch.zeros(3, 2, bt.shape[1] * 16, device=DEV)
    with pytest.raises(RuntimeError, match="code -4"):
        K.attn(q, pool, bt, ln, torch.empty(3, 2048, dtype=BF, device=DEV), small, 0.1, weights=w)


# ---------------------------------------------------------------------------------------------------------------- prefill
def check_prefill(K, lens, new, Hkv, G, D, page, dtype, window, sinks, seed, gap=0, tail=0, qs=None, ws=None, scale=1.5):
    g = gen(seed)
    qs = R.LOG2E / math.sqrt(D) if qs is None else qs
    pool, bt, ln = R.make_cache(lens, Hkv, D, page, dtype, g)
    cu = [gap]
    for n in new:
        cu.append(cu[-1] + n)
    T = cu[-1] + tail
    q = queries(T, G * Hkv, D, dtype, g, scale, pad=2)
    out = torch.full((T, G * Hkv * D + 8), 7.0, dtype=dtype, device=DEV)
    if ws is None:
        ws = K.Workspace(len(lens), Hkv, G, D, bt.shape[1] * page, DEV, new_tokens=T)
    K.prefill(q, torch.tensor(cu, dtype=torch.int32, device=DEV), pool, bt, ln, out[:, :-8], qs, window=window, sinks=sinks, ws=ws)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    assert bool((out[:, -8:] == 7.0).all()) and bool((out[:gap] == 7.0).all()) and bool((out[cu[-1]:] == 7.0).all())
    res = out[:, :-8].reshape(T, G * Hkv, D)
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0:
            continue
        o = res[cu[b]:cu[b + 1]].double()
        hidden = max(m - n, 0)                                     # tokens at negative positions
        assert bool((o[:hidden] == 0).all())
        k, v = R.rows_of(pool, bt[b], n)
        for i0 in range(hidden, m, 512):
            i1 = min(m, i0 + 512)
            ref, _, A, S = R.attend(q[cu[b] + i0:cu[b] + i1].double(), k, v, torch.arange(n - m + i0, n - m + i1), qs, window, sinks)
            err, tol = (o[i0:i1] - ref).abs(), bound(ref, A, S, D, n, dtype, True)
            assert bool((err <= tol).all()), (b, n, m, float((err / tol).max()), float(err.max()))


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 7, 8, 12, 16, 33])
@pytest.mark.parametrize("D,page,dtype", [(128, 16, BF), (64, 32, FP), (128, 64, FP), (64, 128, BF)])
def test_prefill_groups_and_lengths(K, G, D, page, dtype):
    check_prefill(K, [1, 5, 130, 64, 0, 257, 300, 17], [1, 5, 130, 1, 0, 100, 33, 16], 2, G, D, page, dtype, 0, 0, G + D, gap=3, tail=5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (5, 4), (64, 0), (100, 4), (128, 128), (129, 130), (300, 1), (5000, 4)])
@pytest.mark.parametrize("dtype,D,page,G", [(BF, 128, 16, 4), (FP, 64, 32, 6)])
def test_prefill_window_and_sinks(K, window, sinks, dtype, D, page, G):
    check_prefill(K, [700, 90, 1300, 513], [700, 20, 333, 1], 2, G, D, page, dtype, window, sinks, window + sinks)


@pytest.mark.parametrize("lens,new,Hkv,G", [([9000], [70], 1, 4), ([4096, 33], [512, 33], 2, 4), ([2500], [2500], 1, 8), ([20000], [3], 2, 1)])
def test_prefill_long(K, lens, new, Hkv, G):
    check_prefill(K, lens, new, Hkv, G, 128, 16, BF, 0, 0, 11)


def test_prefill_more_new_tokens_than_cached(K):
    """tokens at negative positions see nothing and give zeros"""
    check_prefill(K, [4, 0, 30], [10, 7, 30], 2, 4, 128, 16, BF, 0, 0, 12)
    check_prefill(K, [4, 0, 30], [10, 7, 30], 2, 4, 64, 16, FP, 3, 1, 13)


@pytest.mark.parametrize("G,Hkv", [(128, 1), (130, 1), (65, 2), (200, 1)])
def test_prefill_many_heads_per_group(K, G, Hkv):
    check_prefill(K, [150, 9], [20, 9], Hkv, G, 64, 16, BF, 0, 0, 18)


def test_prefill_table_entries_outside_the_pool_read_as_zeros(K):
    g = gen(19)
    pool, bt, ln = R.make_cache([300], 2, 64, 16, BF, g)
    q = queries(40, 8, 64, BF, g)
    bad = bt.clone()
    bad[0, 3], bad[0, 11] = -1, pool.shape[0] + 5
    ref = bad.clone()
    ref[0, 3] = ref[0, 11] = pool.shape[0]
    ws, cu = K.Workspace(1, 2, 4, 64, bt.shape[1] * 16, DEV, new_tokens=40), torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    a, b = torch.empty(40, 512, dtype=BF, device=DEV), torch.empty(40, 512, dtype=BF, device=DEV)
    K.prefill(q, cu, pool, bad, ln, a, 0.2, ws=ws)
    K.prefill(q, cu, torch.cat([pool, torch.zeros_like(pool[:1])]), ref, ln, b, 0.2, ws=ws)
    assert torch.equal(a, b)


@pytest.mark.parametrize("lens,new,Hkv,G,D", [([33280] * 2, [512, 300], 8, 4, 128), ([8000, 5100], [8000, 5100], 4, 8, 64)])
def test_prefill_repeated_calls_agree_bit_for_bit(K, lens, new, Hkv, G, D):
    """split pairs are joined in the order of their pieces, whichever ends last"""
    g = gen(20)
    pool, bt, ln = R.make_cache(lens, Hkv, D, 16, BF, g)
    T = sum(new)
    q = queries(T, Hkv * G, D, BF, g)
    cu = torch.tensor([0, new[0], T], dtype=torch.int32, device=DEV)
    ws = K.Workspace(2, Hkv, G, D, bt.shape[1] * 16, DEV, new_tokens=T)
    first = None
    for _ in range(20):
        out = torch.empty(T, Hkv * G * D, dtype=BF, device=DEV)
        K.prefill(q, cu, pool, bt, ln, out, 0.12, window=3000 if D == 64 else 0, sinks=4, ws=ws)
        first = out if first is None else first
        assert torch.equal(first, out)
    assert int(ws.tickets.abs().max()) == 0


def test_prefill_workspace_is_checked(K):
    g = gen(21)
    pool, bt, ln = R.make_cache([100], 1, 64, 16, BF, g)
    q, cu = queries(100, 4, 64, BF, g), torch.tensor([0, 100], dtype=torch.int32, device=DEV)
    out = torch.empty(100, 256, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="code -4"):
        K.prefill(q, cu, pool, bt, ln, out, 0.1, ws=K.Workspace(1, 1, 4, 64, 112, DEV))
    big = K.Workspace(3, 2, 8, 128, 4096, DEV, weights=True, new_tokens=5000)       # serves smaller calls
    K.prefill(q, cu, pool, bt, ln, out, 0.1, ws=big)
    k, v = R.rows_of(pool, bt[0], 100)
    o, _, A, S = R.attend(q.double(), k, v, torch.arange(100), 0.1, 0, 0)
    assert bool(((out.view(100, 4, 64).double() - o).abs() <= bound(o, A, S, 64, 100, BF, True)).all())


def test_prefill_extreme_scores(K):
    for qs in (2.0, -2.0, 0.0):
        check_prefill(K, [300], [200], 1, 4, 128, 16, BF, 0, 0, 14, qs=qs, scale=20.0)


def test_prefill_many_short_rows(K):
    check_prefill(K, [i % 37 + 1 for i in range(400)], [i % 3 for i in range(400)], 2, 4, 64, 16, BF, 0, 0, 15)


def test_prefill_of_one_token_is_decode(K):
    g = gen(16)
    lens = [5, 64, 1000]
    pool, bt, ln = R.make_cache(lens, 2, 128, 16, BF, g)
    q = queries(3, 8, 128, BF, g)
    ws = K.Workspace(3, 2, 4, 128, bt.shape[1] * 16, DEV, new_tokens=3)
    out = torch.empty(3, 8 * 128, dtype=BF, device=DEV)
    K.prefill(q, torch.arange(4, dtype=torch.int32, device=DEV), pool, bt, ln, out, 0.12, window=50, sinks=2, ws=ws)
    dec = run_attn(K, q, pool, bt, ln, 0.12, 50, 2)
    eps = torch.finfo(BF).eps
    d = (out.view(3, 8, 128).double() - dec.double()).abs()
    # two results, each within its own bound of the definition
    for b, n in enumerate(lens):
        k, v = R.rows_of(pool, bt[b], n)
        o, _, A, S = R.attend(q[b:b + 1].double(), k, v, [n - 1], 0.12, 50, 2)
        assert bool((d[b:b + 1] <= bound(o, A, S, 128, n, BF, True) + bound(o, A, S, 128, n, BF, False)).all())
    assert eps > 0


# --------------------------------------------------------------------------------------------------------------- eviction
def check_evict(K, lens, Hkv, D, page, dtype, budget, sinks, recent, seed, in_place, weights=None, extra=0):
    g = gen(seed)
    B = len(lens)
    pool, bt, ln = R.make_cache(lens, Hkv, D, page, dtype, g, poison=False)
    W = bt.shape[1] * page
    if weights is None:
        weights = torch.rand(B, Hkv, W + 3, generator=g).pow(4).to(DEV)
    weights = weights.to(DEV)
    wcopy = weights.clone()
    before = pool.clone()
    kept = torch.full((B, Hkv, budget), -7, dtype=torch.int32, device=DEV)
    nl = torch.full((B,), -7, dtype=torch.int32, device=DEV)
    nw = torch.full((B, Hkv, budget + extra), -7.0, device=DEV)
    if in_place:
        dst, dbt = pool, bt
        K.evict(pool, bt, ln, weights, budget, sinks, recent, kept, nl, nw)
    else:
        need = -(-budget // page)
        dst = torch.randn(B * need + 2, Hkv, 2, page, D, generator=g).to(dtype).to(DEV)
        dbt = torch.randperm(B * need + 2, generator=g)[:B * need].int().view(B, need).to(DEV)
        dbefore = dst.clone()
        K.evict(pool, bt, ln, weights, budget, sinks, recent, kept, nl, nw, dst_pool=dst, dst_table=dbt)
    torch.cuda.synchronize()
    assert torch.equal(weights.nan_to_num(nan=-3.0), wcopy.nan_to_num(nan=-3.0))
    exp = before.clone() if in_place else dbefore
    for b in range(B):
        n = min(lens[b], weights.shape[2])
        m = min(n, budget)
        assert int(nl[b]) == m
        ref = R.evict_ref(weights[b], n, budget, sinks, recent)
        for h in range(Hkv):
            assert kept[b, h].tolist() == ref[h] + [-1] * (budget - m), (b, h)
            idx = torch.tensor(ref[h], dtype=torch.long, device=DEV)
            got = nw[b, h].double()
            assert torch.equal(got[:m].nan_to_num(nan=-3.0), weights[b, h][idx].double().nan_to_num(nan=-3.0))
            assert bool((got[m:] == 0).all())
            at = torch.arange(m, device=DEV)
            src = before[bt[b, idx // page].long(), h, :, idx % page]
            exp[dbt[b, at // page].long(), h, :, at % page] = src
    assert torch.equal(dst.view(torch.int16), exp.view(torch.int16))
    if not in_place:
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D,page,dtype,Hkv", [(128, 16, BF, 2), (64, 32, FP, 3), (128, 128, FP, 1), (64, 16, BF, 8)])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (16, 4, 4), (33, 4, 16), (64, 0, 0), (64, 32, 32), (200, 4, 100)])
def test_evict(K, in_place, D, page, dtype, Hkv, budget, sinks, recent):
    check_evict(K, [0, 1, 5, 16, 33, 64, 65, 200, 201, 333, 1000], Hkv, D, page, dtype, budget, sinks, recent, budget + D, in_place, extra=5)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget", [([30000], 2000), ([30000], 29000), ([5000, 70000, 64], 4096), ([2049] * 40, 2048)])
def test_evict_long(K, in_place, lens, budget):
    check_evict(K, lens, 2, 64, 16, BF, budget, 4, 64, 21, in_place)


@pytest.mark.parametrize("levels", [0, 3])                      # weights: random, or of few values (many ties)
@pytest.mark.parametrize("lens,Hkv,budget", [([4097, 4100, 64] * 25, 2, 2000), ([8200, 50, 8191, 4096] * 19, 2, 1000), ([17000, 900] * 38, 2, 900),
                                             ([66000], 1, 7000), ([140000, 9, 131073], 2, 6000), ([262200], 1, 262144)])
def test_evict_rows_of_every_size_class(K, lens, Hkv, budget, levels):
    W = -(-max(lens) // 16) * 16 + 3
    g = gen(budget + levels)
    w = torch.randint(0, levels, (len(lens), Hkv, W), generator=g).float() if levels else torch.rand(len(lens), Hkv, W, generator=g)
    check_evict(K, lens, Hkv, 64, 16, BF, budget, 4, 100, 31, False, weights=w)


def test_evict_ties_infinities_nan_and_signs(K):
    """equal weights go to the lower position; -0 equals +0; NaN is the smallest; negative weights and infinities order"""
    g = gen(22)
    n = 1000
    vals = torch.tensor([0.0, -0.0, 1.0, 1.0, -1.0, float("inf"), float("-inf"), float("nan"), 1e-40, -1e-40, 3.0])
    w = vals[torch.randint(0, len(vals), (4, 2, 1008), generator=g)]
    w[1] = 0.25
    w[2] = float("nan")
    w[3, :, ::2] = float("-inf")
    for budget in (1, 50, 300, 700, 999):
        for in_place in (False, True):
            check_evict(K, [n] * 4, 2, 64, 16, BF, budget, 0, budget // 3, 23, in_place, weights=w)


def test_evict_to_other_pages_of_the_same_pool(K):
    g = gen(25)
    lens, Hkv, budget = [300, 90, 40], 2, 64
    pool, bt, ln = R.make_cache(lens, Hkv, 64, 16, BF, g, spare=12, poison=False)
    w = torch.rand(3, Hkv, bt.shape[1] * 16, generator=g).to(DEV)
    used = set(bt[0, :19].tolist()) | set(bt[1, :6].tolist()) | set(bt[2, :3].tolist())
    free = torch.tensor([p for p in range(pool.shape[0]) if p not in used][:12], dtype=torch.int32, device=DEV).view(3, 4)
    kept, nl = torch.empty(3, Hkv, budget, dtype=torch.int32, device=DEV), torch.empty(3, dtype=torch.int32, device=DEV)
    nw, before = torch.empty(3, Hkv, budget, device=DEV), pool.clone()
    K.evict(pool, bt, ln, w, budget, 4, 16, kept, nl, nw, dst_table=free)
    exp = before.clone()
    for b, n in enumerate(lens):
        ref = R.evict_ref(w[b], n, budget, 4, 16)
        for h in range(Hkv):
            idx, at = torch.tensor(ref[h], device=DEV), torch.arange(len(ref[h]), device=DEV)
            assert kept[b, h, :len(ref[h])].tolist() == ref[h]
            exp[free[b, at // 16].long(), h, :, at % 16] = before[bt[b, idx // 16].long(), h, :, idx % 16]
    assert torch.equal(pool, exp)


def test_empty_tables_and_batches(K):
    pool = torch.zeros(2, 1, 2, 16, 64, dtype=BF, device=DEV)
    ws = K.Workspace(2, 1, 4, 64, 0, DEV, weights=True, new_tokens=4)
    bt, ln = torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.tensor([5, 0], dtype=torch.int32, device=DEV)
    q, out, w = torch.ones(2, 4, 64, dtype=BF, device=DEV), torch.ones(2, 256, dtype=BF, device=DEV), torch.zeros(2, 1, 0, device=DEV)
    K.attn(q, pool, bt, ln, out, ws, 0.1, weights=w)
    assert bool((out == 0).all())
    out.fill_(1)
    K.prefill(q, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), pool, bt, ln, out, 0.1, ws=ws)
    assert bool((out == 0).all())
    kept, nl, nw = torch.zeros(2, 1, 3, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV), torch.ones(2, 1, 3, device=DEV)
    K.evict(pool, bt, ln, w, 3, 1, 1, kept, nl, nw)
    assert bool((kept == -1).all()) and bool((nl == 0).all()) and bool((nw == 0).all())
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    K.attn(q[:0], pool, bt[:0], z, out[:0], ws, 0.1)
    K.write(torch.zeros(0, 2, 64, dtype=BF, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), pool)
    K.evict(pool, bt[:0], z, w[:0], 3, 1, 1, kept[:0], nl[:0], nw[:0])
    assert bool((pool == 0).all())


def test_evict_weights_shorter_than_the_table(K):
    """a row is taken as long as its weights at most"""
    w = torch.rand(2, 2, 100, generator=gen(24))
    check_evict(K, [160, 90], 2, 64, 16, BF, 40, 4, 8, 24, False, weights=w)


# ---------------------------------------------------------------------------------------------------------- all together
def serve(K, dev_steps, graph):
    """prompt (write + prefill), steps of decoding that sum weights, eviction in place, more steps: every output against the
    definition on the rows that are then in the cache.  graph: the decode step is captured once and replayed."""
    g = gen(31)
    B, Hkv, G, D, page, budget, sinks, recent = 3, 2, 4, 128, 16, 96, 4, 24
    Hq, width = Hkv * G, 14
    npg = B * width + 2
    pool = torch.full((npg, Hkv, 2, page, D), float("nan"), dtype=BF, device=DEV)
    bt = torch.randperm(npg, generator=g)[:B * width].int().view(B, width).to(DEV)
    prompt = [100, 37, 150]
    T = sum(prompt)
    qs = R.LOG2E / math.sqrt(D)
    ws = K.Workspace(B, Hkv, G, D, width * page, DEV, weights=True, new_tokens=T)
    cu = torch.tensor([0, 100, 137, 287], dtype=torch.int32, device=DEV)
    ln = torch.tensor(prompt, dtype=torch.int32, device=DEV)
    kv = torch.randn(T, 2 * Hkv, D, generator=g).to(BF).to(DEV)
    hist = []                                                      # [b] -> [n, 2 Hkv, D] cached rows (per head: kept ones)
    slots = torch.empty(T, dtype=torch.int64, device=DEV)
    for b in range(B):
        t = torch.arange(prompt[b], device=DEV)
        slots[int(cu[b]):int(cu[b + 1])] = bt[b, t // page].long() * page + t % page
        hist.append(kv[int(cu[b]):int(cu[b + 1])].view(-1, 2, Hkv, D).permute(1, 2, 0, 3).double())
    q = queries(T, Hq, D, BF, g)
    out = torch.empty(T, Hq * D, dtype=BF, device=DEV)
    K.write(kv, slots, pool)
    K.prefill(q, cu, pool, bt, ln, out, qs, ws=ws)
    for b in range(B):
        s = slice(int(cu[b]), int(cu[b + 1]))
        o, _, A, S = R.attend(q[s].double(), hist[b][0], hist[b][1], torch.arange(prompt[b]), qs, 0, 0)
        assert bool(((out[s].view(-1, Hq, D).double() - o).abs() <= bound(o, A, S, D, prompt[b], BF, True)).all())
    weights = torch.zeros(B, Hkv, width * page, device=DEV)
    nkv, nq, nslot = torch.empty(B, 2 * Hkv, D, dtype=BF, device=DEV), torch.empty(B, Hq, D, dtype=BF, device=DEV), torch.empty(B, dtype=torch.int64, device=DEV)
    o1 = torch.empty(B, Hq * D, dtype=BF, device=DEV)

    def body():
        K.write(nkv, nslot, pool)
        K.attn(nq, pool, bt, ln, o1, ws, qs, weights=weights)

    cg = None
    if graph:
        keep = pool.clone(), weights.clone()
        nkv.zero_(), nq.zero_(), nslot.fill_(-1)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            body()
        torch.cuda.current_stream().wait_stream(s)
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            body()
        pool.copy_(keep[0]), weights.copy_(keep[1])
    ref_w = [torch.zeros(Hkv, hist[b].shape[2], dtype=torch.float64, device=DEV) for b in range(B)]
    w_tol = 0.0
    for step in range(dev_steps):
        if step == dev_steps // 2:
            kept = torch.empty(B, Hkv, budget, dtype=torch.int32, device=DEV)
            nl, nw = torch.empty(B, dtype=torch.int32, device=DEV), torch.empty_like(weights)
            K.evict(pool, bt, ln, weights, budget, sinks, recent, kept, nl, nw)
            for b in range(B):
                m, n = int(nl[b]), hist[b].shape[2]
                assert m == min(n, budget)
                idx = kept[b, :, :m].long()
                assert R.evict_ref(weights[b], n, budget, sinks, recent) == idx.tolist()
                hist[b] = hist[b].gather(2, idx[None, :, :, None].expand(2, -1, -1, D))
                ref_w[b] = ref_w[b].gather(1, idx)
            ln.copy_(nl)
            weights.copy_(nw)
        x = torch.randn(B, 2 * Hkv, D, generator=g).to(BF).to(DEV)
        nkv.copy_(x)
        nq.copy_((torch.randn(B, Hq, D, generator=g) * 1.5).to(BF))
        n = ln.long()
        nslot.copy_(bt.long().gather(1, (n // page)[:, None])[:, 0] * page + n % page)
        ln += 1
        if cg is not None:
            cg.replay()
        else:
            body()
        for b in range(B):
            hist[b] = torch.cat([hist[b], x[b].view(2, Hkv, 1, D).double()], 2)
            L = hist[b].shape[2]
            assert L == int(ln[b])
            o, p, A, S = R.attend(nq[b:b + 1].double(), hist[b][0].contiguous(), hist[b][1].contiguous(), [L - 1], qs, 0, 0)
            assert bool(((o1[b].view(1, Hq, D).double() - o).abs() <= bound(o, A, S, D, L, BF, False)).all()), (step, b)
            ref_w[b] = torch.cat([ref_w[b], ref_w[b].new_zeros(Hkv, 1)], 1) + p[0].view(Hkv, G, L).sum(1)
            w_tol = max(w_tol, 2 * float(R.p_error(S, D, L).max()) + (G + 2) * 2.0 ** -24)
            got = weights[b, :, :L].double()
            assert bool(((got - ref_w[b]).abs() <= w_tol * ref_w[b] + (step + 1) * 2.0 ** -24 * ref_w[b]).all())


def test_serving_run(K):
    serve(K, 8, False)


def test_serving_run_captured(K):
    serve(K, 8, True)


def chain(K, sync):
    """writes, prompts, decode steps and evictions one after the other, with torch's own kernels between them"""
    g = gen(51)
    B, Hkv, G, D, page, width, budget = 4, 2, 4, 128, 16, 12, 64
    npg = B * width
    pool = torch.zeros(npg, Hkv, 2, page, D, dtype=BF, device=DEV)
    bt = torch.randperm(npg, generator=g).int().view(B, width).to(DEV)
    ws = K.Workspace(B, Hkv, G, D, width * page, DEV, weights=True, new_tokens=B * 90)
    seen = []

    def done(*t):
        if sync:
            torch.cuda.synchronize()
        seen.extend(x.clone() for x in t)

    for rep in range(6):
        n = 60 + 5 * rep
        kv = torch.randn(B * n, 2 * Hkv, D, generator=g).to(BF).to(DEV)
        q = (torch.randn(B * n, Hkv * G, D, generator=g) * 1.5).to(BF).to(DEV)
        t = torch.arange(n, device=DEV)
        slots = (bt[:, t // page].long() * page + t % page).view(-1)
        cu = torch.arange(B + 1, dtype=torch.int32, device=DEV) * n
        ln = torch.full((B,), n, dtype=torch.int32, device=DEV)
        w = torch.zeros(B, Hkv, width * page, device=DEV)
        out, o1 = torch.empty(B * n, Hkv * G * D, dtype=BF, device=DEV), torch.empty(B, Hkv * G * D, dtype=BF, device=DEV)
        K.write(kv, slots, pool)
        K.prefill(q, cu, pool, bt, ln, out, 0.12, ws=ws)
        done(out)
        for step in range(8):
            m = ln.long()
            K.write(kv[step * B:(step + 1) * B], bt.long().gather(1, (m // page)[:, None])[:, 0] * page + m % page, pool)
            ln += 1
            K.attn(q[step * B:(step + 1) * B], pool, bt, ln, o1, ws, 0.12, weights=w)
            q[(step + 1) * B:(step + 2) * B] += o1.view(B, Hkv * G, D)
            done(o1, w)
            if step % 3 == 2:
                kept = torch.empty(B, Hkv, budget, dtype=torch.int32, device=DEV)
                nl, nw = torch.empty(B, dtype=torch.int32, device=DEV), torch.empty_like(w)
                K.evict(pool, bt, ln, w, budget, 2, 16, kept, nl, nw)
                ln, w = nl, nw
                done(kept, nl, nw)
    torch.cuda.synchronize()
    return seen


def test_kernels_launched_early_keep_the_streams_order(K):
    """the same chain with the host waiting after every call and without any wait: the same bits"""
    a = chain(K, True)
    for _ in range(3):
        b = chain(K, False)
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_side_streams_and_graphs_with_their_own_workspaces(K):
    """two calls at once on two streams, each with its own workspace; then both captured and replayed at once"""
    g = gen(41)
    cases = []
    for i in range(2):
        pool, bt, ln = R.make_cache([700 + 100 * i, 33, 2000], 2, 128, 16, BF, g)
        q = queries(3, 8, 128, BF, g)
        cases.append((q, pool, bt, ln, torch.empty(3, 1024, dtype=BF, device=DEV),
                      K.Workspace(3, 2, 4, 128, bt.shape[1] * 16, DEV), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for q, pool, bt, ln, out, ws, st in cases:
            with torch.cuda.stream(st):
                K.attn(q, pool, bt, ln, out, ws, 0.1)
    torch.cuda.synchronize()
    for q, pool, bt, ln, out, ws, st in cases:
        check_attn(out.view(3, 8, 128), q, pool, bt, ln, 0.1, 0, 0)
        out.zero_()
    graphs = []
    for q, pool, bt, ln, out, ws, st in cases:
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg, stream=st):
            K.attn(q, pool, bt, ln, out, ws, 0.1)
        graphs.append(cg)
    for _ in range(3):
        for cg, c in zip(graphs, cases):
            with torch.cuda.stream(c[-1]):
                cg.replay()
    torch.cuda.synchronize()
    for q, pool, bt, ln, out, ws, st in cases:
        check_attn(out.view(3, 8, 128), q, pool, bt, ln, 0.1, 0, 0)


def test_front_end_refuses_tensors_that_are_not_on_the_device(K):
    pool, bt, ln = R.make_cache([20], 1, 64, 16, BF, gen(42))
    q = queries(1, 4, 64, BF, gen(43))
    ws = K.Workspace(1, 1, 4, 64, bt.shape[1] * 16, DEV)
    with pytest.raises(AssertionError):
        K.attn(q.cpu(), pool, bt, ln, torch.empty(1, 256, dtype=BF), ws, 0.1)
    with pytest.raises(AssertionError):
        K.attn(q, pool, bt.cpu(), ln, torch.empty(1, 256, dtype=BF, device=DEV), ws, 0.1)
