"""The 16-bit paged cache on a GPU in calls that the documentation allows and test_kv16_gpu.py does not make.  Definitions and
tolerances are the ones of that file and of _kv16.py."""
import math

import pytest
import torch

from tests import _kv16 as R
from tests.test_kv16_gpu import BF, DEV, FP, bound, check_attn, check_evict, check_prefill, gen, queries, run_attn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from flagrot_releaser_b200 import kv16
    kv16.lib()
    yield kv16
    assert kv16.device_status() == 0


def carve(shapes):
    """tensors one right behind the other in one buffer (4-byte types)"""
    sizes = [torch.Size(s).numel() for s, _ in shapes]
    buf, out, at = torch.zeros(sum(sizes), dtype=torch.int32, device=DEV), [], 0
    for (s, t), n in zip(shapes, sizes):
        out.append(buf[at:at + n].view(t).view(s))
        at += n
    return out


@pytest.mark.parametrize("order", [[0, 1, 2, 3, 4, 5], [5, 3, 1, 4, 2, 0], [2, 4, 0, 5, 1, 3]])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_takes_tensors_that_touch(K, order, in_place):
    """lengths, weights, table and the three results side by side in one buffer, in any order, are not an overlap"""
    g = gen(61)
    lens, Hkv, page, budget = [100, 7, 333], 2, 16, 64
    pool, table, _ = R.make_cache(lens, Hkv, 64, page, BF, g, poison=False)
    W = table.shape[1] * page
    shapes = [((3,), torch.int32), ((3, Hkv, W), torch.float32), (tuple(table.shape), torch.int32), ((3, Hkv, budget), torch.int32),
              ((3,), torch.int32), ((3, Hkv, budget), torch.float32)]
    t = [None] * 6
    for i, x in zip(order, carve([shapes[i] for i in order])):
        t[i] = x
    ln, w, bt, kept, nl, nw = t
    ln.copy_(torch.tensor(lens)), bt.copy_(table), w.copy_(torch.rand(w.shape, generator=g))
    keep = [x.clone() for x in (ln, w, bt)]
    kw = {} if in_place else dict(dst_pool=torch.zeros_like(pool), dst_table=torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4))
    K.evict(pool, bt, ln, w, budget, 4, 16, kept, nl, nw, **kw)
    assert all(torch.equal(a, b) for a, b in zip(keep, (ln, w, bt)))
    for b, n in enumerate(lens):
        m = min(n, budget)
        ref = R.evict_ref(w[b], n, budget, 4, 16)
        assert int(nl[b]) == m and [x[:m] for x in kept[b].tolist()] == ref
        assert torch.equal(nw[b, :, :m], w[b].gather(1, torch.tensor(ref, device=DEV)))


def test_evict_takes_results_in_the_gaps_of_a_table(K):
    """a table whose rows lie far apart; the results lie between them"""
    g = gen(62)
    lens, Hkv, page, budget = [100, 90], 1, 16, 32
    pool, table, ln = R.make_cache(lens, Hkv, 64, page, BF, g, poison=False)
    width, gap = table.shape[1], 2 * budget + 2
    buf = torch.zeros(2, width + 2 * gap, dtype=torch.int32, device=DEV)
    bt = buf[:, :width]
    bt.copy_(table)
    between = buf.view(-1)[width:]
    kept, nl = between[:2 * budget].view(2, 1, budget), between[2 * budget:2 * budget + 2]
    nw = between[gap:gap + 2 * budget].view(torch.float32).view(2, 1, budget)
    w = torch.rand(2, Hkv, width * page, generator=g).to(DEV)
    K.evict(pool, bt, ln, w, budget, 2, 8, kept, nl, nw)
    assert torch.equal(bt, table) and nl.tolist() == [budget, budget]
    for b, n in enumerate(lens):
        assert kept[b].tolist() == R.evict_ref(w[b], n, budget, 2, 8)


def test_device_status_waits_for_side_streams(K):
    """the status is that of the calls made so far, on streams that the default stream does not wait for too"""
    K.device_status()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            torch.cuda._sleep(400_000_000)                     # a fifth of a second
    assert not any(s.query() for s in streams), "the streams ended too soon for this test"
    assert K.device_status() == 0
    assert all(s.query() for s in streams)


def barred(lens, first, Hkv, D, page, dtype, g, value):
    """a cache whose rows' first `first` keys are barred by `value` in their first channel, which every query multiplies by a
    positive number"""
    pool, bt, ln = R.make_cache(lens, Hkv, D, page, dtype, g)
    pc = pool.cpu()
    for b, n in enumerate(lens):
        for j in range(min(first, n)):
            pc[int(bt[b, j // page]), :, 0, j % page, 0] = value
    return pc.to(DEV), bt, ln


@pytest.mark.parametrize("value", [-math.inf, "lowest"])
@pytest.mark.parametrize("first", [1, 31, 32, 33, 64, 200, 1000])
@pytest.mark.parametrize("G,D,page,dtype", [(4, 128, 16, BF), (1, 64, 64, FP), (12, 64, 16, BF), (12, 128, 32, FP), (24, 128, 16, BF)])
def test_attn_keys_barred_by_infinite_scores(K, G, D, page, dtype, first, value):
    """keys whose score is -inf have weight 0, however many of them come first; a row that has no others gives zeros and adds
    nothing to the weights.  The type's lowest value does the same beside other keys (bf16: the product passes the 32-bit
    range; fp16: scores below -40 000)."""
    g = gen(71)
    lens = [5, 32, 40, 64, 300, 1111, 9000]
    pool, bt, ln = barred(lens, first, 2, D, page, dtype, g, -math.inf)
    given = pool if value != "lowest" else torch.where(pool == -math.inf, torch.full((), torch.finfo(dtype).min, dtype=dtype, device=DEV), pool)
    q = queries(len(lens), 2 * G, D, dtype, g)
    q[..., 0] = q[..., 0].abs() + 4
    w0 = torch.rand(len(lens), 2, bt.shape[1] * page, generator=g).to(DEV)
    w1 = w0.clone()
    qs = R.LOG2E / math.sqrt(D)
    for w in (w1, None):
        out = run_attn(K, q, given, bt, ln, qs, weights=w)
        none = ln <= first
        if value != "lowest":
            assert bool((out[none] == 0).all())
            if w is not None:
                assert torch.equal(w0[none], w1[none])
        assert bool(torch.isfinite(out).all())
        some = (~none).nonzero().flatten()
        check_attn(out[some], q[some], pool, bt[some], ln[some], qs, 0, 0, *((w0[some], w1[some]) if w is not None else ()))


@pytest.mark.parametrize("first", [1, 64, 65, 300])
@pytest.mark.parametrize("G,D,page,dtype", [(4, 128, 16, BF), (12, 64, 64, FP)])
def test_prefill_keys_barred_by_infinite_scores(K, G, D, page, dtype, first):
    g = gen(72)
    lens, new = [5, 40, 300, 1111, 9000], [5, 1, 200, 333, 9]
    pool, bt, ln = barred(lens, first, 2, D, page, dtype, g, -math.inf)
    T = sum(new)
    q = queries(T, 2 * G, D, dtype, g)
    q[..., 0] = q[..., 0].abs() + 4
    cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=DEV)
    ws, qs = K.Workspace(len(lens), 2, G, D, bt.shape[1] * page, DEV, new_tokens=T), R.LOG2E / math.sqrt(D)
    out = torch.full((T, 2 * G * D), 7.0, dtype=dtype, device=DEV)
    K.prefill(q, cu, pool, bt, ln, out, qs, ws=ws)
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = R.rows_of(pool, bt[b], n)
        s = slice(int(cu[b]), int(cu[b + 1]))
        o, _, A, S = R.attend(q[s].double(), k, v, torch.arange(n - m, n), qs, 0, 0)
        err = (out[s].view(m, 2 * G, D).double() - o).abs()
        assert bool((err <= bound(o, A, S, D, n, dtype, True)).all()), (b, n, m)


def prefill_hidden(K, lens, new, Hkv, G, D, page, dtype, window, sinks, seed, give_back):
    """prefill over a cache whose rows that none of the new tokens sees (behind the first one's window, no sinks) hold NaN and
    infinities, keys and values; give_back: the pages that hold only such rows belong to someone else's NaN, or to no pool page"""
    g = gen(seed)
    pool, bt, ln = R.make_cache(lens, Hkv, D, page, dtype, g)
    pc, table = pool.cpu(), bt.cpu()
    for b, (n, m) in enumerate(zip(lens, new)):
        lo = max(max(n - m, 0) + 1 - window, 0)
        for j in range(sinks, min(lo, n)):
            pc[int(table[b, j // page]), :, :, j % page] = (math.nan, math.inf, -math.inf)[j % 3]
        if give_back:
            for i in range(-(-sinks // page), lo // page):
                table[b, i] = (-1, pool.shape[0] + 7, int(bt[b, -1]))[i % 3] if i % 4 else table[b, i]
    given, clean = pc.to(DEV), pool
    T = sum(new)
    q = queries(T, G * Hkv, D, dtype, g, pad=1)
    cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=DEV)
    ws, qs = K.Workspace(len(lens), Hkv, G, D, bt.shape[1] * page, DEV, new_tokens=T), R.LOG2E / math.sqrt(D)
    out = torch.full((T, Hkv * G * D), 7.0, dtype=dtype, device=DEV)
    K.prefill(q, cu, given, table.to(DEV), ln, out, qs, window=window, sinks=sinks, ws=ws)
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = R.rows_of(clean, bt[b], n)
        hidden = max(m - n, 0)
        s = slice(int(cu[b]) + hidden, int(cu[b + 1]))
        assert bool((out[int(cu[b]):s.start] == 0).all())
        if s.start < s.stop:
            o, _, A, S = R.attend(q[s].double(), k, v, torch.arange(n - m + hidden, n), qs, window, sinks)
            err = (out[s].view(-1, Hkv * G, D).double() - o).abs()
            assert bool((err <= bound(o, A, S, D, n, dtype, True)).all()), (b, n, m)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 4), (64, 0), (100, 1), (100, 70), (128, 128), (129, 130), (300, 4), (1000, 4)])
@pytest.mark.parametrize("G,D,page,dtype", [(4, 128, 16, BF), (6, 64, 32, FP), (4, 128, 64, FP), (3, 64, 128, BF), (1, 128, 128, BF)])
@pytest.mark.parametrize("give_back", [False, True])
def test_prefill_rows_that_no_new_token_sees_may_hold_anything(K, window, sinks, G, D, page, dtype, give_back):
    prefill_hidden(K, [700, 90, 1300, 513, 20, 3000], [200, 20, 333, 1, 30, 2], 2, G, D, page, dtype, window, sinks, window + sinks + D, give_back)


def test_prefill_long_cache_behind_a_window_may_hold_anything(K):
    prefill_hidden(K, [20000, 9000], [70, 600], 1, 4, 128, 16, BF, 4096, 4, 5, True)
    prefill_hidden(K, [20000, 9000], [70, 600], 2, 8, 64, 64, FP, 777, 130, 6, True)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 4), (64, 0), (100, 33), (129, 130), (300, 1), (5000, 4)])
@pytest.mark.parametrize("G,D,page,dtype", [(4, 128, 64, FP), (4, 64, 128, BF), (2, 128, 128, BF)])
def test_prefill_window_and_sinks_over_large_pages(K, window, sinks, G, D, page, dtype):
    check_prefill(K, [700, 90, 1300, 513], [700, 20, 333, 1], 2, G, D, page, dtype, window, sinks, window + sinks)


@pytest.mark.parametrize("positions", [32768, 32769, 49153, 65537, 131073])
def test_evict_around_the_sizes_where_clusters_grow(K, positions):
    """80 groups: a cluster grows where its CTAs' registers no longer hold the weights, by rounding up"""
    lens = [positions, 40, positions - 1, 33] + [5] * 36
    w = torch.rand(40, 2, positions, generator=gen(positions))
    w[2] = torch.randint(0, 3, (2, positions), generator=gen(1)).float()
    check_evict(K, lens, 2, 64, 16, BF, 3000, 4, 100, 33, False, weights=w)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_takes_rows_as_long_as_their_weights(K, in_place):
    """weights of 100 entries: longer rows lose their newest tokens, within the budget and above it"""
    w = torch.rand(4, 2, 100, generator=gen(81))
    check_evict(K, [160, 90, 120, 101], 2, 64, 16, BF, 40, 4, 8, 82, in_place, weights=w)
    check_evict(K, [160, 90, 120, 101], 2, 64, 16, BF, 110, 4, 8, 83, in_place, weights=w)


@pytest.mark.parametrize("D,page,dtype", [(128, 16, BF), (128, 64, FP), (128, 128, BF), (64, 32, BF)])
@pytest.mark.parametrize("lens,budget", [([900, 300, 301], 300), ([5000, 700, 90, 2000], 700), ([9000, 64, 2500], 2100), ([12000], 11990)])
def test_evict_in_place_by_clusters(K, D, page, dtype, lens, budget):
    """few rows of large budgets: two, four and eight CTAs move a row together"""
    check_evict(K, lens, 2, D, page, dtype, budget, 4, 100, 34, True)


def test_prefill_and_evict_on_side_streams_and_in_graphs(K):
    """prefill whose pairs are cut along their keys, and evictions in place and to other pages, on three streams at once, each
    with a workspace and results of its own; then captured, and the graphs replayed at once"""
    g = gen(91)
    qs, budget = 0.11, 700
    calls, checks = [], []
    for i, (n, m) in enumerate([(9000, 70), (12000, 33)]):
        pool, bt, ln = R.make_cache([n, 300], 1, 128, 16, BF, g)
        q = queries(m + 5, 4, 128, BF, g)
        cu = torch.tensor([0, m, m + 5], dtype=torch.int32, device=DEV)
        ws = K.Workspace(2, 1, 4, 128, bt.shape[1] * 16, DEV, new_tokens=m + 5)
        out = torch.zeros(m + 5, 512, dtype=BF, device=DEV)
        ref = []
        for b, (s0, s1, L) in enumerate([(0, m, n), (m, m + 5, 300)]):
            k, v = R.rows_of(pool, bt[b], L)
            o, _, A, S = R.attend(q[s0:s1].double(), k, v, torch.arange(L - s1 + s0, L), qs, 0, 0)
            ref.append((o, bound(o, A, S, 128, L, BF, True)))
        o, tol = (torch.cat(x) for x in zip(*ref))
        calls.append(lambda q=q, cu=cu, pool=pool, bt=bt, ln=ln, out=out, ws=ws: K.prefill(q, cu, pool, bt, ln, out, qs, ws=ws))
        checks.append(lambda out=out, o=o, tol=tol, m=m: bool(((out.view(m + 5, 4, 128).double() - o).abs() <= tol).all()))
    for in_place in (True, False):
        lens = [3000, 650, 1200]
        pool, bt, ln = R.make_cache(lens, 2, 128, 16, BF, g, poison=False)
        start, w = pool.clone(), torch.rand(3, 2, bt.shape[1] * 16, generator=g).to(DEV)
        dst = pool if in_place else torch.zeros(3 * 44, 2, 2, 16, 128, dtype=BF, device=DEV)
        dbt = bt if in_place else torch.randperm(132, generator=g).int().view(3, 44).to(DEV)
        kept, nl, nw = torch.empty(3, 2, budget, dtype=torch.int32, device=DEV), torch.empty(3, dtype=torch.int32, device=DEV), torch.empty(3, 2, budget, device=DEV)
        exp, ref = (start if in_place else dst).clone(), [R.evict_ref(w[b], n, budget, 4, 64) for b, n in enumerate(lens)]
        for b in range(3):
            for h in range(2):
                idx = torch.tensor(ref[b][h], device=DEV)
                at = torch.arange(len(idx), device=DEV)
                exp[dbt[b, at // 16].long(), h, :, at % 16] = start[bt[b, idx // 16].long(), h, :, idx % 16]
        kw = {} if in_place else dict(dst_pool=dst, dst_table=dbt)

        def call(pool=pool, bt=bt, ln=ln, w=w, kept=kept, nl=nl, nw=nw, kw=kw, start=start, dst=dst):
            pool.copy_(start)
            if kw:
                dst.zero_()
            K.evict(pool, bt, ln, w, budget, 4, 64, kept, nl, nw, **kw)

        def check(dst=dst, exp=exp, kept=kept, nl=nl, ref=ref, lens=lens):
            return torch.equal(dst, exp) and nl.tolist() == [min(n, budget) for n in lens] and \
                all([x[:len(r)] for x, r in zip(kept[b].tolist(), ref[b])] == ref[b] for b in range(3) for r in ref[b])

        calls.append(call)
        checks.append(check)
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(4):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                c()
    torch.cuda.synchronize()
    assert all(c() for c in checks)
    graphs = []
    for c, s in zip(calls, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            c()
    for _ in range(4):
        for cg, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                cg.replay()
    torch.cuda.synchronize()
    assert all(c() for c in checks)


def test_two_graphs_share_a_workspace_in_turn(K):
    """a decode step and a prompt captured with the same workspace, replayed one after the other on one stream while the lengths
    change under them"""
    g = gen(92)
    lens = [2000, 33, 700]
    pool, bt, ln = R.make_cache(lens, 2, 128, 16, BF, g)
    T, qs = 90, 0.1
    ws = K.Workspace(3, 2, 4, 128, bt.shape[1] * 16, DEV, weights=True, new_tokens=T)
    q1, qn = queries(3, 8, 128, BF, g), queries(T, 8, 128, BF, g)
    cu = torch.tensor([0, 60, 60, T], dtype=torch.int32, device=DEV)
    o1, on = torch.zeros(3, 1024, dtype=BF, device=DEV), torch.zeros(T, 1024, dtype=BF, device=DEV)
    w = torch.zeros(3, 2, bt.shape[1] * 16, device=DEV)
    steps = (lambda: K.attn(q1, pool, bt, ln, o1, ws, qs, weights=w)), (lambda: K.prefill(qn, cu, pool, bt, ln, on, qs, ws=ws))
    graphs = []
    for f in steps:
        f()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            f()
    for now in ([2000, 33, 700], [1, 0, 31], [1500, 20, 64]):
        ln.copy_(torch.tensor(now, dtype=torch.int32))
        for _ in range(3):
            w.zero_()
            for cg in graphs:
                cg.replay()
        check_attn(o1.view(3, 8, 128), q1, pool, bt, torch.tensor(now), qs, 0, 0, torch.zeros_like(w), w)
        for b, (s0, s1) in enumerate([(0, 60), (60, 60), (60, T)]):
            n, m = now[b], s1 - s0
            lost = max(m - n, 0)
            assert bool((on[s0:s0 + lost] == 0).all())
            if m > lost:
                k, v = R.rows_of(pool, bt[b], n)
                o, _, A, S = R.attend(qn[s0 + lost:s1].double(), k, v, torch.arange(n - m + lost, n), qs, 0, 0)
                assert bool(((on[s0 + lost:s1].view(-1, 8, 128).double() - o).abs() <= bound(o, A, S, 128, n, BF, True)).all())
        assert int(ws.tickets.abs().max()) == 0


@pytest.mark.parametrize("captured", [False, True])
def test_calls_that_follow_other_streams_wait_for_all_of_them(K, captured):
    """rows written on two side streams, a copy on a third, and the attention that joins them by events: early launches wait for
    every one of them, eagerly and as branches of a graph"""
    g = gen(93)
    B, Hkv, G, D, page, n = 8, 4, 4, 128, 16, 4000
    width = -(-n // page)
    pool = torch.zeros(B * width, Hkv, 2, page, D, dtype=BF, device=DEV)
    bt = torch.randperm(B * width, generator=g).int().view(B, width).to(DEV)
    t = torch.arange(n, device=DEV)
    slots = (bt[:, t // page].long() * page + t % page).view(B, n)
    kv = [torch.randn(B // 2 * n, 2 * Hkv, D, generator=g).to(BF).to(DEV) for _ in range(2)]
    qs = [queries(B, Hkv * G, D, BF, g) for _ in range(2)]
    q, ln, w = torch.empty_like(qs[0]), torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, Hkv, width * page, device=DEV)
    full = torch.full((B,), n, dtype=torch.int32, device=DEV)
    out = torch.zeros(B, Hkv * G * D, dtype=BF, device=DEV)
    ws = K.Workspace(B, Hkv, G, D, width * page, DEV, weights=True)
    sides = [torch.cuda.Stream() for _ in range(3)]

    def step():
        main = torch.cuda.current_stream()
        pool.zero_(), ln.zero_(), w.zero_(), q.zero_()
        for s in sides:
            s.wait_stream(main)
        for i in range(2):
            with torch.cuda.stream(sides[i]):
                K.write(kv[i], slots[i * B // 2:(i + 1) * B // 2].reshape(-1), pool)
        with torch.cuda.stream(sides[2]):
            q.copy_(qs[0])
            ln.copy_(full)
        for s in sides:
            main.wait_stream(s)
        K.attn(q, pool, bt, ln, out, ws, 0.1, weights=w)

    step()
    torch.cuda.synchronize()
    check_attn(out.view(B, Hkv * G, D), qs[0], pool, bt, full, 0.1, 0, 0, torch.zeros_like(w), w)
    first = out.clone(), w.clone()
    run = step
    if captured:
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            step()
        run = cg.replay
    for _ in range(20):
        run()
    torch.cuda.synchronize()
    assert torch.equal(out, first[0]) and torch.equal(w, first[1])
