"""The 16-bit cache's library without a GPU: exported symbols, argument checks of every C entry (they run on the host, before
any launch) and of the Python front end, and the workspace sizes."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

from flagrot_releaser_b200 import kv16

ROOT = Path(__file__).resolve().parents[1]
A = 0x10000          # a 16-byte aligned address that no check follows


def test_header_symbols_exported():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "flagrot_kv16.h").read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(k16_[a-z0-9_]+)\s*\(", text)))
    assert len(names) >= 9, names
    L = ctypes.CDLL(str(ROOT / "flagrot_releaser_b200" / "lib" / "libflagrot_kv16.so"))
    assert not [n for n in names if not hasattr(L, n)]
    assert kv16.lib().k16_abi_version() == kv16.ABI


def _attn(**kw):
    a = dict(dtype=0, q=A, q_bs=1024, pool=A, npg=16, bt=A, bt_stride=8, width=8, lens=A, B=2, Hkv=2, G=4, D=128, page=16,
             qscale=0.1, window=0, sinks=0, weights=None, w_bs=0, w_hs=0, tickets=A, nt=1 << 20, ws=A, wsb=1 << 40, out=A, o_bs=1024,
             stream=None)
    a.update(kw)
    return kv16.lib().k16_attn(*a.values())


BAD_CACHE = [(dict(D=96), -2), (dict(page=24), -2), (dict(page=256), -2), (dict(Hkv=0), -3), (dict(npg=0), -3), (dict(width=-1), -3),
             (dict(npg=1 << 40), -3), (dict(width=1 << 27), -3), (dict(pool=None), -3), (dict(pool=A + 8), -3), (dict(lens=None), -3),
             (dict(bt=None), -3), (dict(B=-1), -3), (dict(bt_stride=-1), -3)]


@pytest.mark.parametrize("kw,rc", BAD_CACHE + [
    (dict(dtype=2), -2), (dict(G=0), -3), (dict(sinks=-1), -3), (dict(q=None), -3), (dict(q=A + 2), -3), (dict(q_bs=1020), -3),
    (dict(out=None), -3), (dict(out=A + 8), -3), (dict(o_bs=4), -3), (dict(weights=A, w_bs=-1), -3), (dict(weights=A, w_bs=0, w_hs=128), -3), (dict(weights=A, w_bs=256, w_hs=0), -3),
    (dict(o_bs=1016), -3), (dict(o_bs=0), -3), (dict(tickets=None), -4),
    (dict(nt=1), -4), (dict(ws=None), -4), (dict(wsb=16), -4), (dict(B=1 << 28, Hkv=64), -3)])
def test_attn_refusals(kw, rc):
    assert _attn(**kw) == rc


def test_empty_calls_launch_nothing():
    assert _attn(B=0, q=None, out=None) == 0
    assert _prefill(T=0) == 0 and _prefill(B=0) == 0
    assert _write(T=0, kv=None) == 0
    assert _evict(B=0) == 0


def _prefill(**kw):
    a = dict(dtype=0, q=A, q_ts=1024, T=64, cu=A, pool=A, npg=16, bt=A, bt_stride=8, width=8, lens=A, B=2, Hkv=2, G=4, D=128,
             page=16, qscale=0.1, window=0, sinks=0, tickets=A, nt=1 << 20, ws=A, wsb=1 << 40, out=A, o_ts=1024, stream=None)
    a.update(kw)
    return kv16.lib().k16_prefill(*a.values())


@pytest.mark.parametrize("kw,rc", BAD_CACHE + [
    (dict(dtype=-1), -2), (dict(G=0), -3), (dict(sinks=-1), -3), (dict(T=-1), -3), (dict(q=None), -3), (dict(q=A + 4), -3),
    (dict(q_ts=1028), -3), (dict(q_ts=0), -3), (dict(o_ts=512), -3), (dict(cu=None), -3), (dict(out=None), -3), (dict(o_ts=12), -3), (dict(T=1 << 30), -3), (dict(ws=None), -4)])
def test_prefill_refusals(kw, rc):
    assert _prefill(**kw) == rc


def _write(**kw):
    a = dict(kv=A, kv_ts=1024, kv_hs=128, slots=A, T=4, Hkv=2, D=128, page=16, npg=16, pool=A, stream=None)
    a.update(kw)
    return kv16.lib().k16_write(*a.values())


@pytest.mark.parametrize("kw,rc", [(dict(D=32), -2), (dict(page=8), -2), (dict(T=-1), -3), (dict(Hkv=0), -3), (dict(npg=0), -3),
                                   (dict(kv=None), -3), (dict(kv=A + 2), -3), (dict(kv_ts=1020), -3), (dict(kv_hs=4), -3),
                                   (dict(slots=None), -3), (dict(pool=None), -3), (dict(pool=A + 4), -3)])
def test_write_refusals(kw, rc):
    assert _write(**kw) == rc


def _evict(**kw):
    a = dict(pool=A, npg=16, bt=A, bt_stride=8, width=8, lens=A, B=2, Hkv=2, D=128, page=16, weights=A, w_bs=256, w_hs=128,
             w_len=128, budget=64, sinks=4, recent=8, kept=A, new_lens=A, new_weights=A, nw_len=64, dst=A, dst_pages=16, dst_bt=A,
             dst_stride=4, dst_width=4, stream=None)
    a.update(kw)
    return kv16.lib().k16_evict(*a.values())


@pytest.mark.parametrize("kw,rc", BAD_CACHE + [
    (dict(budget=0), -3), (dict(sinks=-1), -3), (dict(recent=-1), -3), (dict(sinks=60), -3), (dict(w_len=-1), -3), (dict(nw_len=63), -3),
    (dict(weights=None), -3), (dict(kept=None), -3), (dict(new_lens=None), -3), (dict(new_weights=None), -3), (dict(dst=None), -3),
    (dict(dst=A + 8), -3), (dict(dst_pages=0), -3), (dict(dst_width=3), -3), (dict(dst_stride=3), -3),
    (dict(dst_bt=None, bt_stride=0), -3)])
def test_evict_refusals(kw, rc):
    assert _evict(**kw) == rc


def test_workspace_sizes_grow_with_the_call():
    L = kv16.lib()
    n = L.k16_ws_bytes(64, 8, 4, 128, 4096, 0, 0)
    assert 0 < n < 1 << 28
    assert L.k16_ws_bytes(64, 8, 4, 128, 4096, 1, 0) >= n + 64 * 8 * 4 * 4096 * 4
    assert L.k16_ws_bytes(64, 8, 4, 128, 4096, 0, 65536) >= n
    assert L.k16_ws_tickets(64, 8, 4, 0) >= 64 * 8
    for bad in ((-1, 8, 4, 128, 64, 0, 0), (1, 0, 4, 128, 64, 0, 0), (1, 8, 0, 128, 64, 0, 5), (1, 8, 4, 100, 64, 0, 0), (1, 8, 4, 128, -1, 0, 0),
                (1, 8, 4, 128, 64, 0, -1)):
        assert L.k16_ws_bytes(*bad) == -3
    assert L.k16_ws_tickets(1, 8, 0, 5) == -3 and L.k16_ws_tickets(-1, 8, 4, 0) == -3
    # a workspace serves every smaller call: the sizes grow in each argument
    base = (3, 2, 3, 64, 100, 0, 50)
    for i, v in ((0, 7), (1, 4), (2, 12), (2, 40), (2, 130), (3, 128), (4, 5000), (5, 1), (6, 9000)):
        more = list(base)
        more[i] = v
        assert L.k16_ws_bytes(*more) >= L.k16_ws_bytes(*base)
        assert L.k16_ws_tickets(more[0], more[1], more[2], more[6]) >= L.k16_ws_tickets(base[0], base[1], base[2], base[6])
    assert kv16.chunk_bytes(16, 128) == L.k16_chunk_bytes(16, 128) == 16 * 128 * 2 * 2


def test_front_end_refuses_before_the_library_is_called():
    pool = torch.zeros(4, 2, 2, 16, 128, dtype=torch.bfloat16)
    q, out = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.zeros(3, 1024, dtype=torch.bfloat16)
    bt, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args in ((q.half(), pool, bt, lens, out), (q[:, :7], pool, bt, lens, out), (q, pool[..., :64], bt, lens, out),
                 (q, pool, bt.long(), lens, out), (q, pool, bt[:2], lens, out), (q, pool, bt, lens[:2], out),
                 (q, pool, bt, lens, out[:, :1000]), (q, pool.float(), bt, lens, out), (q[..., ::2], pool, bt, lens, out)):
        with pytest.raises(AssertionError):
            kv16.attn(*args, None, 0.1)
    kv, slots = torch.zeros(5, 4, 128, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int64)
    for args in ((kv.half(), slots, pool), (kv[:, :3], slots, pool), (kv, slots.int(), pool), (kv, slots[:4], pool), (kv, slots, pool[0])):
        with pytest.raises(AssertionError):
            kv16.write(*args)
    w = torch.zeros(3, 2, 32)
    kept, nl = torch.zeros(3, 2, 16, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    nw = torch.zeros(3, 2, 16)
    for args in ((16, 9, 8, kept, nl, nw), (16, 0, 0, kept[:, :, :8], nl, nw), (16, 0, 0, kept, nl.long(), nw), (16, 0, 0, kept, nl, nw[..., :8]),
                 (0, 0, 0, kept, nl, nw), (16, -1, 0, kept, nl, nw)):
        with pytest.raises(AssertionError):
            kv16.evict(pool, bt, lens, w, *args)
    cu = torch.zeros(4, dtype=torch.int32)
    for args in ((q, cu[:3], pool, bt, lens, out), (q, cu.long(), pool, bt, lens, out), (q, cu, pool, bt, lens, out.float())):
        with pytest.raises(AssertionError):
            kv16.prefill(*args, 0.1)


def test_evict_refuses_results_over_its_inputs():
    pool, bt = torch.zeros(4, 2, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
    w, kept = torch.zeros(3, 2, 32), torch.zeros(3, 2, 16, dtype=torch.int32)
    lens = torch.zeros(8, dtype=torch.int32)
    for a, b in ((0, 0), (0, 2), (2, 0)):
        with pytest.raises(AssertionError, match="new_lens overlaps seq_lens"):
            kv16.evict(pool, bt, lens[a:a + 3], w, 16, 0, 0, kept, lens[b:b + 3], torch.zeros(3, 2, 16))
    with pytest.raises(AssertionError, match="new_weights overlaps weights"):
        kv16.evict(pool, bt, lens[:3], w, 16, 0, 0, kept, lens[3:6], w.view(-1)[96:].view(3, 2, 16))
