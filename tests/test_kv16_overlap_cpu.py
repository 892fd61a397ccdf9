"""k16_evict's checks with a place of its own for every tensor, and its refusal of results that lie over the inputs, over the
tables or over one another.  Everything is refused on the host, before any launch; no address is followed."""
import pytest

from flagrot_releaser_b200 import kv16

M = 1 << 20          # far apart
POOL, TABLE, LENS, WEIGHTS, KEPT, NLENS, NWEIGHTS, DST, DTABLE = (M * i for i in range(1, 10))
# 2 rows, 2 kv heads: weights [2, 2, 128] = 2048 bytes, kept and new_weights [2, 2, 64] = 1024, lengths 8, tables [2, 8] and [2, 4]
W_END, KEPT_END, NW_END, LENS_END, TABLE_END, DTABLE_END = 2048, 1024, 1024, 8, 64, 32


def _evict(**kw):
    a = dict(pool=POOL, npg=16, bt=TABLE, bt_stride=8, width=8, lens=LENS, B=2, Hkv=2, D=128, page=16, weights=WEIGHTS, w_bs=256,
             w_hs=128, w_len=128, budget=64, sinks=4, recent=8, kept=KEPT, new_lens=NLENS, new_weights=NWEIGHTS, nw_len=64, dst=DST,
             dst_pages=16, dst_bt=DTABLE, dst_stride=4, dst_width=4, stream=None)
    a.update(kw)
    return kv16.lib().k16_evict(*a.values())


@pytest.mark.parametrize("kw", [
    dict(new_lens=LENS), dict(new_lens=LENS + LENS_END - 4), dict(new_lens=LENS - 4),
    dict(new_weights=WEIGHTS), dict(new_weights=WEIGHTS + W_END - 4), dict(new_weights=WEIGHTS - NW_END + 4),
    dict(new_weights=LENS - 16), dict(new_lens=WEIGHTS + 1000), dict(kept=WEIGHTS + 4), dict(kept=LENS),
    dict(kept=TABLE), dict(new_lens=TABLE + TABLE_END - 4), dict(new_weights=TABLE - NW_END + 4),
    dict(kept=DTABLE), dict(new_lens=DTABLE + DTABLE_END - 4),
    dict(kept=NWEIGHTS), dict(new_lens=KEPT + KEPT_END - 4), dict(new_weights=NLENS), dict(new_weights=NLENS - NW_END + 4),
    # rows with gaps: the second row of a table, and of weights
    dict(bt_stride=1000, new_lens=TABLE + 4000), dict(bt_stride=1000, new_lens=TABLE + 4000 + 28), dict(bt_stride=1000, new_lens=TABLE + 3996),
    dict(dst_stride=500, new_lens=DTABLE + 2000 + 12), dict(w_bs=5000, new_lens=WEIGHTS + 4 * (5000 + 128 + 127)),
    dict(dst=None, dst_bt=None, dst_pages=0, new_lens=LENS), dict(dst=None, dst_bt=None, dst_pages=0, new_weights=WEIGHTS)])
def test_results_over_inputs_tables_or_one_another(kw):
    assert _evict(**kw) == -3


BAD = [(dict(D=96), -2), (dict(page=24), -2), (dict(Hkv=0), -3), (dict(npg=0), -3), (dict(width=-1), -3), (dict(pool=POOL + 8), -3),
       (dict(lens=None), -3), (dict(bt=None), -3), (dict(B=-1), -3), (dict(bt_stride=-1), -3), (dict(budget=0), -3), (dict(sinks=-1), -3),
       (dict(recent=-1), -3), (dict(sinks=60), -3), (dict(w_len=-1), -3), (dict(w_bs=-1), -3), (dict(w_hs=-1), -3), (dict(nw_len=63), -3),
       (dict(weights=None), -3), (dict(kept=None), -3), (dict(new_lens=None), -3), (dict(new_weights=None), -3), (dict(dst=None), -3),
       (dict(dst=DST + 8), -3), (dict(dst_pages=0), -3), (dict(dst_width=3), -3), (dict(dst_stride=3), -3), (dict(dst_bt=None, bt_stride=0), -3)]


@pytest.mark.parametrize("kw,rc", BAD)
def test_refusals_with_tensors_apart(kw, rc):
    assert _evict(**kw) == rc
