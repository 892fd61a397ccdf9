"""Host side of libflagrot_kv16.so for B200: the 16-bit (bf16 / fp16) paged key-value cache.

The cache of the layers a deployment does not quantise (sliding-window layers, whose caches are small; first and last
layers; the uncompressed arm a quantised format is compared with), with the same block tables, slots and score scaling as
the quantised pages:

  write                 append rows to the pages
  attn                  decode attention, one new token per row; optionally a sliding window with sink tokens, optionally
                        adding the attention weight each cached token receives to a running sum
  prefill               attention of many new tokens per row (causal; the same window and sinks)
  evict                 keep the tokens with the largest sums, in place or into other pages
  Workspace             split partials, merge tickets and scores of attn / prefill; allocate before graph capture

Pool: torch tensor [num_pages, Hkv, 2, page, D], contiguous, bf16 or fp16 (index 0 of the third axis keys, 1 values); D 64 |
128; page 16 | 32 | 64 | 128.  No counterpart in the reference, whose 16-bit rows are a ring of sinks and recent tokens.

The library must exist (built by flagrot_releaser_b200/_build.py): there is no fallback.  FLAGROT_KV16_LIB overrides its
location.  All launches go to torch's current CUDA stream and are asynchronous; the tensors have to be on the current device.
Capture a call in a CUDA graph after it has run once.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch

_PKG = Path(__file__).resolve().parent
ABI = 1
DTYPES = {torch.bfloat16: 0, torch.float16: 1}
PAGES, HEAD_DIMS = (16, 32, 64, 128), (64, 128)
MAX_POS = 1 << 30                # positions are below it


def _lib_path() -> Path:
    return Path(os.environ.get("FLAGROT_KV16_LIB", _PKG / "lib" / "libflagrot_kv16.so"))


_LIB = None


def lib():
    """the loaded library (ctypes).  Raises if it is missing or reports another ABI version."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = _lib_path()
    if not path.exists():
        raise RuntimeError(f"{path} not found: build it with `python -m flagrot_releaser_b200._build`; there is no fallback")
    L = ctypes.CDLL(str(path))
    P, I, LL, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
    L.k16_abi_version.restype = I
    if L.k16_abi_version() != ABI:
        raise RuntimeError(f"libflagrot_kv16 ABI {L.k16_abi_version()} != {ABI}: rebuild ({path})")
    L.k16_last_error.restype = ctypes.c_char_p
    L.k16_chunk_bytes.argtypes = [I, I]
    L.k16_write.argtypes = [P, LL, LL, P, I, I, I, I, LL, P, P]
    L.k16_ws_bytes.argtypes, L.k16_ws_bytes.restype = [I, I, I, I, LL, I, LL], LL
    L.k16_ws_tickets.argtypes, L.k16_ws_tickets.restype = [I, I, I, LL], LL
    L.k16_attn.argtypes = [I, P, LL, P, LL, P, LL, I, P, I, I, I, I, I, F, I, I, P, LL, LL, P, LL, P, LL, P, LL, P]
    L.k16_prefill.argtypes = [I, P, LL, I, P, P, LL, P, LL, I, P, I, I, I, I, I, F, I, I, P, LL, P, LL, P, LL, P]
    L.k16_evict.argtypes = [P, LL, P, LL, I, P, I, I, I, I, P, LL, LL, I, I, I, I, P, P, P, I, P, LL, P, LL, I, P]
    for n in ("k16_chunk_bytes", "k16_write", "k16_attn", "k16_prefill", "k16_evict", "k16_device_status"):
        getattr(L, n).restype = I
    _LIB = L
    return L


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what}: failed (code {rc}, {lib().k16_last_error().decode()})")


def _stream(*tensors):
    """the current stream of the current device, on which every tensor has to be"""
    dev = torch.cuda.current_device()
    for t in tensors:
        assert t.get_device() == dev, f"tensor on {t.device}, current device cuda:{dev}"
    return torch._C._cuda_getCurrentRawStream(dev)


def chunk_bytes(page: int, D: int = 128) -> int:
    """bytes per (page, kv head)"""
    return 4 * page * D


def device_status() -> int:
    """0, or the source line of a bounded device-side wait that gave up; -1 when the device cannot be asked.  Waits for every
    stream of the current device: not during a capture."""
    return lib().k16_device_status()


class Workspace:
    """split partials and scores of attn / prefill for up to `rows` sequences of up to max_len cached tokens (the block
    table's width times the page) and G q heads per kv head, and the merge tickets (zeroed once, left zero by every call).
    weights: attn is called with weights; new_tokens: the most rows of q that prefill is called with (0: attn only).
    Allocate once before CUDA-graph capture; calls that may overlap on the device need workspaces of their own."""

    def __init__(self, rows, Hkv, G, D, max_len, device, weights=False, new_tokens=0):
        L = lib()
        assert rows >= 0 and Hkv > 0 and G > 0 and D in HEAD_DIMS and max_len >= 0 and new_tokens >= 0
        self.nbytes = int(L.k16_ws_bytes(rows, Hkv, G, D, max_len, int(weights), new_tokens))
        self.ntickets = int(L.k16_ws_tickets(rows, Hkv, G, new_tokens))
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        self.tickets = torch.zeros(max(self.ntickets, 1), dtype=torch.int32, device=device)
        self.pbuf, self.ptickets = self.buf.data_ptr(), self.tickets.data_ptr()


def _pool_ok(pool):
    """(num_pages, Hkv, page, D)"""
    assert pool.dim() == 5 and pool.dtype in DTYPES and pool.is_contiguous(), "pool: [num_pages, Hkv, 2, page, D] bf16 | fp16, contiguous"
    npg, Hkv, two, page, D = pool.shape
    assert two == 2 and page in PAGES and D in HEAD_DIMS, "page 16 | 32 | 64 | 128, head dim 64 | 128"
    return npg, Hkv, page, D


def _table_ok(block_table, B):
    """(width, row stride)"""
    assert block_table.dtype == torch.int32 and block_table.dim() == 2
    rows, width = block_table.shape
    st = block_table.stride()
    assert rows == B and (st[1] == 1 or width <= 1), "block_table: int32 [B, width]"
    return width, st[0]


def _lens_ok(lens, B):
    assert lens.dtype == torch.int32 and lens.dim() == 1 and lens.shape[0] == B and (B <= 1 or lens.stride(0) == 1), "seq_lens: int32 [B]"


def _q_ok(q, out, pool, Hkv, D):
    """(rows, G, dtype code, row strides of q and out)"""
    n, Hq, Dq = q.shape
    assert q.dtype == pool.dtype == out.dtype and Dq == D and Hq > 0 and Hq % Hkv == 0, "q: [rows, G Hkv, D] of the pool's type"
    qs, os_ = q.stride(), out.stride()
    assert qs[2] == 1 and (qs[1] == D or Hq == 1) and out.shape[0] == n and out.numel() == n * Hq * D and os_[-1] == 1 and \
        (len(os_) == 2 or os_[1] == D or Hq == 1), "out: [rows, G Hkv D]"
    return n, Hq // Hkv, DTYPES[q.dtype], qs[0] if n > 1 else 0, os_[0] if n > 1 else 0


def write(kv, slots, pool):
    """kv [T, 2 Hkv, D] (K rows of all heads, then V rows; 16-byte aligned rows, any token and row strides that are multiples of
    8 elements) -> pool at slots int64 [T] (slot = page_id * page + offset; < 0 or past the pool skipped).  The slots that are
    written must be distinct."""
    npg, Hkv, page, D = _pool_ok(pool)
    T, rows, Dk = kv.shape
    st = kv.stride()
    assert kv.dtype == pool.dtype and rows == 2 * Hkv and Dk == D and st[2] == 1, "kv: [T, 2 Hkv, D] of the pool's type"
    assert slots.dtype == torch.int64 and slots.dim() == 1 and slots.shape[0] == T and (T <= 1 or slots.stride(0) == 1), "slots: int64 [T]"
    if T == 0:
        return
    stream = _stream(kv, slots, pool)
    _check(lib().k16_write(kv.data_ptr(), st[0] if T > 1 else 0, st[1], slots.data_ptr(), T, Hkv, D, page, npg, pool.data_ptr(), stream),
           "k16_write")


def attn(q, pool, block_table, seq_lens, out, ws, qscale, window=0, sinks=0, weights=None):
    """q [B, G Hkv, D] -> out [B, G Hkv D] (or [B, G Hkv, D]), rows 16-byte aligned; block_table int32 [B, width] (row stride 0
    allowed), seq_lens int32 [B]; qscale = softmax scale * log2(e).  Key j is seen when j < len and (window <= 0 or
    j >= len - window or j < sinks); a row that sees no key, or only such with a score of -inf, gives zeros.  weights fp32
    [B, Hkv, >= width * page] or None: the softmax weights of every seen key, summed over the G heads, are added to it."""
    npg, Hkv, page, D = _pool_ok(pool)
    B, G, dt, qs, os_ = _q_ok(q, out, pool, Hkv, D)
    width, bs = _table_ok(block_table, B)
    _lens_ok(seq_lens, B)
    if B == 0:
        return
    stream = _stream(q, pool, block_table, seq_lens, out, ws.buf)
    wp = wb = wh = 0
    if weights is not None:
        assert weights.dtype == torch.float32 and weights.dim() == 3, "weights: fp32 [B, Hkv, >= width * page]"
        (wB, wH, W), (wb, wh, w1) = weights.shape, weights.stride()
        assert wB == B and wH == Hkv and W >= width * page and (w1 == 1 or W <= 1), "weights: fp32 [B, Hkv, >= width * page]"
        _stream(weights)
        wp = weights.data_ptr()
    window, sinks = min(window, MAX_POS), min(sinks, MAX_POS)
    _check(lib().k16_attn(dt, q.data_ptr(), qs, pool.data_ptr(), npg, block_table.data_ptr(), bs, width, seq_lens.data_ptr(), B, Hkv, G,
                          D, page, qscale, window, sinks, wp, wb, wh, ws.ptickets, ws.ntickets, ws.pbuf, ws.nbytes, out.data_ptr(),
                          os_, stream), "k16_attn")


def prefill(q, cu_q, pool, block_table, seq_lens, out, qscale, window=0, sinks=0, ws=None):
    """q [T, G Hkv, D] -> out [T, G Hkv D], rows 16-byte aligned: row b's new tokens are rows cu_q[b] .. cu_q[b + 1] (int32
    [B + 1]) and the last ones of its seq_lens[b] cached tokens (their keys and values are in the pages already).  The token
    at position p sees key j <= p when window <= 0 or j > p - window or j < sinks; one at a negative position gives zeros;
    rows of out that belong to no sequence are left as they are.  Cached rows that none of a sequence's new tokens sees may
    hold anything (their pages may belong to others by now); the values of those that some see must be finite.  The softmax
    weights are rounded to the pool's type before they meet the values (attn keeps them to 2^-17).  ws: a Workspace made with
    new_tokens."""
    npg, Hkv, page, D = _pool_ok(pool)
    T, G, dt, qs, os_ = _q_ok(q, out, pool, Hkv, D)
    B = block_table.shape[0]
    width, bs = _table_ok(block_table, B)
    _lens_ok(seq_lens, B)
    assert cu_q.dtype == torch.int32 and cu_q.dim() == 1 and cu_q.shape[0] == B + 1 and cu_q.stride(0) == 1, "cu_q: int32 [B + 1]"
    if B == 0 or T == 0:
        return
    assert ws is not None, "ws: a Workspace made with new_tokens"
    stream = _stream(q, cu_q, pool, block_table, seq_lens, out, ws.buf)
    window, sinks = min(window, MAX_POS), min(sinks, MAX_POS)
    _check(lib().k16_prefill(dt, q.data_ptr(), qs, T, cu_q.data_ptr(), pool.data_ptr(), npg, block_table.data_ptr(), bs, width,
                             seq_lens.data_ptr(), B, Hkv, G, D, page, qscale, window, sinks, ws.ptickets, ws.ntickets, ws.pbuf,
                             ws.nbytes, out.data_ptr(), os_, stream), "k16_prefill")


def evict(pool, block_table, seq_lens, weights, budget, sinks, recent, kept, new_lens, new_weights, dst_pool=None,
          dst_table=None):
    """Of every (row, kv head) with more than `budget` cached tokens keeps the first `sinks`, the last `recent` and the
    budget - sinks - recent others with the largest weights (fp32 [B, Hkv, W], as attn sums them; ties: the lower position;
    NaN counts as the smallest), in their order.  A row is taken as min(len, W) tokens long: with W below its length the newest
    ones are dropped, so give weights as wide as attn wants them (W >= width * page) to keep every one.  kept int32 [B, Hkv,
    budget]: the kept positions, then -1; new_lens int32 [B] = min(len, W, budget); new_weights fp32 [B, Hkv, >= budget]: the
    kept tokens' weights, then zeros.  The three results overlap neither one another nor seq_lens, weights and the tables.
    Without dst_table the rows move to the front of the row's own pages (pages must not be shared between rows); with
    it they are copied to the pages of dst_table in dst_pool (default: pool), which must not be among the pages read."""
    npg, Hkv, page, D = _pool_ok(pool)
    B = block_table.shape[0]
    width, bs = _table_ok(block_table, B)
    _lens_ok(seq_lens, B)
    assert weights.dtype == torch.float32 and weights.dim() == 3 and weights.shape[:2] == (B, Hkv), "weights: fp32 [B, Hkv, W]"
    (wb, wh, w1), W = weights.stride(), weights.shape[2]
    assert w1 == 1 or W <= 1
    assert budget >= 1 and sinks >= 0 and recent >= 0 and sinks + recent <= budget, "sinks + recent must fit the budget"
    assert kept.dtype == torch.int32 and kept.shape == (B, Hkv, budget) and kept.is_contiguous(), "kept: int32 [B, Hkv, budget]"
    assert new_lens.dtype == torch.int32 and new_lens.shape == (B,) and new_lens.is_contiguous(), "new_lens: int32 [B]"
    assert new_weights.dtype == torch.float32 and new_weights.is_contiguous() and new_weights.dim() == 3
    assert new_weights.shape[:2] == (B, Hkv) and new_weights.shape[2] >= budget, "new_weights: fp32 [B, Hkv, >= budget]"
    if B == 0:
        return
    nwp, wp = new_weights.data_ptr(), weights.data_ptr()
    assert nwp + new_weights.numel() * 4 <= wp or wp + ((B - 1) * wb + (Hkv - 1) * wh + W) * 4 <= nwp, "new_weights overlaps weights"
    assert abs(new_lens.data_ptr() - seq_lens.data_ptr()) >= 4 * B, "new_lens overlaps seq_lens"
    stream = _stream(pool, block_table, seq_lens, weights, kept, new_lens, new_weights)
    dp = dn = dt = ds = dw = 0
    if dst_table is not None:
        dst = pool if dst_pool is None else dst_pool
        dn, dH, dpage, dD = _pool_ok(dst)
        assert dst.dtype == pool.dtype and (dH, dpage, dD) == (Hkv, page, D), "dst_pool: another pool of the same kind"
        dw, ds = _table_ok(dst_table, B)
        assert dw * page >= budget, "dst_table must cover the budget"
        _stream(dst, dst_table)
        dp, dt = dst.data_ptr(), dst_table.data_ptr()
    else:
        assert dst_pool is None, "dst_pool needs a dst_table"
    _check(lib().k16_evict(pool.data_ptr(), npg, block_table.data_ptr(), bs, width, seq_lens.data_ptr(), B, Hkv, D, page, wp, wb, wh, W,
                           budget, sinks, recent, kept.data_ptr(), new_lens.data_ptr(), nwp, new_weights.shape[2], dp, dn, dt, ds, dw,
                           stream), "k16_evict")
