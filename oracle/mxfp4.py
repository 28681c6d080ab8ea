"""The 4-bit cache by its definition, in 64 bits: what the tests of its kernels compare with.

Rows are quantised in blocks of 32 to FP4 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign) under a power-of-two scale;
pages hold the codes of their tokens, then their scales (include/tvmkv.h)."""
import numpy as np

BLOCK = 32
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
EMPTY_LSE = -5e4


def quantise(rows):
    """(..., d) -> codes (..., d) of 4 bits and scale bytes (..., d / 32)."""
    x = np.asarray(rows, np.float64).reshape(*rows.shape[:-1], -1, BLOCK)
    largest = np.abs(x).max(-1)
    finite = np.isfinite(largest)
    power = np.full(largest.shape, 13)
    for e in range(12, -24, -1):
        power[largest <= 7.0 * 2.0 ** e] = e
    y = np.where(finite[..., None], x, 0.0) / 2.0 ** power[..., None]
    off = np.abs(np.abs(y)[..., None] - GRID)
    least = off.min(-1, keepdims=True)
    ties = off == least
    even = ties & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), ties.argmax(-1)) + 8 * np.signbit(y)
    return code.reshape(rows.shape).astype(np.uint8), np.where(finite, power + 127, 255).astype(np.uint8)


def dequantise(codes, scales):
    values = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return values * np.repeat(scale, BLOCK, -1)


def rounded(rows):
    """Rows as the cache gives them back."""
    return dequantise(*quantise(rows))


def empty_pages(num_pages, h_kv, page_size, d):
    return np.zeros((num_pages, 2, h_kv, page_size, 17 * d // BLOCK), np.uint8)


def _slabs(pages, d):
    n, two, h_kv, page, _ = pages.shape
    flat = pages.reshape(n, two, h_kv, -1)
    cut = page * d // 2
    return flat[..., :cut].reshape(n, two, h_kv, page, d // 2), flat[..., cut:].reshape(n, two, h_kv, page, d // BLOCK)


def append(pages, k, v, position_map):
    """A copy of the pages with the rows k, v (tokens, h_kv, d) in their slots."""
    d, page = k.shape[-1], pages.shape[3]
    codes, scales = (a.copy() for a in _slabs(pages, d))
    slots = np.asarray(position_map)
    keep = slots >= 0
    page_of, at = slots[keep] // page, slots[keep] % page
    for which, rows in enumerate((k, v)):
        c, s = quantise(rows[keep])
        codes[page_of, which, :, at] = c[..., 0::2] | c[..., 1::2] << 4
        scales[page_of, which, :, at] = s
    flat = [a.reshape(*pages.shape[:3], -1) for a in (codes, scales)]
    return np.concatenate(flat, -1).reshape(pages.shape)


def rows_of(pages, d):
    """All rows of a pool in 64 bits: (pages, 2, h_kv, page, d)."""
    packed, scales = _slabs(pages, d)
    codes = np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], d)
    return dequantise(codes, scales)


def attention(q, q_lens, rows, page_indptr, page_values, length_info, causal, sm_scale):
    """Attention of q (queries, h_q, d) over rows_of(pages); returns out and lse in 64 bits."""
    h_q, h_kv, page = q.shape[1], rows.shape[2], rows.shape[3]
    info = np.asarray(length_info)
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], EMPTY_LSE)
    begin = 0
    for b, n in enumerate(q_lens):
        ids = page_values[page_indptr[b]:page_indptr[b + 1]]
        last = info[0][b] if info.ndim == 2 else info[b]
        stored = (len(ids) - 1) * page + last if len(ids) else 0
        at = np.arange(stored)
        if info.ndim == 2 and stored:
            at = np.concatenate((at[:info[2][b]], at[info[1][b]:]))
        if len(at):
            kv = np.moveaxis(rows[ids], 2, 1).reshape(len(ids), h_kv, 2, page, -1)
            kv = np.moveaxis(kv, 3, 1).reshape(len(ids) * page, h_kv, 2, -1)[at]
        for i in range(n):
            see = min(max(len(at) - n + 1 + i, 0), len(at)) if causal else len(at)
            if not see:
                continue
            for h in range(h_q):
                k, v = kv[:see, h // (h_q // h_kv), 0], kv[:see, h // (h_q // h_kv), 1]
                s = k @ q[begin + i, h].astype(np.float64) * (sm_scale / np.log(2.0))
                w = np.exp2(s - s.max())
                out[begin + i, h] = w @ v / w.sum()
                lse[begin + i, h] = s.max() + np.log2(w.sum())
        begin += n
    return out, lse
