"""Eviction by attention weight in 64 bits, from the definitions in include/tvmkv.h."""
import numpy as np

EMPTY_LSE = -5e4


def _stored(page_indptr, length_info, b, page):
    n = page_indptr[b + 1] - page_indptr[b]
    return (n - 1) * page + length_info[b] if n else 0


def attention(q, q_lens, pages, page_indptr, page_values, length_info, causal, sm_scale, key_weights, weight_page_values, observed=0):
    """q (queries, h_q, d), pages (num_pages, 2, h_kv, page, d), key_weights (weight pages, h_kv, page): out, lse, the sums
    afterwards, and how far float32 arithmetic may take each sum (see tests/test_gpu_eviction.py)."""
    h_q, d, h_kv, page = q.shape[1], q.shape[2], pages.shape[2], pages.shape[3]
    group = h_q // h_kv
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], EMPTY_LSE)
    size = np.zeros(q.shape)  # sum w |v|
    sums = key_weights.astype(np.float64)
    slack = np.zeros(sums.shape)
    begin = 0
    for b, n in enumerate(q_lens):
        ids = page_values[page_indptr[b]:page_indptr[b + 1]]
        weight_ids = weight_page_values[page_indptr[b]:page_indptr[b + 1]]
        stored = _stored(page_indptr, length_info, b, page)
        if stored and n:
            kv = np.moveaxis(pages[ids].astype(np.float64), 3, 1).reshape(len(ids) * page, 2, h_kv, d)[:stored]
            first = max(0, n - observed) if observed else 0
            sees = np.arange(stored)[None] < (np.clip(stored - n + 1 + np.arange(n), 0, stored)[:, None] if causal else stored)
            place = (weight_ids[np.arange(stored) // page], np.arange(stored) % page)
            for h in range(h_q):
                k, v = kv[:, 0, h // group], kv[:, 1, h // group]
                x = q[begin:begin + n, h].astype(np.float64)
                s = x @ k.T * (sm_scale / np.log(2.0))
                with np.errstate(invalid="ignore"):
                    reach = np.abs(x) @ np.abs(k).T * (abs(sm_scale) / np.log(2.0))  # what the products' sums go through
                s = np.where(sees, s, -np.inf)
                top = s.max(-1, keepdims=True)
                some = np.isfinite(top[:, 0]) | np.isnan(top[:, 0])
                top = np.where(np.isneginf(top), 0.0, top)
                w = np.where(sees, np.exp2(s - top), 0.0)
                total = w.sum(-1, keepdims=True)
                w = w / np.where(some[:, None], total, 1.0)
                out[begin:begin + n, h] = np.where(some[:, None], w @ np.where(sees.any(0)[:, None], v, 0.0), 0.0)
                size[begin:begin + n, h] = w @ np.abs(np.where(sees.any(0)[:, None], v, 0.0))
                lse[begin:begin + n, h] = np.where(some, (top + np.log2(np.where(some[:, None], total, 1.0)))[:, 0], EMPTY_LSE)
                sums[place[0], h // group, place[1]] += w[first:].sum(0)
                # a score is off by (d + 2) 2^-24 of what its sum goes through, the log-sum-exp by as much as the worst of its
                # row's scores; then the exponent's and the power's own roundings, and those of the additions
                worst = np.where(sees, reach, 0.0).max(-1, keepdims=True)
                rel = np.log(2.0) * ((d + 2) * (reach + worst) + 2 * np.abs(lse[begin:begin + n, h, None]) + 8) * 2.0 ** -23 + (n + group + 4) * 2.0 ** -23
                slack[place[0], h // group, place[1]] += (np.where(sees, rel, 0.0) * w)[first:].sum(0)
        begin += n
    slack += sums * 2.0 ** -23
    return out, lse, sums, slack, size


def select(key_weights, page_indptr, weight_page_values, length_info, keep, max_keep, num_sinks, num_recent):
    h_kv, page = key_weights.shape[1:]
    batch = len(page_indptr) - 1
    kept = np.full((batch, h_kv, max_keep), -1, np.int32)
    for b in range(batch):
        have = _stored(page_indptr, length_info, b, page)
        n = min(have, max(0, min(keep[b], max_keep)))
        recent = min(num_recent, n)
        sinks = min(num_sinks, n - recent)
        places = n - recent
        ids = weight_page_values[page_indptr[b]:page_indptr[b + 1]]
        for h in range(h_kv):
            if have == n:
                kept[b, h, :n] = np.arange(n)
                continue
            w = key_weights[ids, h].reshape(-1)[:have]
            order = sorted(range(sinks, have - recent), key=lambda t: (np.isnan(w[t]), -w[t] if not np.isnan(w[t]) else 0.0, t))
            stays = set(range(sinks)) | set(order[:places - sinks])
            others = iter(sorted(t for t in stays if t >= places))
            kept[b, h, :places] = [t if t in stays else next(others) for t in range(places)]
            kept[b, h, places:n] = np.arange(have - recent, have)
    return kept


def move(pages, key_weights, page_indptr, page_values, weight_page_values, kept):
    """The pools afterwards; key_weights None: K and V only."""
    before, sums_before = pages, key_weights
    pages, page = pages.copy(), pages.shape[3]
    key_weights = None if key_weights is None else key_weights.copy()
    for b in range(len(page_indptr) - 1):
        ids = page_values[page_indptr[b]:page_indptr[b + 1]]
        for h in range(kept.shape[1]):
            for i, t in enumerate(kept[b, h]):
                if i < t < len(ids) * page:
                    pages[ids[i // page], :, h, i % page] = before[ids[t // page], :, h, t % page]
                    if key_weights is not None:
                        w = weight_page_values[page_indptr[b]:page_indptr[b + 1]]
                        key_weights[w[i // page], h, i % page] = sums_before[w[t // page], h, t % page]
    return pages, key_weights
