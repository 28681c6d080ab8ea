"""Workloads of eviction from the paged KV cache by the attention that tokens received: decode and prefill over the cache that
also add up each stored token's attention weight, and the choice of the tokens that stay and their move to the front.

A case is a dict of plain values.  Lengths come from the case alone (`lengths` seeds them), values from `seed`.

Weights.  With s the scaled scores of a query and lse their log-sum-exp, a key's weight is exp(s - lse).  The weights pool
(weight pages, kv heads, page size), float32, holds a sum for each stored token and kv head; an attention call adds to it, over the
query heads of the kv head and the queries that count (the last `observed` of a sequence, 0: all of them).  A sequence's weight
pages are listed beside its K/V pages.

Eviction.  Of a sequence of L tokens n = min(L, keep) stay, for each kv head its own: the first `sinks`, the last `recent`, and of
the others those with the largest weights, of equal ones the first.  The last `recent` move to the end of the n places, in order.
In front of them a token that stays and has a place already keeps it; the other places are filled from front to back with the
others, in order.  `kept` names the token that each place takes, -1 behind the last.
"""
import math
import random

import torch

own = False

EMPTY_LSE = -5e4  # log-sum-exp of a query that sees no key; its output is 0


def _case(name, op, **fields):
    case = dict(
        name=name,
        op=op,               # "decode": one query token a sequence; "prefill": several; "evict": the choice and the move
        q_heads=32, kv_heads=8, head_dim=128, page=16,
        batch=1,
        ctx_lo=0, ctx_hi=0,  # tokens of a sequence in the cache in front of the new ones
        new_lo=0, new_hi=0,  # prefill: queries of a sequence, whose keys are the cache's last
        causal=True,         # a prefill query sees the keys up to its own; otherwise all of them
        observed=0,          # prefill: queries at a sequence's end whose weights count; 0: all
        keep=0, sinks=0, recent=0,
        lengths=1)
    case.update(fields)
    return case


def listed():
    return [
        # One user, one short conversation: latency.
        _case("decode_one_sequence", "decode", ctx_lo=500, ctx_hi=500),
        # 64 users whose caches are kept to a few thousand tokens.
        _case("decode_batch", "decode", batch=64, ctx_lo=1024, ctx_hi=4096, lengths=2),
        # Long documents that have not been evicted from yet, many query heads.
        _case("decode_long_context", "decode", q_heads=64, batch=8, ctx_lo=32768, ctx_hi=65536, lengths=3),
        # A model with odd head groups of dim 64 and larger pages, conversations of every length.
        _case("decode_odd", "decode", q_heads=28, kv_heads=4, head_dim=64, page=32, batch=41, ctx_lo=1, ctx_hi=2500, lengths=4),
        # A draft of five tokens is verified for one user.
        _case("prefill_draft", "prefill", ctx_lo=700, ctx_hi=700, new_lo=5, new_hi=5),
        # Chunks of prompts behind what is cached of them; every query counts.
        _case("prefill_chunks", "prefill", batch=8, ctx_lo=0, ctx_hi=4096, new_lo=128, new_hi=2048, lengths=5),
        # Whole prompts of which the last 32 queries say what stays.
        _case("prefill_observed", "prefill", batch=8, new_lo=500, new_hi=4096, observed=32, page=64, lengths=6),
        # Questions to cached documents, head dim 256.
        _case("prefill_long_document", "prefill", q_heads=16, kv_heads=2, head_dim=256, page=64, batch=2, ctx_lo=20000, ctx_hi=32768,
              new_lo=100, new_hi=300, lengths=7),
        # A conversation reaches its budget.
        _case("evict_one_sequence", "evict", ctx_lo=700, ctx_hi=700, keep=512, sinks=4, recent=64),
        # 64 users, every 64 steps: a few tokens go, most keep their places.
        _case("evict_step", "evict", batch=64, ctx_lo=2112, ctx_hi=2112, keep=2048, sinks=4, recent=256, lengths=8),
        # Prompts shrink to the budget after they were read.
        _case("evict_prompts", "evict", batch=16, ctx_lo=2000, ctx_hi=16384, keep=2048, sinks=4, recent=32, page=64, lengths=9),
        # A long document shrinks to an eighth, head dim 256 and few heads.
        _case("evict_long_document", "evict", kv_heads=2, head_dim=256, batch=1, ctx_lo=131072, ctx_hi=131072, keep=16384, sinks=16,
              recent=1024, lengths=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """A case of the listed ones' ranges: one of the operators, other heads, pages, batches and lengths."""
    limit = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("decode", "prefill", "evict")}
    while True:
        op = rng.choice(["decode", "prefill", "evict"])
        case = _case("", op)
        del case["name"]
        case["q_heads"], case["kv_heads"] = rng.choice([(32, 8), (32, 8), (64, 8), (28, 4), (8, 8), (16, 2), (9, 3), (32, 1), (40, 1)])
        case["head_dim"] = rng.choice([64, 80, 96, 112, 128, 128, 128, 256])
        case["page"] = rng.choice([16, 16, 16, 32, 64, 128])
        case["lengths"] = rng.randint(100, 1 << 20)
        if op == "decode":
            case["batch"] = _log_int(rng, 1, 128)
            case["ctx_lo"] = _log_int(rng, 1, 32768)
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 3 * case["ctx_lo"])
        elif op == "prefill":
            case["batch"] = _log_int(rng, 1, 64)
            case["ctx_lo"] = rng.choice([0, _log_int(rng, 1, 16384)])
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 4096)
            case["new_hi"] = _log_int(rng, 2, 2048)
            case["new_lo"] = _log_int(rng, 1, case["new_hi"])
            case["causal"] = rng.random() < 0.8
            case["observed"] = rng.choice([0, 0, _log_int(rng, 1, 256)])
        else:
            case["batch"] = _log_int(rng, 1, 64)
            case["keep"] = _log_int(rng, 64, 16384)
            case["ctx_lo"] = rng.randint(case["keep"] // 2, 2 * case["keep"])
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 8 * case["keep"])
            case["sinks"] = rng.choice([0, 1, 4, 16])
            case["recent"] = rng.randint(0, case["keep"] // 2)
        if _cost(case) <= limit[op] and _padded_elements(case) <= 3.5e9:
            return case


def _lengths(case):
    """Per sequence: stored tokens, queries."""
    r = random.Random(case["lengths"])
    stored, queries = [], []
    for _ in range(case["batch"]):
        n = r.randint(case["new_lo"], case["new_hi"])
        stored.append(r.randint(case["ctx_lo"], case["ctx_hi"]) + n)
        queries.append(1 if case["op"] == "decode" else n)
    return stored, queries


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def _padded_elements(case):
    """Elements of the largest tensor of the plain form."""
    stored, queries = _lengths(case)
    tokens = case["batch"] * (max(stored) + case["page"])
    scores = tokens * case["q_heads"] * max(queries) if case["op"] == "prefill" else 0
    return max(tokens * case["kv_heads"] * case["head_dim"] * (2 if case["op"] == "evict" else 1), scores)


def work(case):
    stored, queries = _lengths(case)
    d, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    row = hkv * 2 * d * 2  # bytes of a token's K and V
    pages = sum(-(-s // case["page"]) for s in stored)
    if case["op"] == "evict":
        # weights are read, `kept` is written; the recent tokens move, and those of the others that stay and lie behind the n places
        total = 0.0
        for s in stored:
            n = min(s, case["keep"])
            total += 4 * hkv * s
            if s > n:
                r = min(case["recent"], n)
                k = min(case["sinks"], n - r)
                moved = r + (n - r - k) * (s - n) / max(1, s - r - k)
                total += 2 * moved * (row + 4 * hkv)
        return {"bytes": total + 4 * hkv * case["keep"] * case["batch"] + 8 * pages, "flops": 0}
    pairs = counted = 0
    for s, n in zip(stored, queries):
        seen = min(case["observed"] or n, n)
        if case["op"] == "prefill" and case["causal"]:
            pairs += n * s - n * (n - 1) // 2
            counted += seen * s - seen * (seen - 1) // 2
        else:
            pairs += n * s
            counted += seen * s
    # sums are read and written; a score that counts costs one addition more
    return {"bytes": sum(stored) * (row + 8 * hkv) + sum(queries) * hq * (4 * d + 4) + 8 * pages,
            "flops": hq * (4 * d * pairs + counted)}


# ---- inputs --------------------------------------------------------------------------------------------------


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    d, hq, hkv, page = case["head_dim"], case["q_heads"], case["kv_heads"], case["page"]
    stored, queries = _lengths(case)
    counts = [-(-s // page) for s in stored]
    used = sum(counts)
    total = used + max(1, used // 16)
    # Pages of a pool that has been in use: permuted, and their last slots hold other sequences' rows.
    ids, weight_ids = (torch.randperm(total, generator=g, device=device)[:used].int() for _ in range(2))
    pages = torch.empty((total, 2, hkv, page, d), dtype=torch.float16, device=device)
    # K has channels that are larger than others, as trained models have them.
    channel = torch.exp(0.6 * torch.randn((2, hkv, 1, d), generator=g, device=device))
    channel[1] = 1.0
    step = max(1, (1 << 26) // (2 * hkv * page * d))
    for p in range(0, total, step):
        n = min(step, total - p)
        pages[p:p + n] = torch.randn((n, 2, hkv, page, d), generator=g, device=device) * channel
    # Sums of earlier steps: a few tokens hold most of the weight, some were never seen.
    weights = 0.05 * torch.exp(2.0 * torch.randn((total, hkv, page), generator=g, device=device))
    weights = torch.where(torch.rand(weights.shape, generator=g, device=device) < 0.02, 0.0, weights)
    host_indptr = [0]
    for c in counts:
        host_indptr.append(host_indptr[-1] + c)

    def int32(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    state = {"case": dict(case), "pages": pages, "weights": weights, "page_indptr": int32(host_indptr), "page_values": ids,
             "weight_page_values": weight_ids, "length_info": int32([s - (c - 1) * page if c else 0 for s, c in zip(stored, counts)]),
             "max_pages": max(counts)}
    if case["op"] == "evict":
        # The pool that the choice goes by stays as it is, so that every pass moves as much; the sums that move are another.
        state.update(keep=int32([case["keep"]] * case["batch"]), moving=weights.clone(),
                     kept=torch.empty((case["batch"], hkv, case["keep"]), dtype=torch.int32, device=device))
        return state
    q_indptr = [0]
    for n in queries:
        q_indptr.append(q_indptr[-1] + n)
    state.update(q=(1.5 * torch.randn((q_indptr[-1], hq, d), generator=g, device=device)).half(), q_indptr=int32(q_indptr),
                 max_queries=max(queries), sm_scale=d ** -0.5,
                 output=torch.empty((q_indptr[-1], hq, d), dtype=torch.float16, device=device),
                 lse=torch.empty((q_indptr[-1], hq), dtype=torch.float32, device=device))
    return state


# ---- one pass ------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return _evict(case, state) if case["op"] == "evict" else _attend(case, state)


def _run_own(case, s):
    from tvm_amd import kernels
    if case["op"] == "evict":
        kernels.select_kept_tokens(s["weights"], s["page_indptr"], s["weight_page_values"], s["length_info"], s["keep"], s["kept"],
                                   case["sinks"], case["recent"])
        kernels.move_kept_tokens(s["pages"], s["moving"], s["page_indptr"], s["page_values"], s["weight_page_values"], s["kept"])
        return {"kept": s["kept"], "pages": s["pages"], "weights": s["moving"]}
    if case["op"] == "decode":
        kernels.batch_decode_paged_kv_weights(s["q"], s["pages"], s["page_indptr"], s["page_values"], s["length_info"], s["output"],
                                              s["lse"], s["weights"], s["weight_page_values"], s["sm_scale"])
    else:
        kernels.batch_prefill_paged_kv_weights(s["q"], s["q_indptr"], s["pages"], s["page_indptr"], s["page_values"], s["length_info"],
                                               s["output"], s["lse"], s["weights"], s["weight_page_values"], int(case["causal"]),
                                               case["observed"], s["sm_scale"])
    return {"out": s["output"], "lse": s["lse"], "weights": s["weights"]}


def _table(s):
    """Entries of the page table that each sequence's pages have, padded to the most pages, and the stored tokens."""
    counts = s["page_indptr"][1:] - s["page_indptr"][:-1]
    nth = torch.arange(s["max_pages"], device=counts.device)
    entries = s["page_indptr"][:-1, None] + torch.minimum(nth, (counts[:, None] - 1).clamp(min=0))
    stored = torch.where(counts > 0, (counts - 1) * s["pages"].shape[3] + s["length_info"], 0)
    return entries.long().clamp(max=s["page_values"].numel() - 1), stored


def _attend(case, s):
    """All sequences at once, padded to the longest."""
    hkv, page = case["kv_heads"], case["page"]
    device = s["q"].device
    entries, stored = _table(s)
    rows = s["pages"][s["page_values"][entries].long()]
    k, v = (rows[:, :, i].float().transpose(1, 2).flatten(2, 3) for i in (0, 1))  # (batch, kv heads, tokens, head_dim)
    del rows
    token = torch.arange(k.shape[2], device=device)
    there = token < stored[:, None]
    # queries, (batch, kv heads, queries of a head group, head_dim)
    asked = s["q_indptr"][1:] - s["q_indptr"][:-1]
    nth = torch.arange(s["max_queries"], device=device)
    at = (s["q_indptr"][:-1, None] + nth).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][at].float().unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)
    shape = q.shape[2:4]
    see = there[:, None, :].expand(-1, s["max_queries"], -1)
    if case["op"] == "prefill" and case["causal"]:
        see = see & (token < (stored - asked)[:, None, None] + 1 + nth[:, None])
    scores = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, shape) * (s["sm_scale"] * math.log2(math.e))
    scores = scores.masked_fill(~see[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp2(scores - most)
    del scores
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    out = (p.flatten(2, 3) @ v).unflatten(2, shape)
    lse = torch.where(total > 0, most + torch.log2(total), EMPTY_LSE)[..., 0]
    counts = (nth < asked[:, None]) & (nth >= asked[:, None] - (case["observed"] or s["max_queries"]))
    received = (p * counts[:, None, None, :, None]).sum((2, 3))  # (batch, kv heads, tokens)
    b, t = there.nonzero(as_tuple=True)
    s["weights"][s["weight_page_values"][entries].long()[b, t // page], :, t % page] += received.transpose(1, 2)[b, t]
    real = (nth < asked[:, None]).flatten().nonzero()[:, 0]
    out = out.permute(0, 3, 1, 2, 4).flatten(0, 1).flatten(1, 2)[real]
    return {"out": out.half(), "lse": lse.permute(0, 3, 1, 2).flatten(0, 1).flatten(1, 2)[real], "weights": s["weights"]}


def _evict(case, s):
    page, hkv = case["page"], case["kv_heads"]
    entries, stored = _table(s)
    weight_pages = s["weight_page_values"][entries].long()
    received = s["weights"][weight_pages].transpose(1, 2).flatten(2, 3)  # (batch, kv heads, tokens)
    token = torch.arange(received.shape[2], device=received.device)
    n = torch.minimum(stored, s["keep"])[:, None, None]
    stored = stored[:, None, None]
    recent = n.clamp(max=case["recent"])
    sinks = (n - recent).clamp(max=case["sinks"])
    received = torch.where((token < sinks) | (token >= stored - recent), math.inf, received)
    received = torch.where(token < stored, received, -math.inf)
    order = received.sort(dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(received.shape, dtype=torch.bool, device=received.device).scatter_(-1, order, (token < n).expand(received.shape))
    # places in front of the recent tokens: free ones, and the tokens that need one
    free = ~stays & (token < n - recent)
    homeless = stays & (token >= n - recent) & (token < stored - recent)
    nth_free, nth_homeless = free.cumsum(-1) - 1, homeless.cumsum(-1) - 1
    b, h, t = homeless.nonzero(as_tuple=True)
    which = torch.zeros(received.shape, dtype=torch.int64, device=received.device)
    which[b, h, nth_homeless[b, h, t]] = t
    kept = token.expand(received.shape).clone()
    b, h, t = free.nonzero(as_tuple=True)
    kept[b, h, t] = which[b, h, nth_free[b, h, t]]
    kept = torch.where(token >= n - recent, token + stored - n, kept)
    kept = torch.where(token < n, kept, -1)
    s["kept"].fill_(-1)
    width = min(kept.shape[2], case["keep"])
    s["kept"][..., :width] = kept[..., :width]
    # every moved row is read before the first is written
    b, h, to = ((kept >= 0) & (kept != token)).nonzero(as_tuple=True)
    of = kept[b, h, to]
    rows, ids = s["pages"].transpose(1, 2), s["page_values"][entries].long()
    rows[ids[b, to // page], h, :, to % page] = rows[ids[b, of // page], h, :, of % page]
    s["moving"][weight_pages[b, to // page], h, to % page] = s["moving"][weight_pages[b, of // page], h, of % page]
    return {"kept": s["kept"], "pages": s["pages"], "weights": s["moving"]}


# ---- the definition in 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    hkv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["q_heads"] // hkv
    stored, queries = _lengths(case)
    indptr = s["page_indptr"].tolist()
    ids = [s["page_values"][indptr[b]:indptr[b + 1]].long() for b in range(case["batch"])]
    weight_ids = [s["weight_page_values"][indptr[b]:indptr[b + 1]].long() for b in range(case["batch"])]
    if case["op"] == "evict":  # one head of one sequence after the other, the weights sorted on the host
        pages, sums = s["pages"].double(), s["moving"].double()
        for b in range(case["batch"]):
            have, n = stored[b], min(stored[b], case["keep"])
            if n == have:
                continue
            recent = min(case["recent"], n)
            sinks, places = min(case["sinks"], n - recent), n - recent
            at = torch.arange(n, device=pages.device)
            for h in range(hkv):
                w = s["weights"][weight_ids[b], h].reshape(-1)[:have].tolist()
                ranked = sorted(range(sinks, have - recent), key=lambda t: (-w[t], t))
                chosen = set(range(sinks)) | set(ranked[:places - sinks])
                others = iter(sorted(t for t in chosen if t >= places))
                of = [t if t in chosen else next(others) for t in range(places)] + list(range(have - recent, have))
                of = torch.tensor(of, device=pages.device)
                pages[ids[b][at // page], :, h, at % page] = pages[ids[b][of // page], :, h, of % page]
                sums[weight_ids[b][at // page], h, at % page] = sums[weight_ids[b][of // page], h, of % page]
        return {"kept": None, "pages": pages, "weights": sums}
    begin = s["q_indptr"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], EMPTY_LSE, dtype=torch.float64, device=s["q"].device)
    sums = s["weights"].double()
    for b in range(case["batch"]):
        n, keys = queries[b], stored[b]
        if not n or not keys:
            continue
        first_counted = n - min(n, case["observed"] or n)
        for h in range(hkv):
            k = s["pages"][ids[b], 0, h].reshape(-1, d)[:keys].double()
            v = s["pages"][ids[b], 1, h].reshape(-1, d)[:keys].double()
            received = torch.zeros(len(ids[b]) * page, dtype=torch.float64, device=k.device)
            for r in range(0, n, 256):
                q = s["q"][begin[b] + r:begin[b] + min(n, r + 256), h * group:(h + 1) * group].double()
                x = torch.tensordot(q, k, dims=([2], [1])) * s["sm_scale"]
                if case["op"] == "prefill" and case["causal"]:
                    mine = keys - n + r + torch.arange(q.shape[0], device=k.device)
                    x = x.masked_fill((torch.arange(keys, device=k.device) > mine[:, None])[:, None], -math.inf)
                natural = torch.logsumexp(x, -1)
                w = torch.exp(x - natural[..., None])
                at = slice(begin[b] + r, begin[b] + r + q.shape[0])
                out[at, h * group:(h + 1) * group] = torch.tensordot(w, v, dims=([2], [0]))
                lse[at, h * group:(h + 1) * group] = natural / math.log(2.0)
                received[:keys] += w[max(0, first_counted - r):].sum((0, 1))
            sums[weight_ids[b], h] += received.view(-1, page)
    return {"out": out, "lse": lse, "weights": sums}
