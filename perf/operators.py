"""Workloads of the 4-bit paged KV cache: rows quantised as they are written and read back, attention of single
tokens over the cache, attention of prompts and draft chains over it.

The cache's format (block-scaled FP4).  A row is one token's K or V of one kv head, `head_dim` elements in blocks
of 32.  A block is 32 FP4 codes (sign, 2 exponent bits, 1 mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6; element 2i in
the low half of byte i) and one scale byte s that stands for 2^(s - 127); 255 stands for NaN.  The pool is a
uint8 tensor (pages, 2, kv heads, page size, 17 head_dim / 32); the bytes of one (page, K or V, kv head) are the
codes of its tokens, head_dim / 2 bytes each, then their scales, head_dim / 32 bytes each.  A block's scale is
the smallest power of two, 2^-23 to 2^13, at which its largest magnitude is at most 7 (6 is the largest code, 7
the point where it is nearest); codes round to nearest, ties to the even code; a block with a value that is not
finite is NaN.

A case is a dict of plain values.  Lengths come from the case alone (`lengths` seeds them), values from `seed`.
"""
import math
import random

import torch

own = False

BLOCK = 32
EMPTY_LSE = -5e4        # log-sum-exp of a query that sees no key; its output is 0
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, op, **fields):
    case = dict(
        name=name,
        op=op,               # "write": append and read back; "decode": one query token a sequence; "prefill": several
        q_heads=32, kv_heads=8, head_dim=128, page=16,
        batch=1,
        ctx_lo=0, ctx_hi=0,  # tokens of a sequence in the cache in front of the new ones
        new_lo=1, new_hi=1,  # new tokens of a sequence: rows to write, or queries (their keys are the cache's last)
        causal=True,         # a prefill query sees the keys up to its own; otherwise all of them
        sinks=0, evicted=0,  # > 0: sliding windows, `sinks` first tokens stay, up to `evicted` behind them are masked
        lengths=1)
    case.update(fields)
    return case


def listed():
    return [
        # The first answers of one conversation: a single token's rows, a short cache read back.
        _case("write_one_token", "write", ctx_lo=40, ctx_hi=40),
        # A decode step of 64 conversations writes a row each; what they hold is gathered for a reader of fp16 rows.
        _case("write_decode_step", "write", batch=64, ctx_lo=100, ctx_hi=600, lengths=2),
        # Eight prompts enter the cache at once.
        _case("write_prompts", "write", batch=8, new_lo=500, new_hi=4096, page=64, lengths=3),
        # Odd prompt lengths behind cached ones, a model with three kv heads of dim 96.
        _case("write_odd", "write", kv_heads=3, head_dim=96, page=48, batch=13, ctx_lo=1, ctx_hi=300, new_lo=1, new_hi=700, lengths=4),
        # One user, one short conversation: latency.
        _case("decode_one_sequence", "decode", ctx_lo=500, ctx_hi=500),
        # 64 users, contexts from a paragraph to a long document.
        _case("decode_batch", "decode", batch=64, ctx_lo=1024, ctx_hi=8192, lengths=5),
        # Long documents and many query heads: what a cache of 4 bits is for.
        _case("decode_long_context", "decode", q_heads=64, batch=8, ctx_lo=32768, ctx_hi=131072, lengths=6),
        # Endless conversations (windows with attention sinks) of a small model with odd head groups.
        _case("decode_windows", "decode", q_heads=28, kv_heads=4, head_dim=64, page=32, batch=41, ctx_lo=3, ctx_hi=2500, sinks=4,
              evicted=40, lengths=7),
        # A draft of five tokens is verified for one user.
        _case("prefill_draft", "prefill", ctx_lo=700, ctx_hi=700, new_lo=5, new_hi=5),
        # Prompts in chunks behind what is cached of them.
        _case("prefill_chunks", "prefill", batch=8, ctx_lo=0, ctx_hi=4096, new_lo=128, new_hi=2048, lengths=8),
        # Chunks of a few hundred tokens of one long document, head dim 256.
        _case("prefill_long_document", "prefill", q_heads=16, kv_heads=2, head_dim=256, page=64, batch=2, ctx_lo=20000, ctx_hi=32768,
              new_lo=100, new_hi=300, lengths=9),
        # Queries against a cached document that all of them see, every query head its own kv head.
        _case("prefill_not_causal", "prefill", q_heads=8, kv_heads=8, head_dim=64, page=128, batch=19, ctx_lo=1, ctx_hi=3000, new_lo=1,
              new_hi=130, causal=False, lengths=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """A case of the listed ones' ranges: one of the operators, other heads, pages, batches and lengths."""
    limit = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("write", "decode", "prefill")}
    while True:
        op = rng.choice(["write", "decode", "decode", "prefill", "prefill"])
        case = _case("", op)
        del case["name"]
        case["q_heads"], case["kv_heads"] = rng.choice([(32, 8), (32, 8), (64, 8), (28, 4), (8, 8), (16, 2), (9, 3), (32, 1), (40, 1)])
        case["head_dim"] = rng.choice([64, 96, 128, 128, 128, 256])
        case["page"] = rng.choice([16, 16, 16, 32, 48, 64, 128])
        case["lengths"] = rng.randint(100, 1 << 20)
        if op == "write":
            case["batch"] = _log_int(rng, 1, 128)
            case["ctx_lo"] = rng.randint(0, 300)
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 600)
            case["new_hi"] = _log_int(rng, 1, 4096)
            case["new_lo"] = _log_int(rng, 1, case["new_hi"])
        elif op == "decode":
            case["batch"] = _log_int(rng, 1, 128)
            case["ctx_lo"] = _log_int(rng, 1, 32768)
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 3 * case["ctx_lo"])
            if rng.random() < 0.3:
                case["sinks"], case["evicted"] = rng.choice([1, 4, 16]), rng.randint(1, 80)
        else:
            case["batch"] = _log_int(rng, 1, 64)
            case["ctx_lo"] = rng.choice([0, _log_int(rng, 1, 16384)])
            case["ctx_hi"] = case["ctx_lo"] + _log_int(rng, 1, 4096)
            case["new_hi"] = _log_int(rng, 2, 2048)
            case["new_lo"] = _log_int(rng, 1, case["new_hi"])
            case["causal"] = rng.random() < 0.75
            if rng.random() < 0.2:
                case["sinks"], case["evicted"] = rng.choice([1, 4, 16]), rng.randint(1, 80)
        if _cost(case) <= limit[op] and _padded_elements(case) <= 3.5e9:
            return case


def _lengths(case):
    """Per sequence: stored tokens (evicted ones included), new tokens, first token behind the evicted ones."""
    r = random.Random(case["lengths"])
    stored, new, window = [], [], []
    for _ in range(case["batch"]):
        n = r.randint(case["new_lo"], case["new_hi"])
        held = r.randint(case["ctx_lo"], case["ctx_hi"]) + (0 if case["op"] == "decode" else n)
        masked = r.randint(0, case["evicted"]) if case["sinks"] and held > case["sinks"] else 0
        stored.append(held + masked)
        new.append(n)
        window.append(min(case["sinks"], held) + masked)
    return stored, new, window


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 5e14


def _padded_elements(case):
    """Elements of the largest tensor of the plain form."""
    stored, new, _ = _lengths(case)
    tokens = case["batch"] * (max(stored) + case["page"])
    scores = tokens * case["q_heads"] * max(new) if case["op"] == "prefill" else 0
    return max(tokens * case["kv_heads"] * case["head_dim"], scores)


def work(case):
    stored, new, window = _lengths(case)
    d, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    packed, rows = hkv * 2 * (d // 2 + d // BLOCK), hkv * 2 * d * 2  # bytes of a token: in the cache, as fp16 rows
    if case["op"] == "write":
        return {"bytes": sum(new) * (rows + packed) + sum(stored) * (packed + rows) + 4 * (sum(new) + sum(stored)), "flops": 0}
    queries = case["batch"] if case["op"] == "decode" else sum(new)
    tokens, pairs = 0, 0
    for s, n, w in zip(stored, new, window):
        keys = s - (w - min(case["sinks"], s) if case["sinks"] else 0)
        tokens += keys
        n = 1 if case["op"] == "decode" else n
        if case["op"] == "prefill" and case["causal"]:
            seen = min(n, keys)
            pairs += seen * keys - seen * (seen - 1) // 2
        else:
            pairs += n * keys
    pages = sum(-(-s // case["page"]) for s in stored)
    return {"bytes": tokens * packed + queries * hq * (4 * d + 4) + 4 * pages, "flops": 4 * hq * d * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------


def _tables(device):
    """FP4 values of the two codes of a byte; the scale of a scale byte and its inverse."""
    values = _MAGNITUDES + tuple(-m for m in _MAGNITUDES)
    pair = torch.tensor([[values[b & 15], values[b >> 4]] for b in range(256)], dtype=torch.float32)
    scale = torch.tensor([2.0 ** (b - 127) if b < 255 else math.nan for b in range(256)], dtype=torch.float32)
    inverse = torch.tensor([2.0 ** (127 - b) if b < 255 else 0.0 for b in range(256)], dtype=torch.float32)
    return {"pair": pair.to(device), "scale": scale.to(device), "inverse": inverse.to(device)}


def _quantise(rows, tables):
    """Rows (..., head_dim) to codes (..., head_dim / 2) and scale bytes (..., head_dim / 32)."""
    x = rows.float().unflatten(-1, (-1, BLOCK))
    largest = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    mantissa, exponent = torch.frexp(torch.where(finite & (largest > 0), largest, 2.0 ** -24))
    power = (exponent - 2 - (mantissa <= 0.875).int()).clamp(-23, 13)
    scales = torch.where(finite, power + 127, 255)
    y = torch.where(finite[..., None], x, 0.0) * tables["inverse"][scales.long()][..., None]
    a = y.abs()
    codes = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() +
             (a > 5.0).byte() + torch.signbit(y).byte() * 8).flatten(-2).unflatten(-1, (-1, 2))
    return codes[..., 0] + codes[..., 1] * 16, scales.byte()


def _slabs(pages, head_dim):
    """Views of a pool, or of some of its pages: codes (..., page size, head_dim / 2), scales (..., page size, head_dim / 32)."""
    page = pages.shape[-2]
    flat = pages.flatten(-2)
    return (flat[..., :page * head_dim // 2].unflatten(-1, (page, head_dim // 2)),
            flat[..., page * head_dim // 2:].unflatten(-1, (page, head_dim // BLOCK)))


def _values(codes, scales, tables):
    x = tables["pair"][codes.long()].flatten(-2).unflatten(-1, (-1, BLOCK))
    return (x * tables["scale"][scales.long()][..., None]).flatten(-2)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    d, hq, hkv, page = case["head_dim"], case["q_heads"], case["kv_heads"], case["page"]
    stored, new, window = _lengths(case)
    counts = [-(-s // page) for s in stored]
    used = sum(counts)
    total = used + max(1, used // 16)
    tables = _tables(device)
    # Pages of a pool that has been in use: permuted, and their last slots hold other sequences' rows.
    ids = torch.randperm(total, generator=g, device=device)[:used].int()
    pages = torch.empty((total, 2, hkv, page, 17 * d // BLOCK), dtype=torch.uint8, device=device)
    # K has channels that are larger than others, as trained models have them.
    channel = torch.exp(0.6 * torch.randn((2, hkv, 1, d), generator=g, device=device))
    channel[1] = 1.0
    step = max(1, (1 << 26) // (2 * hkv * page * d))
    for p in range(0, total, step):
        n = min(step, total - p)
        rows = (torch.randn((n, 2, hkv, page, d), generator=g, device=device) * channel).half()
        codes, scales = _quantise(rows, tables)
        into_codes, into_scales = _slabs(pages[p:p + n], d)
        into_codes.copy_(codes)
        into_scales.copy_(scales)
    host_indptr = [0]
    for c in counts:
        host_indptr.append(host_indptr[-1] + c)

    def int32(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    last = [s - (c - 1) * page if c else 0 for s, c in zip(stored, counts)]
    length_info = int32([last, window, [min(case["sinks"], s) for s in stored]]) if case["sinks"] else int32(last)
    state = {"case": dict(case), "tables": tables, "pages": pages, "page_indptr": int32(host_indptr), "page_values": ids,
             "length_info": length_info, "max_pages": max(counts), "sm_scale": d ** -0.5}
    if case["op"] == "write":
        # slots of all stored tokens, sequence by sequence, and of the new ones, which are each sequence's last
        at = [host_indptr[b] * page + t for b in range(case["batch"]) for t in range(stored[b])]
        newest = [host_indptr[b] * page + t for b in range(case["batch"]) for t in range(stored[b] - new[b], stored[b])]
        held, fresh = (ids[(int32(v) // page).long()] * page + int32(v) % page for v in (at, newest))
        rows = torch.randn((2, len(newest), hkv, d), generator=g, device=device) * channel.transpose(1, 2)
        state.update(append_map=fresh.int(), read_map=held.int(), k_new=rows[0].half().contiguous(),
                     v_new=rows[1].half().contiguous(),
                     k_rows=torch.empty((len(at), hkv, d), dtype=torch.float16, device=device),
                     v_rows=torch.empty((len(at), hkv, d), dtype=torch.float16, device=device))
        return state
    queries = [1] * case["batch"] if case["op"] == "decode" else new
    q_indptr = [0]
    for n in queries:
        q_indptr.append(q_indptr[-1] + n)
    state.update(q=(1.5 * torch.randn((q_indptr[-1], hq, d), generator=g, device=device)).half(), q_indptr=int32(q_indptr),
                 max_queries=max(queries), output=torch.empty((q_indptr[-1], hq, d), dtype=torch.float16, device=device),
                 lse=torch.empty((q_indptr[-1], hq), dtype=torch.float32, device=device))
    return state


# ---- one pass ------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return _write(case, state) if case["op"] == "write" else _attend(case, state)


def _run_own(case, s):
    from tvm_amd import kernels
    if case["op"] == "write":
        kernels.mxfp4_append(s["pages"], s["k_new"], s["v_new"], s["append_map"])
        kernels.mxfp4_read_kv(s["pages"], s["read_map"], s["k_rows"], s["v_rows"])
        return {"k": s["k_rows"], "v": s["v_rows"]}
    if case["op"] == "decode":
        kernels.mxfp4_batch_decode_paged_kv(s["q"], s["pages"], s["page_indptr"], s["page_values"], s["length_info"], s["output"],
                                            s["lse"], s["sm_scale"])
    else:
        kernels.mxfp4_batch_prefill_paged_kv(s["q"], s["q_indptr"], s["pages"], s["page_indptr"], s["page_values"],
                                             s["length_info"], s["output"], s["lse"], int(case["causal"]), s["sm_scale"])
    return {"out": s["output"], "lse": s["lse"]}


def _write(case, s):
    page, d = case["page"], case["head_dim"]
    codes, scales = _slabs(s["pages"], d)
    at, slot = (s["append_map"] // page).long(), (s["append_map"] % page).long()
    new_codes, new_scales = _quantise(torch.stack((s["k_new"], s["v_new"]), 1), s["tables"])
    codes[at, :, :, slot] = new_codes
    scales[at, :, :, slot] = new_scales
    at, slot = (s["read_map"] // page).long(), (s["read_map"] % page).long()
    rows = _values(codes[at, :, :, slot], scales[at, :, :, slot], s["tables"]).half()
    return {"k": rows[:, 0].contiguous(), "v": rows[:, 1].contiguous()}


def _attend(case, s):
    """All sequences at once, padded to the longest."""
    d, hkv, page = case["head_dim"], case["kv_heads"], case["page"]
    device = s["q"].device
    counts = s["page_indptr"][1:] - s["page_indptr"][:-1]
    windows = s["length_info"].dim() == 2
    last = s["length_info"][0] if windows else s["length_info"]
    stored = torch.where(counts > 0, (counts - 1) * page + last, 0)
    keys = stored - s["length_info"][1] + s["length_info"][2] if windows else stored
    # keys and values, (batch, 2, kv heads, tokens, head_dim)
    nth = torch.arange(s["max_pages"], device=device)
    table = s["page_values"][(s["page_indptr"][:-1, None] + torch.minimum(nth, (counts[:, None] - 1).clamp(min=0))).long().clamp(
        max=s["page_values"].numel() - 1)]
    codes, scales = _slabs(s["pages"][table.long()], d)
    kv = [_values(codes[:, :, i], scales[:, :, i], s["tables"]).transpose(1, 2).flatten(2, 3) for i in (0, 1)]
    token = torch.arange(kv[0].shape[2], device=device)
    logical = token.expand(case["batch"], -1)
    there = token < stored[:, None]
    if windows:
        sinks, first = s["length_info"][2][:, None], s["length_info"][1][:, None]
        there = (token < sinks) | ((token >= first) & there)
        logical = torch.where(token < sinks, token, token - first + sinks)
    # queries, (batch, kv heads, queries of a head group, head_dim)
    asked = s["q_indptr"][1:] - s["q_indptr"][:-1]
    nth = torch.arange(s["max_queries"], device=device)
    at = (s["q_indptr"][:-1, None] + nth).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][at].float().unflatten(2, (hkv, -1)).permute(0, 2, 3, 1, 4)
    shape = q.shape[2:4]
    see = there[:, None, :].expand(-1, s["max_queries"], -1)
    if case["op"] == "prefill" and case["causal"]:
        see = see & (logical[:, None, :] < (keys - asked)[:, None, None] + 1 + nth[:, None])
    scores = (q.flatten(2, 3) @ kv[0].transpose(2, 3)).unflatten(2, shape) * (s["sm_scale"] * math.log2(math.e))
    scores = scores.masked_fill(~see[:, None, None], -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    weights = torch.exp2(scores - most)
    del scores
    total = weights.sum(-1, keepdim=True)
    out = (weights.flatten(2, 3) @ kv[1]).unflatten(2, shape) / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, most + torch.log2(total), EMPTY_LSE)[..., 0]
    real = (nth < asked[:, None]).flatten().nonzero()[:, 0]
    out = out.permute(0, 3, 1, 2, 4).flatten(0, 1).flatten(1, 2)[real]
    return {"out": out.half(), "lse": lse.permute(0, 3, 1, 2).flatten(0, 1).flatten(1, 2)[real]}


# ---- the definition in 64 bits -------------------------------------------------------------------------------


def _fp4(code):
    """A code's value from its bits: sign, two exponent bits with bias 1, one mantissa bit."""
    sign, e, m = (code >> 3) & 1, (code >> 1) & 3, (code & 1).double()
    return torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * 2.0 ** (e - 1).double()) * (1.0 - 2.0 * sign.double())


def _stored_rows(pages, ids, which, head, head_dim):
    """The rows that some pages hold for one head, in 64 bits: (tokens, head_dim)."""
    page = pages.shape[3]
    flat = pages[ids, which, head].reshape(len(ids), -1).long()
    codes = flat[:, :page * head_dim // 2].reshape(-1, head_dim // 2)
    power = (flat[:, page * head_dim // 2:].reshape(-1, head_dim // BLOCK) - 127).repeat_interleave(BLOCK, 1)
    return torch.stack((_fp4(codes & 15), _fp4(codes >> 4)), -1).reshape(-1, head_dim) * 2.0 ** power.double()


def _rounded(rows):
    """Rows as the cache holds them: the nearest of a block's sixteen values, ties to the even code."""
    x = rows.double().unflatten(-1, (-1, BLOCK))
    largest = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(largest, 13.0)
    for e in range(12, -24, -1):
        power = torch.where(largest <= 7.0 * 2.0 ** e, float(e), power)
    y = x.abs() / 2.0 ** power
    best, value = torch.full_like(y, math.inf), torch.zeros_like(y)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: a tie keeps them
        off = (y - _MAGNITUDES[code]).abs()
        value = torch.where(off < best, _MAGNITUDES[code], value)
        best = torch.minimum(best, off)
    return (torch.copysign(value, x) * 2.0 ** power).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    d, hkv, page = case["head_dim"], case["kv_heads"], case["page"]
    stored, new, window = _lengths(case)
    indptr = s["page_indptr"].tolist()
    if case["op"] == "write":
        got = {}
        for which, rows in enumerate((s["k_new"], s["v_new"])):
            whole = torch.empty((len(s["read_map"]), hkv, d), dtype=torch.float64, device=rows.device)
            for h in range(hkv):
                held = _stored_rows(s["pages"], s["page_values"].long(), which, h, d)
                begin, fresh = 0, 0
                for b in range(case["batch"]):
                    mine = held[indptr[b] * page:indptr[b] * page + stored[b]].clone()
                    if new[b]:
                        mine[stored[b] - new[b]:] = _rounded(rows[fresh:fresh + new[b], h])
                    whole[begin:begin + stored[b], h] = mine
                    begin, fresh = begin + stored[b], fresh + new[b]
            got["kv"[which]] = whole
        return got
    hq = case["q_heads"]
    group = hq // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], EMPTY_LSE, dtype=torch.float64, device=s["q"].device)
    begin = s["q_indptr"].tolist()
    for b in range(case["batch"]):
        ids = s["page_values"][indptr[b]:indptr[b + 1]].long()
        at = list(range(stored[b]))
        if case["sinks"]:
            at = at[:min(case["sinks"], stored[b])] + at[window[b]:]
        n, keys = begin[b + 1] - begin[b], len(at)
        if not n or not keys:
            continue
        at = torch.tensor(at, device=ids.device)
        first = keys - n if case["op"] == "prefill" and case["causal"] else None
        for h in range(hkv):
            k = _stored_rows(s["pages"], ids, 0, h, d)[at]
            v = _stored_rows(s["pages"], ids, 1, h, d)[at]
            for r in range(0, n, 512):
                q = s["q"][begin[b] + r:begin[b] + min(n, r + 512), h * group:(h + 1) * group].double()
                x = torch.tensordot(q, k, dims=([2], [1])) * (s["sm_scale"] / math.log(2.0))
                if first is not None:
                    mine = first + r + torch.arange(q.shape[0], device=ids.device)
                    x = x.masked_fill((torch.arange(keys, device=ids.device) > mine[:, None])[:, None], -math.inf)
                top = x.amax(-1, keepdim=True)
                e = torch.exp2(x - torch.where(torch.isinf(top), 0.0, top))
                total = e.sum(-1, keepdim=True)
                rows = slice(begin[b] + r, begin[b] + r + q.shape[0])
                some = total > 0
                out[rows, h * group:(h + 1) * group] = torch.where(some, torch.tensordot(e, v, dims=([2], [0])) / total, 0.0)
                lse[rows, h * group:(h + 1) * group] = torch.where(some, top + torch.log2(total), EMPTY_LSE)[..., 0]
    return {"out": out, "lse": lse}
