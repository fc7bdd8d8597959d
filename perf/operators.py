"""The operators of a serving step over a paged key/value cache in 8 bits, as
they are measured: appending keys and values (`kv_append`, read back with
`kv_read`), attention over the cache (`sdpa_paged`, also with a sliding window
and first tokens that stay visible) and the verification of drafted tokens
(`verify_draft`).

With `own` false every operator is computed in plain torch operations from the
definitions:

  rotation   angle = position * inv_freq[j], interleaved pairs (2j, 2j + 1)
  page       64 positions of a sequence; one scale for the keys and one for the
             values of each (page, kv head): s = f32(max|x| / 127), at least the
             page's former scale where it holds earlier rows
  stored     rint(x / s) within +-127; earlier rows of a page whose scale grew
             become rint(q * s_old / s)
  attention  softmax(q.k / sqrt(d)) v over the keys j <= p of a query at
             position p, with a window w only those with j > p - w or j < sinks
  drafts     accepted while u q(x) < p(x); the next token from max(p - q, 0) at
             the first rejection, from p behind the last one
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64
ROPE_BASE = 500000.0
F64 = torch.float64


def listed():
    return [
        # one decoded token of one chat: the smallest call
        {"name": "append_1_token", "op": "append", "seqs": 1, "past_lo": 77, "past_hi": 77, "new": 1, "ragged": False,
         "kv_heads": 8, "dim": 64},
        # one decoded token for each of many chats, their last pages partly filled
        {"name": "append_96_chats", "op": "append", "seqs": 96, "past_lo": 1, "past_hi": 3000, "new": 1,
         "ragged": False, "kv_heads": 8, "dim": 64},
        # a document's prompt behind a short system prompt
        {"name": "append_prompt_2011", "op": "append", "seqs": 1, "past_lo": 37, "past_hi": 37, "new": 2011,
         "ragged": False, "kv_heads": 8, "dim": 128},
        # one decoded token of one short chat
        {"name": "decode_1_of_300", "op": "sdpa", "seqs": 1, "past_lo": 300, "past_hi": 300, "new": 1,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 0, "sinks": 0},
        # a server's decode step, lengths from a greeting to a long chat
        {"name": "decode_48_chats", "op": "sdpa", "seqs": 48, "past_lo": 17, "past_hi": 8000, "new": 1,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 0, "sinks": 0},
        # one decoded token behind a context as long as the 1B model's
        {"name": "decode_1_of_131000", "op": "sdpa", "seqs": 1, "past_lo": 131000, "past_hi": 131000, "new": 1,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 0, "sinks": 0},
        # the target's pass over up to five drafted tokens a chat
        {"name": "drafts_16_chats", "op": "sdpa", "seqs": 16, "past_lo": 100, "past_hi": 4000, "new": 6,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0, "sinks": 0},
        # the second piece of a long prompt
        {"name": "prompt_1531_of_2048", "op": "sdpa", "seqs": 1, "past_lo": 517, "past_hi": 517, "new": 1531,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 0, "sinks": 0},
        # decode with a window of 1024 and four visible first tokens
        {"name": "window_32_chats", "op": "sdpa", "seqs": 32, "past_lo": 500, "past_hi": 9000, "new": 1,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 1024, "sinks": 4},
        # a document's prompt through a layer with a window
        {"name": "window_prompt_2500", "op": "sdpa", "seqs": 1, "past_lo": 0, "past_hi": 0, "new": 2500,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 64, "window": 512, "sinks": 4},
        # four drafted tokens of one chat
        {"name": "verify_1_chat", "op": "verify", "seqs": 1, "drafts": 4, "ragged": False, "vocab": 128256,
         "temperature": 0.8, "sampled": True},
        # up to seven drafted tokens for each of many chats
        {"name": "verify_40_chats", "op": "verify", "seqs": 40, "drafts": 7, "ragged": True, "vocab": 128256,
         "temperature": 1.0, "sampled": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "sdpa", "sdpa", "sdpa", "verify"])
    if op == "verify":
        return {"op": op, "seqs": _log_int(rng, 1, 32), "drafts": rng.randint(1, 7), "ragged": rng.random() < 0.6,
                "vocab": rng.choice([128256, 128256, 32000, _log_int(rng, 500, 128256)]),
                "temperature": rng.choice([0.6, 0.8, 1.0, 1.3]), "sampled": rng.random() < 0.75}
    heads, kv = rng.choice([(32, 8), (32, 8), (8, 2), (4, 2), (16, 16), (24, 3), (32, 4)])
    dim = rng.choice([64, 64, 128])
    kind = rng.choice(["decode", "decode", "drafts", "prompt"])
    if kind == "prompt":
        seqs, past_hi, new = 1, _log_int(rng, 1, 512), _log_int(rng, 9, 1500)
        past_lo = past_hi
    else:
        seqs, new = _log_int(rng, 1, 40), 1 if kind == "decode" else rng.randint(2, 8)
        past_hi = _log_int(rng, 20, 5000)
        past_lo = max(1, past_hi // rng.choice([1, 3, 20]))
    case = {"op": op, "seqs": seqs, "past_lo": past_lo, "past_hi": past_hi, "new": new, "ragged": kind == "drafts",
            "kv_heads": kv, "dim": dim}
    if op == "sdpa":
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 2048)])
        case |= {"heads": heads, "window": window, "sinks": rng.choice([0, 1, 4, 130]) if window else 0}
    return case


def _sizes(case):
    """Cached and new positions of each sequence of a case (the same for every seed)."""
    r = np.random.default_rng(case["seqs"] * 7919 + case["past_hi"])
    lo, hi = max(case["past_lo"], 1), max(case["past_hi"], 1)
    past = np.exp(r.uniform(math.log(lo), math.log(hi), case["seqs"])).round().astype(np.int64)
    past = np.clip(past, case["past_lo"], case["past_hi"])
    new = r.integers(1, case["new"] + 1, case["seqs"]) if case["ragged"] else np.full(case["seqs"], case["new"])
    return past, new.astype(np.int64)


def _drafts(case):
    r = np.random.default_rng(case["seqs"] * 104729 + case["drafts"])
    if not case["ragged"]:
        return np.full(case["seqs"], case["drafts"], np.int64)
    return r.integers(0, case["drafts"] + 1, case["seqs"]).astype(np.int64)


def _inv_freq(dim):
    j = torch.arange(dim // 2, dtype=F64)
    return (ROPE_BASE ** (-2.0 * j / dim)).float()


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _cache_inputs(case, g):
    """Cached keys (rotated) and values of the padded sequences, then the new rows."""
    past, new = _sizes(case)
    s, kv, d = case["seqs"], case["kv_heads"], case["dim"]
    rows = int(new.sum())
    # keys have a few strong channels, values do not
    gain = torch.exp2(2.0 * torch.rand(kv, d, generator=g, device="cuda") - 1.0)
    length = int(past.max())

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    cached = torch.arange(length, device="cuda")[None, :] < torch.from_numpy(past).cuda()[:, None]
    keep = cached[:, :, None, None]
    k_past = normal(s, length, kv, d).mul_(gain).mul_(keep)
    v_past = normal(s, length, kv, d).mul_(keep)
    out = {"past": past, "new": new, "cached": cached, "k_past": k_past, "v_past": v_past}
    if case["op"] == "append":
        out |= {"k": normal(rows, kv, d) * gain, "v": normal(rows, kv, d)}
    else:
        # the new rows are in the cache already when their queries attend
        out |= {"k": normal(rows, kv, d) * gain, "v": normal(rows, kv, d),
                "q": normal(rows, case["heads"], d)}
    return out


def _rows(past, new):
    """Sequence and position of every new row, as tensors."""
    seq = np.repeat(np.arange(len(past)), new)
    first = np.repeat(np.cumsum(new) - new, new)
    pos = np.repeat(past, new) + np.arange(int(new.sum())) - first
    return torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()


def _quantize_pages(x):
    """[seqs, positions, heads, dim] in whole pages: int8 values and f32 scales [seqs, pages, heads]."""
    s, n, h, d = x.shape
    x = x.view(s, n // PAGE, PAGE, h, d)
    scale = (x.abs().amax((2, 4)).double() / 127.0).float()
    by = scale.double()[:, :, None, :, None]
    q = torch.where(by > 0, torch.round(x.double() / by), torch.zeros((), dtype=F64, device=x.device))
    return torch.clamp(q, -127, 127).to(torch.int8), scale


def _padded(x, pages):
    return torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pages * PAGE - x.shape[1]))


def _verify_inputs(case, g):
    n = _drafts(case)
    rows, vocab = int(n.sum()), case["vocab"]
    s = case["seqs"]
    target = 2.5 * torch.randn(rows + s, vocab, generator=g, device="cuda")
    # the rows that a draft was made for, in the target's order
    of = torch.from_numpy(np.concatenate([np.arange(k) + i + first for i, (first, k) in
                                          enumerate(zip(np.cumsum(n) - n, n))]).astype(np.int64)).cuda()
    # the draft model's distribution is near the target's
    draft = target[of] + 0.7 * torch.randn(rows, vocab, generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device="cuda", dtype=F64).clamp(1e-300, 1 - 1e-16)))
    tokens = (draft.double() / case["temperature"] + noise).argmax(1).to(torch.int32)  # drawn from the draft
    u = torch.rand(rows + s, generator=g, device="cuda")
    return {"n": n, "of": of, "target": target, "draft": draft if case["sampled"] else None, "tokens": tokens, "u": u}


class Buffer:
    """A torch tensor's memory as sqhip.ops takes it."""

    def __init__(self, t):
        self.ptr, self.shape, self.size = t.data_ptr(), tuple(t.shape), t.numel()


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "squirrel-rs_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from sqhip import ops
    return ops


def _filled_pool(case, x, seed):
    """A pool with the cached rows of every sequence in pages in no order, and the plan of the step."""
    ops = _ops()
    past, new = x["past"], x["new"]
    pages = -(-(past + new) // PAGE)
    total = int(pages.sum())
    free = np.random.default_rng(seed).permutation(total + 8).astype(np.uint32)
    tables = np.zeros((len(past), int(pages.max())), np.uint32)
    tables[np.arange(tables.shape[1])[None, :] < pages[:, None]] = free[:total]
    pool = ops.KvPool(1, total + 8, case["kv_heads"], case["dim"], _inv_freq(case["dim"]).numpy())
    if past.any():
        k, v = x["k_past"][x["cached"]].contiguous(), x["v_past"][x["cached"]].contiguous()
        fill = ops.KvPlan(pool, np.zeros_like(past), past, tables)
        ops.kv_append(fill, 0, Buffer(k), Buffer(v), rotated=True)
    return ops.KvPlan(pool, past, new, tables)


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "verify":
        x = _verify_inputs(case, g)
        state |= x
        if own:
            return state
        n = x["n"]
        most = int(n.max()) if len(n) else 0
        first = np.cumsum(n) - n
        # padded (sequence, draft) -> row of the drafts, of the target
        at = first[:, None] + np.minimum(np.arange(most)[None, :], np.maximum(n - 1, 0)[:, None])
        state["draft_row"] = torch.from_numpy(np.minimum(at, max(int(n.sum()) - 1, 0))).cuda()
        state["target_row"] = torch.from_numpy(at + np.arange(len(n))[:, None]).cuda()
        state["first_target"] = torch.from_numpy(first + np.arange(len(n))).cuda()
        state["count"] = torch.from_numpy(n).cuda()
        return state
    x = _cache_inputs(case, g)
    past, new = x["past"], x["new"]
    state |= {"past": past, "new": new}
    state["k"], state["v"] = x["k"], x["v"]
    if case["op"] == "sdpa":
        state["q"] = x["q"]
    if own:
        state["plan"] = _filled_pool(case, x, seed)
        if case["op"] == "append":
            n = int(np.minimum(past + new, case["new"] + PAGE - 1).sum())
            shape = (n, case["kv_heads"], case["dim"])
            state["k_out"], state["v_out"] = (torch.empty(shape, device="cuda") for _ in range(2))
        else:
            ops = _ops()
            ops.kv_append(state["plan"], 0, Buffer(x["k"]), Buffer(x["v"]), rotated=True)
            state["out"] = torch.empty_like(x["q"])
        return state
    state["seq"], state["pos"] = _rows(past, new)
    state["inv_freq"] = _inv_freq(case["dim"]).cuda()
    pages = int((-(-(past + new) // PAGE)).max())
    kq, ks = _quantize_pages(_padded(x["k_past"], pages))
    vq, vs = _quantize_pages(_padded(x["v_past"], pages))
    state |= {"kq": kq, "ks": ks, "vq": vq, "vs": vs}
    if case["op"] == "sdpa":
        _append_plain(state, state["k"].double(), state["v"].double())
        most = int(new.max())
        state["lengths"] = torch.from_numpy(past + new).cuda()
        state["slot"] = state["pos"] - torch.from_numpy(past).cuda()[state["seq"]]
        state["query_pos"] = torch.from_numpy(past).cuda()[:, None] + torch.arange(most, device="cuda")
    return state


# ------------------------------------------------------------------ plain forms


def _rotated(x, pos, inv_freq):
    """x [rows, heads, dim] in 64 bits, rotated by its position."""
    angle = pos.double()[:, None] * inv_freq.double()[None, :]
    c, s = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)


def _append_into(q, scale, x, seq, pos):
    """New rows x (64 bits) into the pages q [seqs, pages, PAGE, heads, dim], scales [seqs, pages, heads]."""
    page, slot = pos // PAGE, pos % PAGE
    s, p, h = scale.shape
    # the largest new magnitude of each page, and whether earlier rows stay in it
    top = torch.zeros(s * p, h, dtype=F64, device=x.device)
    cell = seq * p + page
    top = top.scatter_reduce(0, cell[:, None].expand(-1, h), x.abs().amax(2), "amax").view(s, p, h)
    low = torch.full((s * p,), PAGE, device=x.device, dtype=slot.dtype)
    low = low.scatter_reduce(0, cell, slot, "amin").view(s, p)  # first new slot; PAGE: an untouched page
    fresh = (top / 127.0).float()
    old = torch.where((low > 0)[:, :, None], scale, torch.zeros_like(scale))
    grown = torch.maximum(old, fresh)
    ratio_from, ratio_to = old.double(), grown.double()
    moved = (grown > old) & (low > 0)[:, :, None] & (low < PAGE)[:, :, None]
    # earlier rows of the pages whose scale grew, in the steps of the new scale
    si, pi, hi = torch.nonzero(moved, as_tuple=True)
    part = q[si, pi, :, hi].double()
    part = torch.round(part * ratio_from[si, pi, hi][:, None, None] / ratio_to[si, pi, hi][:, None, None])
    q[si, pi, :, hi] = part.to(torch.int8)
    scale.copy_(grown)
    by = grown[seq, page].double()[:, :, None]
    new = torch.where(by > 0, torch.round(x / by), torch.zeros_like(x))
    q[seq, page, slot] = torch.clamp(new, -127, 127).to(torch.int8)


def _append_plain(state, k, v):
    _append_into(state["kq"], state["ks"], k, state["seq"], state["pos"])
    _append_into(state["vq"], state["vs"], v, state["seq"], state["pos"])


def _values(q, scale):
    """The f32 values that stored integers stand for, [seqs, positions, heads, dim]."""
    x = q.float() * scale[:, :, None, :, None]
    return x.flatten(1, 2)


def _plain_append(state):
    case = state["case"]
    k = _rotated(state["k"], state["pos"], state["inv_freq"])
    _append_plain(state, k, state["v"].double())
    # the last positions of each sequence, as far as a page that was written reaches back
    past, new = state["past"], state["new"]
    last = np.minimum(past + new, case["new"] + PAGE - 1)
    seq = np.repeat(np.arange(len(past)), last)
    pos = np.arange(int(last.sum())) - np.repeat(np.cumsum(last) - last, last) + np.repeat(past + new - last, last)
    seq, pos = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
    page, slot = pos // PAGE, pos % PAGE
    return (state["kq"][seq, page, slot].float() * state["ks"][seq, page][:, :, None],
            state["vq"][seq, page, slot].float() * state["vs"][seq, page][:, :, None])


def _plain_sdpa(state):
    case = state["case"]
    kv, d, g = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    k, v = _values(state["kq"], state["ks"]), _values(state["vq"], state["vs"])
    s, n = k.shape[0], k.shape[1]
    q = _rotated(state["q"], state["pos"], state["inv_freq"]).float()
    m = state["query_pos"].shape[1]
    padded = torch.zeros(s, m, kv, g, d, device=q.device)
    padded[state["seq"], state["slot"]] = q.view(-1, kv, g, d)
    qb = padded.permute(0, 2, 1, 3, 4).reshape(s * kv, m * g, d)
    kb = k.permute(0, 2, 3, 1).reshape(s * kv, d, n)
    vb = v.permute(0, 2, 1, 3).reshape(s * kv, n, d)
    scores = torch.bmm(qb, kb).view(s, kv, m, g, n) / math.sqrt(d)
    at, p = torch.arange(n, device=q.device), state["query_pos"][:, :, None]
    seen = at <= p
    if case["window"]:
        seen &= (at > p - case["window"]) | (at < case["sinks"])
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    out = torch.bmm(w.view(s * kv, m * g, n), vb).view(s, kv, m, g, d).permute(0, 2, 1, 3, 4)
    return out[state["seq"], state["slot"]].reshape(-1, kv * g, d)


def _softmax64(logits, temperature):
    x = logits.double() / temperature
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(state):
    case = state["case"]
    count, tokens, u = state["count"], state["tokens"].long(), state["u"].double()
    s = case["seqs"]
    t = case["temperature"]
    p = _softmax64(state["target"], t)
    q = None if state["draft"] is None else _softmax64(state["draft"], t)
    accepted = torch.zeros(s, dtype=torch.int64, device=u.device)
    # (a batch in which no sequence has a draft only draws)
    if state["draft_row"].shape[1] and len(tokens):
        x = tokens[state["draft_row"]]
        px = p[state["target_row"], x]
        qx = torch.ones_like(px) if q is None else q[state["draft_row"], x]
        there = torch.arange(x.shape[1], device=u.device)[None, :] < count[:, None]
        taken = (u[state["target_row"]] * qx < px) & there
        accepted = torch.cumprod(taken.long(), 1).sum(1)
    w = p[state["first_target"] + accepted]
    rejected = accepted < count
    if len(tokens):
        row = torch.clamp(state["first_target"] - torch.arange(s, device=u.device) + accepted, max=len(tokens) - 1)
        if q is None:
            less = torch.zeros_like(w).scatter_(1, tokens[row][:, None], 1.0)
            less = torch.where(less > 0, w, torch.zeros_like(w))
        else:
            less = q[row]
        w = torch.where(rejected[:, None], torch.clamp(w - less, min=0.0), w)
    cum = torch.cumsum(w, 1)
    at = u[state["first_target"] + count] * cum[:, -1]
    token = (cum <= at[:, None]).sum(1)
    return accepted.cpu().numpy().astype(np.uint32), token.cpu().numpy().astype(np.uint32)


# ------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"append": _plain_append, "sdpa": _plain_sdpa, "verify": _plain_verify}[op](state)
    ops = _ops()
    if op == "append":
        ops.kv_append(state["plan"], 0, Buffer(state["k"]), Buffer(state["v"]))
        ops.kv_read(state["plan"], 0, case["new"] + PAGE - 1, Buffer(state["k_out"]), Buffer(state["v_out"]))
        return state["k_out"], state["v_out"]
    if op == "sdpa":
        ops.sdpa_paged(state["plan"], 0, Buffer(state["q"]), Buffer(state["out"]), case["heads"],
                       window=case["window"], sinks=case["sinks"])
        return state["out"]
    draft = state["draft"]
    return ops.verify_draft(Buffer(state["target"]), None if draft is None else Buffer(draft),
                            Buffer(state["tokens"]), Buffer(state["u"]), state["n"], case["temperature"])


def work(case):
    if case["op"] == "verify":
        n = int(_drafts(case).sum())
        rows = n + case["seqs"] + (n if case["sampled"] else 0)
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}
    past, new = _sizes(case)
    width = case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        read = np.minimum(past + new, case["new"] + PAGE - 1)
        # new rows in and stored, the last rows read back
        return {"bytes": float(2 * width * (5 * new.sum() + 5 * read.sum())),
                "flops": float(width * (10 * new.sum() + 2 * read.sum()))}
    length = past + new
    most = np.minimum(length, case["window"] + new - 1 + case["sinks"]) if case["window"] else length
    pairs = 0.0
    for a, n in zip(past, new):
        p = np.arange(a, a + n, dtype=np.float64)
        seen = p + 1
        if case["window"]:
            w0 = np.maximum(p - case["window"] + 1, 0)
            seen = p + 1 - w0 + np.minimum(w0, case["sinks"])
        pairs += float(seen.sum())
    q_bytes = 8.0 * float(new.sum()) * case["heads"] * case["dim"]
    return {"bytes": q_bytes + 2.0 * width * float(most.sum()), "flops": 4.0 * case["dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------ 64-bit results


def _exact_cache(past, new, seq, x_past, x_new):
    """A sequence's stored values after the new rows were appended, in 64 bits: [positions, heads, dim]."""
    length = int(past + new)
    out = torch.zeros(length, *x_new.shape[1:], dtype=F64, device=x_new.device)
    for start in range(0, length, PAGE):
        end = min(start + PAGE, length)
        a, b = max(start, min(int(past), end)), end  # new rows of the page
        old, fresh = x_past[seq, start:a].double(), x_new[a - int(past):b - int(past)]
        s = torch.zeros(x_new.shape[1], dtype=F64, device=x_new.device)
        q = old
        if len(old):
            s = (old.abs().amax((0, 2)) / 127.0).float().double()
            q = torch.clamp(torch.round(old / s[:, None]), -127, 127)
        if len(fresh):
            t = torch.maximum(s, (fresh.abs().amax((0, 2)) / 127.0).float().double())
            if len(old):
                q = torch.where((t > s)[:, None], torch.round(q * s[:, None] / t[:, None]), q)
            q = torch.cat([q, torch.clamp(torch.round(fresh / t[:, None]), -127, 127)])
            s = t
        out[start:end] = q * s[:, None]
    return out


def _exact_rotation(x, first, dim):
    """Rows at positions first, first + 1, ...: the pairs as complex numbers times exp(i angle)."""
    pos = torch.arange(first, first + len(x), device=x.device, dtype=F64)
    angle = torch.outer(pos, _inv_freq(dim).to(x.device).double())[:, None, :]
    z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], dim // 2, 2).contiguous())
    return torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)).flatten(-2)


def exact(case, seed):
    g = _generator(seed)
    if case["op"] == "verify":
        return _exact_verify(case, _verify_inputs(case, g))
    x = _cache_inputs(case, g)
    past, new = x["past"], x["new"]
    first = np.cumsum(new) - new
    d, g_heads = case["dim"], case.get("heads", 0) // case["kv_heads"]
    ks, vs, outs = [], [], []
    for i in range(case["seqs"]):
        a, n = int(past[i]), int(new[i])
        k, v = x["k"][first[i]:first[i] + n].double(), x["v"][first[i]:first[i] + n].double()
        if case["op"] == "append":
            k = _exact_rotation(k, a, d)
        k = _exact_cache(a, n, i, x["k_past"], k)
        v = _exact_cache(a, n, i, x["v_past"], v)
        if case["op"] == "append":
            last = min(a + n, case["new"] + PAGE - 1)
            ks.append(k[a + n - last:])
            vs.append(v[a + n - last:])
            continue
        q = _exact_rotation(x["q"][first[i]:first[i] + n], a, d)
        p = torch.arange(a, a + n, device="cuda")[:, None]
        at = torch.arange(a + n, device="cuda")[None, :]
        hidden = at > p
        if case["window"]:
            hidden |= (at <= p - case["window"]) & (at >= case["sinks"])
        out = torch.empty_like(q)
        for h in range(case["heads"]):
            j = h // g_heads
            s = (q[:, h].contiguous() @ k[:, j].t().contiguous()) / math.sqrt(d)
            w = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1)
            out[:, h] = w @ v[:, j].contiguous()
        outs.append(out)
    if case["op"] == "append":
        return torch.cat(ks), torch.cat(vs)
    return torch.cat(outs)


def _exact_verify(case, x):
    """Sequence by sequence, draft by draft, on the host."""
    n = x["n"]
    accepted, token = np.zeros(len(n), np.uint32), np.zeros(len(n), np.uint32)
    tokens, u = x["tokens"].cpu().numpy(), x["u"].cpu().numpy().astype(np.float64)
    row_t, row_d = 0, 0

    def probabilities(row):
        z = row.cpu().numpy().astype(np.float64) / case["temperature"]
        z = np.exp(z - z.max())
        return z / z.sum()

    for i in range(len(n)):
        w = None
        for j in range(int(n[i])):
            p, t = probabilities(x["target"][row_t + j]), tokens[row_d + j]
            q = np.zeros_like(p) if x["draft"] is None else probabilities(x["draft"][row_d + j])
            if x["draft"] is None:
                q[t] = 1.0
            if not u[row_t + j] * q[t] < p[t]:
                w = np.maximum(p - q, 0.0)
                break
            accepted[i] += 1
        if w is None:
            w = probabilities(x["target"][row_t + int(n[i])])
        cum = np.cumsum(w)
        token[i] = np.searchsorted(cum, u[row_t + int(n[i])] * cum[-1], side="right")
        row_t, row_d = row_t + int(n[i]) + 1, row_d + int(n[i])
    return accepted, token
