"""What the decoder operators are measured on: the paged key/value cache, the attention that reads it and the sampler.

`listed()` names the cases, `draw(rng)` makes more of the same ranges, `prepare(case, seed)` makes a case's inputs on the GPU,
`run(state)` is one pass (elementary torch operations, or the library's operators where `own` is true), `work(case)` counts
what a pass cannot do without and `exact(case, seed)` gives the outputs in 64 bits.

Operators ("op" of a case):
  cache   keys and values of new tokens are written into the pages of a cache (bf16, or 8 bits with one scale per token and
          head) and rows are read back
  attend  attention of each sequence's new tokens over its cached keys and values, with an optional sliding window beside
          a few first tokens that stay visible
  sample  one token per row of logits: temperature, top-k, top-p, min-p, drawn with a given uniform number
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

LN_NONE = float("-inf")


def _package():
    if "obs_localvocal_amd" in sys.modules:
        return sys.modules["obs_localvocal_amd"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("obs_localvocal_amd", os.path.join(root, "obs-localvocal_amd", "__init__.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["obs_localvocal_amd"] = mod
    spec.loader.exec_module(mod)
    return mod


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _cache(name, kind, seqs, q_lo, q_hi, past_lo, past_hi, kv_heads, dim, page, source, whole):
    c = dict(op="cache", kind=kind, seqs=seqs, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, heads=kv_heads, kv_heads=kv_heads,
             dim=dim, page=page, source=source, whole=whole, window=0, sinks=0)
    return dict(c, name=name) if name else c


def _attend(name, kind, seqs, q_lo, q_hi, past_lo, past_hi, heads, kv_heads, dim, page, window=0, sinks=0):
    c = dict(op="attend", kind=kind, seqs=seqs, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, heads=heads, kv_heads=kv_heads,
             dim=dim, page=page, window=window, sinks=sinks)
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, dtype, mix):
    c = dict(op="sample", rows=rows, vocab=vocab, dtype=dtype, mix=mix)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decode step of 64 streams of a 20-head decoder: one token each goes into the cache (latency)
        _cache("cache-step-64", "e4m3", 64, 1, 1, 30, 447, 20, 64, 32, "bf16", False),
        # prompts of several requests written at once behind cached prefixes, then whole sequences read back (migrating or
        # saving them)
        _cache("cache-prompts", "int8", 16, 130, 1021, 0, 3001, 8, 128, 16, "f32", True),
        # one stream's next token over a short text context: the smallest call
        _attend("attend-one-short", "bf16", 1, 1, 1, 223, 223, 20, 20, 64, 16),
        # the decode step of 64 streams over contexts as long as an encoder's output, in 8 bits
        _attend("attend-step-64", "e4m3", 64, 1, 1, 99, 1499, 20, 20, 64, 32),
        # few requests with long contexts and grouped heads: the key axis has to be split to fill the card
        _attend("attend-step-long", "int8", 8, 1, 1, 9001, 32767, 32, 8, 128, 64),
        # prompts of ragged lengths over ragged cached prefixes
        _attend("attend-prompts", "bf16", 8, 17, 448, 0, 1000, 20, 20, 64, 16),
        # one piece of a long document's prefill
        _attend("attend-chunk-long", "bf16", 1, 2048, 2048, 14336, 14336, 32, 8, 128, 64),
        # streaming decoders that keep a window and the first tokens; pages behind the window have been given back
        _attend("window-step-32", "e4m3", 32, 1, 1, 2900, 65535, 32, 8, 128, 16, window=2048, sinks=4),
        # a streaming decoder's prompt with a window shorter than the chunk
        _attend("window-chunk", "bf16", 3, 600, 1777, 100, 6000, 20, 20, 64, 32, window=512, sinks=16),
        # one stream that falls back to sampling
        _sample("sample-one", 1, 51866, "f32", False),
        # a batch of streams with settings of their own, greedy ones among them
        _sample("sample-64", 64, 51866, "f32", True),
        # a large batch over a large vocabulary with logits in 16 bits: many ties
        _sample("sample-256-wide", 256, 128000, "bf16", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "window", "sample"])
    if op == "sample":
        vocab = _log_int(rng, 1000, 128000)
        rows = _log_int(rng, 1, 256)
        return _sample(None, rows, vocab, rng.choice(["f32", "bf16"]), rng.choice([False, True]))
    kind = rng.choice(["bf16", "e4m3", "int8"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 6, 8, 12, 16, 20])
    page = rng.choice([1, 8, 16, 32, 64, 128, 256])
    if op == "cache":
        seqs = _log_int(rng, 1, 64)
        most = max(2, 16000 // seqs)
        q_hi = _log_int(rng, 1, min(most, 2000))
        return _cache(None, kind, seqs, max(1, q_hi // rng.choice([1, 2, 7])), q_hi, 0, _log_int(rng, 1, most), kv_heads, dim, page,
                      rng.choice(["bf16", "f32"]), rng.choice([False, True]))
    group = rng.choice([1, 1, 2, 3, 4, 5, 8])
    window, sinks = (0, 0) if op == "attend" else (_log_int(rng, 16, 4096), rng.choice([0, 1, 4, 16, 70]))
    if rng.random() < 0.6:  # single tokens, or the few of a draft that is checked
        seqs = _log_int(rng, 1, 64)
        q_hi = rng.choice([1, 1, 1, 2, 5])
        past = _log_int(rng, 1, max(2, 700000 // (seqs * kv_heads)) if op == "attend" else 65000)
        return _attend(None, kind, seqs, rng.choice([1, q_hi]), q_hi, past // rng.choice([1, 2, 9]), past, group * kv_heads, kv_heads, dim, page,
                       window, sinks)
    seqs = rng.choice([1, 1, 2, 3, 6])
    q_hi = _log_int(rng, 16, 1900 // seqs)
    past = _log_int(rng, 1, max(2, min(12000, 250000000 // (q_hi * seqs * kv_heads * group))))
    return _attend(None, kind, seqs, max(1, q_hi // rng.choice([1, 2, 5])), q_hi, past // rng.choice([1, 2, 9]), past, group * kv_heads, kv_heads,
                   dim, page, window, sinks)


def _spread(lo, hi, n, step):
    """n whole numbers over lo .. hi in a fixed, mixed order, both ends among them."""
    return [hi if n == 1 else lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _coprime(n, near):
    while math.gcd(n, near) != 1:
        near += 1
    return near


def _lengths(case):
    """New tokens and cached tokens before them, per sequence."""
    n = case["seqs"]
    return _spread(case["q_lo"], case["q_hi"], n, _coprime(n, 5)), _spread(case["past_lo"], case["past_hi"], n, _coprime(n, 7))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _codes(kind, x):
    """Cache contents a program has in hand: codes (as bytes for 8 bits) and scales of the rows of x [..., dim] (f32)."""
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    amax = x.abs().amax(-1)
    if kind == "e4m3":
        s = torch.exp2(torch.ceil(torch.log2((amax.double() / 448).clamp_min(2.0 ** -126)))).float()
        return (x / s[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), s
    s = (amax / 127).clamp_min(2.0 ** -126)
    return torch.round(x.double() / s[..., None].double()).to(torch.int8).view(torch.uint8), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = 2.0 * normal(rows, vocab)
        # a peaked head (what a decoder is sure of) and suppressed tokens
        x[:, : min(vocab, 4096)] += 3.0 * torch.rand(rows, 1, device="cuda", generator=g) * normal(rows, min(vocab, 4096))
        off = torch.rand(vocab, device="cuda", generator=g) < 0.02
        x[:, off] = LN_NONE
        perm = torch.randperm(vocab, device="cuda", generator=g)
        s["logits"] = x[:, perm].to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16).contiguous()
        s["u"] = torch.rand(rows, device="cuda", generator=g, dtype=torch.float64)
        r = torch.arange(rows, device="cuda")
        if case["mix"]:
            s["temperature"] = torch.tensor([0.8, 1.0, 0.0, 0.6, 1.3], device="cuda")[r % 5]
            s["top_k"] = torch.tensor([0, 40, 200, 1, 1000, 7], device="cuda", dtype=torch.int32)[r % 6]
            s["top_p"] = torch.tensor([1.0, 0.95, 0.8, 0.5], device="cuda")[r % 4]
            s["min_p"] = torch.tensor([0.0, 0.05, 0.01], device="cuda")[r % 3]
        else:
            s["temperature"] = torch.full((rows,), 0.8, device="cuda")
            s["top_k"] = torch.full((rows,), 50, device="cuda", dtype=torch.int32)
            s["top_p"] = torch.full((rows,), 0.95, device="cuda")
            s["min_p"] = torch.full((rows,), 0.02, device="cuda")
        return s

    kind, hk, dim, page, window, sinks = (case[k] for k in ("kind", "kv_heads", "dim", "page", "window", "sinks"))
    q, past = _lengths(case)
    kv = [a + b for a, b in zip(q, past)]
    cols = max((n + page - 1) // page for n in kv)
    # pages that some visible position needs, in an order of their own; the others were given back
    live = []
    for b, n in enumerate(kv):
        low = max(0, past[b] - window + 1) if window else 0
        live.append([c for c in range((n + page - 1) // page) if (c + 1) * page > low or c * page < sinks])
    total = sum(len(x) for x in live)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(kv), cols), -1, dtype=torch.int32)
    at = 0
    for b, cs in enumerate(live):
        table[b, torch.tensor(cs, dtype=torch.int64)] = order[at:at + len(cs)]
        at += len(cs)
    s["table"] = table.cuda()
    s["cu_q"] = torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"], rows = max(q), max(kv), sum(q)
    # keys and values differ from head to head in size, as a model's do
    size = torch.exp(0.5 * normal(hk))[:, None, None]
    s["k"], s["k_scale"] = _codes(kind, size * normal(total, hk, page, dim))
    s["v"], s["v_scale"] = _codes(kind, size * normal(total, hk, page, dim))
    if case["op"] == "attend":
        s["q"] = (1.3 * normal(rows, case["heads"], dim)).to(torch.bfloat16)
    else:
        t = torch.float32 if case["source"] == "f32" else torch.bfloat16
        s["k_new"] = (size[:, 0] * normal(rows, hk, dim)).to(t)
        s["v_new"] = (size[:, 0] * normal(rows, hk, dim)).to(t)
        if case["whole"]:
            s["cu_read"] = torch.tensor(np.concatenate([[0], np.cumsum(kv)]), dtype=torch.int32, device="cuda")
            s["n_read"], s["max_read"] = sum(kv), max(kv)
        else:
            s["cu_read"], s["n_read"], s["max_read"] = s["cu_q"], rows, max(q)
    if own:
        as_kind = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[kind]
        s["handle"] = _package().KvCache(s["k"].view(as_kind), s["v"].view(as_kind), s["k_scale"], s["v_scale"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if op == "sample":
        return _run_sample(s)
    return _run_cache(s) if op == "cache" else _run_attend(s)


def _values(kind, codes, scale):
    """The f32 values that gathered codes [..., dim] stand for."""
    if kind == "bf16":
        return codes.float()
    c = codes.view(torch.float8_e4m3fn if kind == "e4m3" else torch.int8).float()
    return c * scale[..., None]


def _rows(cu, kv_len, table, page, n):
    """Page and row inside it of each of the n rows of a batch."""
    t = torch.arange(n, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu[1:], t, right=True)
    pos = (kv_len[b] - (cu[1:][b] - t)).long()
    return table[b, pos // page].long(), pos % page


def _run_cache(s):
    case = s["case"]
    kind, page = case["kind"], case["page"]
    out_type = torch.float32 if case["source"] == "f32" else torch.bfloat16
    if own:
        pkg, cache = _package(), s["handle"]
        cache.write(s["k_new"], s["v_new"], pkg.KvBatch(s["cu_q"], s["kv_len"], s["table"], s["max_q"], s["max_kv"]))
        return cache.read(pkg.KvBatch(s["cu_read"], s["kv_len"], s["table"], s["max_read"], s["max_kv"]), s["n_read"], out_type)
    pages, offs = _rows(s["cu_q"], s["kv_len"], s["table"], page, s["k_new"].shape[0])
    for name in ("k", "v"):
        x = s[name + "_new"]
        if kind == "bf16":
            s[name][pages, :, offs] = x.to(torch.bfloat16)
            continue
        x = x.float()
        amax = x.abs().amax(-1)
        if kind == "e4m3":  # the smallest power of two under which the row is at most 448 = 1.75 x 2^8
            m, e = torch.frexp(amax)
            scale = torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875)).clamp_min(-126))
            code = (x / scale[..., None]).to(torch.float8_e4m3fn)
        else:  # the quotient in 64 bits: halves between two codes are what they are
            scale = (amax / 127).clamp_min(2.0 ** -126)
            code = torch.round(x.double() / scale[..., None].double()).to(torch.int8)
        s[name][pages, :, offs] = code.view(torch.uint8)
        s[name + "_scale"][pages, :, offs] = scale
    pages, offs = _rows(s["cu_read"], s["kv_len"], s["table"], page, s["n_read"])
    return tuple(_values(kind, s[n][pages, :, offs], None if kind == "bf16" else s[n + "_scale"][pages, :, offs]).to(out_type) for n in ("k", "v"))


def _run_attend(s):
    case = s["case"]
    kind, page, window, sinks, heads, hk, dim = (case[k] for k in ("kind", "page", "window", "sinks", "heads", "kv_heads", "dim"))
    if own:
        batch = _package().KvBatch(s["cu_q"], s["kv_len"], s["table"], s["max_q"], s["max_kv"])
        return s["handle"].attend(s["q"], batch, window=window, sinks=sinks)
    cu, kv_len, table, max_q = s["cu_q"].long(), s["kv_len"].long(), s["table"], s["max_q"]
    seqs, rows = table.shape[0], s["q"].shape[0]
    n_q = cu[1:] - cu[:-1]
    # the key positions that some row of a sequence sees: all, or the first ones and the stretch under the windows
    if window:
        span = min(s["max_kv"], window + max_q - 1)
        low = (kv_len - n_q - window + 1).clamp_min(0)
        tail = low[:, None] + torch.arange(span, device="cuda")
        first = torch.arange(min(sinks, s["max_kv"]), device="cuda")
        key = torch.cat([first.expand(seqs, -1), tail], 1)
        once = torch.cat([torch.ones_like(first, dtype=torch.bool).expand(seqs, -1), tail >= sinks], 1)
    else:
        key = torch.arange(s["max_kv"], device="cuda").expand(seqs, -1)
        once = torch.ones_like(key, dtype=torch.bool)
    pages = torch.gather(table, 1, (key // page).clamp_max(table.shape[1] - 1)).long()
    there = once & (key < kv_len[:, None]) & (pages >= 0)
    pages, offs = pages.clamp_min(0), key % page
    k, v = (_values(kind, s[n][pages, :, offs], None if kind == "bf16" else s[n + "_scale"][pages, :, offs]) for n in ("k", "v"))
    # queries as [seqs, kv_heads, group * max_q, dim], rows behind a sequence's end repeated from the last
    row = cu[:-1, None] + torch.arange(max_q, device="cuda").clamp_max(n_q[:, None] - 1)
    group = heads // hk
    q = s["q"][row].float().view(seqs, max_q, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, hk, group * max_q, dim)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(1.0 / math.sqrt(dim))
    pos = kv_len[:, None] - (cu[1:, None] - row)
    see = there[:, None, :] & (key[:, None, :] <= pos[:, :, None])
    if window:
        see &= (key[:, None, :] > pos[:, :, None] - window) | (key[:, None, :] < sinks)
    score.view(seqs, hk, group, max_q, -1).masked_fill_(~see[:, None, None], LN_NONE)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top).exp_()
    out = torch.matmul(p, v.transpose(1, 2).contiguous()).div_(p.sum(-1, keepdim=True))
    out = out.view(seqs, hk, group, max_q, dim).permute(0, 3, 1, 2, 4).reshape(seqs, max_q, heads, dim)
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu[1:], t, right=True)
    return out[b, t - cu[b]].to(torch.bfloat16)


def _run_sample(s):
    if own:
        return _package().sample_logits(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    x, vocab = s["logits"].double(), s["logits"].shape[1]
    greedy = s["temperature"] <= 0
    x = x / torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    # highest first, equal ones by their index
    val, idx = torch.sort(x, dim=1, descending=True, stable=True)
    w = (val - val[:, :1]).exp()
    rank = torch.arange(vocab, device="cuda")
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"])
    w_k = torch.where(rank < k[:, None], w, 0.0)
    cum = w_k.cumsum(1)
    top_p = s["top_p"].double()[:, None]
    keep = (w_k > 0) & ((cum - w_k < top_p * cum[:, -1:]) | (top_p >= 1)) & (w >= s["min_p"].double()[:, None])
    keep = torch.where(greedy[:, None], rank == 0, keep)
    # the kept ones in the order of their index, and the draw
    w_i = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, 0.0))
    cum = w_i.cumsum(1)
    ids = ((cum < s["u"][:, None] * cum[:, -1:]) | (cum <= 0)).sum(1, keepdim=True).clamp_max(vocab - 1)
    logprob = x.gather(1, ids) - val[:, :1] - w.sum(1, keepdim=True).log()
    return ids[:, 0].int(), logprob[:, 0].float()


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 40 * case["rows"], "flops": 4 * n}
    q, past = _lengths(case)
    hk, dim = case["kv_heads"], case["dim"]
    row = dim * 2 if case["kind"] == "bf16" else dim + 4  # one head's key or value in the cache
    if case["op"] == "cache":
        wide = dim * (4 if case["source"] == "f32" else 2)
        read = sum(a + b for a, b in zip(q, past)) if case["whole"] else sum(q)
        return {"bytes": 2 * hk * (sum(q) * (wide + row) + read * (row + wide)), "flops": 2 * hk * dim * (2 * sum(q) + read)}
    seen = pairs = 0
    for n, p in zip(q, past):
        w, s = case["window"] or n + p, case["sinks"]
        low = max(0, p - w + 1)
        seen += n + p - low + min(s, low)
        pos = np.arange(p, p + n, dtype=np.int64)
        pairs += int((np.minimum(pos + 1, w) + np.minimum(np.maximum(pos + 1 - w, 0), s)).sum())
    return {"bytes": 2 * hk * row * seen + 4 * dim * case["heads"] * sum(q), "flops": 4 * dim * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _held(s, name, b, key):
    """f64 values [len(key), kv_heads, dim] of the cached keys or values of sequence b at positions `key`."""
    case = s["case"]
    at = s["table"][b].long()[key // case["page"]]
    codes = s[name][at, :, key % case["page"]]
    if case["kind"] == "bf16":
        return codes.double()
    codes = codes.view(torch.float8_e4m3fn).float().double() if case["kind"] == "e4m3" else codes.view(torch.int8).double()
    return codes * s[name + "_scale"][at, :, key % case["page"]].double().unsqueeze(-1)


def _quantised(kind, x):
    """The f64 values that rows x [n, heads, dim] (f64) have once they were held in the cache."""
    if kind == "bf16":
        return x.float().to(torch.bfloat16).double()
    if kind == "int8":
        step = torch.clamp((x.abs().amax(-1, keepdim=True) / 127).float(), min=2.0 ** -126).double()
        return torch.round(x / step) * step
    most = x.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(most.clamp_min(1e-300))) - 8)
    step = torch.where(most > 448 * step, 2 * step, step).clamp_min(2.0 ** -126)
    y = x / step
    grain = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # the distance of e4m3's values around y
    return torch.round(y / grain) * grain * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    q, past = _lengths(case)
    if case["op"] == "cache":
        start = np.concatenate([[0], np.cumsum(q)])
        outs = []
        for name in ("k", "v"):
            parts = []
            for b, n in enumerate(q):
                new = _quantised(case["kind"], s[name + "_new"][start[b]:start[b + 1]].double())
                old = _held(s, name, b, torch.arange(past[b] if case["whole"] else 0, device="cuda"))
                parts.append(torch.cat([old, new]))
            outs.append(torch.cat(parts))
        return tuple(outs)
    heads, hk, dim, window, sinks = (case[k] for k in ("heads", "kv_heads", "dim", "window", "sinks"))
    out = torch.empty(sum(q), heads, dim, dtype=torch.float64, device="cuda")
    row = 0
    for b, n in enumerate(q):
        i = torch.arange(past[b], past[b] + n, device="cuda")
        low = max(0, past[b] - window + 1) if window else 0
        j = torch.arange(past[b] + n, device="cuda")
        j = j[(j >= low) | (j < sinks)]
        hidden = j[None, :] > i[:, None]
        if window:
            hidden |= (j[None, :] <= i[:, None] - window) & (j[None, :] >= sinks)
        k, v = _held(s, "k", b, j), _held(s, "v", b, j)
        for h in range(heads):
            a = s["q"][row:row + n, h].double() @ k[:, h // (heads // hk)].t() / math.sqrt(dim)
            a = torch.softmax(a.masked_fill(hidden, LN_NONE), dim=1)
            out[row:row + n, h] = a @ v[:, h // (heads // hk)]
        row += n
    return out


def _exact_sample(s):
    """Row by row on the host."""
    logits = s["logits"].float().cpu().numpy().astype(np.float64)
    u = s["u"].cpu().numpy()
    temperature, top_k, top_p, min_p = (s[k].cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p"))
    ids, logprobs = [], []
    for r, l in enumerate(logits):
        greedy = temperature[r] <= 0
        x = l if greedy else l / np.float64(temperature[r])
        p = np.exp(x - x.max())
        if greedy:
            pick = int(np.argmax(l))
        else:
            order = np.argsort(-x, kind="stable")
            order = order[: top_k[r]] if 0 < top_k[r] < len(order) else order
            if top_p[r] < 1:
                mass = np.cumsum(p[order])
                order = order[: int(np.searchsorted(mass, np.float64(top_p[r]) * mass[-1])) + 1]
            order = np.sort(order[p[order] >= np.float64(min_p[r])])
            mass = np.cumsum(p[order])
            pick = int(order[min(int(np.searchsorted(mass, u[r] * mass[-1])), len(order) - 1)])
        ids.append(pick)
        logprobs.append(x[pick] - x.max() - math.log(p.sum()))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64)
