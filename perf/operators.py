"""The operators of the 8-bit cache: keys and values stored as 8-bit codes with a scale per token and head, read back as
values, and attended to by decoding rows and by chunks of new tokens.

A row x of ``width`` numbers (one token's key or value of one head) is held as
    scale = max(max |x| / 127, 2^-120), a 32-bit number,   code = the whole number nearest to x / scale (ties to even),
and stands for code * scale.  Pages are ``[pages, heads, page_size, width]`` (codes) and ``[pages, heads, page_size]`` (scales); a
block table says which page holds which positions of a request.  The query of a request at position p sees the keys up to p
(with a window w the last w of them); its result is softmax(q . k * hd^-0.5) v over them, a sink (a number per head) joining
the denominator where there is one.

Sizes are those of the models of the engine's benchmark and tests: 16 heads of 128 (a GPT of 1.3 B), 25 heads of 64 (GPT-2 XL's),
8 heads of 32 (the reference server's), 16 heads over 4 key/value heads of 128 (a grouped model of width 2,048).
"""
import math

import torch

own = False

FLOOR = 2.0 ** -120
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ------------------------------------------------------------------------------------------------------
def case(name, kind, dtype, heads, kv_heads, width, page, requests, low, high, new=0, new_high=0, window=0, sinks=False):
    """``requests`` requests that hold ``low``..``high`` tokens; ``new``..``new_high`` of them are this step's (kinds "write" and
    "chunk"; at decoding the last one is)."""
    return {"name": name, "kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "width": width, "page": page,
            "requests": requests, "low": low, "high": high, "new": new, "new_high": max(new, new_high), "window": window,
            "sinks": sinks}


def listed():
    return [
        # the smallest store: a decode step's eight tokens
        case("write 8 tokens", "write", "bfloat16", 16, 16, 128, 16, 8, 1024, 1999, 1),
        # a whole prompt stored in one step
        case("write 2048 tokens", "write", "bfloat16", 16, 16, 128, 16, 1, 2048, 2048, 2048),
        # the contexts of a busy server read back, contexts as they come
        case("read 23 requests", "read", "bfloat16", 25, 25, 64, 16, 23, 90, 1100),
        # a long context in 32-bit
        case("read 32767 f32", "read", "float32", 8, 8, 32, 16, 1, 32767, 32767),
        # one user's chat: latency
        case("decode 1", "decode", "bfloat16", 16, 16, 128, 16, 1, 1100, 1100),
        # a busy server
        case("decode 64", "decode", "bfloat16", 16, 16, 128, 16, 64, 120, 1400),
        # a few users with long documents, query heads that share keys
        case("decode grouped long", "decode", "bfloat16", 16, 4, 128, 16, 5, 7000, 30011),
        # the reference server's slots in 32-bit
        case("decode 16 f32", "decode", "float32", 8, 8, 32, 16, 16, 300, 2000),
        # drafted tokens of several requests checked in one step, an odd number of heads
        case("chunk of few rows", "chunk", "bfloat16", 25, 25, 64, 16, 12, 100, 1000, 2, 7),
        # prompt portions with a sliding window and a sink, query heads that share keys
        case("chunk window sinks", "chunk", "bfloat16", 16, 4, 128, 32, 3, 1500, 5000, 60, 190, 1024, True),
        # a portion of a long prompt
        case("chunk 512 behind 8192", "chunk", "bfloat16", 16, 16, 128, 16, 1, 8704, 8704, 512),
        # the reference's long prompt in 32-bit
        case("chunk 512 f32", "chunk", "float32", 8, 8, 32, 16, 1, 4608, 4608, 512),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    group = rng.choice([1, 1, 2, 4, 8])
    kv_heads = rng.choice([1, 2, 3, 4, 8]) if group > 1 else rng.choice([1, 2, 5, 8, 16, 25])
    width = rng.choice([24, 32, 64, 80, 128]) if kind in ("write", "read") else rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([8, 16, 16, 32, 64])
    new = new_high = window = 0
    sinks = False
    if kind == "write":
        requests = _log_uniform(rng, 1, 40)
        new = _log_uniform(rng, 1, 2000 // requests)
        new_high = min(2 * new, 2000 // requests)
        low = new_high + _log_uniform(rng, 1, 1000)
        high = low + _log_uniform(rng, 1, 1000)
    elif kind == "read":
        requests = _log_uniform(rng, 1, 32)
        high = _log_uniform(rng, 16, 32000 // requests)
        low = max(1, rng.randrange(high // 4, high + 1))
    else:
        window = rng.choice([0, 0, 0, _log_uniform(rng, 16, 1500)])
        sinks = rng.random() < 0.25
        requests = _log_uniform(rng, 1, 48) if kind == "decode" else _log_uniform(rng, 1, 10)
        high = _log_uniform(rng, 8, 48000 // requests if kind == "decode" else 8000 // requests)
        low = max(1, rng.randrange(high // 8, high + 1))
        if kind == "chunk":
            new = _log_uniform(rng, 2, 256)
            new_high = min(2 * new, 300)
            low, high = low + new_high, high + new_high
    return {k: v for k, v in case("", kind, dtype, group * kv_heads, kv_heads, width, page, requests, low, high, new, new_high,
                                  window, sinks).items() if k != "name"}


def _spread(low, high, n, turn):
    """n whole numbers over low..high, the same for a case whatever the seed."""
    return [low + int((high - low + 1) * ((i + 1) * turn % 1.0)) for i in range(n)]


def _lengths(c):
    """(tokens held, tokens of this step) of every request."""
    total = _spread(c["low"], c["high"], c["requests"], 0.6180339887498949)
    if c["kind"] == "decode":
        return total, [1] * len(total)
    if c["kind"] == "read":
        return total, list(total)
    return total, _spread(c["new"], c["new_high"], c["requests"], 0.7548776662466927)


def work(c):
    total, new = _lengths(c)
    size, G, W = TYPES[c["dtype"]].itemsize, c["kv_heads"], c["width"]
    held = 2 * G * (W + 4)                        # one token's codes and scales
    if c["kind"] == "write":                      # rows in; codes, scales and the values they stand for out
        return {"bytes": sum(new) * (2 * G * W * 2 * size + held), "flops": sum(new) * 2 * G * W * 4}
    if c["kind"] == "read":
        return {"bytes": sum(total) * (held + 2 * G * W * size), "flops": sum(total) * 2 * G * W}
    pairs = seen = 0
    for t, n in zip(total, new):
        w = c["window"] or t
        pairs += sum(min(w, p + 1) for p in range(t - n, t))
        seen += min(t, w + n - 1)
    return {"bytes": seen * held + sum(new) * 2 * c["heads"] * W * size, "flops": 4 * pairs * c["heads"] * W}


# ---- what a program has in hand before the call ---------------------------------------------------------------------
def _cache(c, pages, g):
    """Codes and scales of normal rows whose channels differ in size, as keys' and values' do."""
    size = torch.exp(0.5 * torch.randn(c["kv_heads"], 1, c["width"], device="cuda", generator=g))
    rows = torch.randn(pages, c["kv_heads"], c["page"], c["width"], device="cuda", generator=g).mul_(size)
    scales = (rows.abs().amax(-1).double() / 127).clamp_min(FLOOR).float()
    return torch.round(rows / scales[..., None]).clamp_(-127, 127).to(torch.int8), scales


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, (total, new) = TYPES[c["dtype"]], _lengths(c)
    need = [-(-t // c["page"]) for t in total]
    most = max(need)
    order = torch.randperm(sum(need) + 3, device="cuda", generator=g).to(torch.int32)      # pages lie anywhere; a few are free
    table = torch.full((len(total), most), -1, dtype=torch.int32, device="cuda")
    count = torch.tensor(need, device="cuda")
    slot = torch.arange(most, device="cuda")[None] < count[:, None]
    table[slot] = order[:sum(need)]
    s = {"case": c, "table": table, "most": max(total), "rows": sum(new), "new_most": max(new)}
    s["total"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    s["start"] = torch.tensor([t - n for t, n in zip(total, new)], dtype=torch.int32, device="cuda")
    s["cu_rows"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda")
    n = torch.tensor(new, device="cuda")
    s["row_seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), n).to(torch.int32)
    s["positions"] = (torch.arange(sum(new), device="cuda") - s["cu_rows"][s["row_seq"].long()] + s["start"][s["row_seq"].long()]).to(torch.int32)
    s["k_codes"], s["k_scales"] = _cache(c, len(order), g)
    s["v_codes"], s["v_scales"] = _cache(c, len(order), g)
    if c["kind"] in ("write", "read"):
        s["k_out"] = torch.zeros(s["k_codes"].shape, dtype=dtype, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    if c["kind"] == "write":
        p, q = s["positions"].long(), s["row_seq"].long()
        s["slots"] = (table[q, p // c["page"]] * c["page"] + p % c["page"]).to(torch.int32)
        wide = c["kv_heads"] * c["width"]
        size = torch.exp(0.5 * torch.randn(2 * wide, device="cuda", generator=g))
        s["kv"] = (torch.randn(sum(new), 2 * wide, device="cuda", generator=g) * size).to(dtype)
    if c["kind"] in ("decode", "chunk"):
        s["q"] = torch.randn(sum(new), c["heads"] * c["width"], device="cuda", generator=g).to(dtype)
        s["sinks"] = torch.randn(c["heads"], device="cuda", generator=g) if c["sinks"] else None
        s["out"] = torch.zeros_like(s["q"])
    return s


# ---- the operators --------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["kind"] == "write":
        wide = c["kv_heads"] * c["width"]
        _store(s["kv"][:, :wide], s["k_codes"], s["k_scales"], s["slots"])
        _store(s["kv"][:, wide:], s["v_codes"], s["v_scales"], s["slots"])
    if c["kind"] in ("write", "read"):
        place = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
        held = place < s["total"][:, None]
        if c["kind"] == "write":
            held = held & (place >= s["start"][:, None])
        request, place = torch.nonzero(held, as_tuple=True)
        page, slot = s["table"][request, place // c["page"]].long(), place % c["page"]
        for at in "kv":
            values = s[at + "_codes"][page, :, slot].float() * s[at + "_scales"][page, :, slot][..., None]
            s[at + "_out"][page, :, slot] = values.to(s[at + "_out"].dtype)
        return (s["k_out"], s["v_out"], s["k_scales"], s["v_scales"]) if c["kind"] == "write" else (s["k_out"], s["v_out"])
    return _attend(s)


def _store(rows, codes, scales, slots):
    """Rows as codes and scales into their slots; the quotients in 64 bits, since half steps are common among 16-bit values."""
    pages, heads, page, width = codes.shape
    x = rows.reshape(-1, heads, width).double()
    scale = (x.abs().amax(-1) / 127).clamp_min(FLOOR).float()
    code = torch.round(x / scale.double()[..., None]).clamp(-127, 127).to(torch.int8)
    slots = slots.long()
    codes[slots // page, :, slots % page] = code
    scales[slots // page, :, slots % page] = scale


def _attend(s):
    c = s["case"]
    G, W, S = c["kv_heads"], c["width"], len(s["total"])
    M = c["heads"] // G
    at = torch.arange(s["most"], device="cuda")
    page, slot = s["table"][:, at // c["page"]].clamp_min(0).long(), (at % c["page"]).expand(S, -1)
    k = s["k_codes"][page, :, slot].float() * s["k_scales"][page, :, slot][..., None]      # [S, keys, G, W]
    v = s["v_codes"][page, :, slot].float() * s["v_scales"][page, :, slot][..., None]
    i = torch.arange(s["new_most"], device="cuda")
    row = (s["cu_rows"][:S, None] + i).clamp_max(s["rows"] - 1).long()
    live = i < (s["total"] - s["start"])[:, None]
    p = s["start"][:, None] + i
    q = s["q"][row].float().view(S, len(i), G, M, W).permute(0, 2, 3, 1, 4).reshape(S, G, M * len(i), W)
    scores = (q @ k.permute(0, 2, 3, 1)).view(S, G, M, len(i), -1) * W ** -0.5
    seen = at <= p[..., None]
    if c["window"]:
        seen = seen & (at > p[..., None] - c["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = s["sinks"].view(1, G, M, 1, 1)
        top = torch.maximum(top, sink)
    e = torch.exp(scores - top)
    norm = e.sum(-1, keepdim=True)
    if c["sinks"]:
        norm = norm + torch.exp(sink - top)
    out = ((e / norm).view(S, G, M * len(i), -1) @ v.permute(0, 2, 1, 3)).view(S, G, M, len(i), W)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, len(i), -1)
    s["out"][row[live]] = out[live].to(s["out"].dtype)
    return s["out"]


def _run_own(s):
    from cbis_b200.kernels import ops
    c = s["case"]
    H, G, W, page = c["heads"], c["kv_heads"], c["width"], c["page"]
    k, v = ops.Q8Pages(s["k_codes"], s["k_scales"]), ops.Q8Pages(s["v_codes"], s["v_scales"])
    if c["kind"] == "write":
        ops.kv_write_q8(s["kv"], 0, G * W, k, v, s["slots"], G, W, page)
        # with a window of one key the first token read is the first of this step
        ops.kv_read_q8(k, v, s["k_out"], s["v_out"], s["table"], s["start"], s["total"], s["new_most"], window=1)
        return s["k_out"], s["v_out"], s["k_scales"], s["v_scales"]
    if c["kind"] == "read":
        ops.kv_read_q8(k, v, s["k_out"], s["v_out"], s["table"], s["start"], s["total"], s["most"])
        return s["k_out"], s["v_out"]
    if "scratch" not in s:       # an engine keeps these, and the pages that a long chunk's keys and values are read back into
        floats, counters = ops.attention_q8_scratch(s["rows"], s["new_most"], len(s["total"]), H, G, W, s["most"], s["q"].dtype)
        s["scratch"] = torch.empty(floats, dtype=torch.float32, device="cuda")
        s["counters"] = torch.zeros(counters, dtype=torch.int32, device="cuda")
        if c["kind"] == "chunk":
            s["work"] = tuple(torch.empty(s["k_codes"].shape, dtype=s["q"].dtype, device="cuda") for _ in "kv")
    if c["kind"] == "decode":
        ops.paged_decode_q8(s["q"], -1, -1, k, v, s["table"], s["row_seq"], s["positions"], None, s["out"], s["scratch"],
                            s["counters"], H, G, W, page, W ** -0.5, c["window"], s["most"], sinks=s["sinks"])
    else:
        ops.paged_prefill_q8(s["q"], k, v, s["table"], s["cu_rows"], s["start"], s["total"], s["positions"], s["out"], 0,
                             len(s["total"]), 0, s["rows"], s["new_most"], H, G, W, page, W ** -0.5, c["window"], s["most"],
                             s["scratch"], s["counters"], s["work"], sinks=s["sinks"])
    return s["out"]


# ---- the definition in 64 bits, request by request ------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    G, W, M = c["kv_heads"], c["width"], c["heads"] // c["kv_heads"]
    total, new = _lengths(c)
    table = s["table"].tolist()
    if c["kind"] in ("write", "read"):
        outs = [s["k_out"].double(), s["v_out"].double()]
        held = [[s["k_codes"].double(), s["k_scales"].double()], [s["v_codes"].double(), s["v_scales"].double()]]
        if c["kind"] == "write":
            kv = s["kv"].double().view(-1, 2, G, W)
            largest = kv.abs().max(dim=3).values
            scale = torch.maximum(largest / 127.0, torch.full_like(largest, FLOOR)).to(torch.float32).double()
            code = torch.round(kv / scale.unsqueeze(3))
        row = 0
        for r, (t, n) in enumerate(zip(total, new)):
            first = t - n if c["kind"] == "write" else 0
            for at in range(first - first % c["page"], t, c["page"]):
                a, b, number = max(first, at), min(t, at + c["page"]), table[r][at // c["page"]]
                for x in range(2):
                    codes, scales = held[x][0][number, :, a - at:b - at], held[x][1][number, :, a - at:b - at]
                    if c["kind"] == "write":
                        codes.copy_(code[row + a - first:row + b - first, x].transpose(0, 1))
                        scales.copy_(scale[row + a - first:row + b - first, x].transpose(0, 1))
                    outs[x][number, :, a - at:b - at] = codes * scales.unsqueeze(2)
            row += n
        return (outs[0], outs[1], held[0][1], held[1][1]) if c["kind"] == "write" else (outs[0], outs[1])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for r, (t, n) in enumerate(zip(total, new)):
        pages = torch.tensor(table[r][:-(-t // c["page"])], device="cuda")
        key, value = ((codes[pages].double() * scales[pages].double().unsqueeze(3)).transpose(1, 2).reshape(-1, G, W)[:t]
                      for codes, scales in ((s["k_codes"], s["k_scales"]), (s["v_codes"], s["v_scales"])))
        back = torch.arange(t - n, t, device="cuda").view(-1, 1) - torch.arange(t, device="cuda").view(1, -1)
        hidden = (back < 0) | (back >= (c["window"] or t + 1))
        for h in range(c["heads"]):
            query = s["q"][row:row + n, h * W:(h + 1) * W].double()
            logits = torch.einsum("nw,tw->nt", query, key[:, h // M]) / math.sqrt(W)
            logits[hidden] = -math.inf
            if c["sinks"]:
                logits = torch.cat([logits, s["sinks"][h].double().expand(n, 1)], dim=1)
            weights = torch.softmax(logits, dim=1)[:, :t]
            out[row:row + n, h * W:(h + 1) * W] = torch.einsum("nt,tw->nw", weights, value[:, h // M])
        row += n
    return out
