"""The operators of a bounded key-value cache, as cases that can be measured: attention with a sliding window and sink
tokens, attention that accumulates the weight every cached position receives, and the eviction that goes by it.

`run` computes a case in its plain form (elementary torch operations) where `own` is false, and through AttnEngine where
it is true.  A case is a dict of plain values:

    op      "sinks" | "track" | "evict"
    heads   "b": 32 query / 8 kv heads of 128, window 4096;  "r": 16 / 4 heads of 256, window 1024
    store   "ring" (window layer, ring of 2 windows + sink buffers), "slots" (one partition per sequence), "paged"
    n_seq   sequences; rows: query rows of each; ctx: positions cached before those rows, by the longest sequence
    spread  sequence i holds ctx - (i * 7919) % spread positions, at least one for an eviction
    n_sink, budget, n_recent   as the calls take them
"""
import math

import torch

own = False

DEV = "cuda"
HEADS = {"b": (32, 8, 128, 4096), "r": (16, 4, 256, 1024)}        # query heads, kv heads, head_dim, window
PAGE = 256
SINK_TILE = 128                                                    # sink buffers hold whole tiles of positions


def listed():
    return [
        # one user chatting far past the window: the smallest call, where launch latency counts
        {"name": "sinks_decode_1", "op": "sinks", "heads": "b", "store": "ring", "n_seq": 1, "rows": 1, "ctx": 20000,
         "spread": 1, "n_sink": 4},
        # a full batch of ragged streams, some of them still shorter than the window
        {"name": "sinks_decode_64", "op": "sinks", "heads": "b", "store": "ring", "n_seq": 64, "rows": 1, "ctx": 32768,
         "spread": 31000, "n_sink": 4},
        # eight speculative rounds at once over a paged cache whose middle pages need not be resident
        {"name": "sinks_verify_8x8", "op": "sinks", "heads": "b", "store": "paged", "n_seq": 8, "rows": 8, "ctx": 12003,
         "spread": 9000, "n_sink": 16},
        # a prompt chunk of the usual length deep in a stream
        {"name": "sinks_prompt_512", "op": "sinks", "heads": "b", "store": "ring", "n_seq": 1, "rows": 512, "ctx": 16384,
         "spread": 1, "n_sink": 4},
        # a ragged last chunk in the wide-head geometry, the sinks read in place
        {"name": "sinks_prompt_r_201", "op": "sinks", "heads": "r", "store": "slots", "n_seq": 1, "rows": 201, "ctx": 4999,
         "spread": 1, "n_sink": 64},
        # one conversation decoding inside its budget
        {"name": "track_decode_1", "op": "track", "heads": "b", "store": "slots", "n_seq": 1, "rows": 1, "ctx": 4095,
         "spread": 1},
        # a serving batch of ragged conversations on pages
        {"name": "track_decode_48", "op": "track", "heads": "b", "store": "paged", "n_seq": 48, "rows": 1, "ctx": 32700,
         "spread": 32000},
        # the last rows of a prompt choose what is kept of it
        {"name": "track_prompt_r_32", "op": "track", "heads": "r", "store": "slots", "n_seq": 1, "rows": 32, "ctx": 16352,
         "spread": 1},
        # every chunk of a long prompt counts: the largest call
        {"name": "track_prompt_512", "op": "track", "heads": "b", "store": "slots", "n_seq": 1, "rows": 512, "ctx": 32256,
         "spread": 1},
        # the regular trim of one conversation that ran 64 tokens over
        {"name": "evict_step_r", "op": "evict", "heads": "r", "store": "slots", "n_seq": 1, "ctx": 4160, "spread": 1,
         "budget": 4096, "n_sink": 4, "n_recent": 512},
        # a batch cut to a quarter
        {"name": "evict_32", "op": "evict", "heads": "b", "store": "slots", "n_seq": 32, "ctx": 8192, "spread": 6500,
         "budget": 2048, "n_sink": 4, "n_recent": 256},
        # a long prompt reduced once, after it was read
        {"name": "evict_prompt_128k", "op": "evict", "heads": "b", "store": "paged", "n_seq": 1, "ctx": 131072, "spread": 1,
         "budget": 8192, "n_sink": 16, "n_recent": 1000},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sinks", "sinks", "track", "track", "evict"])
    c = {"op": op, "heads": rng.choice(["b", "r"])}
    if op == "sinks":
        c["store"] = rng.choice(["ring", "slots", "paged"])
        kind = rng.choice(["decode", "verify", "prompt"])
        c["rows"] = {"decode": 1, "verify": rng.randint(2, 8), "prompt": _log(rng, 9, 512)}[kind]
        c["n_seq"] = 1 if kind == "prompt" else _log(rng, 1, 64 if kind == "decode" else 16)
        c["ctx"] = _log(rng, 1, 32768 if c["store"] == "ring" else max(64, min(32768, 700000 // c["n_seq"])))
        c["n_sink"] = rng.choice([0, 1, 4, 4, rng.randint(2, 64), 128])
    elif op == "track":
        c["store"] = rng.choice(["slots", "paged"])
        c["rows"] = 1 if rng.random() < 0.6 else _log(rng, 2, 512)
        c["n_seq"] = _log(rng, 1, 48) if c["rows"] == 1 else 1
        c["ctx"] = _log(rng, 1, min(32000, 700000 // c["n_seq"]))
    else:
        c["store"] = rng.choice(["slots", "paged"])
        c["n_seq"] = _log(rng, 1, 32)
        c["ctx"] = _log(rng, 2, 260000 // c["n_seq"])
        c["budget"] = _log(rng, 1, c["ctx"])
        c["n_sink"] = min(rng.choice([0, 4, 16]), c["budget"])
        c["n_recent"] = rng.randint(0, (c["budget"] - c["n_sink"]) // 2)
    c["spread"] = rng.randint(1, c["ctx"])
    return c


# ---- shapes -------------------------------------------------------------------------------------------------------------

def _lens(c):
    return [max(1 if c["op"] == "evict" else 0, c["ctx"] - (i * 7919) % c["spread"]) for i in range(c["n_seq"])]


def _rec(hd):
    return hd + hd // 16


def _capacity(c):
    n = c["ctx"] + c.get("rows", 0)
    return n + (-n) % PAGE


def _seen(c, p, r):
    """How many positions row r of a sequence with p cached positions before its rows sees."""
    if c["op"] == "track":
        return p + r + 1
    lo = max(0, p + r + 1 - HEADS[c["heads"]][3])
    return p + r + 1 - lo + min(c["n_sink"], lo)


def work(c):
    hq, hkv, hd, win = HEADS[c["heads"]]
    rec, lens = _rec(hd), _lens(c)
    if c["op"] == "evict":
        total, kept, moved = sum(lens), sum(min(n, c["budget"]) for n in lens), 0
        for n in lens:
            moved += min(n, c["budget"])
        # every score once, the list of what stays, and the records and scores that stay, read and written
        return {"bytes": hkv * (4 * total + 4 * kept + 4 * kept + 4 * moved * rec), "flops": 0}
    rows, flops, cached = c["rows"], 0, 0
    for p in lens:
        if c["op"] == "sinks":
            lo = max(0, p + 1 - win)
            cached += p + rows - lo + min(c["n_sink"], lo)
        else:
            cached += p + rows
        flops += (4 if c["op"] == "sinks" or rows == 1 else 6) * hq * hd * sum(_seen(c, p, r) for r in range(rows))
    nbytes = 2 * cached * hkv * rec + 2 * 2 * c["n_seq"] * rows * hq * hd
    if c["op"] == "track":
        nbytes += 8 * cached * hkv                      # the sums, read and written
    return {"bytes": nbytes, "flops": flops}


# ---- inputs -------------------------------------------------------------------------------------------------------------

def _quantise(x):
    """q8_0 records of fp32 vectors [..., hd]: hd/32 fp16 scales, then hd int8 values."""
    *lead, hd = x.shape
    b = x.reshape(*lead, hd // 32, 32)
    d = b.abs().amax(-1) / 127.0
    q = torch.round(b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))[..., None]).clamp(-127, 127).to(torch.int8)
    return torch.cat([d.to(torch.float16).view(torch.uint8).reshape(*lead, hd // 16),
                      q.reshape(*lead, hd).view(torch.uint8)], -1)


def _records(gen, n, hd):
    out = torch.empty(n, _rec(hd), dtype=torch.uint8, device=DEV)
    step = 1 << 19
    for a in range(0, n, step):
        m = min(step, n - a)
        out[a:a + m] = _quantise(torch.randn(m, hd, generator=gen, device=DEV))
    return out


def _inputs(c, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    hq, hkv, hd, win = HEADS[c["heads"]]
    n_seq, cap, lens = c["n_seq"], _capacity(c), _lens(c)
    s = {"case": c, "lens": lens, "cap": cap, "pos": torch.tensor(lens, dtype=torch.int32, device=DEV)}
    parts = 2 * n_seq if c["op"] == "evict" else n_seq             # an eviction writes into partitions of its own
    if c["store"] == "ring":
        s["shape"] = (n_seq, hkv, 2 * win, _rec(hd))
    elif c["store"] == "slots":
        s["shape"] = (parts, hkv, cap, _rec(hd))
    else:
        per = cap // PAGE
        need = [(n + c.get("rows", 0) + PAGE - 1) // PAGE for n in lens]
        if c["op"] == "evict":
            need += [(min(n, c["budget"]) + PAGE - 1) // PAGE for n in lens]
        order = torch.randperm(sum(need), generator=gen, device=DEV).to(torch.int32)
        s["table"] = torch.full((parts, per), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, m in enumerate(need):
            s["table"][i, :m] = order[at:at + m]
            at += m
        s["shape"] = (sum(need), hkv, PAGE, _rec(hd))
    n_rec = s["shape"][0] * s["shape"][1] * s["shape"][2]
    for name in ("k", "v"):
        if c["op"] == "evict":
            r = torch.randint(0, 256, (n_rec, _rec(hd)), generator=gen, device=DEV, dtype=torch.uint8)
        else:
            r = _records(gen, n_rec, hd)
        s[name] = r.reshape(s["shape"])
    if c["op"] == "evict":
        # what accumulated weights look like: a heavy tail, many positions near nothing, some that never got any
        u = torch.rand(parts, hkv, cap, generator=gen, device=DEV)
        s["score"] = torch.where(u < 0.05, torch.zeros_like(u), u ** 8)
        s["kept"] = torch.full((n_seq, hkv, c["budget"]), -7, dtype=torch.int32, device=DEV)
        s["pos_out"] = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
        s["src"] = torch.arange(n_seq, dtype=torch.int32, device=DEV)
        s["dst"] = s["src"] + n_seq
        return s
    # queries and the first cached keys lean the same way: the first tokens draw much of the attention
    lean = torch.randn(hkv, hd, generator=gen, device=DEV)
    q = torch.randn(n_seq, c["rows"], hkv, hq // hkv, hd, generator=gen, device=DEV) * 1.5 + 0.2 * lean[:, None]
    s["q"] = q.reshape(n_seq, c["rows"], hq, hd).to(torch.float16)
    s["out"] = torch.zeros(n_seq, c["rows"], hq, hd, dtype=torch.float16, device=DEV)
    first = _quantise(torch.randn(n_seq, hkv, 4, hd, generator=gen, device=DEV) + lean[:, None])
    if c["op"] == "sinks" and c["store"] == "ring":
        room = max(SINK_TILE, c["n_sink"] + (-c["n_sink"]) % SINK_TILE)
        for name in ("sink_k", "sink_v"):
            s[name] = _records(gen, n_seq * hkv * room, hd).reshape(n_seq, hkv, room, _rec(hd))
        s["sink_k"][:, :, :4] = first
        for i, p in enumerate(lens):
            if p + c["rows"] <= 2 * win:                            # the ring still holds the first positions itself
                m = min(room, 2 * win)
                s["k"][i, :, :m] = s["sink_k"][i, :, :m]
                s["v"][i, :, :m] = s["sink_v"][i, :, :m]
    elif c["store"] == "paged":
        for i in range(n_seq):
            s["k"][s["table"][i, 0].long(), :, :4] = first[i]
    else:
        s["k"][:n_seq, :, :4] = first
    if c["op"] == "track":
        u = torch.rand(n_seq, hkv, cap, generator=gen, device=DEV)
        held = torch.arange(cap, device=DEV)[None, None] < s["pos"][:, None, None]
        s["score"] = torch.where(held, 4 * u ** 8, torch.zeros_like(u))
        s["score_out"] = torch.zeros_like(u)
    return s


def prepare(c, seed):
    s = _inputs(c, seed)
    if not own:
        return s
    from bruce_engine_b200 import capi
    from bruce_engine_b200.engine import AttnEngine
    from bruce_engine_b200.layout import G_B, G_R, F16
    g = {"b": G_B, "r": G_R}[c["heads"]].with_(q_dtype=F16, out_dtype=F16, slot_ctx=s["cap"],
                                               n_slots=2 * c["n_seq"] if c["op"] == "evict" else c["n_seq"])
    e = s["eng"] = AttnEngine(g, torch.cuda.current_device())
    s["ids"] = torch.arange(c["n_seq"], dtype=torch.int32, device=DEV)
    if c["store"] == "paged":
        s["pages"] = capi.CPages(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["shape"][0],
                                 s["table"].shape[0], s["table"].shape[1], PAGE)
    if c["op"] == "evict":
        s["part"] = e.alloc_evict_part(c["n_seq"])
    elif c["op"] == "track":
        s["part"] = e.alloc_track_part(c["n_seq"], c["rows"], sum(s["lens"]) + c["n_seq"] * c["rows"])
    else:
        s["part"] = e.alloc_part(c["n_seq"], c["rows"])
        s["sinks"] = e.sinks(c["n_sink"], s.get("sink_k"), s.get("sink_v"))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    c, e = s["case"], s["eng"]
    if c["op"] == "sinks":
        if c["store"] == "paged":
            e.attn_sinks_paged(s["out"], s["q"], s["pages"], s["sinks"], s["pos"], s["part"], rows=c["rows"], ktab=s["ids"])
        else:
            e.attn_sinks(s["out"], s["q"], s["k"], s["v"], s["sinks"], s["pos"], s["part"], rows=c["rows"],
                         kslot=s["ids"], is_swa=c["store"] == "ring")
        return s["out"]
    if c["op"] == "track":
        if c["store"] == "paged":
            e.attn_track_paged(s["out"], s["score_out"], s["score"], s["q"], s["pages"], s["pos"], s["part"],
                               rows=c["rows"], ktab=s["ids"])
        else:
            e.attn_track(s["out"], s["score_out"], s["score"], s["q"], s["k"], s["v"], s["pos"], s["part"],
                         rows=c["rows"], kslot=s["ids"])
        return {"out": s["out"], "score": s["score_out"]}
    if c["store"] == "paged":
        e.evict_paged(s["pages"], s["score"], s["kept"], s["pos_out"], s["pos"], s["part"], c["budget"],
                      n_sink=c["n_sink"], n_recent=c["n_recent"], ktab=s["src"], ktab_dst=s["dst"])
    else:
        e.evict(s["k"], s["v"], s["score"], s["kept"], s["pos_out"], s["pos"], s["part"], c["budget"],
                n_sink=c["n_sink"], n_recent=c["n_recent"], kslot=s["src"], kslot_dst=s["dst"])
    return _evicted(s)


def _evicted(s):
    """What an eviction wrote: the lists, the counts, and the partitions (or pages) it filled."""
    c, n, b = s["case"], s["case"]["n_seq"], s["case"]["budget"]
    r = {"kept": s["kept"], "pos": s["pos_out"], "score": s["score"][n:, :, :b]}
    if c["store"] == "paged":
        r.update(k=s["k"], v=s["v"])
    else:
        r.update(k=s["k"][n:, :, :b], v=s["v"][n:, :, :b])
    return r


def _values(rec, hd):
    nb = hd // 32
    d = rec[..., :2 * nb].contiguous().view(torch.float16).to(torch.float32)
    x = rec[..., 2 * nb:].contiguous().view(torch.int8).to(torch.float32)
    return (x.reshape(*x.shape[:-1], nb, 32) * d[..., None]).reshape(x.shape)


def _cached(s, i, idx, name):
    """Records [kv head][len(idx)][record] of positions idx of sequence i."""
    c = s["case"]
    if c["store"] == "slots":
        return s[name][i][:, idx]
    if c["store"] == "paged":
        return s[name][s["table"][i].long()[idx // PAGE], :, idx % PAGE].transpose(0, 1)
    ring = s[name][i][:, idx % s["shape"][2]]
    keep = s["sink_" + name]
    room = keep.shape[2]
    return torch.where((idx < room)[None, :, None], keep[i][:, idx.clamp(max=room - 1)], ring)


def _plain(s):
    c = s["case"]
    hq, hkv, hd, win = HEADS[c["heads"]]
    if c["op"] == "evict":
        return _plain_evict(s)
    g, rows, out = hq // hkv, c["rows"], torch.empty_like(s["q"])
    score = s["score_out"].clone() if c["op"] == "track" else None
    for i, p in enumerate(s["lens"]):
        if c["op"] == "sinks":
            lo = max(0, p + 1 - win)
            idx = torch.cat([torch.arange(min(c["n_sink"], lo), device=DEV), torch.arange(lo, p + rows, device=DEV)])
        else:
            idx = torch.arange(p + rows, device=DEV)
        k, v = _values(_cached(s, i, idx, "k"), hd), _values(_cached(s, i, idx, "v"), hd)
        at = (p + torch.arange(rows, device=DEV))[:, None]
        see = idx[None] <= at
        if c["op"] == "sinks":
            see = see & ((idx[None] > at - win) | (idx[None] < c["n_sink"]))
        q = s["q"][i].float().reshape(rows, hkv, g, hd).permute(1, 2, 0, 3).reshape(hkv, g * rows, hd)
        a = (q @ k.transpose(1, 2) / math.sqrt(hd)).reshape(hkv, g, rows, -1)
        a = torch.where(see, a, torch.full_like(a, -math.inf))
        w = torch.exp(a - a.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        o = w.reshape(hkv, g * rows, -1) @ v
        out[i] = o.reshape(hkv, g, rows, hd).permute(2, 0, 1, 3).reshape(rows, hq, hd).to(torch.float16)
        if score is not None:
            score[i, :, :p + rows] = w.sum((1, 2))
            score[i, :, :p] += s["score"][i, :, :p]
    return out if score is None else {"out": out, "score": score}


def _plain_evict(s):
    c, n_seq, b = s["case"], s["case"]["n_seq"], s["case"]["budget"]
    for i, n in enumerate(s["lens"]):
        m = min(n, b)
        if n > b:
            f = s["score"][i, :, :n].clone()
            f[:, :c["n_sink"]] = math.inf
            f[:, n - c["n_recent"]:] = math.inf
            keep = torch.sort(f, dim=1, descending=True, stable=True).indices[:, :b].sort(1).values
        else:
            keep = torch.arange(n, device=DEV).expand(s["kept"].shape[1], n)
        s["kept"][i, :, :m] = keep.to(torch.int32)
        s["kept"][i, :, m:] = -1
        s["score"][n_seq + i, :, :m] = torch.gather(s["score"][i], 1, keep)
        h = torch.arange(keep.shape[0], device=DEV)[:, None]
        for x in (s["k"], s["v"]):
            if c["store"] == "paged":
                j = torch.arange(m, device=DEV)[None]
                rec = x[s["table"][i].long()[keep // PAGE], h, keep % PAGE]
                x[s["table"][n_seq + i].long()[j // PAGE], h, j % PAGE] = rec
            else:
                x[n_seq + i, :, :m] = x[i][h, keep]
    s["pos_out"].copy_(s["pos"].clamp(max=b))
    return _evicted(s)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(c, seed):
    if c["op"] == "evict":
        return None                                     # whole numbers and copies: nothing is computed
    s = _inputs(c, seed)
    hq, hkv, hd, win = HEADS[c["heads"]]
    g, rows = hq // hkv, c["rows"]
    out = torch.zeros(c["n_seq"], rows, hq, hd, dtype=torch.float64, device=DEV)
    score = torch.zeros(c["n_seq"], hkv, s["cap"], dtype=torch.float64, device=DEV)
    for i, p in enumerate(s["lens"]):
        n = p + rows
        for h in range(hkv):
            val = []
            for name in ("k", "v"):
                if c["store"] == "paged":
                    r = s[name][s["table"][i, :(n + PAGE - 1) // PAGE].long(), h].reshape(-1, _rec(hd))[:n]
                elif c["store"] == "slots":
                    r = s[name][i, h, :n]
                else:
                    # positions that fell out of the ring read as whatever has replaced them: hidden below
                    r = s[name][i, h].repeat(n // (2 * win) + 1, 1)[:n].clone()
                    m = min(n, s["sink_" + name].shape[2])
                    r[:m] = s["sink_" + name][i, h, :m]
                d = r[:, :hd // 16].contiguous().view(torch.float16).double().repeat_interleave(32, 1)
                val.append(r[:, hd // 16:].contiguous().view(torch.int8).double() * d)
            key = torch.arange(n, device=DEV)
            for j in range(g):
                head = h * g + j
                a = s["q"][i, :, head].double() @ val[0].T * hd ** -0.5
                row = p + torch.arange(rows, device=DEV)
                hide = key[None, :] > row[:, None]
                if c["op"] == "sinks":
                    hide |= (key[None, :] <= row[:, None] - win) & (key[None, :] >= c["n_sink"])
                w = torch.softmax(a.masked_fill(hide, -math.inf), -1)
                out[i, :, head] = w @ val[1]
                score[i, h, :n] += w.sum(0)
            if c["op"] == "track":
                score[i, h, :p] += s["score"][i, h, :p].double()
    return out if c["op"] == "sinks" else {"out": out, "score": score}
