"""The paged K/V cache's operators as cases to measure: appending a ragged batch's keys and values (rotated on the way) to
pages of bf16 or of 4 bits, reading rows back, and attention over the pages with a sliding window and sink tokens.

`run` with `own` false computes them with elementary torch operations in f32; with `own` true it makes the calls a user makes.
"""
import math

import torch

own = False

D = 128
SCALE = 1.0 / math.sqrt(D)


def listed():
    return [
        # a decode step's append: one token of each of 16 sequences, heads shared 4 to 1 (latency)
        {"name": "append-step-bf16", "op": "append", "fmt": "bf16", "seqs": 16, "heads": 32, "kv_heads": 8, "page_rows": 16,
         "max_q": 1, "max_kv": 4001, "pairing": "half"},
        # one block of 3 latent frames of the 14B video model (40 heads) at the end of a 21-frame window
        {"name": "append-block-bf16", "op": "append", "fmt": "bf16", "seqs": 1, "heads": 40, "kv_heads": 40, "page_rows": 64,
         "max_q": 4680, "max_kv": 32760, "pairing": "interleaved"},
        # ragged prompts into 4-bit pages, read back as the values they stand for
        {"name": "append-ragged-q4", "op": "append", "fmt": "q4", "seqs": 7, "heads": 40, "kv_heads": 8, "page_rows": 32,
         "max_q": 1021, "max_kv": 2777, "pairing": "half"},
        # the whole 21-frame window of the 1.3B video model out of 4-bit pages, for the dense attention call
        {"name": "read-window-q4", "op": "read", "fmt": "q4", "seqs": 1, "heads": 12, "kv_heads": 12, "page_rows": 128,
         "max_q": 32760, "max_kv": 32760},
        # a few ragged sequences out of bf16 pages
        {"name": "read-ragged-bf16", "op": "read", "fmt": "bf16", "seqs": 5, "heads": 8, "kv_heads": 8, "page_rows": 16,
         "max_q": 333, "max_kv": 1501},
        # a single short sequence's decode step, no shared heads (latency)
        {"name": "decode-short-bf16", "op": "attend", "fmt": "bf16", "seqs": 1, "heads": 12, "kv_heads": 12, "page_rows": 16,
         "max_q": 1, "max_kv": 777, "block": 1, "window": 0, "sink": 0},
        # a serving batch's decode step over ragged lengths
        {"name": "decode-batch-bf16", "op": "attend", "fmt": "bf16", "seqs": 32, "heads": 32, "kv_heads": 8, "page_rows": 64,
         "max_q": 1, "max_kv": 9001, "block": 1, "window": 0, "sink": 0},
        # long streams under a sliding window with sink tokens: the pages in between are given back
        {"name": "decode-window-bf16", "op": "attend", "fmt": "bf16", "seqs": 6, "heads": 40, "kv_heads": 8, "page_rows": 32,
         "max_q": 1, "max_kv": 100003, "block": 1, "window": 8190, "sink": 4},
        # a block of frames of the 1.3B video model against a rolling cache: 5 blocks of window, the first block as sink
        {"name": "block-window-bf16", "op": "attend", "fmt": "bf16", "seqs": 1, "heads": 12, "kv_heads": 12, "page_rows": 64,
         "max_q": 4680, "max_kv": 42120, "block": 4680, "window": 5, "sink": 1},
        # the serving batch on 4-bit pages
        {"name": "decode-batch-q4", "op": "attend", "fmt": "q4", "seqs": 32, "heads": 32, "kv_heads": 8, "page_rows": 64,
         "max_q": 1, "max_kv": 20011, "block": 1, "window": 0, "sink": 0},
        # one short stream on 4-bit pages, 5 heads to a key head (latency)
        {"name": "decode-short-q4", "op": "attend", "fmt": "q4", "seqs": 1, "heads": 40, "kv_heads": 8, "page_rows": 16,
         "max_q": 1, "max_kv": 1999, "block": 1, "window": 0, "sink": 0},
        # ragged prompt chunks on 4-bit pages, causal by token under a sliding window with sinks
        {"name": "chunk-ragged-q4", "op": "attend", "fmt": "q4", "seqs": 3, "heads": 40, "kv_heads": 8, "page_rows": 64,
         "max_q": 1501, "max_kv": 12007, "block": 1, "window": 4100, "sink": 5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    fmt = rng.choice(["bf16", "q4"])
    kv_heads, group = rng.choice([(12, 1), (40, 1), (8, 4), (8, 5), (2, 8), (1, 12), (4, 2), (2, 16), (3, 7)])
    case = {"op": op, "fmt": fmt, "seqs": _log(rng, 1, 24), "heads": kv_heads * group, "kv_heads": kv_heads,
            "page_rows": rng.choice([16, 32, 64, 128])}
    if op != "attend":
        case["max_kv"] = _log(rng, 1, 20000)
        tokens = 4000000 // (128 * (kv_heads * (group + 2)) * 4)
        case["max_q"] = min(case["max_kv"], max(1, _log(rng, 1, max(2, 4 * tokens // case["seqs"]))))
        if op == "append":
            case["pairing"] = rng.choice(["interleaved", "half"])
        while case["seqs"] * case["max_kv"] * kv_heads > 32760 * 20:
            case["seqs"] = (case["seqs"] + 1) // 2
            if case["seqs"] == 1:
                case["max_kv"] = (case["max_kv"] + 1) // 2
            case["max_q"] = min(case["max_q"], case["max_kv"])
        return case
    case["max_kv"] = _log(rng, 1, 40000)
    case["max_q"] = rng.choice([1, 1, rng.randint(1, 12), _log(rng, 1, 3000)])
    case["max_q"] = min(case["max_q"], case["max_kv"])
    case["block"] = rng.choice([1, 1, 1, rng.randint(2, 400), 1560])
    case["window"] = rng.choice([0, 0, 1 + _log(rng, 1, 9000) // case["block"]])
    case["sink"] = rng.choice([0, rng.randint(1, 8)]) if case["window"] else 0
    while case["seqs"] * case["max_kv"] * kv_heads > 32 * 9001 * 8 or \
            case["seqs"] * case["heads"] * case["max_q"] * case["max_kv"] > 12 * 4680 * 20000:
        if case["seqs"] > 1:
            case["seqs"] = (case["seqs"] + 1) // 2
        else:
            case["max_kv"] = (case["max_kv"] + 1) // 2
            case["max_q"] = min(case["max_q"], case["max_kv"])
    return case


def _lengths(case):
    """Cached tokens and new tokens of each sequence: the first has the most, the others are spread below."""
    kv, nq = [], []
    for i in range(case["seqs"]):
        cut = (i * 0.6180339887) % 1.0
        kv.append(max(1, int(case["max_kv"] * (1.0 - 0.6 * cut))))
        nq.append(min(kv[-1], max(1, int(case["max_q"] * (1.0 - 0.7 * cut)))))
    return kv, nq


def _span(case, first, last):
    """Keys that positions first..last see between them: [0, a) and [b, c)."""
    blk, win, sink = case["block"], case["window"], case["sink"]
    end = (last // blk + 1) * blk
    lo = max(0, first // blk - win + 1) * blk if win else 0
    return min(sink * blk, lo), lo, end


def _pages(case, kv, nq):
    """Which pages of each sequence hold something that the call reads or writes."""
    rows, need = case["page_rows"], []
    for n, q in zip(kv, nq):
        pages = (n + rows - 1) // rows
        if case["op"] == "attend":
            a, b, _ = _span(case, n - q, n - 1)
            need.append([p for p in range(pages) if p * rows < a or (p + 1) * rows > b])
        else:
            need.append(list(range(pages)))
    return need


def _pack(codes):
    """Codes 0..15 [..., 128] as bytes [..., 64]: the even value in the low half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    kv, nq = _lengths(case)
    seqs, hk, rows = case["seqs"], case["kv_heads"], case["page_rows"]
    need = _pages(case, kv, nq)
    most = max((n + rows - 1) // rows for n in kv)
    pool = sum(len(p) for p in need) + 2
    order = torch.randperm(pool, generator=host).to(torch.int32)
    table = torch.full((seqs, most), -1, dtype=torch.int32)
    at = 0
    for s, pages in enumerate(need):
        table[s, torch.tensor(pages)] = order[at: at + len(pages)]
        at += len(pages)
    cu = torch.zeros(seqs + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(nq).cumsum(0)
    total = int(cu[-1])
    st = {"case": dict(case), "table": table.to(dev), "kv_len": torch.tensor(kv, dtype=torch.int32).to(dev), "cu": cu.to(dev),
          "total": total, "max_q": max(nq), "max_kv": max(kv)}
    shape = (pool, hk, rows)
    if case["fmt"] == "bf16":
        for n in ("k", "v"):
            st[n] = torch.randn(*shape, D, generator=gen, device=dev, dtype=torch.bfloat16)
        st["k_scale"] = st["v_scale"] = None
    else:
        for n in ("k", "v"):
            st[n] = torch.randint(0, 256, (*shape, D // 2), generator=gen, device=dev, dtype=torch.uint8)
            step = 0.15 + 0.2 * torch.rand(*shape, generator=gen, device=dev)
            zero = step * (0.5 + 0.5 * torch.randn(*shape, generator=gen, device=dev))
            st[n + "_scale"] = torch.stack([step, zero], -1).to(torch.bfloat16)
    # the fused projection's rows: q, k and v side by side
    width = (case["heads"] + 2 * hk) * D
    if case["op"] == "append":
        proj = torch.randn(total, width, generator=gen, device=dev, dtype=torch.bfloat16)
        q, k, v = proj.split([case["heads"] * D, hk * D, hk * D], 1)
        st["q"], st["new_k"], st["new_v"] = q.view(total, -1, D), k.view(total, hk, D), v.view(total, hk, D)
        turn = torch.arange(D // 2, dtype=torch.float64, device=dev) * (-2.0 / D)
        angle = torch.arange(max(kv), dtype=torch.float64, device=dev)[:, None] * (10000.0 ** turn)
        angle = angle.repeat_interleave(2, 1) if case["pairing"] == "interleaved" else angle.repeat(1, 2)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        st["q"] = torch.randn(total, case["heads"], D, generator=gen, device=dev, dtype=torch.bfloat16)
    return st


# ---- the calls a user makes -------------------------------------------------------------------------------------------

def _own(st):
    from fastvideo_rs_b200 import paged
    from fastvideo_rs_b200.sdpa import BlockCausal
    case = st["case"]
    if "handle" not in st:  # what a program keeps beside its cache: the pool and the batch's tables
        st["handle"] = (paged.PagedKv(st["k"], st["v"], st["k_scale"], st["v_scale"]),
                        paged.PagedBatch(st["table"], st["kv_len"], st["cu"], max_q=st["max_q"], max_kv=st["max_kv"]))
    kv, batch = st["handle"]
    if case["op"] == "attend":
        return paged.attend(kv, batch, st["q"], BlockCausal(case["block"], case["window"], case["sink"]), scale=SCALE)
    if case["op"] == "read":
        k, v = paged.read(kv, batch, rows=st["total"])
        return {"k": k, "v": v}
    q = paged.append(kv, batch, st["new_k"], st["new_v"], q=st["q"], cos=st["cos"], sin=st["sin"], pairing=case["pairing"])
    if case["fmt"] == "bf16":
        return {"q": q, "k": st["k"], "v": st["v"]}
    k, v = paged.read(kv, batch, rows=st["total"])
    return {"q": q, "k": k, "v": v}


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _tokens(st):
    """Sequence and position of each token of the batch."""
    cu, dev = st["cu"].long(), st["cu"].device
    t = torch.arange(st["total"], device=dev)
    seq = torch.searchsorted(cu[1:], t, right=True)
    return seq, t - cu[1:][seq] + st["kv_len"].long()[seq], t - cu[seq]


def _rotate(x, cos, sin, pairing):
    x = x.float()
    if pairing == "interleaved":
        other = torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)
    else:
        other = torch.cat([-x[..., D // 2:], x[..., : D // 2]], -1)
    return x * cos[:, None] + other * sin[:, None]


def _quantize(x):
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()  # (a true division, not a product with 1 / 15)
    zero = (lo + 8.0 * step).to(torch.bfloat16).float()
    codes = torch.round((x - zero[..., None]) / step[..., None]).clamp(-8, 7)
    codes = torch.where(step[..., None] > 0, codes, torch.zeros_like(codes))
    return (codes + 8).to(torch.uint8), torch.stack([step, zero], -1).to(torch.bfloat16)


def _values(codes, scale):
    """What 4-bit rows stand for, f32."""
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    s = scale.float()
    return s[..., 1:] + s[..., :1] * both


def _plain_append(st):
    case = st["case"]
    seq, pos, _ = _tokens(st)
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotate(st["q"], cos, sin, case["pairing"]).to(torch.bfloat16)
    k = _rotate(st["new_k"], cos, sin, case["pairing"])
    page, row = st["table"].long()[seq, pos // case["page_rows"]], pos % case["page_rows"]
    if case["fmt"] == "bf16":
        st["k"][page, :, row] = k.to(torch.bfloat16)
        st["v"][page, :, row] = st["new_v"]
        return {"q": q, "k": st["k"], "v": st["v"]}
    for name, x in (("k", k), ("v", st["new_v"].float())):
        codes, scale = _quantize(x)
        st[name][page, :, row] = _pack(codes)
        st[name + "_scale"][page, :, row] = scale
    return {"q": q, **_plain_read(st)}


def _plain_read(st):
    case = st["case"]
    seq, pos, _ = _tokens(st)
    page, row = st["table"].long()[seq, pos // case["page_rows"]], pos % case["page_rows"]
    if case["fmt"] == "bf16":
        return {"k": st["k"][page, :, row], "v": st["v"][page, :, row]}
    return {n: _values(st[n][page, :, row], st[n + "_scale"][page, :, row]).to(torch.bfloat16) for n in ("k", "v")}


def _gather(st, name):
    """[seqs, kv_heads, keys, 128] f32 of every sequence, out of its pages."""
    page = st["table"].long().clamp(min=0)
    x = st[name][page] if st["case"]["fmt"] == "bf16" else _values(st[name][page], st[name + "_scale"][page])
    return x.float().permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attend(st):
    case = st["case"]
    seqs, heads, hk = case["seqs"], case["heads"], case["kv_heads"]
    group, nq = heads // hk, st["max_q"]
    seq, pos, at = _tokens(st)
    q = torch.zeros(seqs, nq, heads, D, device=st["q"].device)
    q[seq, at] = st["q"].float()
    where = torch.full((seqs, nq), -1, dtype=torch.long, device=q.device)
    where[seq, at] = pos
    q = q.view(seqs, nq, hk, group, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    k, v = _gather(st, "k"), _gather(st, "v")
    j = torch.arange(k.shape[2], device=q.device)
    tj, tq = j // case["block"], (where // case["block"])[..., None]
    seen = (tj <= tq) & (where >= 0)[..., None] & (j < st["kv_len"].long()[:, None])[:, None]
    if case["window"]:
        seen &= (tq - tj < case["window"]) | (tj < case["sink"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(SCALE)
    scores = scores.view(seqs, hk, nq, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf).view(seqs, hk, nq * group, -1)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = out.view(seqs, hk, nq, group, D).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[seq, at].to(torch.bfloat16)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    kv, nq = _lengths(case)
    hk, heads, tokens = case["kv_heads"], case["heads"], sum(nq)
    row = 2 * hk * (2 * D if case["fmt"] == "bf16" else D // 2 + 4)  # K and V of one token in the cache
    if case["op"] == "append":
        angles = len({p for n, q in zip(kv, nq) for p in range(n - q, n)})  # rows of the two tables
        moved = tokens * (2 * heads * 2 * D + 2 * hk * 2 * D + row) + angles * 8 * D
        flops = tokens * D * 3 * (heads + hk)
        if case["fmt"] == "q4":
            moved += tokens * (row + 2 * hk * 2 * D)
            flops += tokens * D * 8 * hk
        return {"bytes": moved, "flops": flops}
    if case["op"] == "read":
        return {"bytes": tokens * (row + 2 * hk * 2 * D), "flops": tokens * D * 4 * hk}
    moved, pairs = tokens * heads * 4 * D, 0
    for n, q in zip(kv, nq):
        a, b, c = _span(case, n - q, n - 1)
        moved += (a + min(c, n) - b) * row
        first = n - q
        while first < n:  # rows of one block see the same keys
            last = min(n, (first // case["block"] + 1) * case["block"])
            a, b, c = _span(case, first, first)
            pairs += (last - first) * (a + min(c, n) - b)
            first = last
    return {"bytes": moved, "flops": 4 * D * pairs * heads}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _exact_rows(st, name, s, keys):
    """K or V of sequence s at the given key indices: [kv_heads, keys, 128] f64."""
    rows = st["case"]["page_rows"]
    page = st["table"][s].long()[keys // rows]
    x = st[name][page, :, keys % rows]
    if st["case"]["fmt"] == "q4":
        sc = st[name + "_scale"][page, :, keys % rows].double()
        nib = torch.empty(*x.shape[:-1], D, dtype=torch.float64, device=x.device)
        nib[..., 0::2] = (x % 16).double()
        nib[..., 1::2] = torch.div(x, 16, rounding_mode="floor").double()
        x = (nib - 8.0) * sc[..., 0:1] + sc[..., 1:2]
    return x.double().transpose(0, 1)


def _exact_turn(x, cos, sin, pairing):
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    y = torch.empty_like(x)
    lo, hi = (slice(0, D, 2), slice(1, D, 2)) if pairing == "interleaved" else (slice(0, D // 2), slice(D // 2, D))
    y[..., lo] = x[..., lo] * c[..., lo] - x[..., hi] * s[..., lo]
    y[..., hi] = x[..., lo] * s[..., hi] + x[..., hi] * c[..., hi]
    return y


def _exact_stands(x):
    """The value that each entry's 4-bit code stands for."""
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    step = ((hi - lo) / 15).to(torch.bfloat16).double()
    zero = (lo + 8 * step).to(torch.bfloat16).double()
    return zero + step * ((x - zero) / step).round().clamp(-8, 7).nan_to_num(0.0)


def exact(case, seed):
    st = prepare(case, seed)
    cu, lens = st["cu"].tolist(), st["kv_len"].tolist()
    if case["op"] == "read":
        out = {n: [] for n in ("k", "v")}
        for s, n in enumerate(lens):
            keys = torch.arange(n - (cu[s + 1] - cu[s]), n, device="cuda")
            for name in out:
                out[name].append(_exact_rows(st, name, s, keys).transpose(0, 1))
        return {n: torch.cat(x) for n, x in out.items()}
    if case["op"] == "append":
        pos = torch.cat([torch.arange(n - (cu[s + 1] - cu[s]), n, device="cuda") for s, n in enumerate(lens)])
        cos, sin = st["cos"][pos], st["sin"][pos]
        q, k = (_exact_turn(st[n], cos, sin, case["pairing"]) for n in ("q", "new_k"))
        v = st["new_v"].double()
        if case["fmt"] == "q4":
            return {"q": q, "k": _exact_stands(k), "v": _exact_stands(v)}
        rows, pk, pv = case["page_rows"], st["k"].double(), st["v"].double()
        for s in range(case["seqs"]):
            mine = slice(cu[s], cu[s + 1])
            page = st["table"][s].long()[pos[mine] // rows]
            pk[page, :, pos[mine] % rows] = k[mine]
            pv[page, :, pos[mine] % rows] = v[mine]
        return {"q": q, "k": pk, "v": pv}
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(st["total"], case["heads"], D, dtype=torch.float64, device="cuda")
    for s, n in enumerate(lens):
        first = n - (cu[s + 1] - cu[s])
        a, b, c = _span(case, first, n - 1)
        keys = torch.cat([torch.arange(0, a, device="cuda"), torch.arange(b, min(c, n), device="cuda")])
        tq = torch.arange(first, n, device="cuda")[:, None] // case["block"]
        tk = keys[None] // case["block"]
        hidden = tk > tq
        if case["window"]:
            hidden |= (tq - tk >= case["window"]) & (tk >= case["sink"])
        k, v = _exact_rows(st, "k", s, keys), _exact_rows(st, "v", s, keys)
        for h in range(case["heads"]):
            x = st["q"][cu[s]: cu[s + 1], h].double() @ k[h // group].T * SCALE
            x = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[cu[s]: cu[s + 1], h] = x @ v[h // group]
    return out
