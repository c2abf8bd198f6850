"""What the serving operators around the decoder are measured on: attention of
one new token over a paged key-value cache, appending rows to that cache,
eviction from it by accumulated attention weight, and sampling from logits.

`listed()` are the cases, `draw()` gives more of the same ranges, `prepare()`
makes a case's inputs on the GPU, and `run()` is one pass: in plain torch where
`own` is false, through the framework's entry points where it is true.
"""
import math

import numpy as np
import torch

own = False

LLAMA = {"heads": 32, "kv_heads": 8, "head_dim": 128, "theta": 500000.0}
QWEN = {"heads": 14, "kv_heads": 2, "head_dim": 64, "theta": 1e6}


def listed():
    return [
        # a conversation's first tokens on the small model: latency alone counts
        {"name": "attn_b1_len17", "op": "attention", "batch": 1, "len": 17, "ragged": False, "page": 16, "mass": False,
         **QWEN},
        # continuous batching: 32 sequences of all lengths up to 4096, an empty row among them
        {"name": "attn_b32_ragged4k", "op": "attention", "batch": 32, "len": 4096, "ragged": True, "page": 64,
         "mass": False, **LLAMA},
        # one very long context
        {"name": "attn_b1_131k", "op": "attention", "batch": 1, "len": 131077, "ragged": False, "page": 256,
         "mass": False, **LLAMA},
        # the decode benchmark's own shape with the rotation and the append in the call
        {"name": "rope_b1_2049", "op": "rope_attention", "batch": 1, "len": 2049, "ragged": False, "page": 64,
         "mass": False, **LLAMA},
        # the same for several long sequences whose attention weights are accumulated for eviction
        {"name": "rope_mass_b8_8k", "op": "rope_attention", "batch": 8, "len": 8200, "ragged": True, "page": 16,
         "mass": True, **LLAMA},
        # one token's key and value by themselves
        {"name": "append_1", "op": "append", "rows": 1, "batch": 1, "page": 16, **QWEN},
        # a prompt chunk of several sequences
        {"name": "append_4099", "op": "append", "rows": 4099, "batch": 3, "page": 64, **LLAMA},
        # trimming caches that grew a little past their budget
        {"name": "evict_trim_b8", "op": "evict", "batch": 8, "len": 2113, "ragged": False, "keep": 2048, "recent": 256,
         "page": 64, **LLAMA},
        # long prompts cut down to a budget once they are read
        {"name": "evict_prompt_b4", "op": "evict", "batch": 4, "len": 32771, "ragged": True, "keep": 4096,
         "recent": 512, "page": 64, **LLAMA},
        # one sequence's next token with every filter on
        {"name": "sample_b1", "op": "sample", "batch": 1, "vocab": 151936, "mode": "all"},
        # a batch under nucleus sampling alone
        {"name": "sample_b32_top_p", "op": "sample", "batch": 32, "vocab": 128256, "mode": "top_p"},
        # a server's batch: every request with settings of its own, greedy and unfiltered ones among them
        {"name": "sample_b64_mixed", "op": "sample", "batch": 64, "vocab": 151936, "mode": "mixed"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "rope_attention", "append", "evict", "sample"])
    if op == "sample":
        return {"op": op, "batch": _log_int(rng, 1, 64), "vocab": _log_int(rng, 1000, 151936),
                "mode": rng.choice(["all", "top_k", "top_p", "min_p", "none", "greedy", "mixed"])}
    hd = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.randint(1, 16 if hd < 256 else 8)
    case = {"op": op, "heads": kv * group, "kv_heads": kv, "head_dim": hd, "page": rng.choice([16, 32, 48, 64, 128, 256]),
            "theta": rng.choice([10000.0, 500000.0, 1e6])}
    if op == "append":
        return {**case, "rows": _log_int(rng, 1, max(1, 16_000_000 // ((kv * group + 2 * kv) * hd))),
                "batch": rng.randint(1, 8)}
    length = _log_int(rng, 1, 65536)
    most = 500_000_000 // (4 * kv * hd * length)  # the longest listed cache's bytes
    if op == "evict":
        length = _log_int(rng, 64, 32768)
        most = 400_000_000 // (4 * kv * hd * length)
        keep = _log_int(rng, 16, length)
        return {**case, "batch": min(_log_int(rng, 1, 64), max(1, most)), "len": length, "ragged": rng.random() < 0.5,
                "keep": keep, "recent": rng.randint(0, keep)}
    return {**case, "batch": min(_log_int(rng, 1, 64), max(1, most)), "len": length, "ragged": rng.random() < 0.5,
            "mass": rng.random() < 0.3}


def _lens(case):
    """Slots in use per sequence: all `len`, or spread over the range with an empty row and a row of one."""
    n, b = case["len"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    lens = [1 + int((n - 1) * ((0.6180339887498949 * i) % 1.0)) for i in range(b)]
    lens[0] = n
    if b > 2:
        lens[1], lens[2] = 0, 1
    return lens


def _rows(case):
    """Append: the sequence of each row and the slot it goes to (chunks of equal size, an unused row at the end)."""
    n, b = case["rows"], case["batch"]
    per = -(-n // b)
    seqs = [i // per for i in range(n)]
    slots = [37 * (1 + i // per) + i % per for i in range(n)]
    if n > 4:
        slots[-1] = -1
    return seqs, slots


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        return _prepare_sample(case, s, g, dev)
    hq, hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    b = case["batch"]
    if case["op"] == "append":
        seqs, slots = _rows(case)
        lens = [max([t + 1 for q, t in zip(seqs, slots) if q == i] + [1]) for i in range(b)]
    else:
        lens = _lens(case)
    blocks = [-(-n // page) for n in lens]
    total = sum(blocks)
    perm = torch.randperm(total + 2, generator=g, device=dev).to(torch.int32)
    table = torch.full((b, max(max(blocks), 1)), -1, dtype=torch.int32)
    table = table.to(dev)
    at = torch.cumsum(torch.tensor([0] + blocks[:-1]), 0).to(dev)
    col = torch.arange(table.shape[1], device=dev)
    used = col[None, :] < torch.tensor(blocks, device=dev)[:, None]
    table[used] = perm[(at[:, None] + col[None, :])[used]]
    s["table"] = table
    shape = (total + 2, hkv, page, hd)
    s["k"] = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    s["v"] = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if case["op"] == "append":
        n = case["rows"]
        s["qkv"] = torch.randn((n, (hq + 2 * hkv) * hd), generator=g, device=dev)
        s["q_out"] = torch.zeros((n, hq * hd), device=dev)
        s["seqs"] = torch.tensor(seqs, dtype=torch.int32, device=dev)
        s["slots"] = torch.tensor(slots, dtype=torch.int32, device=dev)
        s["pos"] = torch.randint(0, 100000, (n,), generator=g, device=dev, dtype=torch.int32)
    elif case["op"] == "evict":
        ld = case["len"]
        m = torch.exp(2.0 * torch.randn((b, hkv, ld), generator=g, device=dev))
        s["mass"] = torch.where(torch.rand(m.shape, generator=g, device=dev) < 0.1, 0.0, m)  # never attended: ties
        s["slot_pos"] = torch.arange(ld, dtype=torch.int32, device=dev).expand(b, hkv, ld).contiguous()
        s["recent_from"] = s["lens"] - case["recent"]
        s["mass_out"], s["pos_out"] = torch.zeros_like(s["mass"]), torch.zeros_like(s["slot_pos"])
        s["lens_out"] = torch.zeros_like(s["lens"])
    else:
        cols = (hq + 2 * hkv) * hd if case["op"] == "rope_attention" else hq * hd
        s["qkv"] = 1.5 * torch.randn((b, cols), generator=g, device=dev)
        s["out"] = torch.zeros((b, hq * hd), device=dev)
        s["pos"] = s["lens"] - 1 + torch.randint(0, 5000, (b,), generator=g, device=dev, dtype=torch.int32)
        s["mass"] = s["slot_pos"] = None
        if case["mass"]:
            s["mass"] = torch.rand((b, hkv, case["len"]), generator=g, device=dev)
            s["slot_pos"] = torch.zeros((b, hkv, case["len"]), dtype=torch.int32, device=dev)
    if own:
        from pesti_b200 import kq, paged
        s["cache"] = paged.PagedCache(kq.default_context(0), s["k"], s["v"])
        if case["op"] != "append":
            s["scratch"] = (s["cache"].evict_scratch(b, case["len"]) if case["op"] == "evict" else
                            s["cache"].scratch(b, hq, case["len"] if case["mass"] else 0))
    return s


def _prepare_sample(case, s, g, dev):
    b, v, mode = case["batch"], case["vocab"], case["mode"]
    s["logits"] = 2.5 * torch.randn((b, v), generator=g, device=dev)
    s["u"] = torch.rand((b,), generator=g, device=dev)
    on = lambda name: [mode in (name, "all") or (mode == "mixed" and i % 6 in (k, 5))  # noqa: E731
                       for i in range(b) for k in [["top_k", "top_p", "min_p"].index(name)]]
    temp = [0.0 if mode == "greedy" or (mode == "mixed" and i % 6 == 3) else (0.7, 0.8, 1.0, 1.3)[i % 4]
            for i in range(b)]
    s["temperature"] = torch.tensor(temp, device=dev)
    s["top_k"] = torch.tensor([(40, 20, 100)[i % 3] if o else 0 for i, o in enumerate(on("top_k"))],
                              dtype=torch.int32, device=dev)
    s["top_p"] = torch.tensor([(0.9, 0.95, 0.8)[i % 3] if o else 1.0 for i, o in enumerate(on("top_p"))], device=dev)
    s["min_p"] = torch.tensor([(0.05, 0.02)[i % 2] if o else 0.0 for i, o in enumerate(on("min_p"))], device=dev)
    s["tokens"] = torch.zeros(b, dtype=torch.int32, device=dev)
    s["prob"] = torch.zeros(b, device=dev)
    s["kept"] = torch.zeros(b, dtype=torch.int32, device=dev)
    if own:
        from pesti_b200 import kq
        s["ctx"] = kq.default_context(0)
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rope_attention": _own_attention, "append": _own_append,
                "evict": _own_evict, "sample": _own_sample}[op](state)
    return {"attention": _attention, "rope_attention": _attention, "append": _append, "evict": _evict,
            "sample": _sample}[op](state)


def _own_attention(s):
    c = s["case"]
    if c["op"] == "attention":
        s["cache"].attention(s["qkv"], s["table"], s["lens"], s["out"], s["scratch"], mass=s["mass"])
        return {"out": s["out"]} if s["mass"] is None else {"out": s["out"], "mass": s["mass"]}
    s["cache"].rope_attention(s["qkv"], s["table"], s["lens"], s["out"], s["scratch"], theta=c["theta"], pos=s["pos"],
                              mass=s["mass"], slot_pos=s["slot_pos"])
    return _attention_outputs(s)


def _own_append(s):
    s["cache"].append(s["qkv"], s["table"], s["slots"], theta=s["case"]["theta"], seqs=s["seqs"], pos=s["pos"],
                      q_out=s["q_out"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_evict(s):
    s["cache"].evict(s["table"], s["lens"], s["lens_out"], s["mass"], s["slot_pos"], s["mass_out"], s["pos_out"],
                     s["case"]["keep"], s["scratch"], recent_from=s["recent_from"])
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"], "mass": s["mass_out"], "slot_pos": s["pos_out"]}


def _own_sample(s):
    from pesti_b200 import sampling
    sampling.sample(s["ctx"], s["logits"], s["u"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"],
                    top_p=s["top_p"], min_p=s["min_p"], prob=s["prob"], kept=s["kept"])
    return {"tokens": s["tokens"], "prob": s["prob"], "kept": s["kept"]}


def _attention_outputs(s):
    out = {"out": s["out"], "k": s["k"], "v": s["v"]}
    return out if s["mass"] is None else {**out, "mass": s["mass"], "slot_pos": s["slot_pos"]}


# ---- plain forms ---------------------------------------------------------------------


def _rope(x, pos, theta):
    """Pairs (i, i + hd/2) of x [n][heads][hd] turned by pos * theta^(-2i/hd); the angles in 64 bits."""
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = pos.double()[:, None] * theta ** (-i / half)
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _attention(s):
    c = s["case"]
    hq, hkv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, table = s["lens"].long(), s["table"].long()
    b = lens.shape[0]
    q = s["qkv"][:, :hq * hd].view(b, hq, hd)
    rope = c["op"] == "rope_attention"
    if rope:
        rows = s["qkv"].view(b, hq + 2 * hkv, hd)
        q = _rope(rows[:, :hq], s["pos"], c["theta"])
        live = (lens > 0).nonzero()[:, 0]
        last = lens[live] - 1
        at = table[live, last // page]
        s["k"][at, :, last % page] = _rope(rows[:, hq:hq + hkv], s["pos"], c["theta"])[live].half()
        s["v"][at, :, last % page] = rows[live, hq + hkv:].half()
    n = table.shape[1] * page
    pages = table.clamp(min=0)
    k = s["k"][pages].transpose(1, 2).reshape(b, hkv, n, hd).float()
    v = s["v"][pages].transpose(1, 2).reshape(b, hkv, n, hd).float()
    dead = (torch.arange(n, device=q.device)[None, :] >= lens[:, None])[:, None, None, :]
    scores = (q.reshape(b, hkv, hq // hkv, hd) @ k.transpose(2, 3)) / math.sqrt(hd)
    scores = scores.masked_fill(dead, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    s["out"].copy_((p @ v.masked_fill(dead.transpose(2, 3), 0.0)).reshape(b, hq * hd))
    if s["mass"] is not None:
        m = s["mass"]
        col = torch.arange(m.shape[2], device=m.device)[None, None, :]
        if rope:
            new = (col == lens[:, None, None] - 1) & (lens[:, None, None] > 0)
            m.masked_fill_(new, 0.0)
            s["slot_pos"].copy_(torch.where(new, s["pos"][:, None, None], s["slot_pos"]))
        m += p.sum(2)[:, :, :m.shape[2]]
    if rope:
        return _attention_outputs(s)
    return {"out": s["out"]} if s["mass"] is None else {"out": s["out"], "mass": s["mass"]}


def _append(s):
    c = s["case"]
    hq, hkv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    live = (s["slots"] >= 0).nonzero()[:, 0]
    rows = s["qkv"][live].view(-1, hq + 2 * hkv, hd)
    turned = _rope(rows[:, :hq + hkv], s["pos"][live], c["theta"])
    slot = s["slots"][live].long()
    at = s["table"][s["seqs"][live].long(), slot // page].long()
    s["q_out"][live] = turned[:, :hq].reshape(live.shape[0], -1)
    s["k"][at, :, slot % page] = turned[:, hq:].half()
    s["v"][at, :, slot % page] = rows[:, hq + hkv:].half()
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _evict(s):
    c = s["case"]
    page, keep, hkv = c["page"], c["keep"], c["kv_heads"]
    lens, mass, spos = s["lens"].long(), s["mass"], s["slot_pos"]
    b, _, ld = mass.shape
    col = torch.arange(ld, device=mass.device)
    valid = (col < lens[:, None])[:, None, :]
    key = torch.where(spos >= s["recent_from"][:, None, None], math.inf, mass.nan_to_num(-math.inf))
    # kept: the `keep` greatest, ties to the lowest slot; free slots behind the last come after everything
    key = torch.where(valid, key.double(), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    rank = torch.zeros_like(order).scatter_(2, order, col.expand(b, hkv, ld))
    kept = (rank < keep) & valid
    holes = ~kept & (col < keep) & valid
    movers = kept & (col >= keep)
    hb, hh, hole = holes.nonzero(as_tuple=True)  # in order of (sequence, head, slot), and as many as the movers
    _, _, src = movers.nonzero(as_tuple=True)
    table = s["table"].long()
    ps, pd = table[hb, src // page], table[hb, hole // page]
    s["k"][pd, hh, hole % page] = s["k"][ps, hh, src % page]
    s["v"][pd, hh, hole % page] = s["v"][ps, hh, src % page]
    head = valid & (col < keep)
    s["mass_out"].copy_(torch.where(head, mass, s["mass_out"]))
    s["pos_out"].copy_(torch.where(head, spos, s["pos_out"]))
    s["mass_out"][hb, hh, hole] = mass[hb, hh, src]
    s["pos_out"][hb, hh, hole] = spos[hb, hh, src]
    s["lens_out"].copy_(s["lens"].clamp(max=keep))
    return {"k": s["k"], "v": s["v"], "lens": s["lens_out"], "mass": s["mass_out"], "slot_pos": s["pos_out"]}


def _sample(s):
    z = s["logits"].double()
    z = torch.where(torch.isnan(z), -math.inf, z)
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    top, order = torch.sort(z, dim=-1, descending=True, stable=True)
    d = torch.where(top == top[:, :1], 0.0, (top - top[:, :1]) / torch.where(greedy, 1.0, t))
    w = torch.exp(d)
    rank = torch.arange(z.shape[1], device=z.device)[None, :]
    k = s["top_k"].long()[:, None]
    keep = ((k <= 0) | (rank < k)) & ~(greedy & (rank > 0)) & (top > -math.inf)
    mass = torch.cumsum(torch.where(keep, w, 0.0), dim=-1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (mass - w < p * mass[:, -1:]) | (rank == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    chance = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run_ = torch.cumsum(chance, dim=-1)
    total = run_[:, -1:]
    token = (run_ > s["u"].double()[:, None] * total).int().argmax(-1)
    some = total[:, 0] > 0
    s["tokens"].copy_(torch.where(some, token, -1))
    s["prob"].copy_(torch.where(some, chance.gather(1, token[:, None])[:, 0] / total[:, 0], 0.0))
    s["kept"].copy_(keep.sum(-1))
    return {"tokens": s["tokens"], "prob": s["prob"], "kept": s["kept"]}


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": 4 * n + 32 * case["batch"], "flops": 4 * n}
    hq, hkv, hd, b = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
    if op == "append":
        n = case["rows"]
        return {"bytes": n * ((hq + 2 * hkv) * hd * 4 + hq * hd * 4 + 2 * hkv * hd * 2 + 16),
                "flops": 3 * n * (hq + hkv) * hd}
    lens = _lens(case)
    slots = sum(lens)
    if op == "evict":
        keep = case["keep"]
        cut = [n for n in lens if n > keep]
        old = [max(n - case["recent"], 1) for n in cut]
        # rows that move: the protected ones behind `keep`, and of the others there the share that is kept
        moved = sum(min(case["recent"], n - keep) + max(0, o - keep) * max(0, keep - case["recent"]) / o
                    for n, o in zip(cut, old))
        return {"bytes": 8 * hkv * slots + 8 * hkv * sum(min(n, keep) for n in lens) + moved * hkv * 4 * hd * 2,
                "flops": hkv * slots}
    row = (hq + 2 * hkv) * hd if op == "rope_attention" else hq * hd
    return {"bytes": 4 * hkv * hd * slots + 4 * b * (row + hq * hd) + (8 * hkv * slots if case["mass"] else 0)
            + 4 * sum(-(-n // case["page"]) for n in lens),
            "flops": 4 * hq * hd * slots}


# ---- the definitions in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rope_attention": _exact_attention, "append": _exact_append,
            "evict": _exact_evict, "sample": _exact_sample}[case["op"]](s, case)


def _turn(vec, pos, theta):
    """One head vector (or rows of them) as complex numbers, turned."""
    half = vec.shape[-1] // 2
    z = torch.complex(vec[..., :half].double(), vec[..., half:].double())
    freq = torch.exp(torch.arange(half, device=vec.device, dtype=torch.float64) * (-math.log(theta) / half))
    z = z * torch.polar(torch.ones_like(freq), pos * freq)
    return torch.cat([z.real, z.imag], -1)


def _exact_attention(s, case):
    hq, hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rope = case["op"] == "rope_attention"
    out = torch.zeros((case["batch"], hq * hd), dtype=torch.float64, device=s["qkv"].device)
    mass = s["mass"].double() if s["mass"] is not None else None
    kp, vp = (s["k"].double(), s["v"].double()) if rope else (None, None)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pos = int(s["pos"][b])
        vec = s["qkv"][b].view(-1, hd)
        ids = s["table"][b, :-(-n // page)].long()
        if rope:
            at, r = int(ids[(n - 1) // page]), (n - 1) % page
            k_new = _turn(vec[hq:hq + hkv], pos, case["theta"])
            kp[at, :, r], vp[at, :, r] = k_new, vec[hq + hkv:].double()
            # the cache holds f16: what is attended is the rounded row
            s["k"][at, :, r], s["v"][at, :, r] = k_new.to(torch.float16), vec[hq + hkv:].to(torch.float16)
        for h in range(hkv):
            k, v = (s[x][ids, h].reshape(-1, hd)[:n].double() for x in "kv")
            q = vec[h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            if rope:
                q = _turn(q, pos, case["theta"])
            p = torch.softmax(torch.einsum("gd,nd->gn", q, k) / hd ** 0.5, -1)
            out[b].view(hq, hd)[h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.einsum("gn,nd->gd", p, v)
            if mass is not None:
                if rope:
                    mass[b, h, n - 1] = 0.0
                mass[b, h, :n] += p.sum(0)
    found = {"out": out}
    if rope:
        found.update(k=kp, v=vp)
    if mass is not None:
        found["mass"] = mass
        if rope:
            found["slot_pos"] = None
    return found


def _exact_append(s, case):
    hq, hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    q, k, v = s["q_out"].double(), s["k"].double(), s["v"].double()
    slots, seqs, pos = (s[x].long() for x in ("slots", "seqs", "pos"))
    ok = slots >= 0
    vec = s["qkv"].view(-1, hq + 2 * hkv, hd).double()
    new = _turn(vec[:, :hq + hkv], pos.double()[:, None, None], case["theta"])
    q[ok] = new[ok][:, :hq].flatten(1)
    page_of = s["table"].long()[seqs[ok], slots[ok].div(page, rounding_mode="floor")]
    k[page_of, :, slots[ok].remainder(page)] = new[ok][:, hq:]
    v[page_of, :, slots[ok].remainder(page)] = vec[ok][:, hq + hkv:]
    return {"q": q, "k": k, "v": v}


def _exact_evict(s, case):
    """What stays is moved, not computed: the rows by a walk over every head's slots."""
    keep, page, hkv = case["keep"], case["page"], case["kv_heads"]
    mass, spos = s["mass"].cpu().numpy(), s["slot_pos"].cpu().numpy()
    table, since = s["table"].cpu().numpy(), s["recent_from"].cpu().numpy()
    mass_out = np.zeros(mass.shape)
    dst, src = [], []
    for b, n in enumerate(s["lens"].tolist()):
        for h in range(hkv):
            m = mass[b, h, :n].astype(np.float64)
            stay = np.arange(n)
            if n > keep:
                m = np.where(spos[b, h, :n] >= since[b], np.inf, m)
                stay = np.sort(np.lexsort((np.arange(n), -m))[:keep])
            left = np.setdiff1d(np.arange(min(n, keep)), stay)
            come = stay[stay >= keep]
            to = np.arange(min(n, keep))
            frm = to.copy()
            frm[left] = come
            mass_out[b, h, to] = mass[b, h, frm]
            dst += [(table[b, i // page], h, i % page) for i in left]
            src += [(table[b, i // page], h, i % page) for i in come]
    k, v = s["k"].clone(), s["v"].clone()
    if dst:
        d, f = (torch.tensor(np.array(x, dtype=np.int64), device=k.device).unbind(1) for x in (dst, src))
        k[d], v[d] = s["k"][f], s["v"][f]
    return {"k": k, "v": v, "lens": None, "mass": mass_out, "slot_pos": None}


def _exact_sample(s, case):
    z = s["logits"].cpu().numpy().astype(np.float64)
    t, k, p, mp, u = (s[x].cpu().numpy().astype(np.float64) for x in ("temperature", "top_k", "top_p", "min_p", "u"))
    prob = np.zeros(case["batch"])
    for b in range(case["batch"]):
        by = np.argsort(-z[b], kind="stable")
        if t[b] <= 0:
            by = by[:1]
        elif k[b] > 0:
            by = by[:int(k[b])]
        w = np.exp((z[b][by] - z[b][by[0]]) / (t[b] if t[b] > 0 else 1.0))
        n = len(by)
        if p[b] < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), p[b] * w.sum())))
        n = max(1, min(n, int((w >= mp[b]).sum())))
        by, w = by[:n], w[:n]
        up = np.argsort(by)
        run_ = np.cumsum(w[up])
        prob[b] = w[up][np.searchsorted(run_, u[b] * run_[-1], side="right")] / run_[-1]
    return {"tokens": None, "prob": prob, "kept": None}
