"""The operators of one decode step that run beside the MoE block: what is measured of each.

  plan    block tables and slot maps of a paged key-value cache, from the sequences' lengths
  rope    RMSNorm of each query and key head, position rotation, and the append of K and V to the cache, in one pass
  attn    attention of one new token per row over the paged cache
  route   expert routing from router logits: softmax or sigmoid scores, balance bias, groups, top-k, weights

`run` computes them in elementary torch operations where `own` is false, and by the framework's entry points
(moe.cc_b200/moe_cuda.py) where it is true.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def _mc():
    """The framework's ctypes binding."""
    m = sys.modules.get("moe_cuda")
    if m is None:
        d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe.cc_b200")
        if d not in sys.path:
            sys.path.insert(0, d)
        import moe_cuda as m
    return m


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one conversation, a short context: what a single-user decode step waits for
        {"name": "attn_one_row", "op": "attn", "dtype": "bf16", "rows": 1, "n_q": 32, "n_kv": 4, "hd": 128, "page": 16,
         "lo": 501, "hi": 501, "empty": False, "lse": False},
        # batched serving: 32 sequences of a 30B-A3B-shaped model, ragged contexts up to 8192
        {"name": "attn_batch32", "op": "attn", "dtype": "bf16", "rows": 32, "n_q": 32, "n_kv": 4, "hd": 128, "page": 16,
         "lo": 1000, "hi": 8192, "empty": False, "lse": False},
        # one document of 131072 tokens: a single row has to fill the GPU
        {"name": "attn_long_row", "op": "attn", "dtype": "f16", "rows": 1, "n_q": 32, "n_kv": 4, "hd": 128, "page": 64,
         "lo": 131072, "hi": 131072, "empty": False, "lse": True},
        # the host driver's fp32 cache, an idle sequence among the rows
        {"name": "attn_f32", "op": "attn", "dtype": "f32", "rows": 9, "n_q": 32, "n_kv": 4, "hd": 128, "page": 16,
         "lo": 3000, "hi": 4096, "empty": True, "lse": True},
        # one decode step of 32 sequences: q, k and v are slices of one packed projection
        {"name": "rope_decode32", "op": "rope", "dtype": "bf16", "cache": "bf16", "rows": 32, "n_q": 32, "n_kv": 4,
         "hd": 128, "rot": 128, "page": 16, "far": 40000, "norm": True},
        # a prefill chunk
        {"name": "rope_prefill4096", "op": "rope", "dtype": "bf16", "cache": "bf16", "rows": 4096, "n_q": 32, "n_kv": 4,
         "hd": 128, "rot": 128, "page": 16, "far": 40000, "norm": True},
        # fp32 activations into a 16-bit cache, an odd number of rows
        {"name": "rope_f32_1001", "op": "rope", "dtype": "f32", "cache": "bf16", "rows": 1001, "n_q": 32, "n_kv": 4,
         "hd": 128, "rot": 128, "page": 16, "far": 40000, "norm": True},
        # one decode step of 32 sequences: one new token each, few new pages
        {"name": "plan_decode32", "op": "plan", "seqs": 32, "past": 8192, "new": 1, "page": 16},
        # a serving step that mixes prefill chunks with decoding sequences
        {"name": "plan_mixed512", "op": "plan", "seqs": 512, "past": 4096, "new": 128, "page": 16},
        # one decode step of 16 tokens, softmax over 128 experts, renormalised top 8
        {"name": "route_softmax16", "op": "route", "dtype": "f32", "rows": 16, "experts": 128, "top": 8, "score": "softmax",
         "groups": 1, "keep": 1, "group_top": 1, "bias": False, "renorm": True, "factor": 1.0},
        # a prefill chunk routed by sigmoid scores with a balance bias and 4 of 8 groups
        {"name": "route_groups4096", "op": "route", "dtype": "f32", "rows": 4096, "experts": 256, "top": 8, "score": "sigmoid",
         "groups": 8, "keep": 4, "group_top": 2, "bias": True, "renorm": True, "factor": 2.5},
        # a large prefill, 16-bit logits (many equal ones), weights as the softmax gives them
        {"name": "route_bf16_16384", "op": "route", "dtype": "bf16", "rows": 16384, "experts": 128, "top": 8, "score": "softmax",
         "groups": 1, "keep": 1, "group_top": 1, "bias": False, "renorm": False, "factor": 1.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope", "plan", "route"])
    if op == "attn":
        dt = rng.choice(["f32", "bf16", "bf16", "f16"])
        n_kv, group, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 16]), rng.choice([64, 80, 96, 128, 128, 256])
        rows = _log(rng, 1, 64)
        # at most the listed cases' bytes of keys and values
        most = int(240e6 / (2 * n_kv * hd * SIZES[dt] * rows))
        hi = _log(rng, 1, max(1, min(131072, most)))
        return {"op": op, "dtype": dt, "rows": rows, "n_q": n_kv * group, "n_kv": n_kv, "hd": hd,
                "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), "lo": max(1, hi // rng.choice([1, 2, 8])), "hi": hi,
                "empty": rows > 1 and rng.random() < 0.3, "lse": rng.random() < 0.5}
    if op == "rope":
        dt = rng.choice(["f32", "bf16", "f16"])
        hd = rng.choice([64, 80, 96, 128, 128, 256])
        n_kv = rng.choice([1, 2, 4, 8])
        n_q = n_kv * rng.choice([1, 2, 4, 7, 8])
        most = int(40e6 / ((n_q + 2 * n_kv) * hd * SIZES[dt]))
        return {"op": op, "dtype": dt, "cache": dt if dt != "f32" else rng.choice(["f32", "bf16", "f16"]),
                "rows": _log(rng, 1, min(4096, most)), "n_q": n_q, "n_kv": n_kv, "hd": hd,
                "rot": rng.choice([hd, hd, hd // 16 * 8]), "page": rng.choice([1, 8, 16, 24, 64]),
                "far": _log(rng, 4200, 131072), "norm": rng.random() < 0.7}
    if op == "plan":
        seqs, page = _log(rng, 1, 1024), rng.choice([1, 8, 16, 24, 64])
        return {"op": op, "seqs": seqs, "past": _log(rng, 1, min(32768, 2000000 * page // seqs)),
                "new": _log(rng, 1, max(1, 32768 // seqs)), "page": page}
    score, experts = rng.choice(["softmax", "sigmoid"]), rng.choice([8, 60, 64, 128, 160, 256, 512])
    groups = rng.choice([1, 1, 4 if experts % 8 == 0 else 2, 8 if experts % 16 == 0 else 1])
    keep = rng.randint((groups + 1) // 2, groups)
    return {"op": op, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "rows": _log(rng, 1, 8192), "experts": experts,
            "top": rng.randint(1, min(10, keep * (experts // groups))), "score": score, "groups": groups, "keep": keep,
            "group_top": rng.choice([1, 2]), "bias": rng.random() < 0.5, "renorm": rng.random() < 0.7,
            "factor": rng.choice([1.0, 2.5])}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _attn_inputs(c, g):
    dev, dt = "cuda", DTYPES[c["dtype"]]
    R, hd, nkv, ps = c["rows"], c["hd"], c["n_kv"], c["page"]
    length = torch.randint(c["lo"], c["hi"] + 1, (R,), generator=g, device=dev, dtype=torch.int32)
    if c["empty"]:
        length[R // 2] = 0
    mp = -(-c["hi"] // ps)
    n_pages = R * mp + 3
    order = torch.randperm(n_pages, generator=g, device=dev)[:R * mp].reshape(R, mp).to(torch.int32)
    # entries past a sequence's last page are not its own
    table = torch.where(torch.arange(mp, device=dev) * ps < length[:, None], order, torch.full_like(order, -1))
    # heads as the norm leaves them: unit mean square times a weight
    k = (1.5 * torch.randn(n_pages, ps, nkv, hd, generator=g, device=dev)).to(dt)
    v = torch.randn(n_pages, ps, nkv, hd, generator=g, device=dev).to(dt)
    q = (1.5 * torch.randn(R, c["n_q"], hd, generator=g, device=dev)).to(dt)
    s = {"q": q, "k": k, "v": v, "table": table, "pos": length - 1, "cap": mp * ps, "scale": 1.0 / math.sqrt(hd),
         "out": torch.empty_like(q), "lse": torch.empty(R, c["n_q"], device=dev) if c["lse"] else None}
    # partial results of a split row: m, l and one fp32 row per query head and part (at most 128 parts)
    s["work"] = torch.empty(R * c["n_q"] * min(128, max(1, -(-s["cap"] // 64))) * (hd + 2) * 4 + 1024, dtype=torch.uint8, device=dev)
    return s


def _rope_inputs(c, g):
    dev, dt, ct = "cuda", DTYPES[c["dtype"]], DTYPES[c["cache"]]
    R, nq, nkv, hd, ps, rot = c["rows"], c["n_q"], c["n_kv"], c["hd"], c["page"], c["rot"]
    qkv = torch.randn(R, (nq + 2 * nkv) * hd, generator=g, device=dev).to(dt)
    n_pages = -(-R // ps) + 5
    i = torch.arange(0, rot, 2, device=dev, dtype=torch.float64)
    angle = torch.arange(c["far"], device=dev, dtype=torch.float64)[:, None] * (1e6 ** (-i / max(rot, 1)))
    table = torch.cat([angle.cos(), angle.sin()], 1).float()
    return {"q": qkv[:, :nq * hd].unflatten(1, (nq, hd)), "k": qkv[:, nq * hd:(nq + nkv) * hd].unflatten(1, (nkv, hd)),
            "v": qkv[:, (nq + nkv) * hd:].unflatten(1, (nkv, hd)), "rope": table,
            "pos": torch.randint(0, c["far"], (R,), generator=g, device=dev, dtype=torch.int32),
            "slot": torch.randperm(n_pages * ps, generator=g, device=dev)[:R].to(torch.int32),
            "q_norm": 1 + 0.2 * torch.randn(hd, generator=g, device=dev) if c["norm"] else None,
            "k_norm": 1 + 0.2 * torch.randn(hd, generator=g, device=dev) if c["norm"] else None, "eps": 1e-6,
            "q_out": torch.empty(R, nq, hd, dtype=ct, device=dev),
            "kc": torch.randn(n_pages, ps, nkv, hd, generator=g, device=dev).to(ct),
            "vc": torch.randn(n_pages, ps, nkv, hd, generator=g, device=dev).to(ct)}


def _plan_inputs(c, g):
    dev, n, ps = "cuda", c["seqs"], c["page"]
    past = torch.randint(0, c["past"] + 1, (n,), generator=g, device=dev, dtype=torch.int32)
    new = torch.ones(n, dtype=torch.int32, device=dev)
    if c["new"] > 1:  # most sequences decode, some bring a piece of a prompt, some are idle
        kind = torch.rand(n, generator=g, device=dev)
        many = torch.randint(1, 2 * c["new"], (n,), generator=g, device=dev, dtype=torch.int32)
        new = torch.where(kind < 0.5, many, torch.where(kind < 0.55, torch.zeros_like(new), new))
    mp = -(-(c["past"] + 2 * c["new"]) // ps)
    cap = 2 * n * c["new"]
    n_pages = n * mp
    pages = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    held = (past.long() + ps - 1) // ps
    at = torch.cumsum(held, 0) - held
    j = torch.arange(mp, device=dev)
    table = torch.where(j < held[:, None], pages[(at[:, None] + j).clamp(max=n_pages - 1)], torch.full((n, mp), -1, dtype=torch.int32, device=dev))
    return {"past": past, "new": new, "page": ps, "n_pages": n_pages, "free": pages[int(held.sum()):].clone(),
            "head": torch.randint(0, 8, (1,), generator=g, device=dev, dtype=torch.int32), "table": table,
            "kv_len": torch.empty(n, dtype=torch.int32, device=dev),
            "rows": torch.empty(3, cap, dtype=torch.int32, device=dev), "head_out": torch.empty(1, dtype=torch.int32, device=dev),
            "status": torch.empty(3, dtype=torch.int32, device=dev)}


def _route_inputs(c, g):
    dev, T, E = "cuda", c["rows"], c["experts"]
    # router logits spread over experts of unequal popularity
    lean = torch.randn(E, generator=g, device=dev)
    x = (1.5 * torch.randn(T, E, generator=g, device=dev) + lean).to(DTYPES[c["dtype"]])
    return {"logits": x, "bias": 0.1 * torch.randn(E, generator=g, device=dev) if c["bias"] else None,
            "idx": torch.empty(T, c["top"], dtype=torch.int32, device=dev), "p": torch.empty(T, c["top"], device=dev)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    make = {"attn": _attn_inputs, "rope": _rope_inputs, "plan": _plan_inputs, "route": _route_inputs}[case["op"]]
    return {"case": dict(case), **make(case, g)}


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _attn_plain(s):
    q, pos, table = s["q"].float(), s["pos"], s["table"].long().clamp(min=0)
    R, nq, hd = q.shape
    nkv = s["k"].shape[2]
    k = s["k"][table].flatten(1, 2).float()                          # [R, cap, n_kv, hd]
    v = s["v"][table].flatten(1, 2).float()
    inside = torch.arange(k.shape[1], device=q.device) <= pos[:, None]
    score = torch.matmul(q.view(R, nkv, nq // nkv, hd), k.permute(0, 2, 3, 1)) * s["scale"]
    score = score.masked_fill(~inside[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    v = v.masked_fill(~inside[:, :, None, None], 0.0)
    out = torch.matmul(e, v.permute(0, 2, 1, 3)) / torch.where(total == 0, torch.ones_like(total), total)
    got = {"out": out.reshape(R, nq, hd).to(s["q"].dtype)}
    if s["lse"] is not None:
        got["lse"] = (top + torch.log(total)).reshape(R, nq)
    return got


def _rotate(x, weight, eps, cs, rot):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    cos, sin = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _rope_plain(s):
    rot = s["rope"].shape[1]
    cs = s["rope"][s["pos"].long()]
    slot = s["slot"].long()
    q = _rotate(s["q"], s["q_norm"], s["eps"], cs, rot).to(s["kc"].dtype)
    s["kc"].view(-1, *s["kc"].shape[2:])[slot] = _rotate(s["k"], s["k_norm"], s["eps"], cs, rot).to(s["kc"].dtype)
    s["vc"].view(-1, *s["vc"].shape[2:])[slot] = s["v"].to(s["vc"].dtype)
    return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}


def _plan_plain(s):
    past, new, ps, table, free = s["past"].long(), s["new"].long(), s["page"], s["table"], s["free"]
    n, mp = table.shape
    held = ((past + ps - 1) // ps).clamp(max=mp)
    need = ((past + new + ps - 1) // ps).clamp(max=mp) - held
    row_end, page_end = torch.cumsum(new, 0), torch.cumsum(need, 0)
    head = s["head"].long()
    # new pages, in the order of the sequences
    j = torch.arange(mp, device=past.device)
    at = head + (page_end - need)[:, None] + j - held[:, None]
    fresh = (j >= held[:, None]) & (j < (held + need)[:, None])
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)].int(), torch.full_like(table, -1))
    table.copy_(torch.where(fresh, page, table))
    # rows
    cap = s["rows"].shape[1]
    i = torch.arange(cap, device=past.device)
    seq = torch.searchsorted(row_end, i, right=True)
    live = seq < n
    seq = seq.clamp(max=n - 1)
    pos = past[seq] + i - (row_end - new)[seq]
    where = table[seq, (pos // ps).clamp(0, mp - 1)].long()
    good = live & (pos // ps < mp) & (where >= 0) & (where < s["n_pages"])
    none = torch.full_like(i, -1)
    asked = page_end[-1:]
    taken = torch.minimum(asked, (free.numel() - head).clamp(min=0))
    return {"table": table, "kv_len": (past + new).int(), "row_seq": torch.where(live, seq, none).int(),
            "row_pos": torch.where(live, pos, none).int(), "row_slot": torch.where(good, where * ps + pos % ps, none).int(),
            "head": (head + taken).int(), "status": torch.cat([row_end[-1:], asked, taken]).int()}


def _route_plain(s):
    c, x = s["case"], s["logits"].double()
    T, E = x.shape
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score + s["bias"].double() if s["bias"] is not None else score
    rank = choice if s["bias"] is not None else x        # without a bias the logits order the scores
    if c["groups"] > 1:
        best = torch.sort(choice.view(T, c["groups"], -1), dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
        in_group = torch.zeros_like(best).scatter(1, kept, 1.0).repeat_interleave(E // c["groups"], 1)
        rank = torch.where(in_group > 0, rank, torch.full_like(rank, -math.inf))
    idx = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
    p = score.gather(1, idx)
    if c["renorm"]:
        p = p / p.sum(-1, keepdim=True)
    return {"idx": idx.int(), "p": (p * c["factor"]).float()}


# ---- the framework's calls -----------------------------------------------------------------------------------------------

def _attn_own(s):
    _mc().paged_attention(s["q"], s["k"], s["v"], s["table"], s["pos"], s["out"], s["work"], s["cap"], s["scale"], lse=s["lse"])
    return {"out": s["out"]} if s["lse"] is None else {"out": s["out"], "lse": s["lse"]}


def _rope_own(s):
    _mc().qk_norm_rope(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["pos"], s["slot"], s["q_out"], rope=s["rope"],
                       q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"])
    return {"q": s["q_out"], "k_cache": s["kc"], "v_cache": s["vc"]}


def _plan_own(s):
    r = s["rows"]
    _mc().kv_plan(s["past"], s["new"], s["page"], s["n_pages"], s["free"], s["table"], r[0], r[1], r[2], kv_len=s["kv_len"],
                  free_head=s["head"], free_head_out=s["head_out"], status=s["status"])
    return {"table": s["table"], "kv_len": s["kv_len"], "row_seq": r[0], "row_pos": r[1], "row_slot": r[2],
            "head": s["head_out"], "status": s["status"]}


def _route_own(s):
    c = s["case"]
    _mc().route(s["logits"], s["idx"], s["p"], bias=s["bias"], score=c["score"], groups=c["groups"], keep_groups=c["keep"],
                group_top=c["group_top"], renorm=c["renorm"], scale=c["factor"])
    return {"idx": s["idx"], "p": s["p"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _attn_own, "rope": _rope_own, "plan": _plan_own, "route": _route_own}[op](state)
    return {"attn": _attn_plain, "rope": _rope_plain, "plan": _plan_plain, "route": _route_plain}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "attn":
        es = SIZES[c["dtype"]]
        keys = (c["rows"] - bool(c["empty"])) * (c["lo"] + c["hi"]) / 2
        qo = 2 * c["rows"] * c["n_q"] * c["hd"] * es
        table = 4 * keys / c["page"]
        return {"bytes": 2 * keys * c["n_kv"] * c["hd"] * es + qo + table + 4 * c["rows"] * (1 + c["lse"] * c["n_q"]),
                "flops": 4 * keys * c["n_q"] * c["hd"]}
    if c["op"] == "rope":
        n = c["rows"] * (c["n_q"] + 2 * c["n_kv"]) * c["hd"]
        return {"bytes": n * (SIZES[c["dtype"]] + SIZES[c["cache"]]) + c["rows"] * (8 + 4 * c["rot"]),
                "flops": c["rows"] * (c["n_q"] + c["n_kv"]) * (3 * c["rot"] + 4 * c["hd"] * bool(c["norm"]))}
    if c["op"] == "plan":
        new = c["new"] if c["new"] == 1 else 0.5 * c["new"] + 0.45
        rows, pages = c["seqs"] * new, c["seqs"] * new / c["page"]
        return {"bytes": 12 * c["seqs"] + 8 * pages + 12 * 2 * c["seqs"] * c["new"] + 4 * min(rows, c["seqs"]), "flops": 0}
    n = c["rows"] * c["experts"]
    return {"bytes": n * SIZES[c["dtype"]] + 8 * c["rows"] * c["top"] + 4 * c["experts"] * bool(c["bias"]), "flops": 4 * n}


# ---- 64 bits, from the definitions ---------------------------------------------------------------------------------------

def _attn_exact(s):
    q, ps = s["q"].double(), s["k"].shape[1]
    R, nq, hd = q.shape
    group = nq // s["k"].shape[2]
    out, lse = torch.zeros_like(q), torch.full((R, nq), -math.inf, dtype=torch.float64, device=q.device)
    for r in range(R):
        n = int(s["pos"][r]) + 1
        if n == 0:
            continue
        pages = s["table"][r, :-(-n // ps)].long()
        k, v = (s[x][pages].reshape(-1, *s[x].shape[2:])[:n].double() for x in ("k", "v"))
        for h in range(nq):
            logit = (k[:, h // group] @ q[r, h]) * s["scale"]
            lse[r, h] = torch.logsumexp(logit, 0)
            out[r, h] = torch.exp(logit - lse[r, h]) @ v[:, h // group]
    return {"out": out, "lse": lse} if s["lse"] is not None else {"out": out}


def _rope_exact(s):
    rot = s["rope"].shape[1]
    angle = s["rope"][s["pos"].long()].double()
    unit = torch.complex(angle[:, :rot // 2], angle[:, rot // 2:])[:, None]
    made = {}
    for name, weight in (("q", s["q_norm"]), ("k", s["k_norm"])):
        x = s[name].double()
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]) * weight.double()
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * unit
        made[name] = torch.cat([z.real, z.imag, x[..., rot:]], -1)
    kc, vc = s["kc"].double(), s["vc"].double()
    ps = kc.shape[1]
    page, off = s["slot"].long() // ps, s["slot"].long() % ps
    kc[page, off] = made["k"]
    vc[page, off] = s["v"].double()
    return {"q": made["q"], "k_cache": kc, "v_cache": vc}


def _route_exact(s):
    c, x = s["case"], s["logits"].double().cpu()
    score = torch.softmax(x, -1) if c["score"] == "softmax" else torch.sigmoid(x)
    bias = torch.zeros(x.shape[1], dtype=torch.float64) if s["bias"] is None else s["bias"].double().cpu()
    choice = score + bias
    size = x.shape[1] // c["groups"]
    order = []
    best = choice.unfold(1, size, size).topk(min(c["group_top"], size), -1).values.sum(-1)
    for t in range(x.shape[0]):
        kept = sorted(range(c["groups"]), key=lambda j: -float(best[t, j]))[:c["keep"]]
        mine = sorted(e for j in kept for e in range(j * size, (j + 1) * size))
        key = x[t].tolist() if s["bias"] is None else choice[t].tolist()
        order.append(sorted(mine, key=lambda e: -key[e])[:c["top"]])
    idx = torch.tensor(order)
    p = torch.gather(score, 1, idx)
    if c["renorm"]:
        p = p / p.sum(1, keepdim=True)
    return {"idx": idx.int(), "p": p * c["factor"]}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return {"attn": _attn_exact, "rope": _rope_exact, "route": _route_exact}[case["op"]](s)
