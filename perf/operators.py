"""The serving operators on device buffers, measured: for each of them the cases of real use, a plain form in elementary
torch operations, and the call that a user makes.

  page_map     block tables and slot maps made on the GPU from the requests' lengths
  page_write   new K and V rows into the pages those slots name
  prefix_attn  attention of one new token per conversation over a prompt all conversations share and their own pages
  sample       a word per row of scores by temperature, top-k, top-p and min-p from a given uniform number

`own` False: the plain form; True: this framework's kernels (nunchi_b200).
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the decode step of 64 conversations: each adds one position, one in `page` of them opens a page
        {"name": "map decode 64", "op": "map", "n": 64, "page": 64, "held_max": 1300, "add_max": 1, "cap": 64},
        # a full intake: prompts of up to 4,000 words of 384 requests mapped at once (odd lengths, some adding nothing)
        {"name": "map prompts 384", "op": "map", "n": 384, "page": 16, "held_max": 700, "add_max": 4000, "cap": 1000000},
        # the K and V rows of that decode step as the projection leaves them (32 bits) into 16-bit pages
        {"name": "write decode 64", "op": "write", "rows": 64, "kv": 8, "d": 64, "src": "f32", "dst": "f16", "page": 64,
         "n_pages": 700, "pad": 3},
        # a prompt's rows, heads of 128, with unused rows at the end of the batch
        {"name": "write prompt 16000", "op": "write", "rows": 16000, "kv": 8, "d": 128, "src": "bf16", "dst": "bf16",
         "page": 32, "n_pages": 900, "pad": 77},
        # one conversation at its start: a short prompt and a few own positions; latency is all that counts
        {"name": "attn 1 short", "op": "attn", "n": 1, "kv": 8, "g": 4, "d": 64, "dt": "f16", "page": 64, "prefix": 37,
         "own_max": 6, "window": 0, "pad": 0},
        # 64 conversations on one prompt of 1,000 words, own contexts of up to 1,000: the engine's batched decode step
        {"name": "attn 64 on 1000", "op": "attn", "n": 64, "kv": 8, "g": 4, "d": 64, "dt": "f16", "page": 64,
         "prefix": 1000, "own_max": 1000, "window": 0, "pad": 0},
        # heads of 128 in few kv heads with a sliding window, an odd prompt, and a batch padded to its captured size
        {"name": "attn 24 window", "op": "attn", "n": 24, "kv": 2, "g": 4, "d": 128, "dt": "bf16", "page": 32,
         "prefix": 9001, "own_max": 2500, "window": 8192, "pad": 3},
        # the largest batch on a long instruction prompt, each conversation still short: the shared part is nearly all
        {"name": "attn 256 on 16384", "op": "attn", "n": 256, "kv": 8, "g": 4, "d": 64, "dt": "f16", "page": 128,
         "prefix": 16384, "own_max": 256, "window": 0, "pad": 0},
        # one conversation's word over the engine's word table, the usual settings
        {"name": "sample 1 k50 p95", "op": "sample", "n": 1, "vocab": 97496, "dt": "f32", "t": 0.8, "k": 50, "p": 0.95,
         "m": 0.0, "mixed": False},
        # 64 conversations by nucleus alone: no top-k to shorten the row first
        {"name": "sample 64 p90", "op": "sample", "n": 64, "vocab": 97496, "dt": "f32", "t": 1.0, "k": 0, "p": 0.9,
         "m": 0.0, "mixed": False},
        # the largest batch, every conversation with its own settings (greedy ones among them), 16-bit scores with ties
        {"name": "sample 256 mixed", "op": "sample", "n": 256, "vocab": 97496, "dt": "bf16", "t": 0.9, "k": 40, "p": 0.92,
         "m": 0.05, "mixed": True},
        # a small word table of odd size, min-p alone
        {"name": "sample 33 small", "op": "sample", "n": 33, "vocab": 1003, "dt": "f16", "t": 1.3, "k": 0, "p": 1.0,
         "m": 0.02, "mixed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["map", "write", "attn", "attn", "sample", "sample"])
    if op == "map":
        n, add = _log(rng, 1, 1000), rng.choice([1, 1, _log(rng, 2, 4000)])
        return {"op": op, "n": n, "page": rng.choice([16, 32, 64, 128]), "held_max": _log(rng, 1, 8000), "add_max": add,
                "cap": min(1000000, n * add + rng.randrange(0, 50))}
    if op == "write":
        d, kv, rows = rng.choice([64, 128]), rng.randint(1, 8), _log(rng, 1, 16000)
        page, dst = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
        return {"op": op, "rows": rows, "kv": kv, "d": d, "src": rng.choice(["f32", dst]), "dst": dst, "page": page,
                "n_pages": (rows + page - 1) // page + rng.randint(1, 200), "pad": rng.randint(0, min(9, rows - 1))}
    if op == "attn":
        n, kv, g, d = _log(rng, 1, 256), rng.randint(1, 8), rng.choice([1, 2, 3, 4, 5, 6, 8, 16]), rng.choice([64, 128])
        g = min(g, 32 // kv)
        prefix, own_max = rng.choice([0, _log(rng, 1, 16384)]), _log(rng, 1, 2500)
        while n * kv * d * own_max > 256 * 8 * 64 * 400:   # no more rows to read than the largest listed case has
            own_max = max(1, own_max // 2)
        return {"op": op, "n": n, "kv": kv, "g": g, "d": d, "dt": rng.choice(["f16", "bf16"]),
                "page": rng.choice([16, 32, 64, 128]), "prefix": prefix // (1 if d == 64 else 2), "own_max": own_max,
                "window": rng.choice([0, 0, _log(rng, 1, 16384)]), "pad": rng.randint(0, 2) if n > 4 else 0}
    v = _log(rng, 500, 130000)
    return {"op": op, "n": min(_log(rng, 1, 256), 256 * 97496 // v), "vocab": v, "dt": rng.choice(["f32", "f16", "bf16"]),
            "t": round(rng.uniform(0.3, 1.6), 3), "k": rng.choice([0, 1, _log(rng, 2, 2000)]),
            "p": rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)]), "m": rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]),
            "mixed": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"map": _prep_map, "write": _prep_write, "attn": _prep_attn, "sample": _prep_sample}[case["op"]](case, g)


def _ints(g, lo, hi, shape):   # lo..hi, both included
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _prep_map(c, g):
    n, page = c["n"], c["page"]
    held = _ints(g, 0, c["held_max"], (n,))
    add = _ints(g, 0 if c["add_max"] > 1 else 1, c["add_max"], (n,))
    # no more tokens than the step's slot arrays hold
    add = torch.minimum(add, (c["cap"] - torch.cumsum(add, 0) + add).clamp(min=0).to(torch.int32)).to(torch.int32)
    width = (c["held_max"] + c["add_max"] + page - 1) // page
    n_pages = n * width + 5
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    # the requests' tables hold the pages of what they have; the rest of the shuffled pages is free
    have = (held + page - 1) // page
    first = torch.cumsum(have, 0) - have
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    table = torch.where(col < have[:, None], order[(first[:, None] + col).clamp(max=n_pages - 1).long()], -1).to(torch.int32)
    used = have.sum()
    at = torch.arange(n_pages, device="cuda")
    free = torch.where(at < n_pages - used, order[(at + used).clamp(max=n_pages - 1)], 0).to(torch.int32)
    z = lambda k: torch.zeros(k, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"case": c, "held": held, "add": add, "table": table, "free": free, "n_free": (n_pages - used).to(torch.int32).reshape(1),
            "n_pages": n_pages, "pos0": 1000, "start": z(n + 1), "len": z(n), "slots": z(c["cap"]), "pos": z(c["cap"]),
            "n_free_out": z(1), "status": z(2)}


def _prep_write(c, g):
    rows, kv, d = c["rows"], c["kv"], c["d"]
    # K and V as columns of the stacked projection's rows, heads after the query's
    big = torch.randn((rows, 3 * kv * d + 8), generator=g, device="cuda", dtype=torch.float32).to(DT[c["src"]])
    k = big[:, kv * d:2 * kv * d].unflatten(1, (kv, d))
    v = big[:, 2 * kv * d:3 * kv * d].unflatten(1, (kv, d))
    slots = torch.randperm(c["n_pages"] * c["page"], generator=g, device="cuda", dtype=torch.int32)[:rows].contiguous()
    if c["pad"]:
        slots[-c["pad"]:] = -1
    shape = (c["n_pages"], kv, c["page"], d)
    pages = [torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(DT[c["dst"]]) for _ in range(2)]
    return {"case": c, "k": k, "v": v, "slots": slots, "k_pages": pages[0], "v_pages": pages[1],
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prep_attn(c, g):
    n, kv, d, page, dt = c["n"], c["kv"], c["d"], c["page"], DT[c["dt"]]
    heads, pp, width = kv * c["g"], (c["prefix"] + page - 1) // page, (c["own_max"] + page - 1) // page
    n_pages = pp + n * width + 3
    shape = (n_pages, kv, page, d)
    # normed and rotated queries and keys are of unit size per component; the prompt's first positions draw the
    # attention that first positions draw
    k = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    v = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    q = torch.randn((n, heads, d), generator=g, device="cuda", dtype=torch.float32) * 1.5
    order = torch.randperm(n_pages, generator=g, device="cuda", dtype=torch.int32)
    length = _ints(g, 0, c["own_max"], (n,))
    length[0] = c["own_max"]
    if c["pad"]:
        length[-c["pad"]:] = -1
    return {"case": c, "q": q.to(dt), "k_pages": k.to(dt), "v_pages": v.to(dt), "prefix": order[:pp].contiguous(),
            "table": order[pp:pp + n * width].reshape(n, width).contiguous(), "len": length, "scale": d ** -0.5,
            "out": torch.zeros((n, heads, d), dtype=dt, device="cuda"), "lse": torch.zeros((n, heads), device="cuda"),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prep_sample(c, g):
    n, v = c["n"], c["vocab"]
    # word scores fall off with the word's rank about as its frequency does, steeper or flatter from row to row
    rank = torch.rand((n, v), generator=g, device="cuda").argsort(1)
    steep = 0.8 + 0.8 * torch.rand((n, 1), generator=g, device="cuda")
    x = -steep * torch.log1p(rank.float()) * 1.5 + 0.6 * torch.randn((n, v), generator=g, device="cuda") + 12.0
    x = torch.where(torch.rand((n, v), generator=g, device="cuda") < 0.01, -math.inf, x)   # words not allowed here
    full = lambda val, t: torch.full((n,), val, dtype=t, device="cuda")  # noqa: E731
    t, k, p, m = full(c["t"], torch.float32), full(c["k"], torch.int32), full(c["p"], torch.float32), full(c["m"], torch.float32)
    if c["mixed"]:
        i = torch.arange(n, device="cuda")
        t = torch.where(i % 5 == 4, 0.0, t * (0.7 + 0.6 * torch.rand(n, generator=g, device="cuda")))
        k = torch.where(i % 3 == 0, 0, k).to(torch.int32)
        p = torch.where(i % 4 == 1, 1.0, p)
        m = torch.where(i % 2 == 0, 0.0, m)
    return {"case": c, "scores": x.to(DT[c["dt"]]), "u": torch.rand(n, generator=g, device="cuda"), "t": t, "k": k, "p": p, "m": m,
            "ids": torch.zeros(n, dtype=torch.int32, device="cuda"), "logprob": torch.zeros(n, device="cuda"),
            "kept": torch.zeros(n, dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"map": _run_map, "write": _run_write, "attn": _run_attn, "sample": _run_sample}[state["case"]["op"]](state)


def _run_map(s):
    c = s["case"]
    if own:
        import nunchi_b200 as nb
        nb.page_map(s["held"], s["add"], s["table"], s["free"], s["n_free"], page=c["page"], n_pages=s["n_pages"], pos0=s["pos0"],
                    start=s["start"], length=s["len"], slots=s["slots"], pos=s["pos"], n_free_out=s["n_free_out"],
                    status=s["status"])
        return {k: s[k] for k in ("table", "start", "len", "slots", "pos", "n_free_out")}
    held, add, page, table = s["held"], s["add"], c["page"], s["table"]
    total, have = held + add, (held + page - 1) // page
    want = (total + page - 1) // page
    need = want - have
    first = torch.cumsum(need, 0) - need
    start = torch.nn.functional.pad(torch.cumsum(add, 0), (1, 0)).to(torch.int32)
    col = torch.arange(table.shape[1], device="cuda", dtype=torch.int32)
    taken = s["n_free"] - 1 - (first[:, None] + col - have[:, None])
    table = torch.where((col >= have[:, None]) & (col < want[:, None]), s["free"][taken.clamp(0, s["free"].numel() - 1).long()], table)
    at = torch.arange(c["cap"], device="cuda", dtype=torch.int32)
    req = torch.searchsorted(start[1:].contiguous(), at, right=True).clamp(max=c["n"] - 1)
    p = held[req] + at - start[req]
    live = at < start[-1]
    slot = table[req, (p // page).clamp(0, table.shape[1] - 1).long()] * page + p % page
    return {"table": table, "start": start, "len": total, "slots": torch.where(live, slot, -1).to(torch.int32),
            "pos": torch.where(live, p + s["pos0"], -1).to(torch.int32), "n_free_out": (s["n_free"] - need.sum()).to(torch.int32)}


def _run_write(s):
    c = s["case"]
    if own:
        import nunchi_b200 as nb
        nb.page_write(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"], status=s["status"])
        return s["k_pages"], s["v_pages"]
    live = s["slots"] >= 0
    slot = s["slots"][live].long()
    for src, dst in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        dst[slot // c["page"], :, slot % c["page"]] = src[live].to(torch.float32).to(dst.dtype)
    return s["k_pages"], s["v_pages"]


def _gather(pages, index, count):
    """The first `count` positions of the pages that `index` (..., pages) names, in 32 bits: (..., kv, count, d)."""
    x = pages[index.long()].float()                                    # (..., pages, kv, page, d)
    return x.movedim(-3, -4).flatten(-3, -2)[..., :count, :]


def _run_attn(s):
    c = s["case"]
    if own:
        import nunchi_b200 as nb
        if "work" not in s:
            s["work"] = nb.prefix_attn_work(s["q"], s["k_pages"], c["prefix"], s["table"])
        nb.prefix_attn(s["q"], s["k_pages"], s["v_pages"], s["prefix"], c["prefix"], s["table"], s["len"], scale=s["scale"],
                       window=c["window"], out=s["out"], lse=s["lse"], work=s["work"], status=s["status"])
        return s["out"], s["lse"]
    n, kv, g, d, P, L = c["n"], c["kv"], c["g"], c["d"], c["prefix"], c["own_max"]
    q = s["q"].float().unflatten(1, (kv, g)) * s["scale"]              # (n, kv, g, d)
    kp, vp = (_gather(s[x], s["prefix"], P) for x in ("k_pages", "v_pages"))      # (kv, P, d)
    ko, vo = (_gather(s[x], s["table"], L) for x in ("k_pages", "v_pages"))       # (n, kv, L, d)
    qk = q.transpose(0, 1).reshape(kv, n * g, d)
    shared = torch.bmm(qk, kp.transpose(1, 2)).reshape(kv, n, g, P).transpose(0, 1)
    score = torch.cat((shared, torch.matmul(q, ko.transpose(2, 3))), -1)          # (n, kv, g, P + L)
    at, end = torch.arange(P + L, device="cuda"), P + s["len"].clamp(min=0)
    low = end - c["window"] if c["window"] else torch.zeros_like(end)
    seen = (at < end[:, None]) & (at >= low[:, None])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.bmm(e[..., :P].transpose(0, 1).reshape(kv, n * g, P), vp).reshape(kv, n, g, d).transpose(0, 1)
    o = (o + torch.matmul(e[..., P:], vo)) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1).flatten(1)
    live = s["len"] >= 0
    return (torch.where(live[:, None, None], o.flatten(1, 2).to(s["out"].dtype), s["out"]), torch.where(live[:, None], lse, s["lse"]))


def _run_sample(s):
    if own:
        import nunchi_b200 as nb
        nb.sample(s["scores"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"], ids=s["ids"],
                  logprob=s["logprob"], kept=s["kept"])
        return s["ids"], s["logprob"], s["kept"]
    # in 64 bits: which word a uniform number names, and which word a nucleus ends at, are decided next to borders
    x = s["scores"].double()
    n, V = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    t, k, p, m, u = s["t"].double(), s["k"].long(), s["p"].double(), s["m"].double(), s["u"].double()
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = xs[:, :1]
    greedy = ~(t > 0)
    ws = torch.where(xs == top, 1.0, torch.exp((xs - top) / torch.where(greedy, 1.0, t)[:, None]))
    ws = torch.where(xs == -math.inf, 0.0, ws)
    at = torch.arange(V, device="cuda")
    k = torch.where((k <= 0) | (k > V), V, k)
    keep = (at < k[:, None]) & (xs > -math.inf)
    cum = torch.cumsum(torch.where(keep, ws, 0.0), 1)
    before = torch.nn.functional.pad(cum[:, :-1], (1, 0))
    keep &= (at == 0) | ~(p < 1)[:, None] | (before < p[:, None] * cum[:, -1:])
    keep &= (at == 0) | ~(m > 0)[:, None] | (ws >= m.clamp(max=1.0)[:, None])
    keep &= ~greedy[:, None] | (at == 0)
    w = torch.zeros_like(x).scatter_(1, order, torch.where(keep, ws, 0.0))
    cum = torch.cumsum(w, 1)
    ids = (cum <= u[:, None] * cum[:, -1:]).sum(1).clamp(max=V - 1)
    ids = torch.where(greedy, order[:, 0], ids)
    xi = x.gather(1, ids[:, None])
    lp = torch.where(xi == top, 0.0, (xi - top) / torch.where(greedy, 1.0, t)[:, None]).squeeze(1) - torch.log(cum[:, -1])
    none = top.squeeze(1) == -math.inf
    return (torch.where(none, -1, ids).to(torch.int32), torch.where(none, -math.inf, torch.where(greedy, 0.0, lp)).float(),
            keep.sum(1).to(torch.int32))


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "map":
        adds = min(c["cap"], c["n"] * (1 if c["add_max"] == 1 else c["add_max"] / 2))
        return {"bytes": 8 * c["cap"] + 20 * c["n"] + 8 * adds / c["page"], "flops": 0}
    if c["op"] == "write":
        size = {"f32": 4, "f16": 2, "bf16": 2}
        return {"bytes": 2 * (c["rows"] - c["pad"]) * c["kv"] * c["d"] * (size[c["src"]] + size[c["dst"]]) + 4 * c["rows"], "flops": 0}
    if c["op"] == "attn":
        n, own_mean = c["n"] - c["pad"], (c["own_max"] + c["own_max"] / max(1, c["n"])) / 2
        shared = c["prefix"]
        if c["window"]:
            own_mean = min(own_mean, c["window"])
            shared = min(shared, c["window"])   # most that a query sees of it
        rows = shared + n * own_mean
        heads = c["kv"] * c["g"]
        return {"bytes": 4 * rows * c["kv"] * c["d"] + 4 * n * heads * (c["d"] + 1),
                "flops": 4 * n * heads * (shared + own_mean) * c["d"]}
    return {"bytes": c["n"] * (c["vocab"] * (4 if c["dt"] == "f32" else 2) + 32), "flops": 0}


# ------------------------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    if case["op"] == "write":
        return _exact_write(case, s)
    return _exact_sample(case, s) if case["op"] == "sample" else None


def _exact_write(c, s):
    """Row by row: the rows' values, unrounded, where their slots say."""
    out = [s["k_pages"].double(), s["v_pages"].double()]
    for src, dst in ((s["k"], out[0]), (s["v"], out[1])):
        flat = dst.transpose(1, 2).reshape(-1, c["kv"], c["d"])        # every position of every page
        for r, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                flat[slot] = src[r].double()
        dst.copy_(flat.reshape(c["n_pages"], c["page"], c["kv"], c["d"]).transpose(1, 2))
    return out


def _exact_attn(c, s):
    """Row by row: every key the row may see, one after the other, and the softmax over them."""
    kv, g, d, page, P = c["kv"], c["g"], c["d"], c["page"], c["prefix"]
    K, V = s["k_pages"].double(), s["v_pages"].double()
    rows = lambda pages, ids: pages[ids.long()].permute(1, 0, 2, 3).reshape(kv, -1, d)  # noqa: E731
    pk, pv = rows(K, s["prefix"])[:, :P], rows(V, s["prefix"])[:, :P]
    out, lse = s["out"].double(), s["lse"].double()
    for i, L in enumerate(s["len"].tolist()):
        if L < 0:
            continue
        held = s["table"][i, :(L + page - 1) // page]
        k, v = torch.cat((pk, rows(K, held)[:, :L]), 1), torch.cat((pv, rows(V, held)[:, :L]), 1)
        if c["window"]:
            k, v = k[:, -c["window"]:], v[:, -c["window"]:]
        if k.shape[1] == 0:
            out[i], lse[i] = 0.0, -math.inf
            continue
        a = torch.einsum("hgd,hpd->hgp", s["q"][i].double().reshape(kv, g, d), k) / math.sqrt(d)
        z = torch.logsumexp(a, 2)
        out[i] = torch.einsum("hgp,hpd->hgd", torch.exp(a - z[..., None]), v).reshape(kv * g, d)
        lse[i] = z.reshape(-1)
    return out, lse


def _exact_sample(c, s):
    """Row by row on the host: the words sorted, cut three times, and walked in their own order."""
    x = s["scores"].double().cpu().numpy()
    u, t, k, p, m = (s[n].double().cpu().numpy() for n in ("u", "t", "k", "p", "m"))
    ids, lps, counts = [], [], []
    for i in range(x.shape[0]):
        words = np.flatnonzero(x[i] > -np.inf)
        if words.size == 0:
            ids.append(-1), lps.append(-np.inf), counts.append(0)
            continue
        words = words[np.argsort(-x[i][words], kind="stable")]
        if not t[i] > 0:
            words = words[:1]
        else:
            e = np.exp((x[i][words] - x[i][words[0]]) / t[i])
            if 0 < k[i] < words.size:
                words, e = words[:int(k[i])], e[:int(k[i])]
            if p[i] < 1:
                n = max(1, int(np.searchsorted(np.cumsum(e), p[i] * e.sum())) + 1)
                words, e = words[:n], e[:n]
            if m[i] > 0:
                words = words[:max(1, int((e >= m[i]).sum()))]
        words = np.sort(words)
        e = np.exp((x[i][words] - x[i][words].max()) / t[i]) if t[i] > 0 else np.ones(1)
        at = min(int(np.searchsorted(np.cumsum(e), u[i] * e.sum(), side="right")), words.size - 1)
        ids.append(int(words[at])), lps.append(float(np.log(e[at] / e.sum()))), counts.append(int(words.size))
    return np.array(ids), np.array(lps, np.float64), np.array(counts)
