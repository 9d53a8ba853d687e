"""The operators of the F16 KV cache beside single-sequence decode attention, with their inputs,
plain forms and 64-bit results, for timing.

  rope    KVCacheF16.store_rope_dev: rotate the query and key heads of n tokens by their positions
          (interleaved or half layout, all or part of the head, scaled frequencies) and store the
          rotated keys and the values as cache rows
  shared  KVCacheF16.attend_shared_dev: one decode token for each of n requests that share a
          prefix of the cache, read once for all, and have rows of their own behind it
  mass    KVCacheF16.attend_mass_dev: causal attention of the last n tokens that also adds up the
          weight every cached row received, per kv head
  keep    KVCacheF16.keep_dev: per layer and kv head, the `budget` rows of most accumulated weight
          (first and newest positions always) copied into a smaller cache
  evict   KVCacheF16.evict_store_dev: per kv head, a new token's row in place of the row of least
          accumulated weight

Queries, keys and values are N(0, 1); accumulated weights fall off as the -0.8th power of a random
rank, the few-heavy, many-light shape that attention gives them.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one decode step of a llama layer: the smallest call, all latency
        {"name": "rope_step", "kind": "rope", "n": 1, "heads": 32, "kv": 8, "hd": 128, "rot": 128, "layout": "interleaved",
         "scaling": "none", "first": 4000, "rows": 4096},
        # a prompt chunk of a model that rotates half of each head, in halves, past its trained context
        {"name": "rope_prompt", "kind": "rope", "n": 4001, "heads": 32, "kv": 8, "hd": 128, "rot": 64, "layout": "half",
         "scaling": "yarn", "first": 100000, "rows": 4096},
        # two short chats behind a system prompt on a small model: latency again
        {"name": "shared_pair", "kind": "shared", "n": 2, "heads": 8, "kv": 2, "hd": 64, "prefix": 300, "most": 17},
        # eight requests behind a document of a few thousand tokens
        {"name": "shared_batch8", "kind": "shared", "n": 8, "heads": 32, "kv": 8, "hd": 128, "prefix": 4001, "most": 640},
        # an odd batch, five query heads to a kv head, heads of 80
        {"name": "shared_odd33", "kind": "shared", "n": 33, "heads": 40, "kv": 8, "hd": 80, "prefix": 9973, "most": 200},
        # many samples over one long context
        {"name": "shared_batch64", "kind": "shared", "n": 64, "heads": 32, "kv": 8, "hd": 128, "prefix": 32768, "most": 1024},
        # a decode step that keeps track of which rows matter
        {"name": "mass_step", "kind": "mass", "n": 1, "heads": 32, "kv": 8, "hd": 128, "ctx": 4096},
        # the last tokens of a long prompt vote on which of its rows to keep
        {"name": "mass_window", "kind": "mass", "n": 32, "heads": 32, "kv": 8, "hd": 128, "ctx": 16001},
        # one layer of a short prompt down to a quarter
        {"name": "keep_layer", "kind": "keep", "layers": 1, "kv": 8, "hd": 128, "len": 2000, "budget": 500},
        # a long prompt's cache of a whole model down to an eighth
        {"name": "keep_model", "kind": "keep", "layers": 24, "kv": 8, "hd": 128, "len": 16384, "budget": 2048},
        # a decode step of a bounded cache
        {"name": "evict_step", "kind": "evict", "kv": 8, "hd": 128, "len": 1024},
        # the same over a long one
        {"name": "evict_long", "kind": "evict", "kv": 8, "hd": 128, "len": 32768},
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "shared", "shared", "shared", "mass", "keep", "evict"])
    hd = rng.choice([32, 64, 80, 96, 128, 128, 128])
    kv = rng.choice([1, 2, 4, 5, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    if kind == "rope":
        n = _logint(rng, 1, 4000)
        return {"kind": kind, "n": n, "heads": heads, "kv": kv, "hd": hd, "rot": 2 * rng.randint(4, hd // 2),
                "layout": rng.choice(["interleaved", "half"]), "scaling": rng.choice(["none", "linear", "yarn", "llama3"]),
                "first": _logint(rng, 1, 1000000), "rows": n + rng.randint(0, 300)}
    if kind == "shared":
        prefix = 0 if rng.random() < 0.1 else _logint(rng, 1, 32768)
        return {"kind": kind, "n": _logint(rng, 1, 64), "heads": min(heads, 40), "kv": kv, "hd": hd, "prefix": prefix,
                "most": _logint(rng, 1, 1024)} if heads <= 40 else draw(rng)
    if kind == "mass":
        ctx = _logint(rng, 1, 16001)
        return {"kind": kind, "n": min(ctx, _logint(rng, 1, 32)), "heads": heads, "kv": kv, "hd": hd, "ctx": ctx}
    if kind == "keep":
        n = _logint(rng, 2, 32768)
        return {"kind": kind, "layers": rng.randint(1, 8), "kv": kv, "hd": hd, "len": n, "budget": rng.randint(1, n)}
    return {"kind": kind, "kv": kv, "hd": hd, "len": _logint(rng, 1, 65536)}


# --- inputs -----------------------------------------------------------------


def _generator(seed, key):
    return torch.Generator(device="cuda").manual_seed(1_000_003 * int(seed) + key)


def _normal(seed, key, *shape):
    return torch.randn(shape, generator=_generator(seed, key), device="cuda")


def _rows16(seed, key, layers, rows, dim):
    out = torch.empty((layers, rows, dim), dtype=torch.float16, device="cuda")
    return out.normal_(generator=_generator(seed, key))


def _ints(seed, key, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=_generator(seed, key), device="cuda", dtype=torch.int32)


def _mass(seed, key, *shape):
    rank = torch.rand(shape, generator=_generator(seed, key), device="cuda").mul_(shape[-1]).add_(1.0)
    return rank.pow_(-0.8)


def _cache(k, v):
    """The cache that holds (layers, rows, dim) keys and values, and each layer's rows as tensors."""
    if own:
        from gopherllm_amd import KVCacheF16
        layers, rows, dim = k.shape
        kv = KVCacheF16(layers, dim, v.shape[2], rows)
        views = [kv.tensors(layer) for layer in range(layers)]
        for layer, (kr, vr) in enumerate(views):
            kr.copy_(k[layer])
            vr.copy_(v[layer])
        return {"cache": kv, "k": [x[0] for x in views], "v": [x[1] for x in views]}
    return {"k": list(k.unbind(0)), "v": list(v.unbind(0))}


THETA = 500000.0
SCALED = {"none": {}, "linear": {"factor": 4.0}, "yarn": {"factor": 16.0, "orig_ctx": 8192},
          "llama3": {"factor": 8.0, "orig_ctx": 8192}}


def _frequencies(rot, scaling):
    """(inverse frequencies, amplitude) in 64 bits."""
    i = np.arange(rot // 2, dtype=np.float64)
    inv = THETA ** (-2.0 * i / rot)
    if scaling == "none":
        return inv, 1.0
    f = SCALED[scaling]["factor"]
    if scaling == "linear":
        return inv / f, 1.0
    orig = SCALED[scaling]["orig_ctx"]
    if scaling == "llama3":  # low and high frequency factors 1 and 4
        turns = orig * inv / (2 * np.pi)
        smooth = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return inv * ((1 - smooth) / f + smooth), 1.0
    edge = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
    lo, hi = max(0, math.floor(edge(32.0))), min(rot - 1, math.ceil(edge(1.0)))
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
    return inv * (ramp / f + (1 - ramp)), 0.1 * math.log(f) + 1.0


def _lengths(case, seed):
    """First row and number of rows of each request's own part: ragged, one as long as any, one empty."""
    n, most = case["n"], case["most"]
    lens = _ints(seed, 7, 1, most, n)
    lens[0] = most
    if n > 2:
        lens[n // 2] = 0
    starts = case["prefix"] + torch.arange(n, device="cuda", dtype=torch.int32) * most
    return starts.to(torch.int32), lens


def _protected(case):
    """(first positions, newest positions) that stay."""
    n = case["len"]
    return min(4, n // 8), min(64, n // 4)


def prepare(case, seed):
    kind, kv, hd = case["kind"], case["kv"], case["hd"]
    dim = kv * hd
    if kind == "rope":
        n = case["n"]
        s = {"q": _normal(seed, 1, n, case["heads"] * hd), "k_new": _normal(seed, 2, n, dim), "v_new": _normal(seed, 3, n, dim),
             "positions": (case["first"] + torch.arange(n, device="cuda")).to(torch.int32),
             "rows": torch.randperm(case["rows"], generator=_generator(seed, 4), device="cuda")[:n].to(torch.int32),
             "out": torch.empty((n, case["heads"] * hd), device="cuda")}
        s |= _cache(_rows16(seed, 5, 1, case["rows"], dim), _rows16(seed, 6, 1, case["rows"], dim))
        if own:
            from gopherllm_amd import Rope
            s["rope"] = Rope(hd, rot_dim=case["rot"], layout=case["layout"], theta=THETA, scaling=case["scaling"],
                             **SCALED[case["scaling"]])
        else:
            inv, amp = _frequencies(case["rot"], case["scaling"])
            s["inv"], s["amp"] = torch.from_numpy(inv).cuda(), amp
    elif kind == "shared":
        rows = case["prefix"] + case["n"] * case["most"]
        starts, lens = _lengths(case, seed)
        s = {"q": _normal(seed, 1, case["n"], case["heads"] * hd), "starts": starts, "lens": lens,
             "out": torch.empty((case["n"], case["heads"] * hd), device="cuda")}
        s |= _cache(_rows16(seed, 5, 1, rows, dim), _rows16(seed, 6, 1, rows, dim))
    elif kind == "mass":
        s = {"q": _normal(seed, 1, case["n"], case["heads"] * hd), "mass": _mass(seed, 8, kv, case["ctx"]),
             "out": torch.empty((case["n"], case["heads"] * hd), device="cuda")}
        s |= _cache(_rows16(seed, 5, 1, case["ctx"], dim), _rows16(seed, 6, 1, case["ctx"], dim))
    elif kind == "keep":
        layers, n, budget = case["layers"], case["len"], case["budget"]
        s = {"mass": _mass(seed, 8, layers, kv, n), "mass_out": torch.zeros((layers, kv, budget), device="cuda"),
             "pos": torch.arange(n, device="cuda", dtype=torch.int32).expand(layers, kv, n).contiguous(),
             "pos_out": torch.zeros((layers, kv, budget), device="cuda", dtype=torch.int32)}
        s |= _cache(_rows16(seed, 5, layers, n, dim), _rows16(seed, 6, layers, n, dim))
        small = torch.zeros((layers, budget, dim), dtype=torch.float16, device="cuda")
        s["to"] = _cache(small, small.clone())
    else:
        n = case["len"]
        order = torch.stack([torch.randperm(n, generator=_generator(seed, 20 + g), device="cuda") for g in range(kv)])
        s = {"k_new": _normal(seed, 2, dim), "v_new": _normal(seed, 3, dim), "mass": _mass(seed, 8, kv, n),
             "pos": order.to(torch.int32), "now": torch.tensor([n], device="cuda", dtype=torch.int32),
             "victims": torch.zeros(kv, device="cuda", dtype=torch.int32)}
        s |= _cache(_rows16(seed, 5, 1, n, dim), _rows16(seed, 6, 1, n, dim))
    s["case"] = dict(case)
    return s


# --- one pass ---------------------------------------------------------------


def _run_own(s):
    c, kv = s["case"], s["cache"]
    kind, hd = c["kind"], c["hd"]
    if kind == "rope":
        kv.store_rope_dev(0, s["rope"], s["q"], s["k_new"], s["v_new"], s["positions"], s["rows"], s["out"])
        return {"q": s["out"], "k": s["k"][0], "v": s["v"][0]}
    if kind == "shared":
        return kv.attend_shared_dev(0, s["q"], c["heads"], c["kv"], hd, 0, c["prefix"], s["starts"], s["lens"], c["most"],
                                    hd ** -0.5, s["out"])
    if kind == "mass":
        kv.attend_mass_dev(0, s["q"], c["heads"], c["kv"], hd, 0, c["ctx"] - 1, hd ** -0.5, s["mass"], s["out"])
        return {"out": s["out"], "mass": s["mass"]}
    sinks, recent = _protected(c)
    if kind == "keep":
        kv.keep_dev(s["to"]["cache"], c["kv"], hd, c["len"], c["budget"], s["mass"], s["pos"], s["mass_out"], s["pos_out"],
                    now=c["len"], sinks=sinks, recent=recent)
        return {"k": s["to"]["k"], "v": s["to"]["v"], "mass": s["mass_out"], "pos": s["pos_out"]}
    kv.evict_store_dev(0, c["kv"], hd, s["k_new"], s["v_new"], 0, c["len"], s["mass"], s["pos"], s["now"],
                       sinks=sinks, recent=recent, rows_out=s["victims"])
    return {"k": s["k"][0], "v": s["v"][0], "mass": s["mass"], "pos": s["pos"], "rows": s["victims"]}


def _rotate(x, hd, rot, layout, cos, sin):
    """x (n, heads * hd), cos and sin (n, rot / 2)."""
    x = x.view(x.shape[0], -1, hd)
    c, s = cos[:, None], sin[:, None]
    out = x.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if layout == "interleaved" else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    return out.view(x.shape[0], -1)


def _finish(w, total):
    return torch.where(total > 0, w / total.clamp_min(1e-38), torch.zeros_like(w))


def _run_rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv"]
    cos, sin = (torch.cos(angle) * s["amp"]).float(), (torch.sin(angle) * s["amp"]).float()
    s["out"].copy_(_rotate(s["q"], c["hd"], c["rot"], c["layout"], cos, sin))
    rows = s["rows"].long()
    s["k"][0][rows] = _rotate(s["k_new"], c["hd"], c["rot"], c["layout"], cos, sin).half()
    s["v"][0][rows] = s["v_new"].half()
    return {"q": s["out"], "k": s["k"][0], "v": s["v"][0]}


def _run_shared(s):
    c, k, v = s["case"], s["k"][0], s["v"][0]
    n, g, hd, t, most = c["n"], c["kv"], c["hd"], c["prefix"], c["most"]
    r = c["heads"] // g
    q = s["q"].view(n, g, r, hd) * hd ** -0.5
    first = torch.bmm(q.permute(1, 0, 2, 3).reshape(g, n * r, hd), k[:t].view(t, g, hd).permute(1, 2, 0).float().contiguous())
    at = torch.arange(most, device="cuda")
    rows = (s["starts"].long()[:, None] + at).clamp_max(k.shape[0] - 1)
    mine = torch.matmul(q, k[rows].view(n, most, g, hd).permute(0, 2, 3, 1).float().contiguous())  # n, g, r, most
    mine = mine.masked_fill((at >= s["lens"].long()[:, None])[:, None, None], -math.inf)
    scores = torch.cat([first.view(g, n, r, t), mine.permute(1, 0, 2, 3)], -1)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    o = torch.bmm(w[..., :t].reshape(g, n * r, t), v[:t].view(t, g, hd).permute(1, 0, 2).float().contiguous()).view(g, n, r, hd)
    o = o + torch.matmul(w[..., t:].permute(1, 0, 2, 3).contiguous(),
                         v[rows].view(n, most, g, hd).permute(0, 2, 1, 3).float().contiguous()).permute(1, 0, 2, 3)
    s["out"].copy_(_finish(o, total).permute(1, 0, 2, 3).reshape(n, -1))
    return s["out"]


def _run_mass(s):
    c, t = s["case"], s["case"]["ctx"]
    n, g, hd = c["n"], c["kv"], c["hd"]
    r = c["heads"] // g
    q = (s["q"].view(n, g, r, hd) * hd ** -0.5).permute(1, 0, 2, 3).reshape(g, n * r, hd)
    scores = torch.bmm(q, s["k"][0].view(t, g, hd).permute(1, 2, 0).float().contiguous()).view(g, n, r, t)
    after = torch.arange(t, device="cuda") > (t - n + torch.arange(n, device="cuda"))[:, None]
    scores = scores.masked_fill(after[None, :, None], -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = torch.bmm(w.view(g, n * r, t), s["v"][0].view(t, g, hd).permute(1, 0, 2).float().contiguous())
    s["mass"].add_(w.sum((1, 2)))
    s["out"].copy_(o.view(g, n, r, hd).permute(1, 0, 2, 3).reshape(n, -1))
    return {"out": s["out"], "mass": s["mass"]}


def _run_keep(s):
    c = s["case"]
    sinks, recent = _protected(c)
    stay = (s["pos"] < sinks) | (s["pos"] >= c["len"] - recent)
    order = torch.sort(s["mass"].masked_fill(stay, math.inf), dim=-1, descending=True, stable=True).indices
    rows = order[..., :c["budget"]].sort(-1).values  # layers, kv, budget
    s["mass_out"].copy_(s["mass"].gather(-1, rows))
    s["pos_out"].copy_(s["pos"].gather(-1, rows))
    layers, n, g, hd = c["layers"], c["len"], c["kv"], c["hd"]
    at = rows.transpose(1, 2)[..., None].expand(layers, c["budget"], g, hd)
    for name in ("k", "v"):
        full = torch.stack(s[name]).view(layers, n, g, hd)
        kept = full.gather(1, at).view(layers, c["budget"], g * hd)
        torch._foreach_copy_(s["to"][name], list(kept.unbind(0)))
    return {"k": s["to"]["k"], "v": s["to"]["v"], "mass": s["mass_out"], "pos": s["pos_out"]}


def _run_evict(s):
    c = s["case"]
    sinks, recent = _protected(c)
    stay = (s["pos"] < sinks) | (s["pos"] >= s["now"] - recent)
    rows = s["mass"].masked_fill(stay, math.inf).sort(dim=-1, stable=True).indices[:, 0]
    s["victims"].copy_(rows)
    g = torch.arange(c["kv"], device="cuda")
    s["k"][0].view(c["len"], c["kv"], c["hd"])[rows, g] = s["k_new"].view(c["kv"], c["hd"]).half()
    s["v"][0].view(c["len"], c["kv"], c["hd"])[rows, g] = s["v_new"].view(c["kv"], c["hd"]).half()
    s["mass"][g, rows] = 0.0
    s["pos"][g, rows] = s["now"]
    return {"k": s["k"][0], "v": s["v"][0], "mass": s["mass"], "pos": s["pos"], "rows": s["victims"]}


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _run_rope, "shared": _run_shared, "mass": _run_mass, "keep": _run_keep, "evict": _run_evict}[s["case"]["kind"]](s)


# --- the definitions in 64 bits ----------------------------------------------


def _attention64(q, k, v):
    """q (hd,), k and v (rows, hd) of one head in 64 bits: (output, weights)."""
    w = torch.softmax(k @ q * q.shape[-1] ** -0.5, 0)
    return w @ v, w


def exact(case, seed):
    kind, kv, hd = case["kind"], case["kv"], case["hd"]
    dim = kv * hd
    if kind == "keep":
        return None  # copies of its inputs
    if kind == "rope":
        n, rot = case["n"], case["rot"]
        inv, amp = _frequencies(rot, case["scaling"])
        angle = torch.from_numpy(np.outer(case["first"] + np.arange(n, dtype=np.float64), inv)).cuda()
        turn = torch.polar(torch.full_like(angle, amp), angle)[:, None]  # a complex factor for each pair
        rows = torch.randperm(case["rows"], generator=_generator(seed, 4), device="cuda")[:n]
        out = []
        for x in (_normal(seed, 1, n, case["heads"] * hd), _normal(seed, 2, n, dim)):
            x = x.double().view(n, -1, hd)
            pairs = x[..., :rot]
            pairs = pairs.reshape(n, -1, rot // 2, 2) if case["layout"] == "interleaved" else \
                pairs.reshape(n, -1, 2, rot // 2).transpose(2, 3)
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y = y.flatten(2) if case["layout"] == "interleaved" else y.transpose(2, 3).flatten(2)
            out.append(torch.cat([y, x[..., rot:]], -1).reshape(n, -1))
        k = _rows16(seed, 5, 1, case["rows"], dim)[0].double()
        v = _rows16(seed, 6, 1, case["rows"], dim)[0].double()
        k[rows], v[rows] = out[1], _normal(seed, 3, n, dim).double()
        return {"q": out[0], "k": k, "v": v}
    if kind == "evict":
        n = case["len"]
        sinks, recent = _protected(case)
        k = _rows16(seed, 5, 1, n, dim)[0].double().view(n, kv, hd)
        v = _rows16(seed, 6, 1, n, dim)[0].double().view(n, kv, hd)
        new_k, new_v = _normal(seed, 2, dim).double().view(kv, hd), _normal(seed, 3, dim).double().view(kv, hd)
        mass = _mass(seed, 8, kv, n).double().cpu().numpy()
        for g in range(kv):
            pos = torch.randperm(n, generator=_generator(seed, 20 + g), device="cuda").cpu().numpy()
            row = min(range(n), key=lambda r: (bool(pos[r] < sinks or pos[r] >= n - recent), mass[g, r]))
            k[row, g], v[row, g] = new_k[g], new_v[g]
            mass[g, row] = 0.0
        return {"k": k.view(n, dim), "v": v.view(n, dim), "mass": mass, "pos": None, "rows": None}
    heads, n = case["heads"], case["n"]
    r = heads // kv
    q = _normal(seed, 1, n, heads * hd).double().view(n, kv, r, hd)
    if kind == "shared":
        t, most = case["prefix"], case["most"]
        rows = t + n * most
    else:
        t, rows = case["ctx"], case["ctx"]
    k = _rows16(seed, 5, 1, rows, dim)[0].view(rows, kv, hd)
    v = _rows16(seed, 6, 1, rows, dim)[0].view(rows, kv, hd)
    out = torch.zeros((n, kv, r, hd), dtype=torch.float64, device="cuda")
    if kind == "shared":
        starts, lens = _lengths(case, seed)
        spans = list(zip(starts.tolist(), lens.tolist()))
        for g in range(kv):
            pk, pv = k[:t, g].double(), v[:t, g].double()
            for i, (a, m) in enumerate(spans):
                if t + m == 0:
                    continue
                kk, vv = torch.cat([pk, k[a:a + m, g].double()]), torch.cat([pv, v[a:a + m, g].double()])
                w = torch.softmax(q[i, g] @ kk.T * hd ** -0.5, -1)
                out[i, g] = w @ vv
        return out.view(n, -1)
    mass = _mass(seed, 8, kv, t).double()
    for g in range(kv):
        kk, vv = k[:, g].double(), v[:, g].double()
        for i in range(n):
            m = t - n + 1 + i
            w = torch.softmax(q[i, g] @ kk[:m].T * hd ** -0.5, -1)
            out[i, g] = w @ vv[:m]
            mass[g, :m] += w.sum(0)
    return {"out": out.view(n, -1), "mass": mass}


# --- what a pass cannot do without -------------------------------------------


def work(case):
    kind, kv, hd = case["kind"], case["kv"], case["hd"]
    row = 2 * kv * hd * 2  # a row of keys and values
    if kind == "rope":
        n, h = case["n"], case["heads"]
        return {"bytes": n * (8 * h * hd + 8 * kv * hd + row + 8), "flops": n * (3 * case["rot"] * (h + kv) + 40 * case["rot"])}
    if kind == "shared":
        n, h, mean = case["n"], case["heads"], (case["most"] + 1) / 2
        return {"bytes": (case["prefix"] + n * mean) * row + 8 * n * h * hd + 8 * n,
                "flops": 4 * n * h * hd * (case["prefix"] + mean)}
    if kind == "mass":
        n, h, t = case["n"], case["heads"], case["ctx"]
        return {"bytes": t * row + 8 * n * h * hd + 8 * kv * t, "flops": 4 * h * hd * (n * t - n * (n - 1) // 2)}
    if kind == "keep":
        n, m = case["layers"] * kv * case["len"], case["layers"] * kv * case["budget"]
        return {"bytes": 8 * n + m * (8 + 2 * 4 * hd), "flops": n}
    n = kv * case["len"]
    return {"bytes": 8 * n + kv * (12 * hd + 12), "flops": n}
