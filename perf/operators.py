"""Paged-cache operators as measured workloads: append (head norms, rotation, write into pages), attention of
a ragged batch of new tokens over the pages, and eviction by accumulated attention weight.

``own`` selects the framework's kernels; otherwise every operator is computed in elementary torch operations."""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------- cases
def _append(name, **kw):
    c = {"op": "append", "dtype": "bf16", "requests": 1, "idle": 0, "chunk": 1, "length": 64, "kv_heads": 8, "group": 4,
         "dim": 128, "page": 16, "norm": True, "rotary": 128, "interleaved": False, "fused": True, "weights": False}
    return {"name": name, **c, **kw} if name else {**c, **kw}


def _attend(name, **kw):
    c = {"op": "attend", "dtype": "bf16", "requests": 1, "idle": 0, "chunked": 0, "chunk": 1, "length": 64,
         "kv_heads": 8, "group": 4, "dim": 128, "page": 16, "weights": False, "causal": True}
    return {"name": name, **c, **kw} if name else {**c, **kw}


def _evict(name, **kw):
    c = {"op": "evict", "dtype": "bf16", "requests": 1, "length": 64, "budget": 32, "first": 4, "last": 8,
         "kv_heads": 8, "dim": 128, "page": 16}
    return {"name": name, **c, **kw} if name else {**c, **kw}


def listed():
    return [
        # one decode step of 64 streams: q and k normed per head, rotated, k and v put into the pages
        _append("append step 64", requests=64, chunk=1, length=2048, weights=True),
        # prompts of four requests enter the cache, straight out of a fused projection
        _append("append prompts 4x2048", requests=4, chunk=2048, length=2048),
        # fp32 heads of an odd width, rotation of their first half in interleaved pairs, no norm
        _append("append fp32 d80", dtype="fp32", requests=3, chunk=259, length=700, kv_heads=4, group=3, dim=80, page=32,
                norm=False, rotary=40, interleaved=True, fused=False),
        # a handful of short streams, two of the batch's places idle: latency decides
        _attend("step 4 short", requests=4, idle=2, length=500, kv_heads=2, group=4, dim=64),
        # a full serving batch at its decode step, lengths from 2048 to 16384
        _attend("step 32 to 16384", requests=32, length=16384),
        # one stream with a very long cache, weights of the keys accumulated for eviction
        _attend("step 65536 weights", length=65536, page=64, weights=True),
        # two long prompts, a chunk of 2048 tokens each on top of what is cached
        _attend("chunk 2x2048 on 8192", requests=2, chunked=2, chunk=2048, length=8192, page=64),
        # chunks of three prompts beside the single tokens of 21 running streams, heads of 96, one query head per kv head
        _attend("mixed 24", requests=24, chunked=3, chunk=509, length=2048, kv_heads=8, group=1, dim=96),
        # a prompt's chunk whose attention weight is kept for every key
        _attend("chunk 1024 weights", requests=2, chunked=2, chunk=1024, length=4096, weights=True),
        # fp32 verification of a lowered model on small ragged chunks
        _attend("chunk fp32 d64", dtype="fp32", requests=3, chunked=2, chunk=301, length=1024, kv_heads=4, group=2, dim=64, page=8),
        # a small cache is cut to 128 keys
        _evict("evict 4 short fp32", dtype="fp32", requests=4, length=500, budget=128, kv_heads=2, dim=64),
        # the caches of 16 long streams are halved
        _evict("evict 16 to 4096", requests=16, length=8192, budget=4096, first=16, last=256, page=64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16]) if kv_heads <= 4 else rng.choice([1, 2, 4])
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if op == "append":
        chunk = _log_int(rng, 1, 2048)
        requests = _log_int(rng, 1, min(64, max(1, 8192 // chunk)))
        rotary = rng.choice([0, dim, dim, 2 * (dim // 4)])
        return _append(None, dtype=dtype, requests=requests, idle=rng.randrange(3), chunk=chunk, length=chunk + _log_int(rng, 1, 2048),
                       kv_heads=kv_heads, group=group, dim=dim, page=page, norm=rng.random() < 0.7, rotary=rotary,
                       interleaved=rng.random() < 0.4, fused=rng.random() < 0.5, weights=rng.random() < 0.5)
    if op == "evict":
        length = _log_int(rng, 16, 16384)
        requests = _log_int(rng, 1, max(1, min(32, 8192 * 16 // length)))
        budget = rng.randint(max(1, length // 8), max(1, length * 3 // 4))
        first, last = rng.randint(0, budget // 4), rng.randint(0, budget // 4)
        return _evict(None, dtype=dtype, requests=requests, length=length, budget=budget, first=first, last=last,
                      kv_heads=kv_heads, dim=dim, page=page)
    if rng.random() < 0.5:  # single tokens
        length = _log_int(rng, 1, 65536)
        requests = _log_int(rng, 1, max(1, min(64, (1 << 19) // length)))
        return _attend(None, dtype=dtype, requests=requests, idle=rng.randrange(3), length=length, kv_heads=kv_heads,
                       group=group, dim=dim, page=page, weights=rng.random() < 0.4)
    chunk = _log_int(rng, 2, 1024)
    length = chunk + _log_int(rng, 1, 6000)
    room = (1 << 29) // (chunk * length * kv_heads * group * (4 if dtype == "fp32" else 1))
    requests = _log_int(rng, 1, max(1, min(24, room)))
    return _attend(None, dtype=dtype, requests=requests, idle=rng.randrange(3), chunked=rng.randint(1, requests), chunk=chunk,
                   length=length, kv_heads=kv_heads, group=group, dim=dim, page=page, weights=rng.random() < 0.4,
                   causal=rng.random() < 0.8)


def _spread(i):
    """1 for the first request, then fractions spread over (0, 1)."""
    return 1.0 if i == 0 else (i * 0.6180339887498949) % 1.0


def _sizes(case):
    """New tokens and cached keys (new ones included) of every request; idle places have none of either."""
    n, keys = [], []
    for r in range(case["requests"]):
        chunked = case["op"] == "append" or (case["op"] == "attend" and r < case["chunked"])
        new = max(1, int(case["chunk"] * (0.5 + 0.5 * _spread(r)))) if chunked else 1
        n.append(0 if case["op"] == "evict" else new)
        keys.append(max(n[-1], 1, int(case["length"] * (0.125 + 0.875 * _spread(r)))))
    idle = case.get("idle", 0)
    return n + [0] * idle, keys + [0] * idle


# ------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _cache(case, keys, g, fill, extra_pages=0):
    """Pools of pages in random order, the table that says which page holds what, and the lengths. Slots that
    no request has written hold `fill`."""
    ps, kv, dim, dtype = case["page"], case["kv_heads"], case["dim"], _TYPES[case["dtype"]]
    count = [(k + ps - 1) // ps for k in keys]
    pages = sum(count) + 3 + extra_pages
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).tolist()
    width = max(max(count), 1)
    rows, at = [], 0
    for c in count:
        rows.append(order[at:at + c] + [-1] * (width - c))
        at += c
    table = torch.tensor(rows, dtype=torch.int32, device="cuda")
    k = _normal((pages, kv, ps, dim), g, dtype)
    v = _normal((pages, kv, ps, dim), g, dtype)
    lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
    used = torch.zeros(pages, ps, dtype=torch.bool, device="cuda")
    slot = torch.arange(width * ps, device="cuda")
    r, j = (slot[None, :] < lens[:, None]).nonzero(as_tuple=True)
    used[table[r, j // ps].long(), j % ps] = True
    if fill is not None:
        k.masked_fill_(~used[:, None, :, None], fill)
        v.masked_fill_(~used[:, None, :, None], fill)
    return {"k": k, "v": v, "table": table, "lens": lens, "used": used, "spare": order[at:]}


def _offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    n, keys = _sizes(case)
    dtype, kv, dim = _TYPES[case["dtype"]], case["kv_heads"], case["dim"]
    heads, total = kv * case.get("group", 1), sum(n)
    if case["op"] == "append":
        c = _cache(case, keys, g, None)
        if case["fused"]:  # views of one projection's output
            qkv = _normal((total, (heads + 2 * kv), dim), g, dtype, 1.5)
            q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        else:
            q, k, v = (_normal((total, h, dim), g, dtype, 1.5) for h in (heads, kv, kv))
        position = torch.cat([torch.arange(kk - x, kk) for x, kk in zip(n, keys)]).to(torch.int32).cuda()
        s = {"q": q, "k": k, "v": v, "cache": c, "cu": _offsets(n), "position": position, "max_q": max(n),
             "weights": torch.rand(c["k"].shape[:3], generator=g, device="cuda") if case["weights"] else None,
             "qw": None, "kw": None, "cos": None, "sin": None, "out": torch.zeros(total, heads, dim, dtype=dtype, device="cuda")}
        if case["norm"]:
            s["qw"], s["kw"] = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda") for _ in range(2))
            s["qw"], s["kw"] = s["qw"].to(dtype), s["kw"].to(dtype)
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = torch.arange(max(keys), device="cuda", dtype=torch.float64)[:, None] * \
                10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        c = _cache(case, keys, g, float("nan"))
        s = {"q": _normal((total, heads, dim), g, dtype, 1.5), "cache": c, "cu": _offsets(n), "max_q": max(n),
             "max_k": max(keys), "weights": None, "out": torch.zeros(total, heads, dim, dtype=dtype, device="cuda")}
        if case["weights"]:
            s["weights"] = torch.zeros(c["k"].shape[:3], device="cuda")
    else:
        ps, budget = case["page"], case["budget"]
        need = (budget + ps - 1) // ps
        c = _cache(case, keys, g, None, need * len(keys))
        w = torch.exp(2 * torch.randn(c["k"].shape[:3], generator=g, device="cuda"))
        w.masked_fill_(torch.rand(w.shape, generator=g, device="cuda") < 0.05, 0.0)  # keys that nobody looked at
        spare = c["spare"][:need * len(keys)]
        s = {"cache": c, "weights": w, "to": torch.tensor(spare, dtype=torch.int32, device="cuda").view(len(keys), need),
             "max_k": max(keys)}
    s["case"] = dict(case)
    return s


# ------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from catopt_b200 import ops
        c, cache = s["case"], s["cache"]
        if c["op"] == "append":
            q = ops.paged_append(s["q"], s["k"], s["v"], cache["k"], cache["v"], cache["table"], cache["lens"], s["cu"],
                                 q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, cos=s["cos"], sin=s["sin"], positions=s["position"],
                                 interleaved=c["interleaved"], weights=s["weights"], out=s["out"])
            return _append_outputs(s, q)
        if c["op"] == "attend":
            o = ops.om_paged_fwd(s["q"], cache["k"], cache["v"], cache["table"], cache["lens"], s["cu"], s["max_q"],
                                 max_k=s["max_k"], causal=c["causal"], weights=s["weights"], out=s["out"])
            return {"o": o} if s["weights"] is None else {"o": o, "weights": s["weights"]}
        kept, lens = ops.paged_evict(cache["k"], cache["v"], s["weights"], cache["table"], cache["lens"], s["to"], c["budget"],
                                     keep_first=c["first"], keep_last=c["last"], max_k=s["max_k"])
        return {"kept": kept, "lens": lens, "k": cache["k"], "v": cache["v"], "weights": s["weights"]}
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[s["case"]["op"]](s)


def _append_outputs(s, q):
    r = {"q": q, "k": s["cache"]["k"], "v": s["cache"]["v"]}
    if s["weights"] is not None:
        r["weights"] = s["weights"]
    return r


def _plain_append(s):
    c, cache = s["case"], s["cache"]
    n = s["cu"][1:] - s["cu"][:-1]
    request = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n.long(), output_size=s["q"].shape[0])
    slot = (cache["lens"] - n)[request] + torch.arange(request.numel(), device="cuda") - s["cu"][request]
    page, at = cache["table"][request, slot // c["page"]].long(), slot % c["page"]

    def turned(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        if s["cos"] is not None:
            cos, sin, rot = s["cos"][s["position"].long()][:, None], s["sin"][s["position"].long()][:, None], c["rotary"]
            if c["interleaved"]:
                a, b = y[..., :rot:2], y[..., 1:rot:2]
                z = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
            else:
                a, b = y[..., :rot // 2], y[..., rot // 2:rot]
                z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
            y = torch.cat((z, y[..., rot:]), -1)
        return y.to(x.dtype)

    s["out"].copy_(turned(s["q"], s["qw"]))
    cache["k"][page, :, at] = turned(s["k"], s["kw"])
    cache["v"][page, :, at] = s["v"]
    if s["weights"] is not None:
        s["weights"][page, :, at] = 0.0
    return _append_outputs(s, s["out"])


def _plain_attend(s):
    c, cache = s["case"], s["cache"]
    ps, kv, group, dim = c["page"], c["kv_heads"], c["group"], c["dim"]
    lens, cu = cache["lens"], s["cu"]
    R, n = lens.numel(), s["cu"][1:] - s["cu"][:-1]
    width = (s["max_k"] + ps - 1) // ps
    table = cache["table"][:, :width].clamp(min=0).long()
    slot = torch.arange(width * ps, device="cuda")
    seen = slot[None, :] < lens[:, None]                                             # [R, K]
    k = cache["k"][table].transpose(2, 1).reshape(R, kv, width * ps, dim).float()
    v = cache["v"][table].transpose(2, 1).reshape(R, kv, width * ps, dim).float()
    v = torch.where(seen[:, None, :, None], v, 0.0)
    row = torch.arange(s["max_q"], device="cuda")
    there = row[None, :] < n[:, None]                                                # [R, T]
    at = (cu[:-1, None] + row[None, :]).clamp(max=max(s["q"].shape[0] - 1, 0)).long()
    q = s["q"][at].float().view(R, s["max_q"], kv, group, dim).permute(0, 2, 3, 1, 4)  # [R, kv, G, T, d]
    scores = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).view(R, kv, group, s["max_q"], -1) * dim ** -0.5
    visible = seen[:, None, :] & there[:, :, None]
    if c["causal"]:
        visible = visible & (slot[None, None, :] <= (lens - n)[:, None, None] + row[None, :, None])
    visible = visible[:, None, None]
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.flatten(2, 3), v).view(R, kv, group, s["max_q"], dim).permute(0, 3, 1, 2, 4)
    s["out"][at[there]] = o[there].reshape(-1, kv * group, dim).to(s["out"].dtype)
    if s["weights"] is None:
        return {"o": s["out"]}
    got = p.sum((2, 3)).view(R, kv, width, ps)                                       # [R, kv, K]
    r, j = seen.view(R, width, ps).any(-1).nonzero(as_tuple=True)
    s["weights"][table[r, j]] += got[r, :, j]
    return {"o": s["out"], "weights": s["weights"]}


def _plain_evict(s):
    c, cache = s["case"], s["cache"]
    ps, budget, first, last = c["page"], c["budget"], c["first"], c["last"]
    lens, kv = cache["lens"].long(), c["kv_heads"]
    R, width = lens.numel(), (s["max_k"] + ps - 1) // ps
    table = cache["table"][:, :width].clamp(min=0).long()
    slot = torch.arange(width * ps, device="cuda")
    w = s["weights"][table].transpose(2, 1).reshape(R, kv, width * ps)
    # what is always kept sorts before every weight, what is not there after
    kind = torch.where((slot < first) | (slot >= (lens - last)[:, None]), 0, 1) + 2 * (slot >= lens[:, None])
    by_weight = torch.sort(w, dim=-1, descending=True, stable=True).indices
    by_kind = torch.sort(torch.gather(kind[:, None].expand(R, kv, -1), -1, by_weight), dim=-1, stable=True).indices
    order = torch.gather(by_weight, -1, by_kind)
    new = lens.clamp(max=budget)
    order = torch.nn.functional.pad(order, (0, max(0, budget - order.shape[-1])))[..., :budget]
    rank = torch.arange(budget, device="cuda")
    there = (rank[None, :] < new[:, None])[:, None]                                    # [R, 1, budget]
    order = torch.where(there, order, width * ps).sort(-1).values
    kept = torch.where(there, order, -1).to(torch.int32)
    r, h, i = there.expand(R, kv, budget).nonzero(as_tuple=True)
    j = order[r, h, i]
    src, dst = table[r, j // ps], s["to"].long()[r, i // ps]
    for pool in (cache["k"], cache["v"], s["weights"]):
        pool[dst, h, i % ps] = pool[src, h, j % ps]
    return {"kept": kept, "lens": new.to(torch.int32), "k": cache["k"], "v": cache["v"], "weights": s["weights"]}


# ------------------------------------------------------------------------------------------- cost and definition
def work(case):
    n, keys = _sizes(case)
    e = 2 if case["dtype"] == "bf16" else 4
    kv, dim, heads = case["kv_heads"], case["dim"], case["kv_heads"] * case.get("group", 1)
    if case["op"] == "append":
        total = sum(n)
        rows = total * (heads + kv)
        return {"bytes": 2 * total * (heads + 2 * kv) * dim * e + total * 4 + (4 * total * case["rotary"] if case["rotary"] else 0) +
                (4 * total * kv if case["weights"] else 0) + (2 * dim * e if case["norm"] else 0),
                "flops": rows * ((4 * dim if case["norm"] else 0) + 3 * case["rotary"])}
    if case["op"] == "attend":
        pairs = sum(x * (k - x) + x * (x + 1) // 2 if case["causal"] else x * k for x, k in zip(n, keys)) * heads
        cells = sum(k for x, k in zip(n, keys) if x) * kv
        flops = 4 * dim * pairs + 5 * pairs
        return {"bytes": 2 * cells * dim * e + 2 * sum(n) * heads * dim * e + (8 * cells if case["weights"] else 0), "flops": flops}
    kept = sum(min(k, case["budget"]) for k in keys) * kv
    return {"bytes": 4 * sum(keys) * kv + 2 * kept * (2 * dim * e + 4), "flops": sum(keys) * kv}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _exact_append(s):
    c, cache = s["case"], s["cache"]
    n, keys = _sizes(c)
    ps, rot = c["page"], c["rotary"]

    def turned(x, w):
        y = x.double()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
        if rot:
            z = y.clone()
            i = torch.arange(rot // 2, device="cuda")
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
            cos, sin = s["cos"].double()[s["position"].long()], s["sin"].double()[s["position"].long()]
            z[:, :, a] = y[:, :, a] * cos[:, None] - y[:, :, b] * sin[:, None]
            z[:, :, b] = y[:, :, a] * sin[:, None] + y[:, :, b] * cos[:, None]
            y = z
        return y

    new_k, new_v = turned(s["k"], s["kw"]), s["v"].double()
    k, v = cache["k"].double(), cache["v"].double()
    w = None if s["weights"] is None else s["weights"].double()
    table, at = cache["table"].tolist(), 0
    for r, (x, total) in enumerate(zip(n, keys)):
        done = 0
        while done < x:  # page by page
            j = total - x + done
            take, page = min(x - done, ps - j % ps), table[r][j // ps]
            k[page, :, j % ps:j % ps + take] = new_k[at:at + take].transpose(0, 1)
            v[page, :, j % ps:j % ps + take] = new_v[at:at + take].transpose(0, 1)
            if w is not None:
                w[page, :, j % ps:j % ps + take] = 0
            done, at = done + take, at + take
    out = {"q": turned(s["q"], s["qw"]), "k": k, "v": v}
    return out if w is None else {**out, "weights": w}


def _exact_attend(s):
    c, cache = s["case"], s["cache"]
    n, keys = _sizes(c)
    ps, group = c["page"], c["group"]
    o = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    w = None if s["weights"] is None else torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (x, total) in enumerate(zip(n, keys)):
        if not x:
            continue
        pages = cache["table"][r, :(total + ps - 1) // ps].long()
        hidden = None
        if c["causal"]:
            hidden = torch.arange(total, device="cuda")[None, :] > torch.arange(total - x, total, device="cuda")[:, None]
        for h in range(c["kv_heads"]):
            k = cache["k"][pages, h].reshape(-1, c["dim"])[:total].double()
            v = cache["v"][pages, h].reshape(-1, c["dim"])[:total].double()
            got = torch.zeros(pages.numel() * ps, dtype=torch.float64, device="cuda")
            for head in range(h * group, (h + 1) * group):
                z = s["q"][at:at + x, head].double() @ k.T / math.sqrt(c["dim"])
                if hidden is not None:
                    z[hidden] = float("-inf")
                p = torch.softmax(z, -1)
                o[at:at + x, head] = p @ v
                got[:total] += p.sum(0)
            if w is not None:
                w[pages, h] += got.view(-1, ps)
        at += x
    return {"o": o} if w is None else {"o": o, "weights": w}


def _exact_evict(s):
    c, cache = s["case"], s["cache"]
    _, keys = _sizes(c)
    ps, kv, budget = c["page"], c["kv_heads"], c["budget"]
    k, v, w = cache["k"].double(), cache["v"].double(), s["weights"].double()
    for r, total in enumerate(keys):
        pages, new = cache["table"][r, :(total + ps - 1) // ps].long(), min(total, budget)
        for h in range(kv):
            if total > budget:
                lo, hi = c["first"], total - c["last"]
                mid = s["weights"][pages, h].reshape(-1)[lo:hi].double()
                heavy = torch.argsort(-mid, stable=True)[:budget - lo - c["last"]].sort().values + lo
                j = torch.cat((torch.arange(lo, device="cuda"), heavy, torch.arange(hi, total, device="cuda")))
            else:
                j = torch.arange(total, device="cuda")
            i = torch.arange(new, device="cuda")
            to = s["to"][r].long()[i // ps]
            for dst, src in ((k, cache["k"]), (v, cache["v"]), (w, s["weights"])):
                dst[to, h, i % ps] = src[pages[j // ps], h, j % ps].double()
    return {"kept": None, "lens": None, "k": k, "v": v, "weights": w}
