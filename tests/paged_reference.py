"""Plain 64-bit forms of the paged-cache operators, request by request, and the bounds of their rounding errors."""
import torch

U32 = 2.0 ** -24          # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_cache(lens, kv_heads, page, d, dtype, device, seed, fill=float("nan"), spare=2, page_gap=0):
    """Pools with the requests' pages in random order; slots nobody has written hold ``fill``."""
    g = torch.Generator().manual_seed(seed)
    count = [(n + page - 1) // page for n in lens]
    pages = sum(count) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width = max(max(count), 1) + 1
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for r, c in enumerate(count):
        table[r, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    pools = []
    for _ in range(2):
        x = torch.randn(pages, kv_heads, page, d, generator=g).to(dtype)
        mask = torch.zeros(pages, page, dtype=torch.bool)
        for r, n in enumerate(lens):
            for j in range(n):
                mask[table[r, j // page], j % page] = True
        x.masked_fill_(~mask[:, None, :, None], fill)
        if page_gap:      # pages further apart than a page is long
            wide = torch.full((pages, kv_heads * page * d + page_gap), fill, dtype=dtype, device=device)
            view = wide[:, :kv_heads * page * d].view(pages, kv_heads, page, d)
            view.copy_(x)
            pools.append(view)
        else:
            pools.append(x.to(device))
    return {"k": pools[0], "v": pools[1], "table": table.to(device), "lens": torch.tensor(lens, dtype=torch.int32, device=device),
            "page": page, "free": order[at:]}


def offsets(new, device):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def rows_of(pool, table, r, h, n):
    """Slots [0, n) of request r, kv head h, in 64 bits."""
    page = pool.shape[2]
    ids = table[r, :(n + page - 1) // page].long()
    return pool[ids, h].reshape(-1, *pool.shape[3:])[:n].double()


def attend(q, cache, new, lens, scale, causal):
    """o, weights, and bounds of their errors for kernels that accumulate in fp32 and round p and o to q's type.

    With dot = scale sum |q_c k_c| of a row at its largest: a score is off by (d + 4) u dot at most (d + 1
    roundings of the sum, the scale and the conversion to base 2), so p / sum p by twice that, by 2^-21 for the two
    exponentials involved, and by (keys + 8) u for the sums and rescalings.  p rounded to the tensor type adds half a
    step of it for the products with v, and o half a step of itself."""
    d, hq, kv = q.shape[2], q.shape[1], cache["k"].shape[1]
    group, bf = hq // kv, q.dtype == torch.bfloat16
    o, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    w, wtol = (torch.zeros(cache["k"].shape[:3], dtype=torch.float64, device=q.device) for _ in range(2))
    page, at = cache["page"], 0
    for r, (x, n) in enumerate(zip(new, lens)):
        for head in range(hq if x and n else 0):
            h = head // group
            k, v = rows_of(cache["k"], cache["table"], r, h, n), rows_of(cache["v"], cache["table"], r, h, n)
            qq = q[at:at + x, head].double()
            s = qq @ k.T * scale
            seen = torch.ones(x, n, dtype=torch.bool, device=q.device)
            if causal:
                seen = torch.arange(n, device=q.device)[None] <= torch.arange(n - x, n, device=q.device)[:, None]
            s = s.masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, -1).nan_to_num(0.0)
            dot = ((qq.abs() @ k.abs().T) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
            rel = 2 * (d + 4) * U32 * dot + 2.0 ** -21 + (n + 8) * U32
            o[at:at + x, head] = p @ v
            spread = p @ v.abs()
            tol[at:at + x, head] = spread * (rel + (half_step(q.dtype) if bf else 0)) + half_step(q.dtype) * (p @ v).abs() + 1e-30
            for j in range(0, n, page):
                m = min(page, n - j)
                w[cache["table"][r, j // page].long(), h, :m] += p.sum(0)[j:j + m]
                wtol[cache["table"][r, j // page].long(), h, :m] += (p * (rel + x * group * U32)).sum(0)[j:j + m] + 1e-30
        at += x
    return o, tol, w, wtol


def turned(x, weight, eps, cos, sin, positions, interleaved):
    """Norm and rotation in 64 bits, and the bound of an fp32 evaluation rounded once: (d + 16) u for norm
    and products, relative to the two terms of the rotation, and half a step of the result."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = y.abs()
    if cos is not None:
        half = cos.shape[1]
        c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
        i = torch.arange(half, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        z, size = y.clone(), y.abs()
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = (y[..., a].abs() + y[..., b].abs())
        y = z
    return y, size * (x.shape[-1] + 16) * U32 + half_step(x.dtype) * y.abs() + 1e-30


def keep(weights, length, budget, first, last):
    """Kept slots of one head: first and last ones, and the heaviest between (ties to the lowest slot, NaN least)."""
    if length <= budget:
        return list(range(length))
    w = [(-float("inf") if x != x else x) for x in weights[:length].tolist()]
    mid = sorted(range(first, length - last), key=lambda j: (-w[j], j))[:budget - first - last]
    return list(range(first)) + sorted(mid) + list(range(length - last, length))
