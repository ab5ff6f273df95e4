"""The paged K/V cache, rotary positions and attention over the cache from their definitions, in 64 bits and without
the package's code.  Caches are dicts of the four buffers."""
import math

import torch

TINY = 2.0 ** -100
E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()   # 0 ... 448


def new_cache(pages, page, Hkv, D, device="cpu", fill=0):
    """A cache whose unwritten rows hold `fill` as codes, and NaN as scales when fill is not 0."""
    shape = (pages, Hkv, page, D)
    k8 = torch.full(shape, fill, dtype=torch.uint8, device=device).view(torch.int8)
    v8 = torch.full(shape, fill, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    s = torch.full(shape[:3], float("nan") if fill else 0.0, device=device)
    return dict(k8=k8, ks=s, v8=v8, vs=s.clone())


def codes(x, most):
    """(codes as numbers, scale) of rows x: nearest with ties away from zero, rows rules of the cache."""
    x = x.double()
    a = x.abs().amax(-1)
    a = torch.where(x.isnan().any(-1), torch.full_like(a, math.nan), a)
    finite = torch.isfinite(a)
    ok = finite & (a >= TINY)
    t = torch.where(ok[..., None], x * most / torch.where(ok, a, torch.ones_like(a))[..., None], torch.zeros_like(x))
    if most == 127:
        near = (t.abs() + 0.5).floor()
    else:
        grid = E4M3.to(x.device)
        near = grid[torch.bucketize(t.abs().contiguous(), (grid[1:] + grid[:-1]) / 2, right=True)]
    scale = torch.where(ok, a / most, torch.where(finite, torch.zeros_like(a), torch.full_like(a, math.nan)))
    return torch.copysign(near, t), scale.float()


def place(cache, table, b, at):
    page = cache["k8"].shape[2]
    at = torch.as_tensor(at, device=table.device).long()
    return table[b].long()[at // page], at % page


def append(cache, k, v, table, lens, counts=None):
    """k, v (B, S, Hkv, D) written at lens[b] ...; in place."""
    for b in range(k.shape[0]):
        n = k.shape[1] if counts is None else int(counts[b])
        if n == 0:
            continue
        p, r = place(cache, table, b, range(int(lens[b]), int(lens[b]) + n))
        for x, name, scale, most in ((k, "k8", "ks", 127), (v, "v8", "vs", 448)):
            c, s = codes(x[b, :n], most)
            if name == "k8":
                cache[name][p, :, r] = c.to(torch.int8)
            else:
                cache[name].view(torch.uint8)[p, :, r] = c.float().to(torch.float8_e4m3fn).view(torch.uint8)
            cache[scale][p, :, r] = s


def rows(cache, table, b, n):
    """K, V of the first n positions of sequence b, (n, Hkv, D) in 64 bits."""
    p, r = place(cache, table, b, range(n))
    return (cache["k8"][p, :, r].double() * cache["ks"][p, :, r].double()[..., None],
            cache["v8"][p, :, r].double() * cache["vs"][p, :, r].double()[..., None])


def attention(q, cache, table, lens, mask=None, counts=None, sm_scale=None):
    """q (B, T, H, D) -> o, lse and, for tolerances, the mean |v| under the weights, the largest sum of |q k| of a
    row's visible scores, and the largest weight * row scale (all per output row)."""
    B, T, H, D = q.shape
    Hkv = cache["k8"].shape[1]
    scale = D ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros((B, T, H, D), dtype=torch.float64, device=q.device)
    mean, lse = torch.zeros_like(o), torch.full((B, H, T), -math.inf, dtype=torch.float64, device=q.device)
    most, top = torch.zeros((B, T, H), dtype=torch.float64, device=q.device), torch.zeros((B, T, H), dtype=torch.float64, device=q.device)
    for b in range(B):
        n, m = int(lens[b]), T if counts is None else int(counts[b])
        if m == 0:
            continue
        k, v = rows(cache, table, b, n + m)
        _, vs = (cache["v8"], cache["vs"])
        p_, r_ = place(cache, table, b, range(n + m))
        vscale = vs[p_, :, r_].double()
        own = torch.ones((m, m), dtype=torch.bool, device=q.device).tril() if mask is None else \
            (mask if mask.dim() == 2 else mask[b if mask.shape[0] > 1 else 0])[:m, :m]
        see = torch.cat((torch.ones((m, n), dtype=torch.bool, device=q.device), own), 1)
        for h in range(H):
            g = h * Hkv // H
            kk, vv = k[:, g], v[:, g]
            s = (q[b, :m, h].double() @ kk.T * scale).masked_fill(~see, -math.inf)
            big = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(big.isinf(), torch.zeros_like(big), big)), torch.zeros_like(s))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, torch.ones_like(total))
            used = see.any(0)                      # what no row sees may hold anything
            vz = torch.where(used[:, None], vv, torch.zeros_like(vv))
            o[b, :m, h] = p @ vz
            mean[b, :m, h] = p @ vz.abs()
            lse[b, h, :m] = (big + torch.log(total))[:, 0]
            kz = torch.where(used[:, None], kk, torch.zeros_like(kk))
            most[b, :m, h] = ((q[b, :m, h].double().abs() @ kz.abs().T) * see).amax(-1) * scale
            top[b, :m, h] = (p * torch.where(used, vscale[:, g], torch.zeros_like(vscale[:, g]))).amax(-1)
    return o, lse, mean, most, top


def rotary(x, positions, w, magnitude, R, interleaved, back=False):
    """x (B, S, H, D), positions (B, S), w (R / 2,) radians per position."""
    x = x.double()
    a = positions.double()[..., None] * w.to(x.device) * (-1 if back else 1)
    c, s = magnitude * a.cos()[:, :, None], magnitude * a.sin()[:, :, None]
    y = x.clone()
    one, two = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    y[..., one], y[..., two] = x[..., one] * c - x[..., two] * s, x[..., two] * c + x[..., one] * s
    return y
