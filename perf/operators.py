"""Measured cases of the serving and position operators: rotary positions (with the backward pass), the paged
int8 / e4m3 K/V cache (append, read, keep) and attention over that cache for single tokens and drafted trees.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, with ``own`` set, through
the framework's entry points; both take the same state.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -100  # rows whose largest magnitude is below this are stored as zero rows


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a batch of prompts far into a long context, frequencies scaled for it (grouped heads)
        dict(name="rotary-prompt", op="rotary", B=4, S=8192, H=32, Hkv=8, D=128, R=128, interleaved=False,
             scaling="ramp", start=120000, dtype="bf16", train=False),
        # a training step: forward and gradient, interleaved pairs on part of the head, an odd length
        dict(name="rotary-train", op="rotary", B=2, S=4095, H=16, Hkv=16, D=96, R=64, interleaved=True,
             scaling="none", start=0, dtype="f16", train=True),
        # one token of each of 64 running sequences written into the cache: latency
        dict(name="append-step", op="append", B=64, S=1, Hkv=8, D=128, page=16, ctx=700, dtype="bf16", ragged=False),
        # ragged prompts written into the cache
        dict(name="append-prompt", op="append", B=4, S=8190, Hkv=8, D=128, page=64, ctx=100, dtype="bf16", ragged=True),
        # a short shared prefix read back, three ragged sequences
        dict(name="read-short", op="read", B=3, Hkv=4, D=96, page=32, ctx=1001, dtype="f16"),
        # long contexts read back in front of a dense attention call
        dict(name="read-long", op="read", B=8, Hkv=8, D=128, page=64, ctx=32760, dtype="bf16"),
        # the accepted path of a small tree of drafts, few sequences: latency
        dict(name="keep-few", op="keep", B=4, Hkv=8, D=128, page=16, ctx=500, T=16, N=5),
        # the same for a full server batch
        dict(name="keep-batch", op="keep", B=256, Hkv=8, D=128, page=64, ctx=200, T=64, N=12),
        # one token over a short context: the smallest attention call
        dict(name="decode-one", op="attend", B=1, T=1, H=32, Hkv=8, D=128, page=16, ctx=1023, dtype="bf16", tree=False,
             ragged=False),
        # one token of each of 16 long sequences
        dict(name="decode-long", op="attend", B=16, T=1, H=32, Hkv=8, D=128, page=64, ctx=32760, dtype="bf16",
             tree=False, ragged=False),
        # a full tree of 64 drafted tokens for each of 8 sequences
        dict(name="tree-64", op="attend", B=8, T=64, H=32, Hkv=8, D=128, page=64, ctx=8190, dtype="bf16", tree=True,
             ragged=False),
        # small trees of unequal size, wide heads without groups
        dict(name="tree-odd", op="attend", B=3, T=13, H=16, Hkv=16, D=256, page=32, ctx=4999, dtype="f16", tree=True,
             ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "read", "keep", "attend", "attend"])
    D = rng.choice([64, 96, 128, 128, 256])
    H, Hkv = rng.choice([(32, 8), (16, 16), (16, 4), (40, 40), (8, 1), (12, 4), (5, 5)])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "f16"])
    if op == "rotary":
        B = _log_int(rng, 1, 64)
        S = _log_int(rng, 1, max(1, min(8192, 4 * 8192 * 40 * 128 // (B * (H + Hkv) * D))))
        train = rng.random() < 0.4
        return dict(op=op, B=B, S=S // 2 + 1 if train else S, H=H, Hkv=Hkv, D=D, R=rng.choice([D, D, D // 2]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "ramp"]),
                    start=rng.choice([0, 4096, 500000]), dtype=dtype, train=train)
    if op == "append":
        B = _log_int(rng, 1, 128)
        S = _log_int(rng, 1, max(1, min(8190, 4 * 8190 * 8 * 128 // (B * Hkv * D))))
        return dict(op=op, B=B, S=S, Hkv=Hkv, D=D, page=page, ctx=_log_int(rng, 1, 1000), dtype=dtype,
                    ragged=rng.random() < 0.5)
    if op == "read":
        B = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, max(1, min(32760, 8 * 32760 * 8 * 128 // (B * Hkv * D))))
        return dict(op=op, B=B, Hkv=Hkv, D=D, page=page, ctx=ctx, dtype=dtype)
    if op == "keep":
        T = _log_int(rng, 2, 64)
        return dict(op=op, B=_log_int(rng, 1, 256), Hkv=min(Hkv, 16), D=min(D, 128), page=page, ctx=_log_int(rng, 1, 250),
                    T=T, N=rng.randint(1, min(T, 12)))
    B = _log_int(rng, 1, 64)
    T = 1 if rng.random() < 0.4 else _log_int(rng, 2, 64)
    most = min(16 * 32760 * 8 * 128 // (B * Hkv * D), 8 * 64 * 32 * 8190 * 128 // (B * T * H * D), 32760)
    return dict(op=op, B=B, T=T, H=H, Hkv=Hkv, D=D, page=page, ctx=_log_int(rng, 1, max(1, most)), dtype=dtype,
                tree=T > 1 and rng.random() < 0.7, ragged=T > 1 and rng.random() < 0.5)


def _lens(c):
    """Context lengths of the case's sequences: fixed by the case, the first one full and the others down to half."""
    r = random.Random("%d %d" % (c["B"], c["ctx"]))
    return [c["ctx"]] + [r.randint((c["ctx"] + 1) // 2, c["ctx"]) for _ in range(c["B"] - 1)]


def _counts(c, n):
    """New tokens of each sequence: all n, or unequal numbers of them in a padded batch."""
    if not c.get("ragged"):
        return [n] * c["B"]
    r = random.Random("%d %d counts" % (c["B"], n))
    return [n] + [r.randint((n + 1) // 2, n) for _ in range(c["B"] - 1)]


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _cache(g, c, lens, new):
    """A paged cache whose written rows hold quantised K and V and whose pages are dealt to the sequences in random
    order; table entries past a sequence's pages are -1."""
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    need = [(n + new + page - 1) // page for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["B"], max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k8 = torch.empty((total, Hkv, page, D), dtype=torch.int8, device="cuda")
    v8 = torch.empty((total, Hkv, page, D), dtype=torch.float8_e4m3fn, device="cuda")
    ks = torch.empty((total, Hkv, page), device="cuda")
    vs = torch.empty((total, Hkv, page), device="cuda")
    offset = torch.randn((Hkv, 1, D), device="cuda", generator=g)   # K has an offset for each channel, as trained keys have
    step = max(1, 32 * 2 ** 20 // (Hkv * page * D))
    for p in range(0, total, step):
        n = min(step, total - p)
        k8[p:p + n], ks[p:p + n] = _to_int8(torch.randn((n, Hkv, page, D), device="cuda", generator=g) + offset)
        v8[p:p + n], vs[p:p + n] = _to_e4m3(torch.randn((n, Hkv, page, D), device="cuda", generator=g))
    return dict(k8=k8, ks=ks, v8=v8, vs=vs, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(c)}
    if c["op"] == "rotary":
        dt = DTYPES[c["dtype"]]
        for name, h in (("q", c["H"]), ("k", c["Hkv"])):
            x = torch.randn((c["B"], c["S"], h, c["D"]), device="cuda", generator=g).to(dt)
            s[name] = x.requires_grad_(c["train"])
            if c["train"]:
                s["d" + name] = torch.randn((c["B"], c["S"], h, c["D"]), device="cuda", generator=g).to(dt)
        first = c["start"] + torch.randint(0, 64, (c["B"], 1), device="cuda", generator=g)
        s["positions"] = (first + torch.arange(c["S"], device="cuda")).to(torch.int32)
        return s
    lens = _lens(c)
    if c["op"] == "append":
        dt = DTYPES[c["dtype"]]
        s.update(_cache(g, c, lens, c["S"]))
        shape = (c["B"], c["S"], c["Hkv"], c["D"])
        s["k"] = (torch.randn(shape, device="cuda", generator=g) + torch.randn(shape[2:], device="cuda", generator=g)).to(dt)
        s["v"] = torch.randn(shape, device="cuda", generator=g).to(dt)
        if c["ragged"]:
            s["counts"] = torch.tensor(_counts(c, c["S"]), dtype=torch.int32, device="cuda")
    elif c["op"] == "read":
        s.update(_cache(g, c, lens, 0))
    elif c["op"] == "keep":
        s.update(_cache(g, c, lens, c["T"]))
        nodes = torch.rand((c["B"], c["T"]), device="cuda", generator=g).argsort(dim=1)[:, :c["N"]]
        s["keep"] = nodes.sort(dim=1).values.to(torch.int32).contiguous()
        s["counts"] = torch.tensor(_counts({**c, "ragged": True}, c["N"]), dtype=torch.int32, device="cuda")
    else:
        s.update(_cache(g, c, lens, c["T"]))
        s["q"] = (1.5 * torch.randn((c["B"], c["T"], c["H"], c["D"]), device="cuda", generator=g)).to(DTYPES[c["dtype"]])
        if c["ragged"]:
            s["counts"] = torch.tensor(_counts(c, c["T"]), dtype=torch.int32, device="cuda")
        if c["tree"]:
            s["mask"] = _trees(g, c["B"], c["T"])
    return s


def _trees(g, B, T):
    """Ancestor masks of B random trees of T nodes (a node's parent comes before it; some nodes are roots)."""
    parent = (torch.rand((B, T), device="cuda", generator=g) * (torch.arange(T, device="cuda") + 1)).long() - 1
    mask = torch.zeros((B, T, T), dtype=torch.bool, device="cuda")
    rows = torch.arange(B, device="cuda")
    for i in range(T):
        up = parent[:, i]
        mask[:, i] = mask[rows, up.clamp(min=0)] & (up >= 0)[:, None]
        mask[:, i, i] = True
    return mask


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _row_max(x):
    """Largest magnitude of each row, and where the row is stored as it is (finite, not tiny)."""
    a = x.abs().amax(-1)
    return a, torch.isfinite(a) & (a >= TINY)


def _scale(a, ok, most):
    one = torch.full_like(a, most)
    return torch.where(ok, a / one, torch.where(torch.isfinite(a), torch.zeros_like(a), torch.full_like(a, float("nan"))))


def _to_int8(x):
    """int8 codes round(127 x / max|x|), ties away from zero, and the scale max|x| / 127 of each row."""
    a, ok = _row_max(x)
    t = torch.where(ok[..., None], x * 127.0 / torch.where(ok, a, 1.0)[..., None], 0.0)
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), _scale(a, ok, 127.0)


def _to_e4m3(x):
    """e4m3 codes of 448 x / max|x| (nearest, ties away from zero) and the scale max|x| / 448 of each row."""
    a, ok = _row_max(x)
    t = torch.where(ok[..., None], x * 448.0 / torch.where(ok, a, 1.0)[..., None], 0.0)
    e = torch.frexp(t).exponent.clamp(min=-5)                 # |t| < 2^e; three fraction bits, steps of 2^-9 at the least
    step = torch.exp2((e - 4).to(x.dtype))
    return (torch.sign(t) * torch.floor(t.abs() / step + 0.5) * step).to(torch.float8_e4m3fn), _scale(a, ok, 448.0)


def _slots(s, at):
    """(page, row in the page) of the positions `at` [B, n] of each sequence."""
    page = s["k8"].shape[2]
    pages = torch.gather(s["table"], 1, (at // page).clamp(max=s["table"].shape[1] - 1).long())
    return pages.clamp(min=0).long(), (at % page).long()


def _gathered(s, n):
    """K and V of the first n positions in fp32, (B, Hkv, n, D); what is behind a sequence's pages is anything."""
    page = s["k8"].shape[2]
    pages = s["table"][:, :(n + page - 1) // page].clamp(min=0).long()
    k = s["k8"][pages].float() * s["ks"][pages][..., None]
    v = s["v8"][pages].float() * s["vs"][pages][..., None]
    return [x.transpose(1, 2).flatten(2, 3)[:, :, :n] for x in (k, v)]


def _frequencies(c, dtype=torch.float64):
    R = c["R"]
    i = torch.arange(0, R, 2, dtype=dtype, device="cuda")
    if c["scaling"] == "ntk":
        return (10000.0 * 4.0 ** (R / (R - 2))) ** (-i / R), 1.0
    w = 10000.0 ** (-i / R)
    if c["scaling"] == "linear":
        return w / 4.0, 1.0
    if c["scaling"] == "ramp":
        r = 8192.0 * w / (2 * math.pi)
        g = ((r - 1.0) / 31.0).clamp(0, 1)
        return w * ((1 - g) / 16.0 + g), 0.1 * math.log(16.0) + 1
    return w, 1.0


def _rotate(x, cos, sin, c):
    R, h = c["R"], c["R"] // 2
    y = x.float()
    x1, x2 = (y[..., 0:R:2], y[..., 1:R:2]) if c["interleaved"] else (y[..., :h], y[..., h:R])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    turned = torch.stack((y1, y2), -1).flatten(-2) if c["interleaved"] else torch.cat((y1, y2), -1)
    return torch.cat((turned, y[..., R:]), -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    w, m = _frequencies(c)
    angle = s["positions"].double()[..., None] * w
    cos, sin = (m * angle.cos()).float()[:, :, None], (m * angle.sin()).float()[:, :, None]
    out = [_rotate(s["q"].detach(), cos, sin, c), _rotate(s["k"].detach(), cos, sin, c)]
    if c["train"]:
        out += [_rotate(s["dq"], cos, -sin, c), _rotate(s["dk"], cos, -sin, c)]
    return out


def _plain_append(s):
    S = s["k"].shape[1]
    i = torch.arange(S, device="cuda")
    new = i < s["counts"][:, None] if "counts" in s else torch.ones((s["lens"].shape[0], S), dtype=torch.bool, device="cuda")
    pages, rows = _slots(s, s["lens"][:, None] + i)
    kc, kscale = _to_int8(s["k"].float())
    vc, vscale = _to_e4m3(s["v"].float())
    s["k8"][pages, :, rows] = torch.where(new[..., None, None], kc, s["k8"][pages, :, rows])
    bits = s["v8"].view(torch.uint8)
    bits[pages, :, rows] = torch.where(new[..., None, None], vc.view(torch.uint8), bits[pages, :, rows])
    s["ks"][pages, :, rows] = torch.where(new[..., None], kscale, s["ks"][pages, :, rows])
    s["vs"][pages, :, rows] = torch.where(new[..., None], vscale, s["vs"][pages, :, rows])
    return [s["k8"], s["ks"], s["v8"], s["vs"]]


def _plain_read(s):
    c = s["case"]
    held = (torch.arange(c["ctx"], device="cuda") < s["lens"][:, None])[:, None, :, None]
    return [torch.where(held, x, 0.0).to(DTYPES[c["dtype"]]).transpose(1, 2).contiguous() for x in _gathered(s, c["ctx"])]


def _plain_keep(s):
    i = torch.arange(s["keep"].shape[1], device="cuda", dtype=torch.int32)
    from_, to = s["lens"][:, None] + torch.where(i < s["counts"][:, None], s["keep"], i), s["lens"][:, None] + i
    (p0, r0), (p1, r1) = _slots(s, from_), _slots(s, to)
    for x in (s["k8"], s["ks"], s["v8"].view(torch.uint8), s["vs"]):
        x[p1, :, r1] = x[p0, :, r0]
    return [s["k8"], s["ks"], s["v8"], s["vs"]]


def _visible(s, n):
    """(B, T, n): the keys each row attends."""
    c = s["case"]
    T = c["T"]
    i, j = torch.arange(T, device="cuda"), torch.arange(n, device="cuda")
    lens = s["lens"].long()[:, None, None]
    t = j[None, None] - lens                                    # number of the drafted token behind a key
    if "mask" in s:
        drafts = torch.gather(s["mask"], 2, t.clamp(0, T - 1).expand(-1, T, -1)) & (t >= 0) & (t < T)
    else:
        drafts = (t >= 0) & (t <= i[:, None])
    seen = (t < 0) | drafts
    if "counts" in s:
        m = s["counts"].long()[:, None, None]
        seen = seen & (t < m) & (i[:, None] < m)
    return seen


def _plain_attend(s):
    c = s["case"]
    g, n = c["H"] // c["Hkv"], c["ctx"] + c["T"]
    k, v = _gathered(s, n)
    seen = _visible(s, n)[:, None, None]                        # (B, 1, 1, T, n)
    written = (torch.arange(n, device="cuda") < (s["lens"] + c["T"])[:, None])[:, None, :, None]
    k, v = torch.where(written, k, 0.0), torch.where(written, v, 0.0)
    q = s["q"].float().unflatten(2, (c["Hkv"], g)).permute(0, 2, 3, 1, 4)
    x = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (g, c["T"])) * c["D"] ** -0.5
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (g, c["T"])) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0].flatten(1, 2)
    return [o.flatten(1, 2).transpose(1, 2).contiguous().to(s["q"].dtype), lse]


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "keep": _plain_keep,
          "attend": _plain_attend}


def _framework(s):
    """The package, and the handle (cache or frequencies) that a program keeps next to its tensors."""
    if "rdna4-sageattention_b200" not in sys.path:
        sys.path.insert(1, "rdna4-sageattention_b200")
    import rdna4_sage
    if "handle" not in s:
        c = s["case"]
        if c["op"] == "rotary":
            more = {"none": {}, "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=4.0),
                    "ramp": dict(scaling="ramp", factor=16.0, original_len=8192, ramp=(1.0, 32.0))}[c["scaling"]]
            s["handle"] = rdna4_sage.Rotary(c["D"], rotary_dim=c["R"], base=10000.0, interleaved=c["interleaved"],
                                            device="cuda", **more)
        else:
            s["handle"] = rdna4_sage.PagedKV(s["k8"], s["ks"], s["v8"], s["vs"])
    return rdna4_sage, s["handle"]


def _own(s):
    sage, handle = _framework(s)
    c = s["case"]
    if c["op"] == "rotary":
        out = sage.rotary(s["q"], s["k"], s["positions"], handle, tensor_layout="NHD")
        if c["train"]:
            return [*out, *torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"]))]
        return list(out)
    if c["op"] == "append":
        sage.paged_kv_append(handle, s["k"], s["v"], s["table"], s["lens"], counts=s.get("counts"), tensor_layout="NHD")
        return [s["k8"], s["ks"], s["v8"], s["vs"]]
    if c["op"] == "read":
        return list(sage.paged_kv_read(handle, s["table"], s["lens"], c["ctx"], dtype=DTYPES[c["dtype"]],
                                       tensor_layout="NHD"))
    if c["op"] == "keep":
        sage.paged_kv_keep(handle, s["table"], s["lens"], s["keep"], counts=s["counts"])
        return [s["k8"], s["ks"], s["v8"], s["vs"]]
    return list(sage.attention_paged_kv(s["q"], handle, s["table"], s["lens"], tree_mask=s.get("mask"),
                                        counts=s.get("counts"), tensor_layout="NHD", return_lse=True))


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["B"] * c["S"] * (c["H"] + c["Hkv"]) * c["D"] * (2 if c["train"] else 1)
        return {"bytes": 4 * n + 4 * c["B"] * c["S"], "flops": 3 * n * c["R"] // c["D"]}
    if c["op"] == "append":
        rows = sum(_counts(c, c["S"])) * c["Hkv"] * 2
        return {"bytes": rows * (3 * c["D"] + 4), "flops": 3 * rows * c["D"]}
    if c["op"] == "read":
        rows, held = 2 * c["B"] * c["ctx"] * c["Hkv"], 2 * sum(_lens(c)) * c["Hkv"]
        return {"bytes": held * (c["D"] + 4) + 2 * rows * c["D"], "flops": held * c["D"]}
    if c["op"] == "keep":
        rows = sum(_counts({**c, "ragged": True}, c["N"])) * c["Hkv"]
        return {"bytes": 2 * rows * (2 * c["D"] + 8), "flops": 0}
    lens, new = _lens(c), _counts(c, c["T"])
    keys = sum(n + m for n, m in zip(lens, new))
    pairs = sum(m * n + m * (m + 1) // 2 for n, m in zip(lens, new))
    moved = keys * c["Hkv"] * (2 * c["D"] + 8) + c["B"] * c["T"] * c["H"] * (4 * c["D"] + 4)
    return {"bytes": moved + (c["B"] * c["T"] ** 2 if c["tree"] else 0), "flops": 4 * pairs * c["H"] * c["D"]}


# ---------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_rotary(s):
    c = s["case"]
    w, m = _frequencies(c)
    turn = m * torch.polar(torch.ones_like(w), s["positions"].double()[..., None] * w)[:, :, None]

    def turned(x, by):
        x = x.detach().double()
        part = x[..., :c["R"]]
        pairs = part.unflatten(-1, (-1, 2)) if c["interleaved"] else part.unflatten(-1, (2, -1)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
        return torch.cat((y, x[..., c["R"]:]), -1)

    return [turned(s[name], turn if name in ("q", "k") else turn.conj()) for name in ("q", "k", "dq", "dk") if name in s]


def _exact_append(s):
    c = s["case"]
    grid = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()   # 0 ... 448
    border = (grid[1:] + grid[:-1]) / 2
    k8, ks, v8, vs = s["k8"].double(), s["ks"].double(), s["v8"].double(), s["vs"].double()
    for b, (n, m) in enumerate(zip(_lens(c), _counts(c, c["S"]))):
        at = torch.arange(n, n + m, device="cuda")
        page, row = s["table"][b].long()[at // c["page"]], at % c["page"]
        for x, code, scale, most in ((s["k"], k8, ks, 127), (s["v"], v8, vs, 448)):
            x = x[b, :m].double()
            a = x.abs().amax(-1, keepdim=True)
            t = x * most / a
            near = (t.abs() + 0.5).floor() if most == 127 else grid[torch.bucketize(t.abs(), border, right=True)]
            code[page, :, row] = torch.copysign(near, t)
            scale[page, :, row] = (a / most)[..., 0]
    return [k8, ks, v8, vs]


def _exact_read(s):
    c = s["case"]
    out = [torch.zeros((c["B"], c["ctx"], c["Hkv"], c["D"]), dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, n in enumerate(_lens(c)):
        at = torch.arange(n, device="cuda")
        page, row = s["table"][b].long()[at // c["page"]], at % c["page"]
        out[0][b, :n] = s["k8"][page, :, row].double() * s["ks"][page, :, row].double()[..., None]
        out[1][b, :n] = s["v8"][page, :, row].double() * s["vs"][page, :, row].double()[..., None]
    return out


def _exact_keep(s):
    c = s["case"]
    to = [x.clone() for x in (s["k8"], s["ks"], s["v8"].view(torch.uint8), s["vs"])]
    table, keep = s["table"].tolist(), s["keep"].tolist()
    for b, (n, m) in enumerate(zip(_lens(c), _counts({**c, "ragged": True}, c["N"]))):
        for i in range(m):
            (p0, r0), (p1, r1) = divmod(n + keep[b][i], c["page"]), divmod(n + i, c["page"])
            for x, y in zip((s["k8"], s["ks"], s["v8"].view(torch.uint8), s["vs"]), to):
                y[table[b][p1], :, r1] = x[table[b][p0], :, r0]
    return [to[0], to[1].double(), to[2].view(torch.float8_e4m3fn).double(), to[3].double()]


def _exact_attend(s):
    c = s["case"]
    B, T, H, D = s["q"].shape
    g = H // c["Hkv"]
    o = torch.zeros((B, T, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, T), -math.inf, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(_lens(c), _counts(c, T))):
        at = torch.arange(n + m, device="cuda")
        page, row = s["table"][b].long()[at // c["page"]], at % c["page"]
        k = s["k8"][page, :, row].double() * s["ks"][page, :, row].double()[..., None]
        v = s["v8"][page, :, row].double() * s["vs"][page, :, row].double()[..., None]
        mine = s["mask"][b, :m, :m] if "mask" in s else torch.ones((m, m), dtype=torch.bool, device="cuda").tril()
        hide = torch.cat((torch.zeros((m, n), dtype=torch.bool, device="cuda"), ~mine), 1)
        for h in range(H):
            x = (s["q"][b, :m, h].double() @ k[:, h // g].T / math.sqrt(D)).masked_fill(hide, -math.inf)
            lse[b, h, :m] = torch.logsumexp(x, -1)
            o[b, :m, h] = torch.softmax(x, -1) @ v[:, h // g]
    return [o, lse]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "read": _exact_read, "keep": _exact_keep,
            "attend": _exact_attend}[case["op"]](s)
