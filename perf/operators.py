"""The operators of a decode step (or of a prompt's chunk) over a cache held in 4 bits, as cases that can be timed and compared.

  gemv       matrix-vector products with int4 weights and a scale (and maybe an offset) for each group of k
  rope       norms of the query and key heads with the rotation in the same pass, keys and queries written out
  append     the same pass with K and V put into the 4-bit cache; the rows are then read back as the values they stand for
  attention  attention of ragged sequences, one query token each or many, over that cache

Layouts, as include/b200lm_ops.h states them:

Weights.  Strips of 16 rows, blocks of 128 k; a block is two tiles of 64 k of 512 bytes, then the scales, then the offsets, as
[8 row pairs][128 / group][row g, row g + 8] 16-bit numbers.  In a tile lane 4g+t owns 16 bytes: byte 4j+i holds
k = 32 (j / 2) + 16 (j % 2) + 4 t + i, row g in the low and row g + 8 in the high nibble, two's complement.

Cache.  For each page and kv head: K codes, K scales, V codes, V scales of 256 positions.  Codes lie in planes of 128 dims (64 at
head size 64), a row of a plane is 64 (32) bytes.  K: byte t w + 4 step + i (w = 16 or 8) holds the dims 32 step + 4 t + i (low) and
16 more (high).  V: unit g of 8 (4) bytes, byte b holds the dims 16 b + g and 8 more; in planes of 128 the units of positions with
bit 1 set are exchanged with those 4 further.  Scales are fp16 pairs (s, m) for each group of dims; a code c stands for s c + m.
"""
import math

import torch

own = False

F32, BF16, F16 = 0, 1, 2
TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODE = {"fp32": F32, "bf16": BF16, "fp16": F16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
PAGE = 256


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # The query, key and value projection of the 1B layer for one user: the smallest call.
        {"name": "gemv-1x1536x1152", "kind": "gemv", "n": 1536, "k": 1152, "group": 32, "cols": 1, "x": "bf16", "y": "bf16", "scale": "bf16", "offset": False},
        # Gate and up of the 4B layer for three users, weights with offsets.
        {"name": "gemv-3x20480x2560", "kind": "gemv", "n": 20480, "k": 2560, "group": 64, "cols": 3, "x": "fp16", "y": "fp16", "scale": "fp16", "offset": True},
        # The head over the whole vocabulary: logits in fp32 of a few sessions.
        {"name": "gemv-2x262144x1152", "kind": "gemv", "n": 262144, "k": 1152, "group": 128, "cols": 2, "x": "fp32", "y": "fp32", "scale": "bf16", "offset": False},
        # One token of one user at the 27B head geometry.
        {"name": "rope-1-27b", "kind": "rope", "tokens": 1, "hq": 32, "hkv": 16, "hd": 128, "rot": 128, "type": "bf16", "far": 4095, "pad": 0},
        # A long prompt's chunk at the 4B head geometry, rows with padding between them.
        {"name": "rope-8191-4b", "kind": "rope", "tokens": 8191, "hq": 8, "hkv": 4, "hd": 256, "rot": 256, "type": "bf16", "far": 131072, "pad": 64},
        # A decode step of 9 users of the 1B model, rows in fp32 as its kernels keep them.
        {"name": "append-9-1b", "kind": "append", "tokens": 9, "seqs": 9, "hq": 4, "hkv": 1, "hd": 256, "rot": 256, "group": 64, "type": "fp32", "far": 8000},
        # A prompt of 2001 tokens at the 27B head geometry enters the cache.
        {"name": "append-2001-27b", "kind": "append", "tokens": 2001, "seqs": 1, "hq": 32, "hkv": 16, "hd": 128, "rot": 128, "group": 128, "type": "bf16", "far": 4096},
        # One user of the 1B model in a short conversation: latency.
        {"name": "attention-1x777", "kind": "attention", "batch": 1, "low": 777, "high": 777, "queries": 1, "hq": 4, "hkv": 1, "hd": 256, "group": 64, "window": 0, "type": "bf16"},
        # A server's decode step on the 4B geometry: 64 conversations of different lengths.
        {"name": "attention-64x8192", "kind": "attention", "batch": 64, "low": 300, "high": 8192, "queries": 1, "hq": 8, "hkv": 4, "hd": 256, "group": 64, "window": 0, "type": "bf16"},
        # Three long documents at the 27B geometry, fp32 as the decode kernels keep their rows.
        {"name": "attention-3x65536", "kind": "attention", "batch": 3, "low": 40001, "high": 65536, "queries": 1, "hq": 32, "hkv": 16, "hd": 128, "group": 128, "window": 0, "type": "fp32"},
        # Five drafted tokens of 16 users are verified on a layer with a window of 1024.
        {"name": "attention-16x5-window", "kind": "attention", "batch": 16, "low": 5, "high": 4097, "queries": 5, "hq": 8, "hkv": 4, "hd": 256, "group": 128, "window": 1024, "type": "fp16"},
        # Chunks of two long prompts meet what the cache holds of them.
        {"name": "attention-2x512-chunk", "kind": "attention", "batch": 2, "low": 4000, "high": 8192, "queries": 512, "hq": 8, "hkv": 4, "hd": 256, "group": 64, "window": 0, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["gemv", "gemv", "rope", "append", "attention", "attention", "attention"])
    if kind == "gemv":
        k = 2 * _log(rng, 64, 10752) if rng.random() < 0.5 else rng.choice([1152, 2560, 5376, 6912, 10240, 21504])
        n = _log(rng, 64, max(64, min(262144, 300_000_000 // k)))
        return {"kind": kind, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "cols": rng.randint(1, 8),
                "x": rng.choice(["fp32", "bf16", "fp16"]), "y": rng.choice(["fp32", "bf16", "fp16"]), "scale": rng.choice(["bf16", "fp16"]), "offset": rng.random() < 0.4}
    hq, hkv, hd = rng.choice([(4, 1, 256), (8, 4, 256), (32, 16, 128), (8, 4, 128), (16, 2, 128), (12, 4, 64)])
    group = 64 if hd == 64 else rng.choice([64, 128])
    typ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "rope":
        return {"kind": kind, "tokens": _log(rng, 1, 8191), "hq": hq, "hkv": hkv, "hd": hd, "rot": rng.choice([hd, hd, hd // 2]), "type": typ, "far": _log(rng, 8192, 131072),
                "pad": rng.choice([0, 8, 64])}
    if kind == "append":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, "tokens": seqs if rng.random() < 0.5 else seqs + _log(rng, 1, 4000), "seqs": seqs, "hq": hq, "hkv": hkv, "hd": hd, "rot": rng.choice([hd, hd, hd // 2]), "group": group,
                "type": typ, "far": _log(rng, 4096, 16384)}
    queries = rng.choice([1, 1, 1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
    high = _log(rng, max(16, queries), 65536 if queries <= 8 else 8192)
    room = min(64 * 8192 * 1024 // (high * hkv * hd), 2 * 8 * 512 * 8192 // (high * hq * queries), 64)
    return {"kind": kind, "batch": _log(rng, 1, max(1, room)), "low": rng.randint(min(high, queries), high), "high": high, "queries": queries, "hq": hq, "hkv": hkv, "hd": hd, "group": group,
            "window": rng.choice([0, 0, 0, 512, 1024]), "type": typ}


# ------------------------------------------------------------------------------------------------- sizes

def _lengths(case):
    """Cached positions of each sequence, from low to high; the longest is not the last."""
    b, low, high = case["batch"], case["low"], case["high"]
    return [high] if b == 1 else [low + (high - low) * ((i * 5 + 3) % b if math.gcd(5, b) == 1 else b - 1 - i) // (b - 1) for i in range(b)]


def _counts(case):
    """Query tokens of each sequence: all of them, or one less where there are several."""
    return [case["queries"] - (1 if case["queries"] > 1 and i % 3 == 1 else 0) for i in range(case["batch"])]


def _planes(hd):
    """(planes, dims of a plane)"""
    return (hd // 128, 128) if hd >= 128 else (1, hd)


def _row_bytes(hd, group):
    """K or V of one position and kv head: codes and scales."""
    return hd // 2 + 4 * (hd // group)


def work(case):
    kind = case["kind"]
    if kind == "gemv":
        n, k, c = case["n"], case["k"], case["cols"]
        weights = n * k // 2 + 2 * n * -(-k // case["group"]) * (2 if case["offset"] else 1)
        return {"bytes": weights + c * (k * SIZE[case["x"]] + n * SIZE[case["y"]]), "flops": 2 * n * k * c}
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if kind in ("rope", "append"):
        t, esz = case["tokens"], SIZE[case["type"]]
        table = t * (4 * case["rot"] + 4) + 8 * hd
        if kind == "rope":
            return {"bytes": 2 * t * (hq + hkv) * hd * esz + table, "flops": 10 * t * (hq + hkv) * hd}
        rows = t * hkv * 2
        return {"bytes": t * (2 * hq + 2 * hkv) * hd * esz + table + rows * (2 * _row_bytes(hd, case["group"]) + 4 * hd), "flops": 10 * t * (hq + 2 * hkv) * hd}
    keys = pairs = 0
    for s, n in zip(_lengths(case), _counts(case)):
        w = case["window"]
        first = max(0, s - n)
        keys += s - (max(0, first + 1 - w) if w else 0)
        pairs += sum(min(p + 1, w) if w else p + 1 for p in range(first, s))
    rows = sum(_counts(case)) * hq * hd * SIZE[case["type"]] * 2
    return {"bytes": keys * hkv * 2 * _row_bytes(hd, case["group"]) + rows, "flops": 4 * hd * hq * pairs}


# ------------------------------------------------------------------------------------------------- inputs

def _image(q, scale, offset, group):
    """Weights, scales and offsets of [n][k] in the operator's layout."""
    n, k = q.shape
    strips, blocks = -(-n // 16), -(-k // 128)
    full = torch.zeros(strips * 16, blocks * 128, dtype=torch.uint8, device=q.device)
    full[:n, :k] = q & 15
    tile = full.view(strips, 2, 8, blocks, 2, 2, 2, 4, 4)          # strip, half, g, block, tile, j / 2, j % 2, t, i
    codes = (tile[:, 0] | tile[:, 1] << 4).permute(0, 2, 3, 1, 6, 4, 5, 7).reshape(strips, blocks, 1024)
    parts = [codes]
    for x in (scale, offset):
        if x is not None:
            g = torch.zeros(strips * 16, blocks * 128 // group, dtype=x.dtype, device=q.device)
            g[:n, :x.shape[1]] = x
            g = g.view(strips, 2, 8, blocks, 128 // group).permute(0, 3, 2, 4, 1).contiguous()
            parts.append(g.view(torch.uint8).reshape(strips, blocks, -1))
    return torch.cat(parts, dim=2).contiguous()


def _pack(k_code, v_code, hd, slot):
    """Codes [..., hd] as bytes [..., planes, bytes of a row] of K and of V; `slot` [...] is the position in the page."""
    planes, dims = _planes(hd)
    k = k_code.view(*k_code.shape[:-1], planes, dims // 32, 2, 4, 4)                   # step, half, t, i
    kb = (k[..., 0, :, :] | k[..., 1, :, :] << 4).transpose(-3, -2).reshape(*k.shape[:-4], dims // 2)
    v = v_code.view(*v_code.shape[:-1], planes, dims // 16, 2, 8)                      # b, half, g
    vb = (v[..., 0, :] | v[..., 1, :] << 4).transpose(-2, -1)                          # [..., planes, g, b]
    if dims == 128:
        turned = (slot >> 1 & 1).bool()[..., None, None, None]
        vb = torch.where(turned, torch.roll(vb, 4, dims=-2), vb)
    return kb, vb.reshape(*vb.shape[:-2], dims // 2)


def _quantise(x, group):
    """Codes and (s, m) pairs of [..., hd]; 64 bits, since a value may lie next to the border of two codes."""
    g = x.unflatten(-1, (-1, group))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, m = ((high - low) / 15).to(torch.float16), low.to(torch.float16)
    c = torch.where(s > 0, ((g - m.to(x.dtype)) / s.to(x.dtype)).round().clamp(0, 15), torch.zeros_like(g))
    return c.to(torch.uint8).flatten(-2), torch.cat([s, m], dim=-1)


def _views(pages, hd, group):
    """K codes, K scales, V codes, V scales as views [page, kv head, ...] of the pages' bytes."""
    planes, dims = _planes(hd)
    codes, scales = PAGE * hd // 2, PAGE * 4 * (hd // group)
    p, h, _ = pages.shape
    at, out = 0, []
    for _ in range(2):
        out.append(pages[:, :, at:at + codes].view(p, h, planes, PAGE, dims // 2))
        out.append(pages[:, :, at + codes:at + codes + scales].view(torch.float16).view(p, h, PAGE, hd // group, 2))
        at += codes + scales
    return out


def _fill(pages, hd, group, gen):
    """Random rows, as keys behind a norm and values have them, into all of the pages."""
    kc, ks, vc, vs = _views(pages, hd, group)
    slot = torch.arange(PAGE, device="cuda")
    for a in range(0, pages.shape[0], 512):
        n = min(512, pages.shape[0] - a)
        k, kp = _quantise(torch.randn(n, pages.shape[1], PAGE, hd, device="cuda", generator=gen), group)
        v, vp = _quantise(torch.randn(n, pages.shape[1], PAGE, hd, device="cuda", generator=gen), group)
        kb, vb = _pack(k, v, hd, slot)
        kc[a:a + n], vc[a:a + n] = kb.transpose(2, 3), vb.transpose(2, 3)
        ks[a:a + n], vs[a:a + n] = kp, vp


def _page_bytes(hd, group):
    return PAGE * 2 * _row_bytes(hd, group)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "gemv":
        n, k, group = case["n"], case["k"], case["group"]
        q = torch.randn(n, k, device="cuda", generator=gen).mul_(2.6).round_().clamp_(-8, 7).to(torch.int8).view(torch.uint8)
        groups = -(-k // group)
        scale = (0.005 + 0.01 * torch.rand(n, groups, device="cuda", generator=gen)).to(TYPE[case["scale"]])
        offset = (0.01 * torch.randn(n, groups, device="cuda", generator=gen)).to(TYPE[case["scale"]]) if case["offset"] else None
        return {"case": case, "w": _image(q, scale, offset, group), "x": torch.randn(case["cols"], k, device="cuda", generator=gen).to(TYPE[case["x"]]),
                "y": torch.empty(case["cols"], n, device="cuda", dtype=TYPE[case["y"]])}
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if kind in ("rope", "append"):
        t, typ, half = case["tokens"], TYPE[case["type"]], case["rot"] // 2
        s = {"case": case, "gains": 1 + 0.1 * torch.randn(2, hd, device="cuda", generator=gen)}
        s["qkv"] = torch.randn(t, (hq + 2 * hkv) * hd + case.get("pad", 0), device="cuda", generator=gen).to(typ)
        turns = torch.arange(case["far"] + 1, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = torch.cos(turns).float(), torch.sin(turns).float()
        s["q"] = torch.empty(t, hq * hd, device="cuda", dtype=typ)
        if kind == "rope":
            # several prompts packed into one batch of rows, the last ones far along
            start = torch.randint(0, case["far"] + 2 - min(t, case["far"]), (1,), device="cuda", generator=gen)
            s["pos"] = ((start + torch.arange(t, device="cuda")) % (case["far"] + 1)).to(torch.int32)
            s["k"] = torch.empty(t, hkv * hd, device="cuda", dtype=typ)
            return s
        # each sequence takes an equal share of the tokens, behind what it holds already
        seqs = case["seqs"]
        seq = torch.arange(t, device="cuda") * seqs // t
        first = torch.searchsorted(seq, torch.arange(seqs, device="cuda"))
        held = torch.randint(0, case["far"] + 1 - -(-t // seqs), (seqs,), device="cuda", generator=gen)
        s["seq"], s["pos"] = seq.to(torch.int32), (held[seq] + torch.arange(t, device="cuda") - first[seq]).to(torch.int32)
        per = -(-(case["far"] + 1) // PAGE)
        # only the pages of the new rows matter here: every sequence's are spread over one pool
        s["table"] = (torch.randperm(seqs * per, device="cuda", generator=gen)).to(torch.int32).view(seqs, per)
        s["pages"] = torch.zeros(seqs * per, hkv, _page_bytes(hd, case["group"]), device="cuda", dtype=torch.uint8)
        s["k"], s["v"] = (torch.empty(t, hkv, hd, device="cuda") for _ in range(2))
        return s
    lengths, counts, per = _lengths(case), _counts(case), -(-case["high"] // PAGE)
    need = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(need), device="cuda", generator=gen).to(torch.int32)
    table, at = torch.zeros(case["batch"], per, device="cuda", dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    pages = torch.empty(sum(need), hkv, _page_bytes(hd, case["group"]), device="cuda", dtype=torch.uint8)
    _fill(pages, hd, case["group"], gen)
    tokens, typ = sum(counts), TYPE[case["type"]]
    starts = torch.tensor([sum(counts[:i]) for i in range(case["batch"] + 1)], device="cuda", dtype=torch.int32)
    s = {"case": case, "pages": pages, "table": table, "lengths": torch.tensor(lengths, device="cuda", dtype=torch.int32), "starts": starts, "tokens": tokens,
         "q": (1.5 * torch.randn(tokens, hq * hd, device="cuda", generator=gen)).to(typ), "out": torch.empty(tokens, hq * hd, device="cuda", dtype=typ)}
    # room for the partial results of split sequences, zero before the first call
    s["room"] = torch.zeros(32 << 20, device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------------------------------------- plain forms

def _norm_rope(x, gain, cos, sin, rot):
    """x [t, heads, hd] in 64 bits, cos and sin [t, 1, rot / 2]."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
    a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], dim=-1)


def _unpack(kc, vc, hd, slot):
    """Codes [..., hd] of bytes [..., planes, bytes of a row]."""
    planes, dims = _planes(hd)
    kb = kc.unflatten(-1, (4, dims // 32, 4))                                          # t, step, i
    k = torch.stack([kb & 15, kb >> 4], dim=-4).permute(*range(kb.dim() - 3), -2, -4, -3, -1)
    vb = vc.unflatten(-1, (8, dims // 16))                                             # unit, b
    if dims == 128:
        vb = torch.where((slot >> 1 & 1).bool()[..., None, None, None], torch.roll(vb, 4, dims=-2), vb)
    v = torch.stack([vb & 15, vb >> 4], dim=-1).permute(*range(vb.dim() - 2), -2, -1, -3)
    return k.reshape(*kc.shape[:-2], hd), v.reshape(*vc.shape[:-2], hd)


def _values(code, pair):
    """s c + m of codes [..., hd] and pairs [..., groups, 2]."""
    c = code.unflatten(-1, (pair.shape[-2], -1)).float()
    return (pair[..., :1].float() * c + pair[..., 1:].float()).flatten(-2)


def _plain_gemv(s):
    case = s["case"]
    n, k, group = case["n"], case["k"], case["group"]
    w = s["w"]
    strips, blocks, _ = w.shape
    t = w[..., :1024].view(strips, blocks, 2, 8, 4, 2, 2, 4)                           # tile, g, t, j / 2, j % 2, i
    q = torch.stack([t & 15, t >> 4], dim=1).permute(0, 1, 4, 2, 3, 6, 7, 5, 8).reshape(strips * 16, blocks * 128)[:n]
    q = ((q ^ 8).to(torch.int8) - 8).float().unflatten(1, (-1, group))
    g = w[..., 1024:].reshape(strips, blocks, -1).view(TYPE[case["scale"]]).view(strips, blocks, -1, 8, 128 // group, 2)
    g = g.permute(2, 0, 5, 3, 1, 4).reshape(g.shape[2], strips * 16, -1)[:, :n].float()
    q = q * g[0][..., None]
    if case["offset"]:
        q = q + g[1][..., None]
    return [(s["x"].float() @ q.flatten(1)[:, :k].T).to(TYPE[case["y"]])]


def _plain_rows(s):
    """Queries and keys behind norm and rotation, in 64 bits: the keys are rounded once, to 32, before their codes are decided."""
    case = s["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    rows = s["qkv"][:, :(hq + 2 * hkv) * hd].double().unflatten(1, (-1, hd))
    at = s["pos"].long()
    cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
    return (_norm_rope(rows[:, :hq], s["gains"][0].double(), cos, sin, case["rot"]), _norm_rope(rows[:, hq:hq + hkv], s["gains"][1].double(), cos, sin, case["rot"]),
            rows[:, hq + hkv:])


def _plain_rope(s):
    typ = s["qkv"].dtype
    q, k, _ = _plain_rows(s)
    return [q.flatten(1).to(typ), k.flatten(1).to(typ)]


def _plain_append(s):
    case = s["case"]
    hd, group = case["hd"], case["group"]
    q, k, v = _plain_rows(s)
    page, slot = s["table"][s["seq"].long(), s["pos"].long() // PAGE].long(), s["pos"].long() % PAGE
    kcode, kpair = _quantise(k.float().double(), group)
    vcode, vpair = _quantise(v, group)
    kb, vb = _pack(kcode, vcode, hd, slot[:, None])
    kc, ks, vc, vs = _views(s["pages"], hd, group)
    kc[page, :, :, slot], vc[page, :, :, slot], ks[page, :, slot], vs[page, :, slot] = kb, vb, kpair, vpair
    kcode, vcode = _unpack(kc[page, :, :, slot], vc[page, :, :, slot], hd, slot[:, None])
    return [q.flatten(1).to(s["qkv"].dtype), _values(kcode, ks[page, :, slot]), _values(vcode, vs[page, :, slot])]


def _plain_attention(s):
    case = s["case"]
    hq, hkv, hd, b, most = case["hq"], case["hkv"], case["hd"], case["batch"], case["queries"]
    per = s["table"].shape[1]
    kc, ks, vc, vs = (x[s["table"].long()] for x in _views(s["pages"], hd, case["group"]))     # [b, per, hkv, ...]
    k, v = _unpack(kc.transpose(3, 4), vc.transpose(3, 4), hd, torch.arange(PAGE, device="cuda"))
    k = _values(k, ks).transpose(1, 2).reshape(b, hkv, 1, per * PAGE, hd)
    v = _values(v, vs).transpose(1, 2).reshape(b, hkv, 1, per * PAGE, hd)
    start, count = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(most, device="cuda")
    row = (start[:, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[row].view(b, most, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4)
    x = (q @ k.transpose(-1, -2)).mul_(hd ** -0.5)                                            # [b, hkv, group, most, keys]
    at = (s["lengths"].long() - count)[:, None] + i
    key = torch.arange(per * PAGE, device="cuda")
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    seen = seen[:, None, None]
    x = x.masked_fill_(~seen, float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    out = (x @ v) / x.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, most, hq * hd)
    return [out[i < count[:, None]].to(s["q"].dtype)]


# ------------------------------------------------------------------------------------------------- the framework's calls

def _own(s):
    import __graft_entry__ as graft
    pkg = graft.load_package()
    case, ops, stream = s["case"], pkg.ops, torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind == "gemv":
        ops.gemv_w4_grouped(s["w"].data_ptr(), s["x"].data_ptr(), s["y"].data_ptr(), case["n"], case["k"], case["group"], ncols=case["cols"], x_type=CODE[case["x"]], y_type=CODE[case["y"]],
                            scale_type=CODE[case["scale"]], has_offset=case["offset"], stream=stream)
        return [s["y"]]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if kind in ("rope", "append"):
        rows = dict(qkv_dev=s["qkv"].data_ptr(), type=CODE[case["type"]], qkv_stride=s["qkv"].stride(0), tokens=case["tokens"], hq=hq, hkv=hkv, hd=hd, rot=case["rot"],
                    q_gain_dev=s["gains"][0].data_ptr(), k_gain_dev=s["gains"][1].data_ptr(), eps=1e-6, cos_dev=s["cos"].data_ptr(), sin_dev=s["sin"].data_ptr(),
                    rope_rows=s["cos"].shape[0], pos_dev=s["pos"].data_ptr(), q_out_dev=s["q"].data_ptr(), q_stride=hq * hd, stream=stream)
    if kind == "rope":
        ops.qk_norm_rope(k_out_dev=s["k"].data_ptr(), k_stride=hkv * hd, **rows)
        return [s["q"], s["k"]]
    cache = pkg.Kv4Cache(s["pages"].data_ptr(), s["pages"].shape[0], s["table"].data_ptr(), s["table"].shape[1], s["table"].shape[0], hkv, hd, case["group"])
    if kind == "append":
        ops.qk_norm_rope_append_kv4(cache=cache, seq_dev=s["seq"].data_ptr(), **rows)
        ops.kv4_read(cache, s["seq"].data_ptr(), s["pos"].data_ptr(), case["tokens"], F32, s["k"].data_ptr(), s["v"].data_ptr(), stream=stream)
        return [s["q"], s["k"], s["v"]]
    ops.attention_kv4(cache, s["q"].data_ptr(), CODE[case["type"]], hq * hd, s["lengths"].data_ptr(), s["starts"].data_ptr() if case["queries"] > 1 else 0, s["tokens"], case["queries"],
                      case["high"], hq, s["out"].data_ptr(), hq * hd, s["room"].data_ptr(), s["room"].numel(), window=case["window"], stream=stream)
    return [s["out"]]


def run(state):
    if own:
        return _own(state)
    return {"gemv": _plain_gemv, "rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------- 64 bits

def _weight_codes(w, n, k):
    """Element (row, column) by the layout's formula, as an index into the image's bytes."""
    out = torch.empty(n, k, device="cuda", dtype=torch.int8)
    col = torch.arange(k, device="cuda")
    c = col % 64
    byte = (col % 128 // 64) * 512 + (c % 16 // 4) * 16 + (2 * (c // 32) + c % 32 // 16) * 4 + c % 4
    for first in range(0, n, 8192):
        row = torch.arange(first, min(n, first + 8192), device="cuda")
        b = w[(row // 16)[:, None], (col // 128)[None], byte[None] + (row % 8 * 64)[:, None]]
        x = torch.where((row % 16 >= 8)[:, None], b // 16, b % 16).to(torch.int8)
        out[row] = torch.where(x >= 8, x - 16, x)
    return out


def _exact_gemv(s):
    case = s["case"]
    n, k, group, w = case["n"], case["k"], case["group"], s["w"]
    col = torch.arange(k, device="cuda")
    per = 128 // group
    both = w[:, :, 1024:].contiguous().view(TYPE[case["scale"]])                       # [strip, block, numbers]
    x = s["x"].double()
    out = torch.empty(case["cols"], n, device="cuda", dtype=torch.float64)
    code = _weight_codes(w, n, k)
    for first in range(0, n, 8192):
        row = torch.arange(first, min(n, first + 8192), device="cuda")
        at = (row % 8 * per * 2 + row % 16 // 8)[:, None] + (col % 128 // group * 2)[None]
        m = code[row].double() * both[(row // 16)[:, None], (col // 128)[None], at].double()
        if case["offset"]:
            m += both[(row // 16)[:, None], (col // 128)[None], at + 16 * per].double()
        out[:, row] = x @ m.T
    return [out]


def _exact_rows(s, first, heads, gain):
    """Heads [first, first + heads) of the rows, normalised and rotated with complex numbers."""
    case = s["case"]
    hd, half = case["hd"], case["rot"] // 2
    x = s["qkv"][:, first * hd:(first + heads) * hd].to(torch.float64).reshape(-1, heads, hd)
    x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + 1e-6) * gain.to(torch.float64)
    turn = torch.complex(s["cos"][s["pos"].long()].double(), s["sin"][s["pos"].long()].double()).unsqueeze(1)
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1)


def _exact_held(x, group):
    """What 4 bits keep of x."""
    t, h, hd = x.shape
    g = x.reshape(t, h, hd // group, group)
    m = g.min(-1).values.half().double()
    s = ((g.max(-1).values - g.min(-1).values) / 15.0).half().double()
    c = torch.clamp(torch.round((g - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None]), 0, 15) * (s > 0)[..., None]
    return (m[..., None] + s[..., None] * c).reshape(t, h, hd)


def _key_value(block, hd, group, n):
    """K and V of the first n positions of pages [pages, bytes] of one kv head, element by element of the layout."""
    planes, dims = _planes(hd)
    d, p = torch.arange(hd, device="cuda"), torch.arange(n, device="cuda")
    plane, e = d // dims, d % dims
    codes = PAGE * hd // 2
    kb = plane * (PAGE * dims // 2) + e % 16 // 4 * (dims // 8) + e // 32 * 4 + e % 4
    khigh = e % 32 >= 16
    unit, vhigh = e % 8, e % 16 >= 8
    wide = dims // 16
    out, slot, page = [], (p % PAGE)[:, None], (p // PAGE)[:, None]
    for at, is_v in ((0, False), (codes + PAGE * 4 * (hd // group), True)):
        if is_v:
            turned = unit[None] ^ (4 * (slot >> 1 & 1)) if dims == 128 else unit[None].expand(n, -1)
            where, high = (plane * (PAGE * dims // 2) + e // 16)[None] + turned * wide, vhigh
        else:
            where, high = kb[None], khigh
        byte = block[page, at + where + slot * (dims // 2)]
        code = torch.where(high[None], byte // 16, byte % 16).double()
        pair = block[:, at + codes:at + codes + PAGE * 4 * (hd // group)].contiguous().view(torch.float16).double()
        number = slot * (hd // group) * 2 + (d // group * 2)[None]
        out.append(pair[page, number] * code + pair[page, number + 1])
    return out


def _exact_attention(s):
    case = s["case"]
    hq, hkv, hd, w = case["hq"], case["hkv"], case["hd"], case["window"]
    out = torch.zeros(s["tokens"], hq, hd, device="cuda", dtype=torch.float64)
    q = s["q"].double().reshape(-1, hq, hd)
    begin = 0
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        rows = slice(begin, begin + count)
        begin += count
        here = s["pages"][s["table"][b, :-(-n // PAGE)].long()]
        gap = torch.arange(n - count, n, device="cuda")[:, None] - torch.arange(n, device="cuda")[None]
        hidden = (gap < 0) | ((gap >= w) if w else (gap < 0))
        for h in range(hkv):
            k, v = _key_value(here[:, h], hd, case["group"], n)
            for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = (q[rows, j] @ k.T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[rows, j] = torch.softmax(x, dim=-1) @ v
    return [out.reshape(s["tokens"], hq * hd)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gemv":
        return _exact_gemv(s)
    if case["kind"] == "attention":
        return _exact_attention(s)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    q, k = _exact_rows(s, 0, hq, s["gains"][0]), _exact_rows(s, hq, hkv, s["gains"][1])
    if case["kind"] == "rope":
        return [q.flatten(1), k.flatten(1)]
    v = s["qkv"][:, (hq + hkv) * hd:(hq + 2 * hkv) * hd].double().reshape(-1, hkv, hd)
    return [q.flatten(1), _exact_held(k.float().double(), case["group"]), _exact_held(v, case["group"])]
