"""The products with packed block weights that are measured: one matrix times a few tokens (matvec), a whole
mixture-of-experts layer for a few tokens (moe), and the rows of an embedding table by their ids (get_rows).

Weights are packed GGUF blocks.  Sizes are those of this repository's tensor tables (4096 / 11008, 2048 / 5632 and
8192 / 28672 wide models with 32000 tokens) or generic.  The plain form decodes the packed weights with elementary
torch operations to 32 bits and multiplies; `exact` decodes element by element in 64 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
# GGmlType ids, and (elements, bytes) of a block
TYPE = {"f32": 0, "f16": 1, "q4_0": 2, "q4_1": 3, "q5_0": 6, "q5_1": 7, "q8_0": 8, "q2_k": 10, "q3_k": 11, "q4_k": 12, "q5_k": 13,
        "q6_k": 14, "iq4_nl": 20, "iq4_xs": 23, "bf16": 30}
BLOCK = {"q4_0": (32, 18), "q4_1": (32, 20), "q5_0": (32, 22), "q5_1": (32, 24), "q8_0": (32, 34), "q2_k": (256, 84), "q3_k": (256, 110),
         "q4_k": (256, 144), "q5_k": (256, 176), "q6_k": (256, 210), "iq4_nl": (32, 18), "iq4_xs": (256, 136)}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
IQ4 = (-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113)


def listed():
    return [
        # the key projection of a small model with shared heads, one token: the call is all latency
        {"name": "matvec q4_0 256x2048 t1", "op": "matvec", "type": "q4_0", "rows": 256, "cols": 2048, "tokens": 1, "x": "f32", "y": "f32", "pad": 0},
        # an attention projection in decoding
        {"name": "matvec q4_k 4096x4096 t1", "op": "matvec", "type": "q4_k", "rows": 4096, "cols": 4096, "tokens": 1, "x": "bf16", "y": "bf16", "pad": 0},
        # the output head over the whole vocabulary
        {"name": "matvec q6_k 32000x4096 t1", "op": "matvec", "type": "q6_k", "rows": 32000, "cols": 4096, "tokens": 1, "x": "f16", "y": "f32", "pad": 0},
        # the widest feed-forward product of a large model
        {"name": "matvec q4_k 28672x8192 t1", "op": "matvec", "type": "q4_k", "rows": 28672, "cols": 8192, "tokens": 1, "x": "f32", "y": "f32", "pad": 0},
        # odd sizes: a pruned model's projection, three sequences, activations inside a wider buffer
        {"name": "matvec iq4_nl 1537x1184 t3", "op": "matvec", "type": "iq4_nl", "rows": 1537, "cols": 1184, "tokens": 3, "x": "f16", "y": "f16", "pad": 40},
        # sixteen sequences decoded together
        {"name": "matvec q4_k 11008x4096 t16", "op": "matvec", "type": "q4_k", "rows": 11008, "cols": 4096, "tokens": 16, "x": "bf16", "y": "bf16", "pad": 0},
        # eight large experts, one token
        {"name": "moe 8x2 4096 11008 t1", "op": "moe", "experts": 8, "top_k": 2, "hidden": 4096, "ff": 11008, "tokens": 1, "x": "bf16",
         "up": "q4_k", "down": "q6_k", "gating": "softmax", "normalize": True},
        # many small experts, one token: latency
        {"name": "moe 64x8 2048 1024 t1", "op": "moe", "experts": 64, "top_k": 8, "hidden": 2048, "ff": 1024, "tokens": 1, "x": "f32",
         "up": "q4_0", "down": "q4_0", "gating": "softmax", "normalize": False},
        # many small experts, sixteen sequences: nearly every expert is in use, with one or two tokens
        {"name": "moe 128x8 2048 768 t16", "op": "moe", "experts": 128, "top_k": 8, "hidden": 2048, "ff": 768, "tokens": 16, "x": "bf16",
         "up": "q4_k", "down": "q5_k", "gating": "softmax", "normalize": True},
        # an odd number of experts, sigmoid gates
        {"name": "moe 9x3 1536 2560 t5", "op": "moe", "experts": 9, "top_k": 3, "hidden": 1536, "ff": 2560, "tokens": 5, "x": "f16",
         "up": "iq4_xs", "down": "q8_0", "gating": "sigmoid", "normalize": True},
        # one token's embedding
        {"name": "get_rows q4_k 32000x4096 n1", "op": "get_rows", "type": "q4_k", "rows": 32000, "cols": 4096, "n": 1, "y": "bf16"},
        # the embeddings of a prompt
        {"name": "get_rows q6_k 32000x8192 n2049", "op": "get_rows", "type": "q6_k", "rows": 32000, "cols": 8192, "n": 2049, "y": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "matvec", "moe", "moe", "get_rows"])
    kind = rng.choice(sorted(BLOCK))
    unit = BLOCK[kind][0]
    if op == "matvec":
        cols = unit * max(1, _log(rng, 256, 28672) // unit)
        rows = _log(rng, 32, max(33, min(32000, 120_000_000 // cols)))
        return {"op": op, "type": kind, "rows": rows, "cols": cols, "tokens": rng.choice([1, 1, 1, 2, 3, 4, 5, 8, 11, 16]),
                "x": rng.choice(["f32", "f16", "bf16"]), "y": rng.choice(["f32", "f16", "bf16"]), "pad": rng.choice([0, 0, 8, 13])}
    if op == "moe":
        down = rng.choice(sorted(BLOCK))
        experts = _log(rng, 4, 128)
        hidden = unit * max(1, _log(rng, 512, 4096) // unit)
        hidden = max(256, hidden // 256 * 256) if unit == 256 else hidden
        most = 200_000_000 // (experts * hidden)
        step = BLOCK[down][0]
        ff = step * max(1, _log(rng, 256, max(257, min(11008, most))) // step)
        return {"op": op, "experts": experts, "top_k": rng.randint(1, min(8, experts)), "hidden": hidden, "ff": ff, "tokens": rng.choice([1, 1, 2, 3, 4, 7, 16]),
                "x": rng.choice(["f32", "f16", "bf16"]), "up": kind, "down": down, "gating": rng.choice(["softmax", "sigmoid"]),
                "normalize": rng.random() < 0.5}
    cols = unit * max(1, _log(rng, 256, 8192) // unit)
    return {"op": op, "type": kind, "rows": _log(rng, 1000, 128000), "cols": cols, "n": _log(rng, 1, 4096), "y": rng.choice(["f32", "f16", "bf16"])}


# ---- inputs -------------------------------------------------------------------------------------

def _half(v):
    return v.to(torch.float16).view(torch.uint8).reshape(-1, 2)


def _packed(kind, blocks, gen):
    """Packed blocks whose decoded values spread like a model's weights (mean near 0, deviation near 0.02): uniform codes,
    scales that vary from block to block, and a minimum near the middle of the codes' range where the type has one."""
    n, size = BLOCK[kind]
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, ((blocks * size + 3) // 4,), dtype=torch.int32, device=DEVICE, generator=gen)
    raw = words.view(torch.uint8)[:blocks * size].view(blocks, size)
    vary = 0.6 + 0.8 * torch.rand(blocks, device=DEVICE, generator=gen)
    slack = 0.9 + 0.2 * torch.rand(blocks, device=DEVICE, generator=gen)
    # deviation of the codes (times the sub-block's whole-number scale where there is one)
    spread = {"q4_0": 4.6, "q4_1": 4.6, "q5_0": 9.2, "q5_1": 9.2, "q8_0": 74.0, "q2_k": 1.1 * 8.7, "q3_k": 2.3 * 18.5, "q4_k": 4.6 * 36.5,
              "q5_k": 9.2 * 36.5, "q6_k": 18.5 * 74.0, "iq4_nl": 69.0, "iq4_xs": 69.0 * 18.5}[kind]
    d = vary * (0.02 / spread)
    at = {"q2_k": 80, "q3_k": 108, "q6_k": 208}.get(kind, 0)
    raw[:, at:at + 2] = _half(d)
    if kind in ("q4_1", "q5_1"):
        raw[:, 2:4] = _half(-(7.5 if kind == "q4_1" else 15.5) * d * slack)
    if kind == "q2_k":
        raw[:, 82:84] = _half(1.5 * d * slack)
        raw[:, :16] = (raw[:, :16] & 15) * 17
    if kind in ("q4_k", "q5_k"):
        raw[:, 2:4] = _half((7.5 if kind == "q4_k" else 15.5) * d * slack)
        raw[:, 8:12] = raw[:, 4:8]
        raw[:, 12:16] = (raw[:, 12:16] & 15) * 17
    return raw.reshape(-1)


def _activations(tokens, cols, kind, gen, pad=0):
    """Normed activations: unit deviation, a few channels eight times as large, and a buffer that may be wider."""
    v = torch.randn(tokens, cols + pad, device=DEVICE, generator=gen)
    v[:, :: max(1, cols // 5)] *= 8.0
    return v.to(DTYPE[kind])[:, :cols]


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 7919 + 11)
    op = case["op"]
    if op == "moe":
        e, h, f = case["experts"], case["hidden"], case["ff"]
        up, down = BLOCK[case["up"]], BLOCK[case["down"]]
        return {"router": torch.randn(e, h, device=DEVICE, generator=gen) * (1.5 / math.sqrt(h)),
                "gate": _packed(case["up"], e * f * h // up[0], gen), "up": _packed(case["up"], e * f * h // up[0], gen),
                "down": _packed(case["down"], e * h * f // down[0], gen), "x": _activations(case["tokens"], h, case["x"], gen)}
    n, _ = BLOCK[case["type"]]
    w = _packed(case["type"], case["rows"] * case["cols"] // n, gen)
    if op == "matvec":
        return {"w": w, "x": _activations(case["tokens"], case["cols"], case["x"], gen, case["pad"])}
    return {"w": w, "ids": torch.randint(0, case["rows"], (case["n"],), device=DEVICE, generator=gen)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "moe":
        t, k = case["tokens"], case["top_k"]
        s["y"] = torch.empty(t, case["hidden"], dtype=DTYPE[case["x"]], device=DEVICE)
        s["ids"] = torch.empty(t, k, dtype=torch.int32, device=DEVICE)
        s["weights"] = torch.empty(t, k, dtype=torch.float32, device=DEVICE)
        s["kept"] = {}       # where a program keeps the layer that it makes of these weights once
    elif case["op"] == "matvec":
        s["y"] = torch.empty(case["tokens"], case["rows"], dtype=DTYPE[case["y"]], device=DEVICE)
    else:
        s["y"] = torch.empty(case["n"], case["cols"], dtype=DTYPE[case["y"]], device=DEVICE)
    return s


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if case["op"] == "matvec":
        if own:
            import gguf_amd
            gguf_amd.matvec(TYPE[case["type"]], s["y"], s["w"], s["x"])
            return s["y"]
        return (s["x"].float() @ _decode(case["type"], s["w"]).view(case["rows"], case["cols"]).t()).to(DTYPE[case["y"]])
    if case["op"] == "get_rows":
        if own:
            import gguf_amd
            gguf_amd.get_rows(TYPE[case["type"]], s["y"], s["w"], s["ids"])
            return s["y"]
        taken = s["w"].view(case["rows"], -1).index_select(0, s["ids"])
        return _decode(case["type"], taken.reshape(-1)).view(case["n"], case["cols"]).to(DTYPE[case["y"]])
    if own:
        import gguf_amd
        layer = s["kept"].get("layer")
        if layer is None:
            layer = s["kept"]["layer"] = gguf_amd.MoeLayer(
                s["router"], (TYPE[case["up"]], s["gate"]), (TYPE[case["up"]], s["up"]), (TYPE[case["down"]], s["down"]),
                hidden=case["hidden"], ff=case["ff"], top_k=case["top_k"], gating=case["gating"], normalize=case["normalize"])
        layer.run(s["y"], s["x"], ids=s["ids"], weights=s["weights"])
        return {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}
    return _moe(case, s)


def _moe(case, s):
    t, k, h, f = case["tokens"], case["top_k"], case["hidden"], case["ff"]
    x = s["x"].float()
    logits = (s["x"].double() @ s["router"].double().t()).float()           # sums in 64 bits: a choice hangs on them
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]   # equal logits: the lowest index first
    if case["gating"] == "softmax":
        p = torch.exp(logits - logits.max(dim=1, keepdim=True)[0])
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    w = torch.gather(p, 1, ids)
    if case["normalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    used, place = torch.unique(ids, return_inverse=True)
    gate, up = (_decode(case["up"], s[n].view(case["experts"], -1).index_select(0, used).reshape(-1)).view(-1, f, h) for n in ("gate", "up"))
    down = _decode(case["down"], s["down"].view(case["experts"], -1).index_select(0, used).reshape(-1)).view(-1, h, f)
    g = torch.matmul(x, gate.transpose(1, 2))                                # [experts in use, tokens, ff]
    a = g / (1.0 + torch.exp(-g)) * torch.matmul(x, up.transpose(1, 2))
    o = torch.matmul(a, down.transpose(1, 2))
    share = torch.zeros(t, used.numel(), device=x.device).scatter_(1, place.view(t, k), w)
    y = (share.t().unsqueeze(2) * o).sum(dim=0)
    return {"y": y.to(DTYPE[case["x"]]), "ids": ids.to(torch.int32), "weights": w}


def _fields(b, at, count=1):
    return b[:, at:at + 2 * count].contiguous().view(torch.float16).float()


def _nibbles(q):
    return torch.stack((q & 15, q >> 4), dim=1)


def _sub_scales(s):
    """The eight 6-bit scales and the eight 6-bit minima that q4_k and q5_k pack into twelve bytes."""
    a, b, c = s[:, 0:4], s[:, 4:8], s[:, 8:12]
    return (torch.cat((a & 63, (c & 15) | ((a >> 6) << 4)), dim=1).float(), torch.cat((b & 63, (c >> 4) | ((b >> 6) << 4)), dim=1).float())


def _signed(b):
    return b.contiguous().view(torch.int8).float()


def _decode(kind, packed):
    """Packed blocks to 32-bit values, block after block."""
    n, size = BLOCK[kind]
    b = packed.view(-1, size)
    m = b.shape[0]
    if kind == "q4_0":
        return (_nibbles(b[:, 2:18]).reshape(m, n).float() - 8.0) * _fields(b, 0)
    if kind == "q4_1":
        return _nibbles(b[:, 4:20]).reshape(m, n).float() * _fields(b, 0) + _fields(b, 2)
    if kind in ("q5_0", "q5_1"):
        at = 2 if kind == "q5_0" else 4
        bits = torch.arange(8, device=b.device, dtype=torch.uint8)
        high = ((b[:, at:at + 4].unsqueeze(2) >> bits) & 1).reshape(m, n)
        q = (_nibbles(b[:, at + 4:at + 20]).reshape(m, n) | (high << 4)).float()
        return (q - 16.0) * _fields(b, 0) if kind == "q5_0" else q * _fields(b, 0) + _fields(b, 2)
    if kind == "q8_0":
        return _signed(b[:, 2:34]) * _fields(b, 0)
    if kind == "iq4_nl":
        table = torch.tensor(IQ4, dtype=torch.float32, device=b.device)
        return table[_nibbles(b[:, 2:18]).reshape(m, n).int()] * _fields(b, 0)
    two = torch.arange(0, 8, 2, device=b.device, dtype=torch.uint8).view(1, 1, 4, 1)
    if kind == "q2_k":
        q = ((b[:, 16:80].reshape(m, 2, 1, 32) >> two) & 3).reshape(m, 16, 16).float()
        s = b[:, :16]
        return (q * (_fields(b, 80) * (s & 15).float()).unsqueeze(2) - (_fields(b, 82) * (s >> 4).float()).unsqueeze(2)).reshape(m, n)
    if kind == "q3_k":
        q = (b[:, 32:96].reshape(m, 2, 1, 32) >> two) & 3
        bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(1, 2, 4, 1)
        q = (q | (((b[:, :32].reshape(m, 1, 1, 32) >> bit) & 1) << 2)).reshape(m, 16, 16).float() - 4.0
        low = torch.cat((b[:, 96:104] & 15, b[:, 96:104] >> 4), dim=1)
        high = ((b[:, 104:108].reshape(m, 1, 4) >> two.view(1, 4, 1)) & 3).reshape(m, 16)
        return (q * (_fields(b, 108) * ((low | (high << 4)).float() - 32.0)).unsqueeze(2)).reshape(m, n)
    if kind in ("q4_k", "q5_k"):
        sc, mn = _sub_scales(b[:, 4:16])
        q = _nibbles(b[:, size - 128:].reshape(m * 4, 32)).reshape(m, 8, 32)
        if kind == "q5_k":
            bit = torch.arange(8, device=b.device, dtype=torch.uint8).view(1, 8, 1)
            q = q | (((b[:, 16:48].reshape(m, 1, 32) >> bit) & 1) << 4)
        return (q.float() * (_fields(b, 0) * sc).unsqueeze(2) - (_fields(b, 2) * mn).unsqueeze(2)).reshape(m, n)
    if kind == "q6_k":
        low = _nibbles(b[:, :128].reshape(m * 2, 64)).reshape(m, 2, 4, 32)      # per half: the low nibbles of 64, then the high ones
        q = (low | (((b[:, 128:192].reshape(m, 2, 1, 32) >> two) & 3) << 4)).reshape(m, 16, 16).float() - 32.0
        return (q * (_fields(b, 208) * _signed(b[:, 192:208])).unsqueeze(2)).reshape(m, n)
    table = torch.tensor(IQ4, dtype=torch.float32, device=b.device)             # iq4_xs
    low = torch.stack((b[:, 4:8] & 15, b[:, 4:8] >> 4), dim=2).reshape(m, 8)
    high = ((b[:, 2:4].unsqueeze(2) >> two.view(1, 1, 4)) & 3).reshape(m, 8)
    s = _fields(b, 0) * ((low | (high << 4)).float() - 32.0)
    q = table[_nibbles(b[:, 8:136].reshape(m * 8, 16)).reshape(m, 8, 32).int()]
    return (q * s.unsqueeze(2)).reshape(m, n)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "moe":
        e, k, h, f, t = (case[n] for n in ("experts", "top_k", "hidden", "ff", "tokens"))
        used = max(k, round(e * (1.0 - (1.0 - k / e) ** t)))      # experts that t tokens choose, on the average
        per = sum(f * h * size / n for n, size in (BLOCK[case["up"]], BLOCK[case["up"]], BLOCK[case["down"]]))
        return {"bytes": used * per + 4 * e * h + 2 * t * h * SIZE[case["x"]] + 8 * t * k, "flops": 6 * t * k * f * h + 2 * t * e * h}
    n, size = BLOCK[case["type"]]
    if op == "matvec":
        r, c, t = case["rows"], case["cols"], case["tokens"]
        return {"bytes": r * c * size / n + t * c * SIZE[case["x"]] + t * r * SIZE[case["y"]], "flops": 2 * r * c * t}
    return {"bytes": case["n"] * (case["cols"] * (size / n + SIZE[case["y"]]) + 8), "flops": 2 * case["n"] * case["cols"]}


# ---- the definition, element by element in 64 bits ------------------------------------------------

def _element_map(kind, dev):
    """For each element e of a block: where its code, its high bits, its scale and its minimum lie."""
    n, size = BLOCK[kind]
    e = torch.arange(n, device=dev)
    if n == 32:
        return e, e % 16, 4 * (e // 16)
    return e, e, e


def _value(kind, blk):
    """Values in 64 bits of blocks blk[m, bytes] (whole numbers of 64 bits), from each element's own index."""
    n, size = BLOCK[kind]
    e, i, shift = _element_map(kind, blk.device)

    def half(at):
        bits = blk[:, at] | (blk[:, at + 1] << 8)
        sign, ex, man = 1.0 - 2.0 * (bits >> 15).double(), (bits >> 10) & 31, (bits & 1023).double()
        normal = torch.ldexp(1.0 + man / 1024.0, ex - 15)
        return (sign * torch.where(ex == 0, man * 2.0 ** -24, normal)).unsqueeze(1)

    def signed(v):
        return torch.where(v > 127, v - 256, v)

    kv = torch.tensor(IQ4, dtype=torch.float64, device=blk.device)
    if kind == "q4_0":
        return half(0) * (((blk[:, 2 + i] >> shift) & 15) - 8).double()
    if kind == "q4_1":
        return half(0) * ((blk[:, 4 + i] >> shift) & 15).double() + half(2)
    if kind == "q5_0":
        return half(0) * ((((blk[:, 6 + i] >> shift) & 15) + 16 * ((blk[:, 2 + e // 8] >> (e % 8)) & 1)) - 16).double()
    if kind == "q5_1":
        return half(0) * (((blk[:, 8 + i] >> shift) & 15) + 16 * ((blk[:, 4 + e // 8] >> (e % 8)) & 1)).double() + half(2)
    if kind == "q8_0":
        return half(0) * signed(blk[:, 2 + e]).double()
    if kind == "iq4_nl":
        return half(0) * kv[(blk[:, 2 + i] >> shift) & 15]
    part, lane, plane = e // 128, e % 32, (e // 32) % 4
    if kind == "q2_k":
        q = (blk[:, 16 + 32 * part + lane] >> (2 * plane)) & 3
        s = blk[:, e // 16]
        return half(80) * (s & 15).double() * q.double() - half(82) * (s >> 4).double()
    if kind == "q3_k":
        q = ((blk[:, 32 + 32 * part + lane] >> (2 * plane)) & 3) - 4 + 4 * ((blk[:, lane] >> (4 * part + plane)) & 1)
        g = e // 16
        s = ((blk[:, 96 + g % 8] >> (4 * (g // 8))) & 15) + 16 * ((blk[:, 104 + g % 4] >> (2 * (g // 4))) & 3) - 32
        return half(108) * s.double() * q.double()
    if kind in ("q4_k", "q5_k"):
        g = e // 32
        j = g % 4
        early = (g < 4).unsqueeze(0)
        x, y, z = blk[:, 4 + j], blk[:, 8 + j], blk[:, 12 + j]
        s = torch.where(early, x % 64, z % 16 + 16 * (x // 64))
        mn = torch.where(early, y % 64, z // 16 + 16 * (y // 64))
        q = (blk[:, size - 128 + 32 * (e // 64) + lane] >> (4 * (g % 2))) & 15
        if kind == "q5_k":
            q = q + 16 * ((blk[:, 16 + lane] >> g) & 1)
        return half(0) * s.double() * q.double() - half(2) * mn.double()
    if kind == "q6_k":
        q = ((blk[:, 64 * part + 32 * (plane % 2) + lane] >> (4 * (plane // 2))) & 15) + 16 * ((blk[:, 128 + 32 * part + lane] >> (2 * plane)) & 3) - 32
        return half(208) * signed(blk[:, 192 + e // 16]).double() * q.double()
    g = e // 32                                                               # iq4_xs
    s = ((blk[:, 4 + g // 2] >> (4 * (g % 2))) & 15) + 16 * ((blk[:, 2 + g // 4] >> (2 * (g % 4))) & 3) - 32
    return half(0) * s.double() * kv[(blk[:, 8 + 16 * g + e % 16] >> (4 * ((e // 16) % 2))) & 15]


def _product64(kind, packed, rows, cols, x):
    """x[t, cols] in 64 bits times the transposed packed matrix, a strip of rows at a time."""
    n, size = BLOCK[kind]
    strip = max(1, 2 ** 24 // cols)
    return torch.cat([x @ _value(kind, packed[at * (cols // n) * size:min(rows, at + strip) * (cols // n) * size].view(-1, size).long()).view(-1, cols).t()
                      for at in range(0, rows, strip)], dim=1)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "matvec":
        return _product64(case["type"], s["w"], case["rows"], case["cols"], s["x"].double())
    if case["op"] == "get_rows":
        return _value(case["type"], s["w"].view(case["rows"], -1)[s["ids"]].view(-1, BLOCK[case["type"]][1]).long()).view(case["n"], case["cols"])
    h, f, k = case["hidden"], case["ff"], case["top_k"]
    x = s["x"].double()
    y, every, gates = torch.zeros_like(x), [], []
    for t in range(case["tokens"]):
        logit = (s["router"].double() * x[t]).sum(dim=1)
        order = sorted(range(case["experts"]), key=lambda e: (-float(logit[e].float()), e))[:k]
        p = torch.softmax(logit, 0) if case["gating"] == "softmax" else torch.sigmoid(logit)
        w = p[order] / p[order].sum() if case["normalize"] else p[order]
        every.append(order)
        gates.append(w)
        for j, e in enumerate(order):
            one = {name: s[name].view(case["experts"], -1)[e] for name in ("gate", "up", "down")}
            g = _product64(case["up"], one["gate"], f, h, x[t:t + 1])
            a = g * torch.sigmoid(g) * _product64(case["up"], one["up"], f, h, x[t:t + 1])
            y[t] += w[j] * _product64(case["down"], one["down"], h, f, a)[0]
    return {"y": y, "ids": torch.tensor(every, dtype=torch.int32), "weights": torch.stack(gates)}
