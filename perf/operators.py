"""The cases by which the descriptor lookup, the gated recurrence and the microscaled 4-bit operators are measured.

The plain forms are elementary torch operations in 32 bits, rounded once at the end; `exact` evaluates the definitions in
64 bits, written apart from them."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 32  # elements that share a scale in the 4-bit format


def listed():
    return [
        # a probe of 64 rays at the scene's 4-bit descriptor table: 16 hits each, latency counts
        dict(name="lookup 4-bit 1k hits", op="lookup", rows=1_000_000, width=96, n=1024, table="micro4", out="f16",
             index="i32", weight=True, hot=0.0, empty=0.1, train=False),
        # one training batch of 160k rays with a decoder outside the renderer: their 16 nearest hits each, both directions
        dict(name="lookup train 2.6M hits f16", op="lookup", rows=1_000_000, width=96, n=2_560_000, table="f16", out="f16",
             index="i32", weight=True, hot=0.0, empty=0.1, train=True),
        # rows of odd width and a skewed index: a few rows take a third of all entries (backdrop primitives, padding)
        dict(name="lookup train skewed bf16", op="lookup", rows=50_021, width=1023, n=16_383, table="bf16", out="bf16",
             index="i64", weight=False, hot=0.3, empty=0.02, train=True),
        # one new hit for each of 64 rays that keep their state: the smallest call
        dict(name="recurrence step 64x1024", op="step", seqs=64, width=1024, groups=1024, x="bf16", gate="bf16"),
        # descriptor rows of 16 hits composited along 160k rays, back to front, slot-major as the hit lists are
        dict(name="recurrence composite train", op="recurrence", layout="time", seqs=160_000, steps=16, width=96, groups=1,
             x="f16", gate="f32", reverse=True, state=False, states=False, train=True),
        # colour and depth of 42 hits along the rays of an 800 x 800 view, ray-major, inference
        dict(name="recurrence colour 640k rays", op="recurrence", layout="batch", seqs=640_000, steps=42, width=4, groups=1,
             x="f32", gate="f32", reverse=True, state=True, states=False, train=False),
        # one long sequence with a gate for each channel, training
        dict(name="recurrence long bf16 train", op="recurrence", layout="batch", seqs=1, steps=65_536, width=256, groups=256,
             x="bf16", gate="bf16", reverse=False, state=True, states=True, train=True),
        # sequences of uneven length packed behind one another, gates shared by 16 channels
        dict(name="recurrence packed bf16", op="recurrence", layout="packed", seqs=613, steps=100_003, width=512, groups=32,
             x="bf16", gate="bf16", reverse=False, state=True, states=True, train=False),
        # the descriptor table of a 3M-primitive scene taken to 4 bits and read back
        dict(name="quantize 3M x 96 f16", op="quantize", rows=3_000_000, width=96, x="f16"),
        # a 64-wide layer over the 4-bit descriptors of 1M primitives
        dict(name="product 1M x 64 x 96", op="product", m=1_000_000, n=64, k=96, x="micro4", out="f16"),
        # a large layer whose input is quantised on the way
        dict(name="product 4096 cubed", op="product", m=4096, n=4096, k=4096, x="bf16", out="bf16"),
        # the same layer for four rows
        dict(name="product 4 x 4096 x 4096", op="product", m=4, n=4096, k=4096, x="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup", "step", "recurrence", "recurrence", "recurrence", "quantize", "product", "product"])
    if op == "lookup":
        train = rng.random() < 0.5
        width = _log(rng, 1, 2048)
        table = rng.choice(["f16", "bf16", "f32"] + ([] if train else ["micro4"]))
        return dict(op=op, rows=_log(rng, 1, min(2_000_000, 100_000_000 // width)), width=width,
                    n=_log(rng, 1, min(3_000_000, 100_000_000 // width)), table=table,
                    out=rng.choice(["f16", "bf16", "f32"]) if table == "micro4" else rng.choice([table, "f32"]),
                    index=rng.choice(["i32", "i64"]), weight=rng.random() < 0.6, hot=rng.choice([0.0, 0.0, 0.3, 0.9]),
                    empty=rng.choice([0.0, 0.1, 0.5]), train=train)
    if op == "step":
        width = _log(rng, 8, 4096)
        share = rng.choice([q for q in (1, 2, 4, 8, 16, width) if width % q == 0])
        x = rng.choice(["f16", "bf16", "f32"])
        return dict(op=op, seqs=_log(rng, 1, 512), width=width, groups=width // share, x=x, gate=rng.choice([x, "f32"]))
    if op == "recurrence":
        layout = rng.choice(["batch", "time", "packed"])
        width = _log(rng, 1, 2048)
        share = rng.choice([q for q in (1, 1, 2, 3, 4, 16, 64, width, width) if width % q == 0])
        steps = _log(rng, 1, min(100_000, 60_000_000 // width))
        seqs = _log(rng, 1, 2000) if layout == "packed" else _log(rng, 1, min(200_000, 60_000_000 // (width * steps)) or 1)
        x = rng.choice(["f16", "bf16", "f32"])
        train = rng.random() < 0.5
        return dict(op=op, layout=layout, seqs=seqs, steps=steps, width=width, groups=width // share, x=x,
                    gate=rng.choice([x, "f32"]), reverse=rng.random() < 0.5, state=rng.random() < 0.5,
                    states=rng.random() < 0.7, train=train)
    if op == "quantize":
        width = _log(rng, 1, 8192)
        return dict(op=op, rows=_log(rng, 1, 200_000_000 // width), width=width, x=rng.choice(["f16", "bf16", "f32"]))
    m, n, k = _log(rng, 1, 8192), _log(rng, 1, 8192), _log(rng, 1, 8192)
    return dict(op=op, m=m, n=n, k=k, x=rng.choice(["micro4", "f16", "bf16", "f32"]), out=rng.choice(["f16", "bf16"]))


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _two(e):
    """2^e in 32 bits, exactly, for whole e from -127 to 127."""
    powers = torch.cat([torch.full((1,), 2.0 ** -127), (torch.arange(1, 255, dtype=torch.int32) << 23).view(torch.float32)])
    return powers.to(e.device)[e.long() + 127]


def _normal(g, *shape, scale=1.0, type=torch.float32):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(type)


def _gates(g, *shape):
    """Gates as a decay or a transmittance has them: most near 1, some near 0."""
    return torch.sigmoid(torch.randn(*shape, device="cuda", generator=g) * 1.5 + 2.0)


def _pack(x):
    """4-bit codes (rows, 16 per block) and scale bytes (rows, padded to a multiple of 4) of a matrix, by the format's definition."""
    codes, exponents = _to_codes(x.float())
    rows, blocks = exponents.shape
    codes = codes.reshape(rows, blocks * BLOCK)
    scales = torch.zeros(rows, -(-blocks // 4) * 4, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = (exponents + 127).to(torch.uint8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, op = case, case["op"]
    s = dict(case)
    if op == "lookup":
        table = _normal(g, c["rows"], c["width"], scale=0.1)
        if c["table"] == "micro4":
            s["codes"], s["scales"] = _pack(table)
        else:
            s["rows_of"] = table.to(TYPES[c["table"]])
        del table
        idx = torch.randint(0, c["rows"], (c["n"],), device="cuda", generator=g)
        u = torch.rand(c["n"], device="cuda", generator=g)
        idx = torch.where(u < c["hot"], idx % 3, idx)  # a few rows that many entries name
        idx = torch.where(torch.rand(c["n"], device="cuda", generator=g) < c["empty"], -1, idx)
        s["idx"] = idx.to(torch.int32 if c["index"] == "i32" else torch.int64)
        s["weight"] = torch.rand(c["n"], device="cuda", generator=g) if c["weight"] else None
        if c["train"]:
            s["dout"] = _normal(g, c["n"], c["width"], type=TYPES[c["out"]])
    elif op == "step":
        s["x"] = _normal(g, c["seqs"], c["width"], type=TYPES[c["x"]])
        s["gate"] = _gates(g, c["seqs"], c["groups"]).to(TYPES[c["gate"]])
        s["state"] = _normal(g, c["seqs"], c["width"])
        s["new"] = torch.empty_like(s["state"])
    elif op == "recurrence":
        B, T, D, G = c["seqs"], c["steps"], c["width"], c["groups"]
        lead = {"batch": (B, T), "time": (T, B), "packed": (T,)}[c["layout"]]
        tensors = {"x": _normal(g, *lead, D, type=TYPES[c["x"]]), "gate": _gates(g, *lead, G).to(TYPES[c["gate"]])}
        if c["train"] and c["states"]:
            tensors["dh"] = _normal(g, *lead, D, type=TYPES[c["x"]])
        for name, t in tensors.items():
            s[name] = t.transpose(0, 1) if c["layout"] == "time" else t
        if c["layout"] == "packed":
            cuts = torch.randint(0, T + 1, (B,), device="cuda", generator=g).sort().values  # rows behind the last cut belong to none
            s["offsets"] = torch.cat([cuts.new_zeros(1), cuts]).to(torch.int32)
        else:
            s["offsets"] = None
        s["state"] = _normal(g, B, D) if c["state"] else None
        if c["train"]:
            s["dlast"] = _normal(g, B, D)
    elif op == "quantize":
        s["x"] = _normal(g, c["rows"], c["width"], scale=0.1, type=TYPES[c["x"]])
    else:
        bound = math.sqrt(6.0 / (c["n"] + c["k"]))
        w = (torch.rand(c["n"], c["k"], device="cuda", generator=g) * 2 - 1) * bound
        s["w_codes"], s["w_scales"] = _pack(w)
        x = _normal(g, c["m"], c["k"])
        if c["x"] == "micro4":
            s["codes"], s["scales"] = _pack(x)
        else:
            s["x_of"] = x.to(TYPES[c["x"]])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(state):
    return {"lookup": _lookup, "step": _step, "recurrence": _recurrence, "quantize": _quantize, "product": _product}[state["op"]](state)


def _lookup(s):
    if own:
        from flare_b200 import embedding, microscale
        table = microscale.Micro4(s["codes"], s["scales"], s["width"]) if s["table"] == "micro4" else s["rows_of"]
        out = embedding.lookup(table, s["idx"], s["weight"], 0.5, dtype=TYPES[s["out"]])
        if not s["train"]:
            return out
        dtable, dweight = embedding.lookup_backward(s["dout"], table, s["idx"], s["weight"], 0.5)
        return {"out": out, "dtable": dtable} | ({"dweight": dweight} if s["weight"] is not None else {})
    idx = s["idx"].long()
    named = idx >= 0
    at = idx.clamp(min=0)
    if s["table"] == "micro4":
        picked = _values(s["codes"][at], s["scales"][at], s["width"])
    else:
        picked = s["rows_of"][at].float()
    factor = torch.where(named, 0.5 if s["weight"] is None else 0.5 * s["weight"], 0.0)[:, None]
    out = (picked * factor).to(TYPES[s["out"]])
    if not s["train"]:
        return out
    dout = s["dout"].float()
    dtable = torch.zeros(s["rows"], s["width"], device=out.device).index_add_(0, at, dout * factor)
    if s["weight"] is None:
        return {"out": out, "dtable": dtable}
    return {"out": out, "dtable": dtable, "dweight": torch.where(named, 0.5 * (dout * picked).sum(1), 0.0)}


def _step(s):
    if own:
        from flare_b200 import recurrence
        return {"h": recurrence.step(s["gate"], s["x"], s["state"], out=s["new"]), "state": s["new"]}
    B, D, G = s["seqs"], s["width"], s["groups"]
    new = (s["gate"].float()[:, :, None] * s["state"].view(B, G, D // G)).view(B, D) + s["x"].float()
    return {"h": new.to(s["x"].dtype), "state": new}


def _doubling(a, x):
    """h_t = a_t h_{t-1} + x_t along the first axis, h before the first step 0: spans of steps are joined pair by pair."""
    span = 1
    while span < x.shape[0]:
        x = torch.cat([x[:span], x[span:] + a[span:] * x[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return x


def _recurrence(s):
    if own:
        from flare_b200 import recurrence
        h, last, saved = recurrence.scan(s["gate"], s["x"], s["state"], offsets=s["offsets"], reverse=s["reverse"],
                                         states=s["states"], training=s["train"])
        out = {"last": last} | ({"h": h} if s["states"] else {})
        if s["train"]:
            dgate, dx, dstate = recurrence.scan_backward(s["gate"], s["x"], saved, s.get("dh"), s["dlast"], s["state"],
                                                         offsets=s["offsets"], reverse=s["reverse"])
            out |= {"dgate": dgate, "dx": dx} | ({"dstate": dstate} if s["state"] is not None else {})
        return out
    B, D, G = s["seqs"], s["width"], s["groups"]
    packed = s["offsets"] is not None
    # time first, channels split by the gate that they share: (T, B or none, G, D / G)
    order = (lambda t: t) if packed else (lambda t: t.transpose(0, 1))
    split = lambda t: t.float().reshape(*t.shape[:-1], G, D // G)  # noqa: E731
    a, x = order(s["gate"]).float()[..., None], split(order(s["x"]))
    state = torch.zeros(B, D, device=x.device) if s["state"] is None else s["state"]
    state = split(state)
    T = x.shape[0]
    if packed:
        off = s["offsets"].long()
        some = off[1:] > off[:-1]
        owner = torch.searchsorted(off, torch.arange(T, device=x.device), right=True) - 1  # B for rows that belong to none
        inside = (owner < B).view(T, 1, 1)
        first = off[:-1] if not s["reverse"] else off[1:] - 1
        final = off[1:] - 1 if not s["reverse"] else off[:-1]
        starts = torch.zeros(T + 1, dtype=torch.bool, device=x.device)
        starts[torch.where(some, first, T)] = True  # an empty sequence marks the row past the end
        starts = starts[:T].view(T, 1, 1)
        before = torch.where(starts & inside, torch.cat([state, state[:1]])[owner], 0.0)  # what enters a first step
        x = torch.where(inside, x, 0.0)
        link = torch.where(starts, 0.0, a)
    else:
        first, final = (0, T - 1) if not s["reverse"] else (T - 1, 0)
        before = torch.zeros_like(x)
        before[first] = state
        link = a
    forth = (lambda t: t.flip(0)) if s["reverse"] else (lambda t: t)
    h = forth(_doubling(forth(link), forth(x + a * before)))
    if packed:
        h = torch.where(inside, h, 0.0)
        last = torch.where(some.view(B, 1, 1), h[torch.where(some, final, 0)], state)
    else:
        last = h[final]
    flat = lambda t: t.reshape(*t.shape[:-2], D)  # noqa: E731
    back = lambda t, like: order(t).to(like.dtype)  # noqa: E731
    out = {"last": flat(last)} | ({"h": back(flat(h), s["x"])} if s["states"] else {})
    if not s["train"]:
        return out
    dh = split(order(s["dh"])) if s["states"] else torch.zeros_like(x)
    dlast = split(s["dlast"])
    if packed:
        dh = torch.where(inside, dh, 0.0).index_add(0, torch.where(some, final, 0), torch.where(some.view(B, 1, 1), dlast, 0.0))
    else:
        dh = dh.clone()
        dh[final] += dlast
    # the gate that carries the gradient of step t is the one of the step after it
    after = forth(torch.cat([forth(link)[1:], torch.zeros_like(link[:1])]))
    lam = forth(_doubling(forth(after).flip(0), forth(dh).flip(0)).flip(0))
    held = forth(torch.cat([torch.zeros_like(h[:1]), forth(h)[:-1]]))
    if packed:
        held = torch.where(starts, before, torch.where(inside, held, 0.0))
        dstate = torch.where(some.view(B, 1, 1), (a * lam)[torch.where(some, first, 0)], dlast)
        lam = torch.where(inside, lam, 0.0)
    else:
        held[first] = state
        dstate = (a * lam)[first]
    out |= {"dgate": back((lam * held).sum(-1), s["gate"]), "dx": back(flat(lam), s["x"])}
    return out | ({"dstate": flat(dstate)} if s["state"] is not None else {})


def _to_codes(x):
    """Codes (rows, blocks, 32) and exponents (rows, blocks) of the 4-bit format: 2^e with e = floor(log2 of the block's largest) - 2,
    elements to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    most = x.abs().amax(2)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(-127, 127)
    v = x.abs() * _two(-e)[:, :, None]
    code = ((v > 0.25).byte() + (v >= 0.75).byte() + (v > 1.25).byte() + (v >= 1.75).byte() + (v > 2.5).byte() + (v >= 3.5).byte()
            + (v > 5).byte())
    return code | (torch.signbit(x).byte() << 3), e


def _values(codes, scales, k):
    """What codes and scales stand for, in 32 bits: (rows, k)."""
    rows, blocks = codes.shape[0], codes.shape[1] // 16
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    nibbles = torch.stack([codes & 15, codes >> 4], 2).reshape(rows, blocks, BLOCK)
    return (level[nibbles.int()] * _two(scales[:, :blocks].int() - 127)[:, :, None]).reshape(rows, -1)[:, :k]


def _quantize(s):
    if own:
        from flare_b200 import microscale
        return microscale.quantize(s["x"]).dequantize(s["x"].dtype)
    codes, e = _to_codes(s["x"].float())
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    v = level[(codes & 7).int()]
    v = torch.where(codes > 7, -v, v) * _two(e)[:, :, None]
    return v.reshape(v.shape[0], -1)[:, :s["width"]].to(s["x"].dtype)


def _product(s):
    if own:
        from flare_b200 import microscale
        w = microscale.Micro4(s["w_codes"], s["w_scales"], s["k"])
        x = microscale.Micro4(s["codes"], s["scales"], s["k"]) if s["x"] == "micro4" else s["x_of"]
        return microscale.product(x, w, dtype=TYPES[s["out"]])
    w = _values(s["w_codes"], s["w_scales"], s["k"])
    x = _values(s["codes"], s["scales"], s["k"]) if s["x"] == "micro4" else _values(*_pack(s["x_of"]), s["k"])
    return (x @ w.T).to(TYPES[s["out"]])


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def _micro_bytes(rows, k):
    return rows * -(-k // BLOCK) * 17


def work(case):
    c, op = case, case["op"]
    size = lambda t: 4 if t == "f32" else 2  # noqa: E731
    if op == "lookup":
        n, rows, width = c["n"], c["rows"], c["width"]
        spread = n * (1 - c["empty"]) * (1 - c["hot"])
        distinct = min(rows, rows * -math.expm1(-spread / rows) + (min(3, rows) if c["hot"] else 0))
        row = _micro_bytes(1, width) if c["table"] == "micro4" else width * size(c["table"])
        b = distinct * row + n * ((4 if c["index"] == "i32" else 8) + (4 if c["weight"] else 0) + width * size(c["out"]))
        f = n * width
        if c["train"]:
            b += n * width * size(c["out"]) + rows * width * 4 + (n * 4 if c["weight"] else 0)
            f += n * width * (4 if c["weight"] else 2)
        return {"bytes": int(b), "flops": int(f)}
    if op == "step":
        e = c["seqs"] * c["width"]
        return {"bytes": e * (8 + 2 * size(c["x"])) + c["seqs"] * c["groups"] * size(c["gate"]), "flops": 2 * e}
    if op == "recurrence":
        e = c["steps"] * (1 if c["layout"] == "packed" else c["seqs"])
        x, gate, ends = e * c["width"] * size(c["x"]), e * c["groups"] * size(c["gate"]), c["seqs"] * c["width"] * 4
        b = x + gate + (x if c["states"] else 0) + ends * (2 if c["state"] else 1)
        f = 2 * e * c["width"]
        if c["train"]:
            b += (x if c["states"] else 0) + x + gate + ends * (2 if c["state"] else 1)
            f += 4 * e * c["width"]
        return {"bytes": b, "flops": f}
    if op == "quantize":
        e = c["rows"] * c["width"]
        return {"bytes": 2 * e * size(c["x"]), "flops": 4 * e}
    m, n, k = c["m"], c["n"], c["k"]
    x = _micro_bytes(m, k) if c["x"] == "micro4" else m * k * size(c["x"])
    return {"bytes": x + _micro_bytes(n, k) + m * n * 2, "flops": 2 * m * n * k}


# ---- in 64 bits -------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"lookup": _exact_lookup, "step": _exact_step, "recurrence": _exact_recurrence, "quantize": _exact_quantize,
            "product": _exact_product}[case["op"]](s)


def _exact_two(e):
    """2^e in 64 bits, from its bits."""
    return ((e + 1023) << 52).view(torch.float64)


def _exact_values(codes, scales, k):
    lo, hi = (codes & 15).long(), (codes >> 4).long()
    n = torch.stack([lo, hi], -1).flatten(1)
    sign, high, low = 1.0 - 2.0 * (n >> 3).double(), (n >> 1) & 3, n & 1
    size = torch.where(high == 0, 0.5 * low, (1.0 + 0.5 * low) * _exact_two(high - 1))
    scale = _exact_two(scales.long() - 127).repeat_interleave(BLOCK, 1)[:, :n.shape[1]]
    return (sign * size * scale)[:, :k]


def _exact_rounded(x):
    """The values of the 4-bit format nearest to x, in 64 bits, by the distance to every level."""
    rows, k = x.shape
    blocks = torch.zeros(rows, -(-k // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    blocks[:, :k] = x.double()
    blocks = blocks.view(rows, -1, BLOCK)
    most = blocks.abs().amax(2, keepdim=True)
    scale = _exact_two(torch.frexp(most.clamp(min=2.0 ** -125)).exponent.long() - 3)
    v = blocks.abs() / scale
    best = torch.zeros_like(v)
    for level in (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0):  # the even codes first: an odd one has to be nearer
        best = torch.where((v - level).abs() < (v - best).abs(), torch.full_like(v, level), best)
    return (best * scale * torch.sign(blocks)).view(rows, -1)[:, :k]


def _exact_lookup(s):
    if s["n"] * s["width"] > 400_000_000:
        return None
    keep = (s["idx"] >= 0).nonzero().squeeze(1)
    at = s["idx"][keep].long()
    if s["table"] == "micro4":
        rows = _exact_values(s["codes"][at], s["scales"][at], s["width"])
    else:
        rows = s["rows_of"][at].double()
    w = torch.full((s["n"],), 0.5, dtype=torch.float64, device=at.device)
    if s["weight"] is not None:
        w = w * s["weight"].double()
    out = torch.zeros(s["n"], s["width"], dtype=torch.float64, device=at.device)
    out[keep] = rows * w[keep, None]
    if not s["train"]:
        return out
    dout = s["dout"][keep].double()
    dtable = torch.zeros(s["rows"], s["width"], dtype=torch.float64, device=at.device)
    dtable.index_add_(0, at, dout * w[keep, None])
    if s["weight"] is None:
        return {"out": out, "dtable": dtable}
    dweight = torch.zeros(s["n"], dtype=torch.float64, device=at.device)
    dweight[keep] = 0.5 * torch.einsum("nd,nd->n", dout, rows)
    return {"out": out, "dtable": dtable, "dweight": dweight}


def _exact_step(s):
    a = s["gate"].double().repeat_interleave(s["width"] // s["groups"], 1)
    new = a * s["state"].double() + s["x"].double()
    return {"h": new, "state": new}


def _exact_recurrence(s):
    """Step by step, all sequences at once; packed ones are laid out to one length by an index."""
    B, T, D, G = s["seqs"], s["steps"], s["width"], s["groups"]
    if s["offsets"] is not None:
        off = s["offsets"].long()
        length = off[1:] - off[:-1]
        T = int(length.max())
        if T * B * D > 700_000_000 or T > 120_000:
            return None
        t = torch.arange(T, device=off.device)[None, :]
        row = torch.where(t < length[:, None], off[:-1, None] + (length[:, None] - 1 - t if s["reverse"] else t), -1)
        take = lambda z: torch.where((row >= 0)[..., None], z.double()[row.clamp(min=0)], 0.0)  # noqa: E731
    else:
        if T * B * D > 700_000_000 or T > 120_000:
            return None
        length = torch.full((B,), T, device=s["x"].device)
        row = torch.arange(T, device=s["x"].device)[None, :].expand(B, T)
        take = lambda z: z.double().flip(1) if s["reverse"] else z.double()  # noqa: E731
    a, x = take(s["gate"]), take(s["x"])
    live = (torch.arange(T, device=x.device)[None, :] < length[:, None])[..., None]
    h0 = torch.zeros(B, D, dtype=torch.float64, device=x.device) if s["state"] is None else s["state"].double()
    wide = lambda z: z[:, :, None].expand(B, G, D // G).reshape(B, D)  # noqa: E731
    hs, h = torch.zeros_like(x), h0
    for t in range(T):
        h = torch.where(live[:, t], wide(a[:, t]) * h + x[:, t], h)
        hs[:, t] = h

    def put(z, like):
        if s["offsets"] is None:
            return z.flip(1) if s["reverse"] else z
        full = torch.zeros(like.shape[0] + 1, z.shape[-1], dtype=torch.float64, device=z.device)
        full[row.reshape(-1)] = torch.where(live, z, 0.0).reshape(-1, z.shape[-1])  # rows of no step go to the extra one
        return full[:-1]

    out = {"last": h} | ({"h": put(hs, s["x"])} if s["states"] else {})
    if not s["train"]:
        return out
    dh = take(s["dh"]) if s["states"] else None
    lam, dx, dgate = s["dlast"].double(), torch.zeros_like(x), torch.zeros_like(a)
    for t in range(T - 1, -1, -1):
        here = lam if dh is None else lam + dh[:, t]
        dx[:, t] = here
        dgate[:, t] = (here * (hs[:, t - 1] if t else h0)).view(B, G, D // G).sum(2)
        lam = torch.where(live[:, t], wide(a[:, t]) * here, lam)
    out |= {"dgate": put(dgate, s["gate"]), "dx": put(dx, s["x"])}
    return out | ({"dstate": lam} if s["state"] is not None else {})


def _exact_quantize(s):
    return None if s["rows"] * s["width"] > 300_000_000 else _exact_rounded(s["x"])


def _exact_product(s):
    w = _exact_values(s["w_codes"], s["w_scales"], s["k"])
    x = _exact_values(s["codes"], s["scales"], s["k"]) if s["x"] == "micro4" else _exact_rounded(s["x_of"])
    return x @ w.T
