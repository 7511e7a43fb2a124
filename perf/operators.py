"""Cases of the 4-bit weight operators and of the expert routing around them.

Five operators, each in its plain form and as a call of this repository's `lowbit_kernel` module:

  quantize   weights [M, K] -> 4-bit codes with a scale (and zero point) per group of `group` columns, and back to the values they stand for
  linear     y[n, m] = sum_k x[n, k] * (q[m, k] - z[m, k // group]) * s[m, k // group]          (z = 8 where there are no zero points)
  grouped    the same product with one weight matrix per expert; the rows of one expert are consecutive (offsets), taken from x by index or in order
  route      logits [T, E] -> the k largest experts of each token, their softmax weights, and the order that puts the rows of one expert together
  combine    out[t] = sum_j weights[t, j] * y[slots[t, j]]

The codes of a row are stored in blocks of 128 columns (64 bytes, sixteen little-endian 32-bit words): word 4 t + w holds the columns
32 w + 8 t + i (i = 0..7); column i of a word is nibble i / 2 where i is even and nibble 4 + i / 2 where it is odd. A row ends on a whole block.
"""
import math
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_module = None


def kernels():
    """This repository's extension module (only where `own` is true)."""
    global _module
    if _module is None:
        sys.path.insert(0, "bgemm-cuda_b200")
        import lowbit_kernel

        _module = lowbit_kernel
    return _module


# ---- the cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one attention projection of a small model, quantised when the model is loaded
        {"name": "quantize 4096x4096", "op": "quantize", "m": 4096, "k": 4096, "group": 128, "dtype": "fp16", "zeros": True},
        # the widest layer of a large model, loaded from bf16, symmetric codes in small groups
        {"name": "quantize 28672x8192", "op": "quantize", "m": 28672, "k": 8192, "group": 64, "dtype": "bf16", "zeros": False},
        # one token through one projection: the smallest call, latency counts
        {"name": "linear 4096x4096 n1", "op": "linear", "n": 1, "m": 4096, "k": 4096, "group": 128, "dtype": "fp16", "zeros": False},
        # a decode step of seven sequences through the widest layer: the weights' bytes count
        {"name": "linear 28672x8192 n7", "op": "linear", "n": 7, "m": 28672, "k": 8192, "group": 64, "dtype": "bf16", "zeros": True},
        # a prompt of 2000 tokens through an up projection: the products count
        {"name": "linear 14336x4096 n2000", "op": "linear", "n": 2000, "m": 14336, "k": 4096, "group": 128, "dtype": "bf16", "zeros": True},
        # one token sent to 8 of 64 experts, read in place by index
        {"name": "grouped 64x4096x2048 s8", "op": "grouped", "slots": 8, "tokens": 1, "experts": 64, "m": 4096, "k": 2048, "group": 128, "dtype": "bf16",
         "zeros": False, "skew": 0.0, "gather": True},
        # a decode step of 100 sequences, 8 of 64 experts each, uneven: some experts get one row, some get dozens; odd sizes
        {"name": "grouped 64x1001x2056 s800", "op": "grouped", "slots": 800, "tokens": 100, "experts": 64, "m": 1001, "k": 2056, "group": 64,
         "dtype": "fp16", "zeros": True, "skew": 0.8, "gather": True},
        # the largest: a prefill batch of 4096 tokens, 2 of 8 experts each, through the up projection
        {"name": "grouped 8x14336x4096 s8192", "op": "grouped", "slots": 8192, "tokens": 4096, "experts": 8, "m": 14336, "k": 4096, "group": 128,
         "dtype": "bf16", "zeros": True, "skew": 0.25, "gather": False},
        # routing of a decode step
        {"name": "route 64x64 top8", "op": "route", "tokens": 64, "experts": 64, "top_k": 8, "dtype": "fp32", "renormalize": True, "padded": 0.0},
        # routing of a long prefill batch with padding rows at its end, many equal logits (bf16)
        {"name": "route 16000x256 top8", "op": "route", "tokens": 16000, "experts": 256, "top_k": 8, "dtype": "bf16", "renormalize": False, "padded": 0.03},
        # the experts' results of a decode step back into 64 rows
        {"name": "combine 64x4096 top8", "op": "combine", "tokens": 64, "m": 4096, "top_k": 8, "dtype": "bf16", "padded": 0.0},
        # the same after a prefill batch, with padding rows; odd width
        {"name": "combine 8000x4104 top4", "op": "combine", "tokens": 8000, "m": 4104, "top_k": 4, "dtype": "fp16", "padded": 0.05},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm; odd and even alike."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _columns(rng, lo, hi):
    """A row length: mostly a multiple of 128 or of 8, now and then any number."""
    k = _spread(rng, lo, hi)
    step = rng.choice([128, 128, 8, 8, 1])
    return max(lo, k // step * step)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "grouped", "grouped", "route", "combine"])
    kind = {"dtype": rng.choice(["fp16", "bf16"])}
    if op == "quantize":
        k = _columns(rng, 128, 8192)
        m = _spread(rng, 64, 28672)
        return {"op": op, "m": m, "k": k, "group": rng.choice([32, 64, 128]), "dtype": rng.choice(["fp16", "bf16", "fp32"]), "zeros": rng.random() < 0.5}
    if op == "linear":
        k, m = _columns(rng, 128, 8192), _spread(rng, 64, 28672)
        n = _spread(rng, 1, max(1, min(4096, 480_000_000_000 // (m * k))))
        return {"op": op, "n": n, "m": m, "k": k, "group": rng.choice([32, 64, 128]), **kind, "zeros": rng.random() < 0.5}
    if op == "grouped":
        k, m, top = _columns(rng, 128, 4096), _spread(rng, 64, 14336), rng.choice([1, 2, 4, 8])
        e = _spread(rng, top, max(top, min(128, 400_000_000 // (m * k))))
        t = _spread(rng, 1, max(1, min(4096, 400_000_000_000 // (m * k * top))))
        return {"op": op, "slots": t * top, "tokens": t, "experts": e, "m": m, "k": k, "group": rng.choice([32, 64, 128]), **kind,
                "zeros": rng.random() < 0.5, "skew": round(rng.uniform(0.0, 1.0), 3), "gather": rng.random() < 0.5}
    if op == "route":
        e = _spread(rng, 8, 256)
        return {"op": op, "tokens": _spread(rng, 1, 16000), "experts": e, "top_k": rng.randint(1, min(8, e)), "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "renormalize": rng.random() < 0.5, "padded": round(rng.choice([0.0, rng.uniform(0.0, 0.2)]), 3)}
    return {"op": op, "tokens": _spread(rng, 1, 8000), "m": _columns(rng, 64, 8192), "top_k": rng.randint(1, 8), **kind,
            "padded": round(rng.choice([0.0, rng.uniform(0.0, 0.2)]), 3)}


# ---- what a program has in hand --------------------------------------------------------------------------------------
def _pack(codes):
    """Codes [..., M, K] (whole numbers 0..15) -> the stored rows, uint8 [..., M, ceil(K / 128) * 64]."""
    k = codes.shape[-1]
    blocks = -(-k // 128)
    padded = torch.zeros(codes.shape[:-1] + (blocks * 128,), dtype=torch.int32, device=codes.device)
    padded[..., :k] = codes
    c = padded.view(codes.shape[:-1] + (blocks, 4, 4, 8)).transpose(-3, -2)           # [..., block, t, w, i]
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=codes.device)
    words = (c << shifts).sum(-1, dtype=torch.int64)
    bytes_ = torch.stack([(words >> (8 * b)) & 255 for b in range(4)], -1).to(torch.uint8)
    return bytes_.reshape(codes.shape[:-1] + (blocks * 64,)).contiguous()


def _weights(c, g, lead):
    """A quantised matrix (or a stack of them, one packed at a time): codes around the middle, scales spread over a factor of a few."""
    m, k, group = c["m"], c["k"], c["group"]
    groups = -(-k // group)
    planes = []
    for _ in range(lead or 1):
        codes = torch.randn(m, k, generator=g, device="cuda").mul_(2.7).add_(7.7).round_().clamp_(0, 15).to(torch.int32)
        planes.append(_pack(codes))
    plane = torch.stack(planes) if lead else planes[0]
    shape = ((lead,) if lead else ()) + (m, groups)
    scales = (torch.randn(shape, generator=g, device="cuda") * 0.4 - 5.2).exp().to(DTYPES[c["dtype"]])
    zeros = torch.randint(5, 12, shape, generator=g, device="cuda", dtype=torch.uint8) if c["zeros"] else None
    return plane, scales, zeros


def _activations(rows, k, dtype, g):
    """Rows of a normalised residual stream: unit variance, a few columns far larger than the others."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    loud = torch.rand(k, generator=g, device="cuda") < 0.004
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def _counts(c):
    """Rows of each expert, largest first: a power law of the rank, the same for every seed."""
    e, s = c["experts"], c["slots"]
    share = [(r + 1.0) ** -c["skew"] for r in range(e)]
    total = sum(share)
    got = [int(s * v / total) for v in share]
    left = s - sum(got)
    return [n + (left // e) + (1 if r < left % e else 0) for r, n in enumerate(got)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "quantize":
        w = torch.randn(c["m"], c["k"], generator=g, device="cuda").mul_(0.02)
        w *= (torch.randn(c["m"], 1, generator=g, device="cuda") * 0.3).exp()          # rows of different size
        s["w"] = w.to(DTYPES[c["dtype"]])
    elif c["op"] == "linear":
        s["plane"], s["scales"], s["zeros"] = _weights(c, g, 0)
        s["x"] = _activations(c["n"], c["k"], DTYPES[c["dtype"]], g)
    elif c["op"] == "grouped":
        s["plane"], s["scales"], s["zeros"] = _weights(c, g, c["experts"])
        order = torch.randperm(c["experts"], generator=g, device="cuda")
        counts = torch.tensor(_counts(c), device="cuda")[order]
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)]).to(torch.int32)
        s["most"] = max(_counts(c))
        s["rows"] = torch.randint(0, c["tokens"], (c["slots"],), generator=g, device="cuda", dtype=torch.int32) if c["gather"] else None
        s["x"] = _activations(c["tokens"] if c["gather"] else c["slots"], c["k"], DTYPES[c["dtype"]], g)
    elif c["op"] == "route":
        logits = torch.randn(c["tokens"], c["experts"], generator=g, device="cuda") * 1.5
        logits[torch.rand(c["tokens"], generator=g, device="cuda") < c["padded"]] = -math.inf
        s["logits"] = logits.to(DTYPES[c["dtype"]])
    else:
        t, k = c["tokens"], c["top_k"]
        s["y"] = torch.randn(t * k, c["m"], generator=g, device="cuda").to(DTYPES[c["dtype"]])
        slots = torch.randperm(t * k, generator=g, device="cuda").to(torch.int32).view(t, k)
        slots[torch.rand(t, generator=g, device="cuda") < c["padded"]] = -1
        s["slots"] = slots
        s["weights"] = torch.rand(t, k, generator=g, device="cuda") + 0.02
        s["weights"] /= s["weights"].sum(-1, keepdim=True)
    return s


# ---- the operators: plain, and the framework's -----------------------------------------------------------------------
def _values(plane, scales, zeros, k, group):
    """(q - z) * s in 32 bits, [..., M, K]."""
    lead = plane.shape[:-1]
    words = plane.view(torch.int32).view(lead + (-1, 4, 4, 1))                          # [..., block, t, w, 1]
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=plane.device)
    q = ((words >> shifts) & 15).transpose(-3, -2).reshape(lead + (-1,))[..., :k].float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, -1)[..., :k]
    return (q - z) * scales.float().repeat_interleave(group, -1)[..., :k]


def _plain_quantize(w, group, with_zeros):
    m, k = w.shape
    kind = torch.float16 if w.dtype == torch.float32 else w.dtype
    groups = -(-k // group)
    v = torch.zeros(m, groups * group, device=w.device)
    v[:, :k] = w.float()
    v = v.view(m, groups, group)
    if with_zeros:
        lo, hi = v.amin(-1).clamp(max=0.0), v.amax(-1).clamp(min=0.0)
        s = ((hi - lo) / 15.0).to(kind)
        f = s.float()
        z = torch.where(f > 0, torch.round(-lo / f).clamp(0, 15), torch.zeros_like(f))
    else:
        s = (v.abs().amax(-1) / 7.0).to(kind)
        f = s.float()
        z = torch.full_like(f, 8.0)
    q = torch.where(f[..., None] > 0, (torch.round(v / f[..., None]) + z[..., None]).clamp(0, 15), z[..., None])
    values = ((q - z[..., None]) * f[..., None]).reshape(m, -1)[:, :k].to(kind)
    return {"values": values, "scales": s, "zeros": z.to(torch.uint8) if with_zeros else None}


def _plain_grouped(s, c):
    w = _values(s["plane"], s["scales"], s["zeros"], c["k"], c["group"])                # [E, M, K]
    x = s["x"].float() if s["rows"] is None else s["x"].float()[s["rows"].long()]       # [slots, K]
    start = s["offsets"][:-1].long()
    count = s["offsets"][1:].long() - start
    at = torch.arange(s["most"], device=x.device)
    place = start[:, None] + at                                                          # [E, most]
    inside = at < count[:, None]
    padded = x[place.clamp(max=c["slots"] - 1)] * inside[..., None]
    y = torch.bmm(padded, w.transpose(1, 2))                                             # [E, most, M]
    out = torch.empty(c["slots"] + 1, c["m"], device=x.device)
    out[torch.where(inside, place, c["slots"])] = y                                      # the last row takes what lies behind each expert's rows
    return out[:-1].to(s["x"].dtype)


def _plain_route(logits, top_k, renormalize):
    t, e = logits.shape
    v = logits.float()
    top, experts = torch.sort(v, dim=-1, descending=True, stable=True)
    top, experts = top[:, :top_k], experts[:, :top_k]
    chosen = top > -math.inf
    first = torch.where(chosen[:, :1], top[:, :1], torch.zeros_like(top[:, :1]))
    up = torch.exp(top - first)
    below = up.sum(-1, keepdim=True) if renormalize else torch.exp(v - first).sum(-1, keepdim=True)
    weights = torch.where(chosen, up / below, torch.zeros_like(up))
    key = torch.where(chosen, experts, torch.full_like(experts, e)).reshape(-1)
    key, order = torch.sort(key, stable=True)                                            # pairs (token, choice) by expert, then in order
    slot = torch.empty_like(order)
    slot[order] = torch.arange(t * top_k, device=v.device)
    rows = torch.where(key < e, order // top_k, -1)
    offsets = torch.searchsorted(key, torch.arange(e + 1, device=v.device))
    offsets[0] = 0
    return {"weights": weights, "experts": torch.where(chosen, experts, -1).int(), "offsets": offsets.int(), "rows": rows.int(),
            "slots": torch.where(chosen, slot.view(t, top_k), -1).int()}


def _plain_combine(y, slots, weights):
    picked = y.float()[slots.clamp(min=0).long()]                                        # [T, k, M]
    scale = torch.where(slots >= 0, weights, torch.zeros_like(weights))
    return (picked * scale[..., None]).sum(1).to(y.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        lib = kernels()
        if c["op"] == "quantize":
            plane, scales, zeros = lib.w4_quantize(s["w"], c["group"], not c["zeros"])
            return {"values": lib.w4_dequantize(plane, scales, zeros, c["k"], c["group"]), "scales": scales, "zeros": zeros}
        if c["op"] == "linear":
            return lib.w4a16_linear_forward(s["x"], s["plane"], s["scales"], s["zeros"], c["group"])
        if c["op"] == "grouped":
            return lib.w4a16_grouped_forward(s["x"], s["plane"], s["scales"], s["zeros"], s["offsets"], s["rows"], c["group"])
        if c["op"] == "route":
            weights, experts, offsets, rows, slots = lib.moe_route(s["logits"], c["top_k"], c["renormalize"])
            return {"weights": weights, "experts": experts, "offsets": offsets, "rows": rows, "slots": slots}
        return lib.moe_combine(s["y"], s["slots"], s["weights"])
    if c["op"] == "quantize":
        return _plain_quantize(s["w"], c["group"], c["zeros"])
    if c["op"] == "linear":
        return (s["x"].float() @ _values(s["plane"], s["scales"], s["zeros"], c["k"], c["group"]).t()).to(s["x"].dtype)
    if c["op"] == "grouped":
        return _plain_grouped(s, c)
    if c["op"] == "route":
        return _plain_route(s["logits"], c["top_k"], c["renormalize"])
    return _plain_combine(s["y"], s["slots"], s["weights"])


def work(case):
    c = case
    size = 4 if c.get("dtype") == "fp32" else 2
    if c["op"] == "quantize":
        groups = c["m"] * -(-c["k"] // c["group"]) * (3 if c["zeros"] else 2)
        # the weights in, the codes out and in again, the values out
        return {"bytes": c["m"] * c["k"] * (size + 0.5 + 0.5 + 2) + 2 * groups, "flops": 4 * c["m"] * c["k"]}
    if c["op"] in ("linear", "grouped"):
        matrix = c["m"] * c["k"] / 2 + c["m"] * -(-c["k"] // c["group"]) * (3 if c["zeros"] else 2)
        if c["op"] == "linear":
            return {"bytes": matrix + 2 * c["n"] * (c["k"] + c["m"]), "flops": 2 * c["n"] * c["m"] * c["k"]}
        used = sum(1 for n in _counts(c) if n)
        rows = min(c["tokens"], c["slots"]) if c["gather"] else c["slots"]
        return {"bytes": used * matrix + 2 * rows * c["k"] + 2 * c["slots"] * c["m"] + 4 * (c["experts"] + 1) + (4 * c["slots"] if c["gather"] else 0),
                "flops": 2 * c["slots"] * c["m"] * c["k"]}
    if c["op"] == "route":
        pairs = c["tokens"] * c["top_k"]
        return {"bytes": c["tokens"] * c["experts"] * size + 16 * pairs + 4 * (c["experts"] + 1), "flops": 4 * c["tokens"] * c["experts"]}
    pairs = c["tokens"] * c["top_k"] * (1 - c["padded"])
    return {"bytes": pairs * c["m"] * 2 + c["tokens"] * c["m"] * 2 + 8 * c["tokens"] * c["top_k"], "flops": 2 * pairs * c["m"]}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------
def _exact_matrix(plane, scales, zeros, k, group):
    """One matrix [M, K] in 64 bits, column by column of the stored layout."""
    col = torch.arange(k, device=plane.device)
    block, w, t, i = col // 128, col % 128 // 32, col % 32 // 8, col % 8
    nibble = torch.where(i % 2 == 0, i // 2, 4 + i // 2)
    byte = block * 64 + 16 * t + 4 * w + nibble // 2
    q = (plane[:, byte].to(torch.int32) >> (4 * (nibble % 2)).to(torch.int32)) & 15
    g = col // group
    z = 8 if zeros is None else zeros[:, g].to(torch.int32)
    return (q - z).double() * scales[:, g].double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        w = s["w"].double()
        kind = torch.float16 if c["dtype"] == "fp32" else DTYPES[c["dtype"]]
        values, scales, zeros = [], [], []
        for first in range(0, c["k"], c["group"]):
            v = w[:, first:first + c["group"]]
            if c["zeros"]:
                lo, hi = torch.minimum(v.min(1).values, torch.zeros(1, dtype=v.dtype, device=v.device)), torch.maximum(
                    v.max(1).values, torch.zeros(1, dtype=v.dtype, device=v.device))
                sc = ((hi - lo) / 15).to(kind).double()
                z = torch.where(sc > 0, (-lo / sc).round().clamp(0, 15), 0.0)
            else:
                sc = (v.abs().max(1).values / 7).to(kind).double()
                z = torch.full_like(sc, 8.0)
            q = torch.where(sc[:, None] > 0, ((v / sc[:, None]).round() + z[:, None]).clamp(0, 15), z[:, None])
            values.append((q - z[:, None]) * sc[:, None])
            scales.append(sc)
            zeros.append(z)
        return {"values": torch.cat(values, 1), "scales": torch.stack(scales, 1), "zeros": torch.stack(zeros, 1).to(torch.uint8) if c["zeros"] else None}
    if c["op"] == "linear":
        return s["x"].double() @ _exact_matrix(s["plane"], s["scales"], s["zeros"], c["k"], c["group"]).t()
    if c["op"] == "grouped":
        out = torch.zeros(c["slots"], c["m"], dtype=torch.float64, device="cuda")
        at = s["offsets"].tolist()
        for e in range(c["experts"]):
            a, b = at[e], at[e + 1]
            if a < b:
                x = s["x"][a:b] if s["rows"] is None else s["x"][s["rows"][a:b].long()]
                out[a:b] = x.double() @ _exact_matrix(s["plane"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e], c["k"], c["group"]).t()
        return out
    if c["op"] == "route":
        v = s["logits"].double()
        p = torch.softmax(v, -1).nan_to_num(0.0)
        chosen = torch.argsort(v, dim=-1, descending=True, stable=True)[:, :c["top_k"]]
        picked = p.gather(1, chosen)
        if c["renormalize"]:
            picked = (picked / picked.sum(-1, keepdim=True)).nan_to_num(0.0)
        return {"weights": picked, "experts": None, "offsets": None, "rows": None, "slots": None}
    out = torch.zeros(c["tokens"], c["m"], dtype=torch.float64, device="cuda")
    for j in range(c["top_k"]):
        slot = s["slots"][:, j].long()
        there = slot >= 0
        out[there] += s["weights"][there, j].double()[:, None] * s["y"][slot[there]].double()
    return out
