"""Plain 64-bit implementations of the 4-bit weight operators and of the expert routing, for tests: written from the formulas
in include/bgemm_b200.h, column by column, without the library."""
from __future__ import annotations

import math

import torch


def half_step(dtype) -> float:
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def row_bytes(K: int) -> int:
    return -(-K // 128) * 64


def position(k: int):
    """(byte of the row, nibble of the byte) of column k."""
    block, w, t, i = k // 128, k % 128 // 32, k % 32 // 8, k % 8
    nibble = i // 2 if i % 2 == 0 else 4 + i // 2
    return block * 64 + 16 * t + 4 * w + nibble // 2, nibble % 2


def pack(codes: torch.Tensor, fill: int = 0) -> torch.Tensor:
    """Codes [.., M, K] (0..15) -> plane uint8 [.., M, row_bytes(K)]; the columns behind K hold `fill`."""
    K = codes.shape[-1]
    total = -(-K // 128) * 128
    full = torch.full(codes.shape[:-1] + (total,), fill, dtype=torch.uint8, device=codes.device)
    full[..., :K] = codes.to(torch.uint8)
    plane = torch.zeros(codes.shape[:-1] + (total // 2,), dtype=torch.uint8, device=codes.device)
    at = [position(k) for k in range(total)]
    for nib in (0, 1):
        cols = [k for k in range(total) if at[k][1] == nib]
        plane[..., [at[k][0] for k in cols]] |= full[..., cols] << (4 * nib)
    return plane


def unpack(plane: torch.Tensor, K: int) -> torch.Tensor:
    at = [position(k) for k in range(K)]
    b = torch.tensor([a for a, _ in at], device=plane.device)
    n = torch.tensor([4 * n for _, n in at], device=plane.device, dtype=torch.uint8)
    return (plane[..., b] >> n) & 15


def spread(v: torch.Tensor, K: int, group: int) -> torch.Tensor:
    return v[..., torch.arange(K, device=v.device) // group]


def values(plane, scales, zeros, K, group) -> torch.Tensor:
    """(q - z) * s in 64 bits."""
    q = unpack(plane, K).double()
    z = 8.0 if zeros is None else spread((zeros & 15).double(), K, group)
    return (q - z) * spread(scales.double(), K, group)


def quantize(w: torch.Tensor, group: int, symmetric: bool, kind):
    """(codes, scales, zeros) of [M, K] weights; 32-bit arithmetic as the formulas say."""
    M, K = w.shape
    w = w.float()
    G = -(-K // group)
    codes = torch.zeros(M, K, dtype=torch.uint8, device=w.device)
    scales = torch.zeros(M, G, dtype=kind, device=w.device)
    zeros = torch.full((M, G), 8, dtype=torch.uint8, device=w.device)
    for g in range(G):
        v = w[:, g * group:(g + 1) * group]
        lo, hi = v.amin(1).clamp(max=0), v.amax(1).clamp(min=0)
        if symmetric:
            s = (torch.maximum(-lo, hi) * torch.tensor(1.0 / 7.0, dtype=torch.float32, device=w.device)).to(kind)
        else:
            s = ((hi - lo) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=w.device)).to(kind)
        f = s.float()
        ok = f > 0
        safe = torch.where(ok, f, torch.ones_like(f))
        z = torch.full_like(f, 8.0) if symmetric else torch.where(ok, torch.round(-lo / safe).clamp(0, 15), torch.zeros_like(f))
        q = torch.where(ok[:, None], torch.round(v / safe[:, None]), torch.zeros_like(v)) + z[:, None]
        codes[:, g * group:(g + 1) * group] = q.clamp(0, 15).to(torch.uint8)
        scales[:, g] = s
        zeros[:, g] = z.to(torch.uint8)
    return codes, scales, None if symmetric else zeros


def linear(x, w) -> torch.Tensor:
    return x.double() @ w.t()


def linear_tolerance(x, y, plane, scales, zeros, K, group) -> torch.Tensor:
    """How far a kernel's result may be from `y` = linear(x, values(..)), element by element:
      * one rounding of the result: u |y| (u = half a step of the 16-bit type, 2^-25 below the normal numbers of fp16);
      * the weights' own rounding, where a kernel rounds them: u sum |w x|, and 2^-25 sum |x| for weights below fp16's normals;
      * 32-bit sums: at most 128 additions inside a scale group and one per group outside, each off by 2^-23 of the running
        sum (the tensor cores may truncate), whose parts are bounded by (q + z + 2 * 128) s |x| where 128 + q is summed."""
    u = half_step(x.dtype)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    q = unpack(plane, K).double()
    z = 8.0 if zeros is None else spread((zeros & 15).double(), K, group)
    s = spread(scales.double().abs(), K, group)
    ax = x.double().abs()
    weights = ((q - z).abs() * s)
    parts = (q + z + (256.0 if x.dtype == torch.bfloat16 else 0.0)) * s
    steps = 128 + scales.shape[-1] + 16
    return u * y.abs() + tiny + u * (ax @ weights.t()) + tiny * ax.sum(1, keepdim=True) + steps * 2.0 ** -23 * (ax @ parts.t())


def rounded(plane, scales, zeros, K, group) -> torch.Tensor:
    """values(..) as the tensor-core kernel multiplies them: each rounded once to the scales' type (in 64 bits)."""
    return values(plane, scales, zeros, K, group).to(scales.dtype).double()


def linear_bound(x, y, plane, scales, zeros, K, group, tensor) -> torch.Tensor:
    """How far one kernel's result may be from `y`, element by element. tensor: the tensor-core kernel, y = linear(x, rounded(..));
    otherwise the streaming kernel, which rounds no weight, y = linear(x, values(..)). Both:
      * one rounding of the result: u |y| (u = half a step of the 16-bit type, 2^-25 below the normal numbers of fp16);
      * one product of 16 columns adds 16 parts to a sum, each addition off by at most 2^-23 of it (the tensor cores may truncate):
        17 * 2^-23 a product with its start.
    Tensor cores: ceil(K / 16) such products on parts |w x|, and up to 8 partial sums added up, 2^-24 each.
    Streaming: group / 16 products (and 4 roundings where the group's sums meet scale and zero point) on parts (q + z) s |x|,
    (q + z + 256) s |x| for bf16, whose codes are summed as 128 + q; the groups and the sums of up to 12 warps meet by additions of
    2^-24 of sums no larger than sum |w x|."""
    u = half_step(x.dtype)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    ax = x.double().abs()
    mag = ax @ (rounded if tensor else values)(plane, scales, zeros, K, group).abs().t()
    if tensor:
        sums = (17 * -(-K // 16) * 2.0 ** -23 + 8 * 2.0 ** -24) * mag
    else:
        q = unpack(plane, K).double()
        z = 8.0 if zeros is None else spread((zeros & 15).double(), K, group)
        parts = ax @ ((q + z + (256.0 if x.dtype == torch.bfloat16 else 0.0)) * spread(scales.double().abs(), K, group)).t()
        sums = (17 * (group // 16) + 4) * 2.0 ** -23 * parts + (scales.shape[-1] + 16) * 2.0 ** -24 * mag
    return u * (y.abs() + sums) + tiny + sums


def route(logits, top_k, renormalize):
    """(weights float64 [T, k], experts, offsets, rows, slots) by plain loops over tokens."""
    T, E = logits.shape
    v = logits.double().cpu().tolist()
    weights = torch.zeros(T, top_k, dtype=torch.float64)
    experts = torch.full((T, top_k), -1, dtype=torch.int32)
    slots = torch.full((T, top_k), -1, dtype=torch.int32)
    by_expert = [[] for _ in range(E)]
    for t in range(T):
        allowed = [e for e in range(E) if v[t][e] > -math.inf]          # NaN compares false
        order = sorted(allowed, key=lambda e: (-v[t][e], e))[:top_k]
        if not order:
            continue
        top = v[t][order[0]]
        share = lambda e: 1.0 if v[t][e] == top else math.exp(v[t][e] - top)          # noqa: E731
        total = sum(share(e) for e in (order if renormalize else allowed))
        for j, e in enumerate(order):
            experts[t, j] = e
            weights[t, j] = share(e) / total
            by_expert[e].append((t, j))
    offsets, rows = [0], []
    for e in range(E):
        for t, j in by_expert[e]:
            slots[t, j] = len(rows)
            rows.append(t)
        offsets.append(len(rows))
    rows += [-1] * (T * top_k - len(rows))
    return weights, experts, torch.tensor(offsets, dtype=torch.int32), torch.tensor(rows, dtype=torch.int32), slots


def combine(y, slots, weights):
    T, k = slots.shape
    out = torch.zeros(T, y.shape[1], dtype=torch.float64, device=y.device)
    mag = torch.zeros_like(out)
    for j in range(k):
        s = slots[:, j].long()
        ok = (s >= 0) & (s < y.shape[0])
        part = weights[ok, j].double()[:, None] * y[s[ok]].double()
        out[ok] += part
        mag[ok] += part.abs()
    return out, mag
