"""Plain 64-bit forms of the operations that serve a model token by token, for the tests beside this file."""
import torch

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0, "e2m1": 6.0}
_MANTISSA = {"e4m3": (3, -6), "e5m2": (2, -14), "e2m1": (1, 0)}          # bits, exponent of the smallest normal


def element_table(elem):
    """What every code of an element type stands for, fp64."""
    if elem == "e2m1":
        half = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        return torch.tensor(half + [-v for v in half], dtype=torch.float64)
    codes = torch.arange(256, dtype=torch.uint8)
    return codes.view({"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}[elem]).double()


def quantise(x, elem):
    """x [..., D] -> (values of the elements in units of their block's scale, fp64 [..., D/32, 32]; scale codes int64 [..., D/32])."""
    b = x.detach().cpu().double().reshape(*x.shape[:-1], -1, 32)
    amax = b.abs().amax(-1)
    fine = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(fine, amax, 0.0))                       # amax = m 2^e
    top = LARGEST[elem]
    mt, et = torch.frexp(torch.tensor(top, dtype=torch.float64))
    e = (e - et + (m > mt)).clamp(min=-126)
    e = torch.where(amax > 0, e, -126).long()
    y = torch.ldexp(torch.where(fine.unsqueeze(-1), b, 0.0), -e.unsqueeze(-1))
    bits, low = _MANTISSA[elem]
    _, ey = torch.frexp(y)
    step = (ey - 1).clamp(min=low) - bits
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)              # (round takes ties to even)
    return y, torch.where(fine, e + 127, 255)


def values(code, scale, elem):
    """uint8 codes and scale codes -> fp64 [..., D]."""
    code, scale = code.cpu(), scale.cpu().long()
    if elem == "e2m1":
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2)
    v = element_table(elem)[code.long()].reshape(*scale.shape, 32)
    s = torch.ldexp(torch.ones(scale.shape, dtype=torch.float64), scale - 127)
    s = torch.where(scale == 255, float("nan"), torch.where(scale == 0, 0.0, s))
    return (v * s.unsqueeze(-1)).flatten(-2)


def gather(buf, table, length):
    """[pages, H, page, n] through one sequence's table -> [H, length, n]."""
    page = buf.shape[2]
    at = torch.arange(length)
    p = table.cpu().long()[at // page]
    return buf.cpu()[p, :, at % page].transpose(0, 1)


def attention(q, k, v, seen, sm_scale):
    """One sequence: q [Hq,T,D], k, v [Hkv,n,D] fp64, seen bool [T,n] -> out [Hq,T,D], log2 denominators [Hq,T], sum p |v| / sum p, the
    largest sum |q k| sm_scale of each row, and the largest p |v| / sum p of each row."""
    G = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    s = (q @ k.transpose(1, 2)) * sm_scale
    mag = ((q.abs() @ torch.nan_to_num(k).abs().transpose(1, 2)) * sm_scale * seen).amax(-1) if k.shape[1] else torch.zeros(q.shape[:2], dtype=torch.float64)
    s = torch.where(seen, s, float("-inf"))
    none = ~seen.any(-1)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    p = torch.where(seen, torch.exp(s - torch.where(none, 0.0, lse).unsqueeze(-1)), 0.0)
    # (a key that a row does not see has no part in it, whatever its value is)
    vz = torch.nan_to_num(v)
    o, a = p @ vz, p @ vz.abs()
    big = (torch.nan_to_num(p) * vz.abs().amax(-1).unsqueeze(1)).amax(-1) if k.shape[1] else torch.zeros(q.shape[:2], dtype=torch.float64)
    for h, t in torch.nonzero(torch.isnan(p).any(-1) | ((p @ torch.isnan(v).any(-1, keepdim=True).double()).squeeze(-1) > 0)).tolist():
        o[h, t] = (p[h, t].unsqueeze(-1) * torch.where(seen[t].unsqueeze(-1), v[h], 0.0)).sum(0)
    o[:, none] = 0.0
    return o, torch.where(none, float("-inf"), lse / torch.log(torch.tensor(2.0, dtype=torch.float64))), a, mag, big


def norm_rope(x, weight, norm, eps, cos, sin, rows, interleaved):
    """x fp64 [B,H,L,D] logical; weight fp64 broadcastable or None; norm None, "head" or "across"; rows int64 [B,L,R/2]: the table row of every pair."""
    x = x.double().clone()
    if norm is not None:
        ms = (x * x).mean(-1, keepdim=True) if norm == "head" else (x * x).mean((1, 3), keepdim=True)
        x = x / torch.sqrt(ms + eps)
        if weight is not None:
            x = x * weight
    size = x.abs()
    if cos is not None:
        h = rows.shape[-1]
        there = ((rows >= 0) & (rows < cos.shape[0])).all(-1, keepdim=True)
        r = rows.clamp(0, cos.shape[0] - 1)
        i = torch.arange(h)
        c, s = (torch.where(there, t.double()[r, i], float("nan")).unsqueeze(1) for t in (cos, sin))
        at = (torch.arange(0, 2 * h, 2), torch.arange(1, 2 * h, 2)) if interleaved else (torch.arange(h), torch.arange(h, 2 * h))
        a, b = x[..., at[0]], x[..., at[1]]
        x[..., at[0]], x[..., at[1]] = a * c - b * s, b * c + a * s
        both = a.abs() + b.abs()
        size[..., at[0]], size[..., at[1]] = both, both
    return x, size
