"""The 8-bit KV cache in plain NumPy-like torch, 64 bits, CPU: what its
operators are tested against."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def scale_exponent(top: float) -> int:
    """The least e >= -100 with top <= 448 * 2^e."""
    e = -100
    while top > 448.0 * 2.0 ** e:
        e += 1
    return e


def e4m3_round(x: torch.Tensor) -> torch.Tensor:
    """float64 -> nearest e4m3 value (ties to even), |x| <= 448."""
    mag = x.abs().clamp(min=2.0 ** -6)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.floor(torch.log2(mag)) - 3)
    return torch.round(x / step) * step


def seal(x: torch.Tensor, block: int):
    """bf16 ``[B, H, n, D]`` -> (code values float64, scales float64 [B, H, n / block])."""
    b, h, n, d = x.shape
    y = x.double().cpu().reshape(b, h, n // block, block * d)
    codes, scales = torch.zeros_like(y), torch.zeros(b, h, n // block, dtype=torch.float64)
    for i in range(b):
        for j in range(h):
            for k in range(n // block):
                row = y[i, j, k]
                if not torch.isfinite(row).all():
                    scales[i, j, k] = math.nan
                    continue
                scales[i, j, k] = 2.0 ** scale_exponent(float(row.abs().max()))
                codes[i, j, k] = e4m3_round(row / scales[i, j, k])
    return codes.reshape(b, h, n, d), scales


def open_rows(codes: torch.Tensor, scale: torch.Tensor, sealed: int, tail: torch.Tensor, block: int) -> torch.Tensor:
    """The rows a cache stands for, float64."""
    c = codes[:, :, :sealed].cpu().double()
    s = scale[:, :, : sealed // block].cpu().double().repeat_interleave(block, 2)
    return torch.cat([c * s.unsqueeze(-1), tail.cpu().double()], 2)


def attention(q, k, v, vis, scale):
    """float64 (out [B, Tq, Hq, D], lse [B, Hq, Tq]); k, v [B, Hkv, T, D].  A
    key that a row does not see takes no part, whatever its values are."""
    b, hq, tq, d = q.shape
    hkv = k.shape[1]
    out = torch.zeros(b, tq, hq, d, dtype=torch.float64)
    lse = torch.full((b, hq, tq), -math.inf, dtype=torch.float64)
    qd = q.cpu().double()
    for i in range(b):
        for h in range(hq):
            kk, vv = k[i, h // (hq // hkv)], v[i, h // (hq // hkv)]
            for t in range(tq):
                on = vis[i, t]
                if not on.any():
                    continue
                s = (kk[on] @ qd[i, h, t]) * scale
                lse[i, h, t] = torch.logsumexp(s, 0)
                out[i, t, h] = torch.softmax(s, 0) @ vv[on]
    return out, lse


def mass(q, lse, k, vis, scale):
    """float64 [B, Hkv, T]: the weight each key received."""
    b, hq, tq, d = q.shape
    hkv, total = k.shape[1], k.shape[2]
    got = torch.zeros(b, hkv, total, dtype=torch.float64)
    qd, ld = q.cpu().double(), lse.cpu().double()
    for i in range(b):
        for h in range(hq):
            s = (qd[i, h] @ k[i, h // (hq // hkv)].T) * scale
            w = torch.where(vis[i] & (ld[i, h] > -math.inf).unsqueeze(-1), torch.exp(s - ld[i, h].unsqueeze(-1)),
                            torch.zeros((), dtype=torch.float64))
            got[i, h // (hq // hkv)] += w.sum(0)
    return got


def keep_heaviest(m: torch.Tensor, length: int, budget: int, sinks: int, recent: int) -> torch.Tensor:
    b, h = m.shape[:2]
    out = torch.zeros(b, h, budget, dtype=torch.int32)
    for i in range(b):
        for j in range(h):
            w = [-math.inf if x != x else x for x in m[i, j, :length].tolist()]
            least = [x != x for x in m[i, j, :length].tolist()]
            mid = sorted(range(sinks, length - recent), key=lambda t: (least[t], -w[t], t))
            kept = list(range(sinks)) + mid[: budget - sinks - recent] + list(range(length - recent, length))
            out[i, j] = torch.tensor(sorted(kept), dtype=torch.int32)
    return out
