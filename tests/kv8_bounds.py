"""How far an attention over the 8-bit KV cache may be off, row by row.

The definition in 64 bits, with what its error bounds need:

* A probability (times its value's scale) is rounded to fp16, half a step, 2^-11
  relative; scores and the log-sum-exp are off by at most 4e-4 together (the
  log-sum-exp's own tolerance is 2e-4), so an output element is off by at most
  (2^-11 + 4e-4) sum p|v| < 2^-10 sum p|v|.
* Probabilities times scale of less than 2^-14 are rounded to steps of 2^-24 in
  units of which the row's largest has at least 2^7: half a step is 2^-32 of it,
  and n keys of them, times codes of up to 448, add up to less than
  n 2^-23 max p * scale, where 448 scale is at most twice the largest |v| of a
  block: n 2^-30 max p max|v|.  Values of a tail row below 2^-17 of their scale are
  rounded too, half a step of 2^-24, below 2^-32 of the row's largest: inside
  the same term.
* The output is bf16: half a step, 2^-8 relative (below the least normal number
  half a step of 2^-133).

These bounds take every error at its worst and in one direction.  Errors of
different keys are independent, so a row as a whole is held to more: the rounding
of the sum to bf16 and an error of the log-sum-exp are at most 2^-8 + 2e-4 of
the row's norm, and sum_j e_j p_j v_j with independent |e_j| <= 2^-11 + 2e-4 has
a norm whose standard deviation is at most (2^-11 + 2e-4) sqrt(sum p^2 |v|^2); four
of them are allowed.
"""
import math

import torch


def attention(q, k, v, vis, scale):
    """q ``[B, Hq, Tq, D]``, k and v ``[B, Hkv, T, D]``, vis bool ``[B, Tq, T]``
    (any device): a dict of 64-bit tensors."""
    b, hq, tq, d = q.shape
    hkv, total = k.shape[1], k.shape[2]
    x = torch.einsum("bhgrd,bhkd->bhgrk", q.double().view(b, hkv, hq // hkv, tq, d), k.double()) * scale
    seen = vis[:, None, None].expand_as(x)
    x = torch.where(seen, x, torch.full((), -math.inf, dtype=torch.float64, device=x.device))
    lse = torch.logsumexp(x, -1) if total else x.sum(-1) - math.inf
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse).unsqueeze(-1))
    # Largest |v| of the keys that a row sees.
    top = v.double().abs().amax(-1) if total else v.double().sum(-1)
    vmax = torch.where(seen, top[:, :, None, None, :], torch.zeros((), dtype=torch.float64, device=x.device))
    rows = lambda t: t.reshape(b, hq, tq, *t.shape[4:])
    out = {
        "out": torch.einsum("bhgrk,bhkd->bhgrd", p, v.double()),
        "spread": torch.einsum("bhgrk,bhkd->bhgrd", p, v.double().abs()),
        "least": total * 2.0 ** -30 * p.amax(-1) * vmax.amax(-1) if total else lse * 0,
        "rms": torch.sqrt(torch.einsum("bhgrk,bhk->bhgr", p * p, v.double().square().sum(-1))),
        "lse": lse,
        "mass": p.sum((2, 3)),
    }
    return {n: t if n == "mass" else rows(t) for n, t in out.items()}


def off(out, want):
    """What breaks the bounds: None, or a text.  out ``[B, Tq, Hq, D]``."""
    got = out.double().transpose(1, 2).to(want["out"].device)
    o = want["out"]
    err = (got - o).abs()
    each = 2.0 ** -8 * o.abs() + 2.0 ** -10 * want["spread"] + want["least"].unsqueeze(-1) + 2.0 ** -134
    if not bool((err <= each).all()):
        return f"an element is off by {float((err / each).nan_to_num(math.inf).max()):.3g} times its bound"
    d = o.shape[-1]
    norm = ((2.0 ** -8 + 2e-4) * o.norm(dim=-1) + 4 * (2.0 ** -11 + 2e-4) * want["rms"]
            + math.sqrt(d) * (want["least"] + 2.0 ** -134))
    if not bool((err.norm(dim=-1) <= norm).all()):
        return f"a row is off by {float((err.norm(dim=-1) / norm).nan_to_num(math.inf).max()):.3g} times its bound"
    return None


def lse_off(lse, want):
    w = want["lse"]
    got = lse.double().to(w.device)
    empty = torch.isinf(w)
    if not torch.equal(empty, torch.isinf(got)):
        return "rows that see nothing"
    worst = float((got - w)[~empty].abs().max()) if bool((~empty).any()) else 0.0
    return None if worst <= 2e-4 else f"log-sum-exp off by {worst:.3g}"
