"""Work of the 8-bit KV cache: sealing, tree attention, attention mass, eviction.

Four operators over one cache of B requests and Hkv heads.  Keys and values
of the first ``sealed`` tokens are e4m3 codes with one power-of-two scale per
block of ``bt`` tokens and head; the rows after them (the open block and the
pass's own rows) are bf16, the tail.

* ``seal``       bf16 rows to codes and scales
* ``attention``  masked GQA attention over the cache, with its log-sum-exp
* ``mass``       attention weight that each cached token received, added up
* ``evict``      the heaviest tokens of each head kept, the cache compacted
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
DEV = "cuda"


def _case(name, op, **kw):
    base = {"op": op, "batch": 1, "hq": 32, "hkv": 4, "dim": 128, "block": 64, "rows": 1, "sealed": 0,
            "tail": 0, "mask": "tree", "empty": 0, "budget": 0, "sinks": 0, "recent": 0}
    base.update(kw)
    if name:
        base["name"] = name
    return base


def listed():
    return [
        # Decoding fills one block of the open tail every 64 tokens: the smallest seal.
        _case("seal_one_block", "seal", sealed=64),
        # The cache of a long prompt sealed after its prefill.
        _case("seal_prompt", "seal", sealed=32768),
        # One new token after a 512-token prompt: latency.
        _case("decode_short", "attention", sealed=512, tail=17, rows=1),
        # One new token over a long context: bandwidth.
        _case("decode_long", "attention", sealed=131072, tail=41, rows=1),
        # A small verification tree (seed + 7 nodes) over 4,096 tokens and more.
        _case("verify_tree_8", "attention", sealed=4096, tail=55, rows=8),
        # The 64-node verification tree over a 4,096-token context, one request and eight.
        _case("verify_tree_65", "attention", sealed=4096, tail=65, rows=65),
        _case("verify_batch_65", "attention", batch=8, sealed=4096, tail=65, rows=65),
        # A chunk of a long prompt behind what is cached already: the most arithmetic.
        _case("prefill_chunk", "attention", sealed=16384, tail=1007, rows=1000, mask="causal"),
        # The weights that one token's attention, and a tree's, gives a long context.
        _case("mass_decode", "mass", sealed=65536, tail=33, rows=1),
        _case("mass_tree_65", "mass", batch=8, sealed=4096, tail=65, rows=65),
        # A cache that grew a little over its budget; a long prompt cut to an eighth.
        _case("evict_some", "evict", sealed=4096, tail=63, budget=4000, sinks=4, recent=128),
        _case("evict_prompt", "evict", batch=4, sealed=65536, tail=21, budget=8192, sinks=16, recent=1024),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["seal", "attention", "attention", "attention", "mass", "evict"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 128])
    block = rng.choice([32, 64, 128])
    batch = rng.choice([1, 1, 2, 3, 8])
    # Tokens of all requests and heads together stay within the largest listed cache.
    tokens = _spread(rng, 1, max(2, 4 * 131072 // (batch * hkv)))
    c = _case("", op, batch=batch, hq=hkv * group, hkv=hkv, dim=dim, block=block)
    if op == "seal":
        c["sealed"] = max(block, min(tokens, 131072 // batch // hkv * 4) // block * block)
        return c
    tail = rng.randint(0, block + 70)
    c["tail"] = min(tail, tokens)
    c["sealed"] = (tokens - c["tail"]) // block * block
    if op == "evict":
        c["tail"] = max(1, c["tail"])
        total = c["sealed"] + c["tail"]
        c["budget"] = rng.randint(1, total)
        c["sinks"] = rng.randint(0, min(16, c["budget"]))
        c["recent"] = rng.randint(0, (c["budget"] - c["sinks"]))
        return c
    # Pairs of (query head row, key) stay within the largest listed case's.
    most = 32 * 1000 * 17000 // (batch * hkv * group * max(1, tokens))
    c["rows"] = _spread(rng, 1, max(1, min(1024, most)))
    c["mask"] = rng.choice(["tree", "causal", "any", "none"])
    if c["mask"] in ("tree", "causal"):
        # The pass's own rows are the last of the tail.
        c["rows"] = max(1, min(c["rows"], 1024))
        c["tail"] = max(c["tail"], c["rows"])
    elif c["sealed"] + c["tail"] == 0:
        c["tail"] = 1
    c["empty"] = rng.choice([0, 0, 1]) if c["mask"] != "none" else 0
    return c


# ---------------------------------------------------------------------------
# What a user's program holds before the call


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 11)


def _channel_rows(shape, gen, spread):
    """Rows whose channels differ in size, as normalised and rotated keys (and values) do."""
    gain = torch.exp(spread * torch.randn(shape[-1], generator=gen, device=DEV))
    return (torch.randn(shape, generator=gen, device=DEV) * gain).to(torch.bfloat16)


def _seal_plain(x, block):
    b, h, n, d = x.shape
    blocks = x.float().view(b, h, n // block, block * d)
    top = blocks.abs().amax(-1)
    frac, power = torch.frexp(top)
    # 448 = 0.875 * 2^9: the least power of two that brings the block within e4m3's range.
    power = torch.where(frac > 0.875, power - 8, power - 9).clamp(min=-100)
    power = torch.where(top == 0, torch.full_like(power, -100), power)
    scale = ((power + 127).to(torch.int32) << 23).view(torch.float32)  # 2^power, exactly
    codes = (blocks / scale.unsqueeze(-1)).to(E4M3).view(b, h, n, d)
    return codes, scale


def _visible(case, gen):
    """bool [batch, rows, columns] of the masked columns (all from prefix on), and the prefix."""
    b, rows, total = case["batch"], case["rows"], case["sealed"] + case["tail"]
    kind = case["mask"]
    if kind == "none":
        return None, total
    if kind == "any":
        vis = torch.rand(b, rows, total, generator=gen, device=DEV) < 0.6
        prefix = 0
    elif kind == "causal":
        vis = torch.ones(rows, rows, dtype=torch.bool, device=DEV).tril().expand(b, rows, rows).clone()
        prefix = total - rows
    else:
        # A random tree in which every node's parent comes before it: ancestors are the
        # powers of the parent matrix, squared until they reach every depth.
        up = torch.rand(b, rows, generator=gen, device=DEV) * torch.arange(rows, device=DEV)
        grid = torch.eye(rows, device=DEV).expand(b, rows, rows).clone()
        grid.scatter_(2, up.floor().long().unsqueeze(-1), 1.0)
        for _ in range(max(1, rows).bit_length()):
            grid = (torch.matmul(grid, grid) > 0).float()
        vis, prefix = grid.bool(), total - rows
    if case["empty"]:
        # The last row is padding: it sees nothing (its prefix is masked by bits too).
        if prefix:
            vis = torch.cat([torch.ones(b, rows, prefix, dtype=torch.bool, device=DEV), vis], -1)
            prefix = 0
        vis[:, -1] = False
    return vis, prefix


def _pack(vis):
    b, rows, cols = vis.shape
    words = (cols + 31) // 32
    wide = torch.zeros(b, rows, words * 32, dtype=torch.int64, device=DEV)
    wide[..., :cols] = vis
    out = (wide.view(b, rows, words, 32) << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32).contiguous()


def prepare(case, seed):
    gen = _generator(seed)
    b, hq, hkv, d, block = case["batch"], case["hq"], case["hkv"], case["dim"], case["block"]
    sealed, tail = case["sealed"], case["tail"]
    s = {"case": dict(case)}
    k = _channel_rows((b, hkv, sealed, d), gen, 0.5)
    v = _channel_rows((b, hkv, sealed, d), gen, 0.3)
    if case["op"] == "seal":
        s["k"], s["v"] = k, v
        s["k_codes"] = torch.zeros(b, hkv, sealed, d, dtype=E4M3, device=DEV)
        s["v_codes"] = torch.zeros_like(s["k_codes"])
        s["k_scale"] = torch.zeros(b, hkv, sealed // block, device=DEV)
        s["v_scale"] = torch.zeros_like(s["k_scale"])
        return s
    s["k_codes"], s["k_scale"] = _seal_plain(k, block)
    s["v_codes"], s["v_scale"] = _seal_plain(v, block)
    del k, v
    s["k_tail"] = _channel_rows((b, hkv, tail, d), gen, 0.5)
    s["v_tail"] = _channel_rows((b, hkv, tail, d), gen, 0.3)
    total = sealed + tail
    if case["op"] == "evict":
        # Most tokens received little weight, many none at all: ties.
        m = torch.exp(2.0 * torch.randn(b, hkv, total, generator=gen, device=DEV))
        m = torch.where(torch.rand(b, hkv, total, generator=gen, device=DEV) < 0.25, torch.zeros_like(m), m)
        s["mass"] = m
        return s
    s["q"] = _channel_rows((b, hq, case["rows"], d), gen, 0.3)
    vis, s["prefix"] = _visible(case, gen)
    s["bits"] = None if vis is None else _pack(vis)
    s["scale"] = d ** -0.5
    if case["op"] == "mass":
        # What the attention call before it returned, and what earlier passes added up.
        s["lse"] = _attend(s, values=False)["lse"]
        s["mass"] = torch.rand(b, hkv, total, generator=gen, device=DEV) * case["rows"]
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _open(codes, scale, tail):
    """The rows that the cache stands for, in 32 bits."""
    b, h, n, d = codes.shape
    block = n // scale.shape[2] if n else 1
    rows = codes.float().view(b, h, -1, block * d) * scale.unsqueeze(-1) if n else codes.float()
    return torch.cat([rows.view(b, h, n, d), tail.float()], 2)


def _mask(s, total):
    """bool [batch, 1, rows, total] from the packed words."""
    c = s["case"]
    if s["bits"] is None:
        return torch.ones(1, 1, 1, total, dtype=torch.bool, device=DEV)
    cols = torch.arange(total - s["prefix"], device=DEV)
    on = ((s["bits"][..., cols // 32] >> (cols % 32)) & 1).bool()
    front = torch.ones(c["batch"], c["rows"], s["prefix"], dtype=torch.bool, device=DEV)
    return torch.cat([front, on], -1).unsqueeze(1)


def _scores(s, k):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    b, rows, d, total = c["batch"], c["rows"], c["dim"], k.shape[2]
    q = s["q"].float().reshape(b, c["hkv"], group * rows, d)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    x = x.view(b, c["hq"], rows, total)
    return x.masked_fill_(~_mask(s, total), -math.inf)


def _attend(s, values=True):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    k = _open(s["k_codes"], s["k_scale"], s["k_tail"])
    x = _scores(s, k)
    del k
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    if not values:
        return {"lse": lse}
    v = _open(s["v_codes"], s["v_scale"], s["v_tail"])
    b, rows, d = c["batch"], c["rows"], c["dim"]
    o = torch.matmul(x.view(b, c["hkv"], group * rows, -1), v).view(b, c["hq"], rows, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return {"out": o.transpose(1, 2).to(torch.bfloat16), "lse": lse}


def _mass(s):
    c = s["case"]
    k = _open(s["k_codes"], s["k_scale"], s["k_tail"])
    x = _scores(s, k)
    low = s["lse"].unsqueeze(-1)
    x = torch.where(low == -math.inf, torch.zeros_like(x), (x - low).exp_())
    group = c["hq"] // c["hkv"]
    got = x.view(c["batch"], c["hkv"], group * c["rows"], -1).sum(2)
    return {"mass": s["mass"] + got}


def _evict(s):
    c = s["case"]
    total, budget, sinks, recent = c["sealed"] + c["tail"], c["budget"], c["sinks"], c["recent"]
    key = s["mass"].clone()
    key[..., :sinks] = math.inf
    key[..., total - recent:] = math.inf
    # Among equal weights the earlier token stays: a stable sort.
    keep = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.sort(keep, dim=-1).values
    k = _open(s["k_codes"], s["k_scale"], s["k_tail"])
    v = _open(s["v_codes"], s["v_scale"], s["v_tail"])
    at = keep.unsqueeze(-1).expand(-1, -1, -1, c["dim"])
    k, v = k.gather(2, at).to(torch.bfloat16), v.gather(2, at).to(torch.bfloat16)
    full = budget // c["block"] * c["block"]
    kc, ks = _seal_plain(k[:, :, :full], c["block"])
    vc, vs = _seal_plain(v[:, :, :full], c["block"])
    return {"keep": keep.to(torch.int32), "k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs,
            "k_tail": k[:, :, full:].contiguous(), "v_tail": v[:, :, full:].contiguous(),
            "mass": s["mass"].gather(2, keep)}


def _seal(s):
    kc, ks = _seal_plain(s["k"], s["case"]["block"])
    vc, vs = _seal_plain(s["v"], s["case"]["block"])
    return {"k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs}


# ---------------------------------------------------------------------------
# One pass


def run(s):
    op = s["case"]["op"]
    if own:
        return _run_own(s, op)
    if op == "seal":
        return _seal(s)
    if op == "attention":
        return _attend(s)
    if op == "mass":
        return _mass(s)
    return _evict(s)


def _run_own(s, op):
    from specfit_b200 import ops

    c = s["case"]
    if op == "seal":
        ops.kv8_seal(s["k"], s["v"], s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        return {n: s[n] for n in ("k_codes", "v_codes", "k_scale", "v_scale")}
    rows = ops.Kv8Rows(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], c["sealed"], s["k_tail"],
                       s["v_tail"], c["block"])
    if op == "attention":
        out, lse = ops.kv8_tree_attention(s["q"], rows, s["bits"], s["prefix"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "mass":
        mass = s["mass"].clone()
        ops.kv8_attention_mass(s["q"], s["lse"], rows, s["bits"], s["prefix"], mass, scale=s["scale"])
        return {"mass": mass}
    keep = ops.kv_keep_heaviest(s["mass"], c["sealed"] + c["tail"], c["budget"], sinks=c["sinks"],
                                recent=c["recent"])
    new, mass = ops.kv8_compact(rows, keep, mass=s["mass"])
    return {"keep": keep, "k_codes": new.k_codes, "v_codes": new.v_codes, "k_scale": new.k_scale,
            "v_scale": new.v_scale, "k_tail": new.k_tail, "v_tail": new.v_tail, "mass": mass}


# ---------------------------------------------------------------------------
# What a pass cannot do without


def _pairs(case):
    """(query row, key) pairs of one request and head that are visible."""
    rows, total = case["rows"], case["sealed"] + case["tail"]
    kind = case["mask"]
    if kind == "none":
        return rows * total
    if kind == "any":
        return 0.6 * rows * total
    inside = rows * (rows + 1) / 2 if kind == "causal" else rows * (1 + math.log(rows))
    return rows * (total - rows) + inside


def work(case):
    b, hq, hkv, d, block = case["batch"], case["hq"], case["hkv"], case["dim"], case["block"]
    heads, sealed, tail, rows = b * hkv, case["sealed"], case["tail"], case["rows"]
    if case["op"] == "seal":
        return {"bytes": 2 * heads * sealed * (3 * d) + 8 * heads * sealed // block, "flops": 0}
    one = heads * (sealed * d + 4 * sealed // block + 2 * tail * d)  # K or V of the cache
    if case["op"] == "evict":
        n = case["budget"]
        full = n // block * block
        new = heads * (full * d + 4 * full // block + 2 * (n - full) * d)
        read = 2 * heads * n * d  # kept rows, 8 bits each
        return {"bytes": 4 * heads * (sealed + tail) + 4 * heads * n + read + 2 * new + 4 * heads * n, "flops": 0}
    masked = 0 if case["mask"] == "none" else b * rows * ((rows if case["mask"] != "any" else sealed + tail) / 8)
    q = 2 * b * hq * rows * d
    if case["op"] == "mass":
        return {"bytes": one + q + 4 * b * hq * rows + masked + 8 * heads * (sealed + tail),
                "flops": 2 * d * b * hq * _pairs(case)}
    return {"bytes": 2 * one + 2 * q + 4 * b * hq * rows + masked, "flops": 4 * d * b * hq * _pairs(case)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits, apart from the above


def _exact_rows(codes, scale, tail, block):
    wide = torch.repeat_interleave(scale.double(), block, dim=2)
    return torch.cat((codes.to(torch.float64) * wide[..., None], tail.to(torch.float64)), dim=2)


def _exact_seal(x, block):
    b, h, n, d = x.shape
    y = x.double().reshape(b, h, n // block, block, d)
    top = y.abs().amax((3, 4))
    # 2^i, exactly, for the integers -110 .. 130.
    twos = ((torch.arange(-110, 131, device=DEV) + 1023) << 52).view(torch.float64)
    e = torch.searchsorted(448.0 * twos, top.reshape(-1)).clamp(min=10)  # the first that is not below
    scale = twos[e].reshape(top.shape)
    z = y / scale[:, :, :, None, None]
    # e4m3: three bits of fraction down to 2^-6, steps of 2^-9 below; ties to even.
    step = torch.frexp(z.abs().clamp(min=2.0 ** -6)).exponent.long() - 4  # |z| = f * 2^exponent, f in [1/2, 1)
    step = ((step + 1023) << 52).view(torch.float64)
    return (torch.round(z / step) * step).reshape(b, h, n, d), scale


def exact(case, seed):
    s = prepare(case, seed)
    b, hq, hkv, d, rows = case["batch"], case["hq"], case["hkv"], case["dim"], case["rows"]
    block = case["block"]
    if case["op"] == "seal":
        kc, ks = _exact_seal(s["k"], block)
        vc, vs = _exact_seal(s["v"], block)
        return {"k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs}
    k = _exact_rows(s["k_codes"], s["k_scale"], s["k_tail"], block)
    v = _exact_rows(s["v_codes"], s["v_scale"], s["v_tail"], block)
    total = k.shape[2]
    if case["op"] == "evict":
        n = case["budget"]
        m = s["mass"].double().cpu()
        keep = torch.zeros(b, hkv, n, dtype=torch.long)
        index = torch.arange(total)
        always = (index < case["sinks"]) | (index >= total - case["recent"])
        for i in range(b):
            for h in range(hkv):
                rank = sorted(range(total), key=lambda j: (not bool(always[j]), -m[i, h, j].item(), j)) \
                    if total <= 512 else None
                if rank is None:
                    import numpy as np
                    rank = np.lexsort((index.numpy(), -m[i, h].numpy(), ~always.numpy())).tolist()
                keep[i, h] = torch.tensor(sorted(rank[:n]))
        keep = keep.to(DEV)
        pick = keep[..., None].expand(b, hkv, n, d)
        k, v = k.gather(2, pick), v.gather(2, pick)
        full = n - n % block
        kc, ks = _exact_seal(k[:, :, :full], block)
        vc, vs = _exact_seal(v[:, :, :full], block)
        return {"keep": None, "k_codes": kc, "v_codes": vc, "k_scale": ks, "v_scale": vs,
                "k_tail": k[:, :, full:], "v_tail": v[:, :, full:], "mass": s["mass"].double().gather(2, keep)}
    q = s["q"].double().view(b, hkv, hq // hkv, rows, d)
    bits = s["bits"]
    seen = torch.ones(b, rows, total, dtype=torch.bool, device=DEV)
    if bits is not None:
        lanes = torch.arange(32, device=DEV)
        flat = ((bits.long()[..., None] >> lanes) & 1).reshape(b, rows, -1)
        seen[:, :, s["prefix"]:] = flat[:, :, : total - s["prefix"]] == 1
    x = torch.einsum("bhgrd,bhkd->bhgrk", q, k) * s["scale"]
    x = torch.where(seen[:, None, None], x, torch.tensor(-math.inf, dtype=torch.float64, device=DEV))
    if case["op"] == "mass":
        w = torch.exp(x - s["lse"].double().view(b, hkv, -1, rows)[..., None])
        w = torch.where(seen[:, None, None], w, torch.zeros((), dtype=torch.float64, device=DEV))
        return {"mass": s["mass"].double() + w.sum((2, 3))}
    lse = torch.logsumexp(x, -1)
    w = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    o = torch.einsum("bhgrk,bhkd->brhgd", w, v)
    return {"out": o.reshape(b, rows, hq, d), "lse": lse.reshape(b, hq, rows)}
