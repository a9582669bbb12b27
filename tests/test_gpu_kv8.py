"""The 8-bit KV cache's operators on a GPU against 64-bit plain ones
(``kv8_reference``).

Tolerances, derived before the first run:

* codes, scales, rows read back, kept indices: exact.
* attention output: bf16, so half a step, 2^-8 relative, of the result; before
  it each probability is rounded to fp16 or bf16 (at most 2^-9 relative) and
  its product summed, so the sum is off by at most 2^-9 * sum p|v| <= 2^-9 *
  max|v|; fp32 sums add less than 2^-16 of the same.  Together |err| <=
  2^-8 |o| + 2^-8 max|v|.
* log-sum-exp: scores are fp32 sums of exact products.  A sum of D = 128 terms
  with |q|, |k| as drawn has partial sums below 64 after scaling, so an fp32
  (or a tensor core's, at least 22 bits) accumulation is off by at most
  128 * 2^-22 * 64 < 2^-9; the exponential sum adds 2^-20.  Typical errors
  grow with the square root: 2e-4 is asked for.
* mass: each weight is exp(s - lse), relative error that of s and lse: 4e-4.
"""
import ctypes
import math

import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from specfit_b200 import ops as _ops

    return _ops


def make_rows(ops, b, hkv, d, block, sealed, tail, seed, room=0, k_size=0.5, v_size=0.7):
    """A cache with its bf16 origin sealed by the reference (buffers with
    ``room`` spare tokens, the tail a view of a larger buffer)."""
    g = torch.Generator().manual_seed(seed)
    def rows(n, size):
        gain = torch.exp(size * torch.randn(d, generator=g))
        return (torch.randn(b, hkv, n, d, generator=g) * gain).to(torch.bfloat16)
    parts = []
    for size in (k_size, v_size):
        x = rows(sealed, size)
        # Blocks of quite different magnitudes, and a block of zeros.
        mult = 2.0 ** torch.randint(-3, 4, (b, hkv, max(1, sealed // block)), generator=g)
        if sealed >= 4 * block:
            mult[:, :, 2] = 0.0
        if sealed:
            x = (x.float() * mult.repeat_interleave(block, 2).unsqueeze(-1)).to(torch.bfloat16) if size == v_size else x
        codes, scale = ref.seal(x, block)
        cb = torch.full((b, hkv, sealed + room, d), 3.0).to(ref.E4M3)
        cb[:, :, :sealed] = codes.float().to(ref.E4M3)
        sb = torch.ones(b, hkv, (sealed + room) // block)
        sb[:, :, : sealed // block] = scale.float()
        tb = torch.full((b, hkv, tail + 3, d), 9.0).to(torch.bfloat16)
        tb[:, :, :tail] = rows(tail, size)
        parts.append((cb.to(DEV), sb.to(DEV), tb.to(DEV)[:, :, :tail]))
    (kc, ks, kt), (vc, vs, vt) = parts
    return ops.Kv8Rows(kc, vc, ks, vs, sealed, kt, vt, block)


def opened(rows):
    return (ref.open_rows(rows.k_codes, rows.k_scale, rows.sealed, rows.k_tail, rows.block),
            ref.open_rows(rows.v_codes, rows.v_scale, rows.sealed, rows.v_tail, rows.block))


def pack(vis):
    b, r, n = vis.shape
    words = max(1, (n + 31) // 32)
    w = torch.zeros(b, r, words * 32, dtype=torch.int64)
    w[..., :n] = vis.long()
    x = (w.view(b, r, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def queries(b, hq, rows, d, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    return torch.randn(b, hq, rows, d, generator=g).to(torch.bfloat16).to(DEV)


def masks(kind, b, rows, total, seed):
    """(bits on the GPU or None, prefix, visibility)."""
    g = torch.Generator().manual_seed(seed + 2000)
    if kind == "none":
        return None, total, torch.ones(b, rows, total, dtype=torch.bool)
    if kind == "any":
        vis = torch.rand(b, rows, total, generator=g) < 0.5
        vis[:, rows // 2] = False  # a row that sees nothing
        return pack(vis).to(DEV), 0, vis
    vis = torch.ones(rows, rows, dtype=torch.bool).tril().expand(b, rows, rows).clone()
    if kind == "tree":
        vis = torch.zeros(b, rows, rows, dtype=torch.bool)
        for i in range(rows):
            if i:
                p = int(torch.randint(0, i, (1,), generator=g))
                vis[:, i] = vis[:, p]
            vis[:, i, i] = True
    full = torch.ones(b, rows, total, dtype=torch.bool)
    full[:, :, total - rows:] = vis
    return pack(vis).to(DEV), total - rows, full


def check_attention(out, lse, want, wlse, vmax):
    out, lse = out.double().cpu(), lse.double().cpu()
    off = (out - want).abs()
    assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * vmax).all()), float(off.max())
    empty = torch.isinf(wlse)
    assert torch.equal(empty, torch.isinf(lse))
    assert float((lse - wlse)[~empty].abs().max()) <= 2e-4 if (~empty).any() else True


# ------------------------------------------------------------------ sealing


@pytest.mark.parametrize("b,hkv,d,block,blocks", [(1, 4, 128, 64, 1), (2, 3, 64, 32, 5), (1, 1, 16, 128, 2),
                                                  (1, 2, 112, 128, 3), (3, 1, 80, 32, 1)])
def test_seal_matches_the_definition(ops, b, hkv, d, block, blocks):
    g = torch.Generator().manual_seed(7 * d + blocks)
    x = torch.randn(2, b, hkv, blocks * block, d, generator=g)
    x = (x * torch.exp(2 * torch.randn(2, b, hkv, blocks * block, 1, generator=g))).to(torch.bfloat16)
    x[0, 0, 0, :block] = 0                       # a block of zeros
    x[1, 0, 0, 0, 0], x[1, 0, 0, 0, 1] = 448.0 * 4, 3.389e38 * 0.5  # far apart in one block
    if blocks > 1:
        x[0, 0, 0, block + 1, 3] = float("nan")
        x[1, 0, 0, block + 2, 5] = float("-inf")
        x[0, 0, -1, -block:] *= 1e-38            # below the smallest scale
    cap = (blocks + 2) * block
    codes = torch.full((2, b, hkv, cap, d), 5.0).to(ref.E4M3).to(DEV)
    scale = torch.full((2, b, hkv, blocks + 2), 5.0, device=DEV)
    xd = x.to(DEV)
    ops.kv8_seal(xd[0], xd[1], codes[0], codes[1], scale[0], scale[1], first_block=1)
    for i in range(2):
        want, wscale = ref.seal(x[i], block)
        got, gscale = codes[i].cpu().double(), scale[i].cpu().double()
        assert torch.equal(torch.nan_to_num(gscale[:, :, 1:-1], nan=-1.0), torch.nan_to_num(wscale, nan=-1.0))
        assert torch.equal(got[:, :, block:-block], want)
        # What lies around the sealed blocks is as it was.
        assert bool((got[:, :, :block] == 5).all()) and bool((got[:, :, -block:] == 5).all())
        assert bool((gscale[:, :, 0] == 5).all()) and bool((gscale[:, :, -1] == 5).all())


def test_seal_takes_strided_rows_and_is_idempotent(ops):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(2, 128, 3, 64, generator=g).to(torch.bfloat16).to(DEV)  # token-major rows
    k = wide.permute(0, 2, 1, 3)
    kc = torch.zeros(2, 3, 128, 64, device=DEV).to(ref.E4M3)
    ks = torch.zeros(2, 3, 4, device=DEV)
    vc, vs = torch.zeros_like(kc), torch.zeros_like(ks)
    ops.kv8_seal(k, k, kc, vc, ks, vs)
    want, wscale = ref.seal(k.cpu(), 32)
    assert torch.equal(kc.cpu().double(), want) and torch.equal(ks.cpu().double(), wscale)
    none = torch.zeros(2, 3, 0, 64, dtype=torch.bfloat16, device=DEV)
    rows = ops.Kv8Rows(kc, vc, ks, vs, 128, none, none, 32)
    back, _ = ops.kv8_read(rows)
    assert torch.equal(back.cpu().double(), want * wscale.repeat_interleave(32, 2).unsqueeze(-1))
    ops.kv8_seal(back, back, kc, vc, ks, vs)
    again, _ = ops.kv8_read(rows)
    assert torch.equal(again, back)


def test_read_ranges(ops):
    rows = make_rows(ops, 2, 2, 48, 32, 96, 11, 5, room=32)
    k, v = opened(rows)
    for first, count in ((0, 107), (0, 0), (90, 17), (96, 11), (106, 1), (31, 2)):
        gk, gv = ops.kv8_read(rows, first, count)
        assert torch.equal(gk.cpu().double(), k[:, :, first:first + count])
        assert torch.equal(gv.cpu().double(), v[:, :, first:first + count])


# ---------------------------------------------------------------- attention

ATTENTION = [
    # b, hq, hkv, d, block, sealed, tail, rows, mask
    (1, 32, 4, 128, 64, 512, 17, 1, "tree"),
    (1, 32, 4, 128, 64, 0, 1, 1, "causal"),
    (1, 32, 4, 128, 64, 64, 0, 1, "none"),
    (2, 8, 8, 64, 32, 32, 5, 3, "causal"),
    (1, 5, 1, 128, 128, 256, 40, 7, "tree"),
    (3, 16, 2, 128, 32, 352, 70, 33, "any"),
    (1, 8, 1, 128, 64, 640, 65, 65, "tree"),
    (2, 16, 2, 128, 64, 1024, 66, 65, "tree"),
    (1, 4, 2, 16, 32, 96, 9, 4, "any"),
    (1, 6, 2, 48, 64, 128, 31, 5, "causal"),
    (1, 8, 2, 112, 128, 128, 130, 20, "any"),
    (1, 8, 2, 128, 64, 192, 200, 150, "causal"),
    (1, 8, 1, 128, 64, 0, 300, 257, "causal"),
    (1, 16, 1, 128, 32, 2080, 17, 16, "any"),
    # At most eight query rows for a KV head.
    (2, 4, 2, 112, 32, 288, 45, 4, "any"),
    (1, 3, 1, 64, 64, 640, 70, 2, "tree"),
    (2, 7, 7, 128, 128, 512, 33, 7, "causal"),
    # No tail, and codes that end inside a block of 128 keys.
    (2, 16, 2, 128, 32, 96, 0, 65, "any"),
    (1, 8, 1, 128, 64, 704, 0, 130, "any"),
]


@pytest.mark.parametrize("b,hq,hkv,d,block,sealed,tail,rows,mask", ATTENTION)
def test_attention_and_mass(ops, b, hq, hkv, d, block, sealed, tail, rows, mask):
    seed = hq + d + sealed + rows
    cache = make_rows(ops, b, hkv, d, block, sealed, tail, seed, room=block)
    k, v = opened(cache)
    q = queries(b, hq, rows, d, seed)
    bits, prefix, vis = masks(mask, b, rows, sealed + tail, seed)
    out, lse = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
    want, wlse = ref.attention(q, k, v, vis, d ** -0.5)
    check_attention(out, lse, want, wlse, float(v.abs().max()))
    before = torch.rand(b, hkv, sealed + tail + 5, device=DEV)
    got = ops.kv8_attention_mass(q, lse, cache, bits, prefix, before.clone())
    wmass = ref.mass(q, wlse, k, vis, d ** -0.5)
    add = (got - before).double().cpu()
    assert torch.equal(got[..., sealed + tail:], before[..., sealed + tail:])
    # The sum is rounded into `before`: half a step of the sum, below 2^-24 * (1 + mass).
    assert bool(((add[..., : sealed + tail] - wmass).abs() <= 4e-4 * wmass + 2.0 ** -22 * (1 + wmass)).all())
    # The same call, the same bits.
    out2, lse2 = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    assert torch.equal(got, ops.kv8_attention_mass(q, lse, cache, bits, prefix, before.clone()))


def _long(ops, b, hkv, d, block, sealed, tail, seed):
    """A long cache, made on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = [(torch.randn(b, hkv, sealed, d, generator=g, device=DEV) * 60).to(ref.E4M3) for _ in range(2)]
    scale = [torch.full((b, hkv, sealed // block), 2.0 ** -6, device=DEV) for _ in range(2)]
    scale[1][:, :, ::3] = 2.0 ** -4
    tails = [torch.randn(b, hkv, tail, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    return ops.Kv8Rows(codes[0], codes[1], scale[0], scale[1], sealed, tails[0], tails[1], block)


@pytest.mark.parametrize("b,hq,hkv,d,rows,sealed,tail", [(1, 32, 4, 128, 1, 65536, 33), (1, 16, 2, 128, 65, 8192, 65),
                                                         (1, 16, 2, 128, 40, 4096, 40), (2, 16, 2, 64, 20, 8192, 20),
                                                         (1, 8, 1, 128, 300, 4096, 300),
                                                         (2, 16, 4, 128, 65, 8192, 97),
                                                         (2, 8, 2, 128, 180, 12288, 200)])
def test_attention_over_long_caches(ops, b, hq, hkv, d, rows, sealed, tail):
    cache = _long(ops, b, hkv, d, 64, sealed, tail, rows)
    q = queries(b, hq, rows, d, rows)
    bits, prefix, vis = masks("tree" if rows > 1 else "none", b, rows, sealed + tail, rows)
    out, lse = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
    k, v = opened(cache)
    k, v = k.to(DEV), v.to(DEV)
    qd = q.double().view(b, hkv, hq // hkv, rows, d)
    s = torch.einsum("bhgrd,bhkd->bhgrk", qd, k) * d ** -0.5
    s = s.masked_fill(~vis.to(DEV)[:, None, None], -math.inf)
    wlse = torch.logsumexp(s, -1)
    w = torch.exp(s - wlse.unsqueeze(-1))
    want = torch.einsum("bhgrk,bhkd->brhgd", w, v).reshape(b, rows, hq, d)
    check_attention(out, lse, want.cpu(), wlse.reshape(b, hq, rows).cpu(), float(v.abs().max()))
    mass = ops.kv8_attention_mass(q, lse, cache, bits, prefix, torch.zeros(b, hkv, sealed + tail, device=DEV))
    wmass = w.sum((2, 3))
    assert bool(((mass.double() - wmass).abs() <= 4e-4 * wmass + 1e-12).all())
    # Every row's weights sum to one.
    assert abs(float(mass.double().sum()) / (b * hq * rows) - 1) < 1e-4


@pytest.mark.parametrize("rows,hq", [(2, 8), (70, 8), (8, 1)])
def test_masked_garbage_stays_out(ops, rows, hq):
    """NaN and infinities in keys and values that a row does not see change
    nothing for it; rows that see them answer NaN."""
    b, hkv, d, block, sealed, tail = 1, 1, 128, 64, 256, 96
    cache = make_rows(ops, b, hkv, d, block, sealed, tail, 5)
    k, v = opened(cache)
    cache.k_scale[0, 0, 1] = math.nan       # a sealed block that held a NaN key
    cache.v_scale[0, 0, 2] = math.nan       # ... and one with a NaN value
    cache.k_tail[0, 0, 3, 7] = math.nan
    cache.k_tail[0, 0, 4, 0] = math.inf
    cache.v_tail[0, 0, 5, 1] = math.nan
    cache.v_tail[0, 0, 6, 100] = -math.inf
    total = sealed + tail
    vis = torch.ones(b, rows, total, dtype=torch.bool)
    garbage = torch.zeros(total, dtype=torch.bool)
    garbage[block:3 * block] = True
    garbage[sealed + 3:sealed + 7] = True
    vis[:, :, garbage] = False
    vis[:, 0, sealed + 5] = True            # this row sees a NaN value
    q = queries(b, hq, rows, d, 5)
    out, lse = ops.kv8_tree_attention(q, cache, pack(vis).to(DEV), 0, return_lse=True)
    want, wlse = ref.attention(q, k, v, vis, d ** -0.5)
    assert bool(torch.isnan(out[:, 0]).all()) and bool(torch.isnan(lse[:, :, 0]).all())
    check_attention(out[:, 1:], lse[:, :, 1:], want[:, 1:], wlse[:, :, 1:], float(v.abs().max()))
    vis[:, 0, sealed + 5] = False
    out, lse = ops.kv8_tree_attention(q, cache, pack(vis).to(DEV), 0, return_lse=True)
    mass = ops.kv8_attention_mass(q, lse, cache, pack(vis).to(DEV), 0, torch.zeros(b, hkv, total, device=DEV))
    assert bool(torch.isfinite(mass).all()) and float(mass[..., garbage.to(DEV)].abs().max()) == 0
    # One sealed block's keys, then its values, seen by one row each.
    for blk in (1, 2):
        on = vis.clone()
        on[:, 1, blk * block] = True
        o, l = ops.kv8_tree_attention(q, cache, pack(on).to(DEV), 0, return_lse=True)
        assert bool(torch.isnan(o[:, 1]).all())
        assert torch.equal(o[:, 0], out[:, 0]) and bool(torch.isfinite(o[:, 2:]).all())


def test_every_row_empty(ops):
    cache = make_rows(ops, 2, 2, 64, 32, 64, 5, 8)
    q = queries(2, 4, 3, 64, 8)
    bits = torch.zeros(2, 3, 3, dtype=torch.int32, device=DEV)
    out, lse = ops.kv8_tree_attention(q, cache, bits, 0, return_lse=True)
    assert float(out.abs().max()) == 0 and bool((lse == -math.inf).all())
    mass = ops.kv8_attention_mass(q, lse, cache, bits, 0, torch.zeros(2, 2, 69, device=DEV))
    assert float(mass.abs().max()) == 0


def test_large_scores_and_extreme_queries(ops):
    """Scores far from zero, and query rows of very different sizes."""
    cache = make_rows(ops, 1, 1, 128, 64, 256, 20, 9)
    k, v = opened(cache)
    q = queries(1, 8, 4, 128, 9)
    q[:, 1] *= 2.0 ** 6
    q[:, 2] *= 2.0 ** -40
    q[:, 3] = 0
    q[:, 4, :, ::2] *= 2.0 ** -20
    out, lse = ops.kv8_tree_attention(q, cache, None, 276, return_lse=True)
    want, wlse = ref.attention(q, k, v, torch.ones(1, 4, 276, dtype=torch.bool), 128 ** -0.5)
    # Head 1's scores are 2^6 times larger: its softmax is a few keys' and the
    # score error 2^6 times larger too (relative 2^-18 of |s| < 2^11).
    small = [0, 2, 3, 4, 5, 6, 7]
    check_attention(out[:, :, small], lse[:, small], want[:, :, small], wlse[:, small], float(v.abs().max()))
    assert float((lse.double().cpu() - wlse)[:, 1].abs().max()) <= 2e-2
    assert float((out.double().cpu() - want)[:, :, 1].abs().max()) <= 2.0 ** -5 * float(v.abs().max())


def test_strided_inputs(ops):
    """q as a view of [B, T, Hq, D], a padded cache, bits of a wider buffer, out given."""
    cache = make_rows(ops, 2, 2, 128, 64, 128, 9, 4, room=192)
    k, v = opened(cache)
    q = queries(2, 8, 9, 128, 4).transpose(1, 2).contiguous().transpose(1, 2)
    assert not q.is_contiguous()
    bits, prefix, vis = masks("tree", 2, 9, 137, 4)
    wide = torch.zeros(4, 9, bits.shape[2], dtype=torch.int32, device=DEV)
    wide[::2] = bits
    out = torch.empty(4, 9, 8, 128, dtype=torch.bfloat16, device=DEV)
    res, lse = ops.kv8_tree_attention(q, cache, wide[::2], prefix, out=out[::2], return_lse=True)
    want, wlse = ref.attention(q, k, v, vis, 128 ** -0.5)
    check_attention(out[::2], lse, want, wlse, float(v.abs().max()))


# ----------------------------------------------------------------- eviction


@pytest.mark.parametrize("b,h,length,budget,sinks,recent", [
    (1, 1, 1, 1, 0, 0), (1, 1, 7, 3, 1, 1), (2, 3, 100, 40, 4, 8), (1, 2, 2048, 1000, 0, 0), (1, 1, 2049, 1, 0, 0),
    (2, 1, 5000, 4999, 3, 3), (1, 2, 20000, 777, 16, 100), (1, 1, 70001, 8192, 4, 1024), (1, 1, 64, 12, 4, 8),
    (1, 2, 50, 50, 0, 0), (1, 1, 33, 0, 0, 0)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_keep_heaviest(ops, b, h, length, budget, sinks, recent, kind):
    g = torch.Generator().manual_seed(length + budget)
    m = torch.exp(2 * torch.randn(b, h, length + 9, generator=g))
    if kind == "ties":
        m = torch.round(m)
    if kind == "odd":
        pick = torch.rand(m.shape, generator=g)
        m[pick < 0.1] = math.nan
        m[(pick >= 0.1) & (pick < 0.2)] = 0.0
        m[(pick >= 0.2) & (pick < 0.3)] = -0.0
        m[(pick >= 0.3) & (pick < 0.4)] *= -1
        m[(pick >= 0.4) & (pick < 0.45)] = math.inf
        m[(pick >= 0.45) & (pick < 0.5)] = -math.inf
    got = ops.kv_keep_heaviest(m.to(DEV), length, budget, sinks=sinks, recent=recent)
    assert torch.equal(got.cpu(), ref.keep_heaviest(m, length, budget, sinks, recent))


@pytest.mark.parametrize("b,hkv,d,block,sealed,tail,n", [(1, 4, 128, 64, 512, 30, 200), (2, 2, 64, 32, 96, 7, 31),
                                                         (1, 1, 16, 128, 256, 1, 256), (1, 2, 112, 32, 0, 20, 5),
                                                         (2, 1, 128, 64, 128, 0, 128)])
def test_compact(ops, b, hkv, d, block, sealed, tail, n):
    rows = make_rows(ops, b, hkv, d, block, sealed, tail, n, room=block)
    g = torch.Generator().manual_seed(n)
    keep = torch.stack([torch.stack([torch.randperm(sealed + tail, generator=g)[:n].sort().values
                                     for _ in range(hkv)]) for _ in range(b)]).to(torch.int32).to(DEV)
    mass = torch.rand(b, hkv, sealed + tail + 4, device=DEV)
    new, nm = ops.kv8_compact(rows, keep, mass=mass)
    assert new.length == n and new.sealed == n // block * block
    at = keep.long().cpu()
    assert torch.equal(nm.cpu(), mass.cpu().gather(2, at))
    for codes, scale, tl, x in ((new.k_codes, new.k_scale, new.k_tail, opened(rows)[0]),
                                (new.v_codes, new.v_scale, new.v_tail, opened(rows)[1])):
        picked = x.gather(2, at.unsqueeze(-1).expand(-1, -1, -1, d))
        want, wscale = ref.seal(picked[:, :, : new.sealed], block)
        assert torch.equal(codes.cpu().double(), want) and torch.equal(scale.cpu().double(), wscale)
        assert torch.equal(tl.cpu().double(), picked[:, :, new.sealed:])


def test_compact_ignores_indices_outside_the_cache(ops):
    rows = make_rows(ops, 1, 1, 64, 32, 64, 3, 2)
    keep = torch.tensor([[[0, 66, 67, -1, 2 ** 30]]], dtype=torch.int32, device=DEV)
    new, m = ops.kv8_compact(rows, keep, mass=torch.ones(1, 1, 67, device=DEV))
    k, _ = opened(rows)
    assert torch.equal(new.k_tail.cpu().double()[0, 0, :2], k[0, 0, [0, 66]])
    assert float(new.k_tail[0, 0, 2:].abs().max()) == 0
    assert m.flatten().tolist() == [1, 1, 0, 0, 0]


# ----------------------------------------------------------- as one program


def test_decode_evict_decode(ops):
    """Attention with its mass, an eviction, and attention over what is left."""
    b, hq, hkv, d, block = 1, 16, 2, 128, 64
    cache = make_rows(ops, b, hkv, d, block, 512, 40, 12)
    q = queries(b, hq, 3, d, 12)
    bits, prefix, vis = masks("causal", b, 3, 552, 12)
    out, lse = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
    mass = ops.kv8_attention_mass(q, lse, cache, bits, prefix, torch.zeros(b, hkv, 552, device=DEV))
    keep = ops.kv_keep_heaviest(mass, 552, 200, sinks=4, recent=16)
    new, nm = ops.kv8_compact(cache, keep, mass=mass)
    k, v = opened(cache)
    at = keep.long().cpu().unsqueeze(-1).expand(-1, -1, -1, d)
    vis2 = torch.ones(b, 1, 200, dtype=torch.bool)
    q2 = queries(b, hq, 1, d, 13)
    out2, lse2 = ops.kv8_tree_attention(q2, new, None, 200, return_lse=True)
    nk, nv = opened(new)
    # A row that was codes already (index < 512) keeps its values but for the
    # smallest of a block, which are off by half of e4m3's least step, 2^-10 of
    # the scale.  A row that was bf16 and enters a block is rounded to e4m3 for
    # the first time: half a step, 2^-4 relative (finfo.eps / 2 = 2^-3 / 2).
    old = k.gather(2, at)
    least = 2.0 ** -10 * float(new.k_scale.max())
    first_time = (at >= 512).double()
    assert bool(((nk - old).abs() <= least + first_time * 2.0 ** -4 * old.abs()).all())
    want, wlse = ref.attention(q2, nk, nv, vis2, d ** -0.5)
    check_attention(out2, lse2, want, wlse, float(nv.abs().max()))
    assert abs(float(nm.sum()) - float(mass.gather(2, keep.long()).sum())) < 1e-3


def test_streams_and_graph_replay(ops):
    """On a side stream, and captured: two graphs, replayed in turn with new inputs."""
    cache = make_rows(ops, 1, 4, 128, 64, 2048, 8, 3)
    bits, prefix, _ = masks("tree", 1, 8, 2056, 3)
    qa, qb = queries(1, 32, 8, 128, 31), queries(1, 32, 8, 128, 32)
    want = [ops.kv8_tree_attention(x, cache, bits, prefix, return_lse=True) for x in (qa, qb)]
    mass = [ops.kv8_attention_mass(x, w[1], cache, bits, prefix, torch.zeros(1, 4, 2056, device=DEV))
            for x, w in zip((qa, qb), want)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.kv8_tree_attention(qa, cache, bits, prefix)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0][0])
    held = []
    for _ in range(2):
        q = qa.clone()
        m = torch.zeros(1, 4, 2056, device=DEV)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            m.zero_()
            o, l = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
            ops.kv8_attention_mass(q, l, cache, bits, prefix, m)
        held.append((graph, q, m, o, l))
    for i, src in ((0, qb), (1, qa), (0, qa), (1, qb)):
        graph, q, m, o, l = held[i]
        q.copy_(src)
        graph.replay()
        w = 0 if src is qa else 1
        assert torch.equal(o, want[w][0]) and torch.equal(l, want[w][1]) and torch.equal(m, mass[w])


def test_offsets_past_32_bits(ops):
    """A cache whose byte offsets pass 2^31: the last head of the last request."""
    b, hkv, d, sealed = 2, 9, 128, 131072 * 8  # 2 * 9 * 2^20 * 128 B = 2.4 GB of K
    kc = torch.zeros(b, hkv, sealed, d, dtype=torch.uint8, device=DEV)
    code = torch.tensor([1.0]).to(ref.E4M3).view(torch.uint8).item()
    kc[-1, -1, -1] = code
    codes = kc.view(ref.E4M3)
    ks = torch.ones(b, hkv, sealed // 64, device=DEV)
    none = torch.zeros(b, hkv, 0, d, dtype=torch.bfloat16, device=DEV)
    rows = ops.Kv8Rows(codes, codes, ks, ks, sealed, none, none, 64)
    q = torch.full((b, hkv, 1, d), 4.0, dtype=torch.bfloat16, device=DEV)
    out, lse = ops.kv8_tree_attention(q, rows, None, sealed, return_lse=True)
    s = 4 * d * d ** -0.5  # the one key's score; the others' are 0
    w = math.exp(s) / (math.exp(s) + sealed - 1)
    assert abs(float(lse[-1, -1, 0]) - math.log(math.exp(s) + sealed - 1)) < 1e-3
    assert abs(float(out[-1, 0, -1, 0]) - w) <= 2.0 ** -8
    assert float(out[-1, 0, 0].abs().max()) == 0 and abs(float(lse[0, 0, 0]) - math.log(sealed)) < 1e-3
    mass = ops.kv8_attention_mass(q, lse, rows, None, sealed, torch.zeros(b, hkv, sealed, device=DEV))
    assert abs(float(mass[-1, -1, -1]) - w) < 1e-3
    keep = ops.kv_keep_heaviest(mass, sealed, 64, sinks=0, recent=0)
    assert int(keep[-1, -1, -1]) == sealed - 1
    new, _ = ops.kv8_compact(rows, keep)
    assert float(new.k_codes[-1, -1, -1, 0].float()) * float(new.k_scale[-1, -1, 0]) == 1.0
    k, _ = ops.kv8_read(rows, sealed - 2, 2)
    assert k[-1, -1, :, 5].tolist() == [0.0, 1.0]


@pytest.mark.parametrize("rows", [1, 65])
def test_heads_and_requests_that_share_memory(ops, rows):
    """A cache whose heads (or requests) are one tensor expanded is read like
    its copy, whichever kernel its strides allow."""
    one = make_rows(ops, 1, 1, 128, 64, 320, 70, 31)
    k, v = opened(one)
    for b, h in ((1, 2), (3, 1), (2, 2)):
        parts = [t.expand(b, h, *t.shape[2:]) for t in (one.k_codes, one.v_codes, one.k_scale, one.v_scale)]
        tails = [t.expand(b, h, *t.shape[2:]) for t in (one.k_tail, one.v_tail)]
        cache = ops.Kv8Rows(*parts, 320, *tails, 64)
        q = queries(b, 4 * h, rows, 128, 31)
        bits, prefix, vis = masks("any", b, rows, 390, 31)
        out, lse = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
        kk, vv = k.expand(b, h, *k.shape[2:]), v.expand(b, h, *v.shape[2:])
        want, wlse = ref.attention(q, kk, vv, vis, 128 ** -0.5)
        check_attention(out, lse, want, wlse, float(v.abs().max()))
        mass = ops.kv8_attention_mass(q, lse, cache, bits, prefix, torch.zeros(b, h, 390, device=DEV))
        wmass = ref.mass(q, wlse, kk, vis, 128 ** -0.5)
        assert bool(((mass.double().cpu() - wmass).abs() <= 4e-4 * wmass + 2.0 ** -22 * (1 + wmass)).all())


@pytest.mark.parametrize("rows", [1, 9, 70, 130])
def test_scores_that_rise_and_fall_along_the_cache(ops, rows):
    """Each block's scores lie far above (or below) the ones before, for every
    second row the other way round: the reference maximum moves all the time.
    Scores reach 30 here, so their partial sums stay below the 64 that the
    log-sum-exp's tolerance was derived for."""
    b, hq, hkv, d, sealed, tail = 1, 2, 1, 128, 1408, 70
    g = torch.Generator().manual_seed(rows)
    u = torch.where(torch.rand(d, generator=g) < 0.5, -1.0, 1.0)
    size = torch.linspace(-2.5, 2.5, sealed + tail)
    size[::7] *= 0.5
    k = (size[:, None] * u + 0.05 * torch.randn(sealed + tail, d, generator=g)).to(torch.bfloat16)[None, None]
    v = torch.randn(1, 1, sealed + tail, d, generator=g).to(torch.bfloat16)
    codes, scale = zip(*(ref.seal(x[:, :, :sealed], 64) for x in (k, v)))
    cache = ops.Kv8Rows(*(c.float().to(ref.E4M3).to(DEV) for c in codes), *(s.float().to(DEV) for s in scale), sealed,
                        *(x[:, :, sealed:].contiguous().to(DEV) for x in (k, v)), 64)
    k, v = opened(cache)
    sign = torch.where(torch.arange(rows) % 2 == 0, 1.0, -1.0) * torch.linspace(1.0, 0.3, rows)
    q = (sign[None, None, :, None] * u).expand(b, hq, rows, d).to(torch.bfloat16).contiguous().to(DEV)
    bits, prefix, vis = masks("any", b, rows, sealed + tail, 3)
    for use, pre, seen in ((bits, prefix, vis), (None, sealed + tail, torch.ones_like(vis))):
        out, lse = ops.kv8_tree_attention(q, cache, use, pre, return_lse=True)
        want, wlse = ref.attention(q, k, v, seen, d ** -0.5)
        check_attention(out, lse, want, wlse, float(v.abs().max()))
        mass = ops.kv8_attention_mass(q, lse, cache, use, pre, torch.zeros(b, hkv, sealed + tail, device=DEV))
        wmass = ref.mass(q, wlse, k, seen, d ** -0.5)
        assert bool(((mass.double().cpu() - wmass).abs() <= 4e-4 * wmass + 2.0 ** -22 * (1 + wmass)).all())
