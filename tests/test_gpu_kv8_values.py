"""The 8-bit KV cache's operators where magnitudes lie far apart: keys that a row
does not see hold large finite values, and rows see values that are small beside
others of the same cache.  Held to the bounds that ``kv8_bounds`` derives; the
weight of a token to the relative error of its exponentials, 4e-4."""
import math

import pytest
import torch

import kv8_bounds as kb
import kv8_reference as ref
import test_gpu_kv8 as shapes

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from specfit_b200 import ops as _ops

    return _ops


def sealed_cache(ops, k, v, sealed, block):
    """bf16 rows ``[B, Hkv, T, D]`` as a cache whose first ``sealed`` are codes."""
    parts = []
    for x in (k, v):
        codes, scale = ref.seal(x[:, :, :sealed], block)
        parts.append((codes.float().to(ref.E4M3).to(DEV), scale.float().to(DEV), x[:, :, sealed:].contiguous().to(DEV)))
    (kc, ks, kt), (vc, vs, vt) = parts
    return ops.Kv8Rows(kc, vc, ks, vs, sealed, kt, vt, block)


def opened(rows):
    return (ref.open_rows(rows.k_codes, rows.k_scale, rows.sealed, rows.k_tail, rows.block).to(DEV),
            ref.open_rows(rows.v_codes, rows.v_scale, rows.sealed, rows.v_tail, rows.block).to(DEV))


def pack(vis):
    b, r, n = vis.shape
    words = max(1, (n + 31) // 32)
    w = torch.zeros(b, r, words * 32, dtype=torch.int64)
    w[..., :n] = vis.long()
    x = (w.view(b, r, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32).to(DEV)


def draw(b, hq, hkv, rows, total, d, seed, k_size=1.0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, hq, rows, d, generator=g).to(torch.bfloat16)
    k = (k_size * torch.randn(b, hkv, total, d, generator=g)).to(torch.bfloat16)
    v = torch.randn(b, hkv, total, d, generator=g).to(torch.bfloat16)
    return q.to(DEV), k, v


def compare(ops, q, cache, vis):
    """Attention and weights of one call against the definition."""
    d = q.shape[-1]
    k, v = opened(cache)
    bits = pack(vis)
    out, lse = ops.kv8_tree_attention(q, cache, bits, 0, return_lse=True)
    want = kb.attention(q, k, v, vis.to(DEV), d ** -0.5)
    assert kb.off(out, want) is None, kb.off(out, want)
    assert kb.lse_off(lse, want) is None, kb.lse_off(lse, want)
    check_weights(ops, q, cache, vis, lse, want)


def check_weights(ops, q, cache, vis, lse, want):
    b, hkv = cache.shape[:2]
    mass = ops.kv8_attention_mass(q, lse, cache, pack(vis), 0, torch.zeros(b, hkv, cache.length, device=DEV)).double()
    bad = (mass - want["mass"]).abs() > 4e-4 * want["mass"] + 2.0 ** -100
    assert not bool(bad.any()), (int(bad.sum()), mass[bad][:4], want["mass"][bad][:4])


# Query heads of one KV head, rows, head_dim: what the form for many query rows takes.
MANY = [(8, 9, 128), (8, 33, 128)]


# What the forms for few take: at most eight packed rows, sixteen, more than one tile of them.
FEW = [(8, 1, 128), (2, 3, 112), (1, 2, 64), (4, 3, 128), (5, 7, 48), (8, 9, 64)]


@pytest.mark.parametrize("hq,rows,d", FEW)
@pytest.mark.parametrize("where", ["tail", "codes"])
@pytest.mark.parametrize("size", [1e4, 1e12, 1e30])
def test_large_keys_and_values_of_an_unseen_key_stay_out(ops, hq, rows, d, where, size):
    unseen_large(ops, hq, rows, d, where, size, keys=True)


@pytest.mark.parametrize("hq,rows,d", [f for f in FEW if f[1] > 1])
def test_rows_that_see_small_values_only(ops, hq, rows, d):
    small_beside_large(ops, hq, rows, d)


@pytest.mark.parametrize("hq,rows,d", FEW)
def test_values_that_shrink_while_scores_grow(ops, hq, rows, d):
    shrinking(ops, hq, rows, d)


@pytest.mark.parametrize("hq,hkv,rows,sealed,tail,d", [(32, 4, 1, 65536, 33, 128), (32, 4, 8, 4096, 55, 128),
                                                       (4, 1, 3, 1024, 20, 64), (16, 2, 40, 8192, 40, 64),
                                                       (8, 8, 1, 2048, 90, 128)])
def test_long_caches(ops, hq, hkv, rows, sealed, tail, d):
    long_cache(ops, hq, hkv, rows, sealed, tail, d)


@pytest.mark.parametrize("hq,rows,d", FEW + MANY)
def test_weights_beside_a_large_unseen_key(ops, hq, rows, d):
    """The weights alone, by the definition's log-sum-exp."""
    sealed, tail = 128, 37
    q, k, v = draw(1, hq, 1, rows, sealed + tail, d, 15)
    k[:, :, sealed + 5] = 1e12
    vis = torch.ones(1, rows, sealed + tail, dtype=torch.bool)
    vis[:, :, sealed + 5] = False
    cache = sealed_cache(ops, k, v, sealed, 64)
    want = kb.attention(q, *opened(cache), vis.to(DEV), d ** -0.5)
    check_weights(ops, q, cache, vis, want["lse"].float(), want)


def test_rows_of_zeros_and_tail_keys_far_apart(ops):
    """Tail rows of quite different sizes, seen: rows of zeros, keys 2^20 apart."""
    for hq, rows, d in FEW + MANY:
        q, k, v = draw(1, hq, 1, rows, 150, d, 14)
        k[:, :, 100::5] = (k[:, :, 100::5].float() * 2.0 ** -20).to(torch.bfloat16)
        v[:, :, 96::3] = (v[:, :, 96::3].float() * 2.0 ** -50).to(torch.bfloat16)
        k[:, :, 98], v[:, :, 99] = 0, 0
        vis = torch.ones(1, rows, 150, dtype=torch.bool)
        vis[:, -1] = False
        vis[:, -1, 96::3] = True  # small values and a row of zeros only
        compare(ops, q, sealed_cache(ops, k, v, 96, 32), vis)


@pytest.mark.parametrize("hq,rows,d", MANY)
@pytest.mark.parametrize("where", ["tail", "codes"])
@pytest.mark.parametrize("size", [1e3, 1e9, 1e30])
def test_large_values_of_an_unseen_key_stay_out_many_rows(ops, hq, rows, d, where, size):
    unseen_large(ops, hq, rows, d, where, size, keys=False)


def unseen_large(ops, hq, rows, d, where, size, keys):
    sealed, tail, block = 448, 41, 64
    total = sealed + tail
    q, k, v = draw(1, hq, 1, rows, total, d, 11)
    hidden = [sealed + 3, sealed + 20, total - 1] if where == "tail" else list(range(64, 128)) + [300]
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    v[:, :, hidden] = size
    if keys:
        k[:, :, hidden] = size
    if where == "codes":
        hidden = list(range(64, 128)) + list(range(256, 320))  # whole blocks: a scale is a block's
    vis[:, :, hidden] = False
    compare(ops, q, sealed_cache(ops, k, v, sealed, block), vis)


def test_rows_that_see_small_values_only_many_rows(ops):
    small_beside_large(ops, 8, 16, 128)


def small_beside_large(ops, hq, rows, d):
    """Every second row sees the large values, the others only the small ones,
    2^40 below."""
    sealed, tail, block = 512, 70, 64
    total = sealed + tail
    q, k, v = draw(1, hq, 1, rows, total, d, 12)
    large = torch.zeros(total, dtype=torch.bool)
    large[128:256] = True
    large[sealed + 10:sealed + 13] = True
    v[:, :, large] = (v[:, :, large].float() * 2.0 ** 40).to(torch.bfloat16)
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    vis[:, ::2, large] = False
    compare(ops, q, sealed_cache(ops, k, v, sealed, block), vis)


def test_values_that_shrink_while_scores_grow_many_rows(ops):
    shrinking(ops, 8, 16, 128)


def shrinking(ops, hq, rows, d):
    """Blocks of values 2^6 smaller each, scores 3 higher each: the last blocks
    decide the softmax, the first were the largest values."""
    sealed, tail, block = 640, 30, 64
    total = sealed + tail
    q, k, v = draw(1, hq, 1, rows, total, d, 13, k_size=0.05)
    u = torch.ones(d)
    step = torch.arange(total) // block
    k = (k.float() + step[None, None, :, None] * (3.0 / math.sqrt(d)) * u).to(torch.bfloat16)
    q = (torch.ones_like(q.float()) + 0.05 * q.float()).to(torch.bfloat16)
    v = (v.float() * torch.pow(2.0, -6.0 * step)[None, None, :, None]).to(torch.bfloat16)
    cache = sealed_cache(ops, k, v, sealed, block)
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    vis[:, 1::2, 320:] = False
    compare(ops, q, cache, vis)


@pytest.mark.parametrize("hq,hkv,rows,sealed,tail", [(32, 4, 65, 8192, 65), (8, 1, 300, 4096, 300),
                                                     (16, 2, 100, 16384, 0)])
def test_long_caches_many_rows(ops, hq, hkv, rows, sealed, tail):
    long_cache(ops, hq, hkv, rows, sealed, tail, 128)


def long_cache(ops, hq, hkv, rows, sealed, tail, d):
    """Averages over thousands of keys are far smaller than the values."""
    total = sealed + tail
    g = torch.Generator(device=DEV).manual_seed(rows + sealed)
    codes = [(torch.randn(1, hkv, sealed, d, generator=g, device=DEV) * 60).to(ref.E4M3) for _ in range(2)]
    scale = [torch.full((1, hkv, sealed // 64), 2.0 ** -6, device=DEV) for _ in range(2)]
    scale[1][:, :, ::3] = 2.0 ** -4
    tails = [torch.randn(1, hkv, tail, d, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    cache = ops.Kv8Rows(codes[0], codes[1], scale[0], scale[1], sealed, tails[0], tails[1], 64)
    q = torch.randn(1, hq, rows, d, generator=g, device=DEV).to(torch.bfloat16)
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    if tail >= rows:
        vis[:, :, total - rows:] = torch.ones(rows, rows, dtype=torch.bool).tril()
    compare(ops, q, cache, vis)


@pytest.mark.parametrize("hq,rows,d", FEW + MANY)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_not_a_number_in_queries_and_keys(ops, hq, rows, d, what):
    """A tail key whose K or V row holds one answers NaN to the rows that see it
    (whatever the sign of the product), a query row that holds one answers NaN, and
    the others stay what they are."""
    sealed, tail = 64, 38
    total = sealed + tail
    q, k, v = draw(1, hq, 1, rows, total, d, 16)
    clean = sealed_cache(ops, k, v, sealed, 32)
    key, value = sealed + 7, sealed + 33
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    vis[:, :, [key, value]] = False
    want, wlse = ops.kv8_tree_attention(q, clean, pack(vis), 0, return_lse=True)
    k[:, :, key, 3], v[:, :, value, d - 1] = what, what
    cache = sealed_cache(ops, k, v, sealed, 32)
    out, lse = ops.kv8_tree_attention(q, cache, pack(vis), 0, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    for at in (key, value):
        on = vis.clone()
        on[:, 0, at] = True
        out, lse = ops.kv8_tree_attention(q, cache, pack(on), 0, return_lse=True)
        assert bool(torch.isnan(out[:, 0]).all()) and bool(torch.isnan(lse[:, :, 0]).all())
        assert torch.equal(out[:, 1:], want[:, 1:]) and torch.equal(lse[:, :, 1:], wlse[:, :, 1:])
    if rows > 1:
        some = q.clone()
        some[:, :, -1, d // 2] = what
        out, lse = ops.kv8_tree_attention(some, cache, pack(vis), 0, return_lse=True)
        assert bool(torch.isnan(out[:, -1]).all()) and bool(torch.isnan(lse[:, :, -1]).all())
        assert torch.equal(out[:, :-1], want[:, :-1]) and torch.equal(lse[:, :, :-1], wlse[:, :, :-1])
    # A weight per key: NaN for the seen key, none for those that no row sees.
    on = vis.clone()
    on[:, :, key] = True
    mass = ops.kv8_attention_mass(q, wlse, cache, pack(on), 0, torch.zeros(1, 1, total, device=DEV))[0, 0]
    assert bool(torch.isnan(mass[key])) and bool(torch.isfinite(mass[:key]).all()) and float(mass[value]) == 0


@pytest.mark.parametrize("b,hq,hkv,d,block,sealed,tail,rows,mask", shapes.ATTENTION)
def test_every_shape_to_the_row(ops, b, hq, hkv, d, block, sealed, tail, rows, mask):
    """The operators' shapes, held to bounds that a row of zeros does not meet."""
    seed = hq + d + sealed + rows + 1
    cache = shapes.make_rows(ops, b, hkv, d, block, sealed, tail, seed, room=block)
    q = shapes.queries(b, hq, rows, d, seed)
    bits, prefix, vis = shapes.masks(mask, b, rows, sealed + tail, seed)
    out, lse = ops.kv8_tree_attention(q, cache, bits, prefix, return_lse=True)
    want = kb.attention(q, *opened(cache), vis.to(DEV), d ** -0.5)
    assert kb.off(out, want) is None, kb.off(out, want)
    assert kb.lse_off(lse, want) is None, kb.lse_off(lse, want)


@pytest.mark.parametrize("hq,rows,d", FEW + MANY)
def test_scales_that_are_no_powers_of_two(ops, hq, rows, d):
    """Codes of another maker, scaled by their largest value over 448."""
    sealed, block = 512, 64
    g = torch.Generator().manual_seed(21)
    q = torch.randn(1, hq, rows, d, generator=g).to(torch.bfloat16).to(DEV)
    codes, scales = [], []
    for _ in range(2):
        x = torch.randn(1, 1, sealed // block, block, d, generator=g) * torch.rand(1, 1, sealed // block, 1, 1, generator=g)
        s = x.abs().amax((3, 4)) / 448
        codes.append((x / s[..., None, None]).reshape(1, 1, sealed, d).to(ref.E4M3).to(DEV))
        scales.append(s.to(DEV))
    none = torch.zeros(1, 1, 0, d, dtype=torch.bfloat16, device=DEV)
    cache = ops.Kv8Rows(*codes, *scales, sealed, none, none, block)
    vis = torch.rand(1, rows, sealed, generator=g) < 0.8
    compare(ops, q, cache, vis)
    out, lse = ops.kv8_tree_attention(q, cache, None, sealed, return_lse=True)
    want = kb.attention(q, *opened(cache), torch.ones_like(vis).to(DEV), d ** -0.5)
    assert kb.off(out, want) is None and kb.lse_off(lse, want) is None


def nodes_of(call):
    """Kernels of a captured call."""
    import ctypes

    for _ in range(2):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    n = ctypes.c_size_t()
    assert ctypes.CDLL("libcuda.so.1").cuGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None,
                                                       ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("b,hq,hkv,rows,sealed,tail,shared", [
    (1, 8, 1, 1, 64, 5, False),       # one range
    (1, 32, 4, 1, 512, 17, False),    # ranges joined by a cluster
    (1, 32, 4, 1, 16384, 17, False),  # and by a second kernel
    (2, 8, 8, 100, 64, 70, False),    # many rows, one range
    (1, 32, 4, 65, 4096, 65, False),  # many rows, many ranges; weights in one part
    (1, 8, 1, 65, 640, 65, False),    # weights of a short cache in parts
    (1, 16, 2, 65, 320, 70, True),    # heads that share memory: the form for few rows
    (1, 8, 1, 0, 64, 5, False),       # nothing to do
])
def test_launches_are_counted(ops, b, hq, hkv, rows, sealed, tail, shared):
    total = sealed + tail
    q, k, v = draw(b, hq, hkv, rows, total, 128, 17)
    cache = sealed_cache(ops, k, v, sealed, 64)
    if shared:
        parts = [t[:, :1].expand(b, hkv, *t.shape[2:]) for t in (cache.k_codes, cache.v_codes, cache.k_scale,
                                                                  cache.v_scale)]
        cache = ops.Kv8Rows(*parts, sealed, cache.k_tail, cache.v_tail, 64)
    _, lse = ops.kv8_tree_attention(q, cache, None, total, return_lse=True)
    mass = torch.zeros(b, hkv, total, device=DEV)
    for call in (lambda: ops.kv8_tree_attention(q, cache, None, total),
                 lambda: ops.kv8_attention_mass(q, lse, cache, None, total, mass)):
        before = ops.LAUNCHES[0]
        call()
        assert ops.LAUNCHES[0] - before == (nodes_of(call) if rows else 0)


# (KV heads so many that one range holds all keys, or few: ranges are joined.)
@pytest.mark.parametrize("hq,hkv,rows,d", [(8, 1, 1, 128), (4, 1, 3, 64), (8, 1, 9, 128), (224, 224, 2, 128),
                                           (128, 128, 40, 64), (148, 148, 70, 128)])
@pytest.mark.parametrize("first", [0.0, 2.0 ** -60])
def test_values_of_zeros_before_large_ones(ops, hq, hkv, rows, d, first):
    """Blocks of zeros (or of 2^-60), then values of 2^60, all seen: the first blocks'
    share of the weights stays when the reference moves by more than fp32's exponents."""
    sealed, tail, block = 512, 40, 64
    total = sealed + tail
    q, k, v = draw(1, hq, hkv, rows, total, d, 18)
    v[:, :, :256] = (v[:, :, :256].float() * first).to(torch.bfloat16)
    v[:, :, 256:] = (v[:, :, 256:].float() * 2.0 ** 60).to(torch.bfloat16)
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    compare(ops, q, sealed_cache(ops, k, v, sealed, block), vis)


@pytest.mark.parametrize("hq,hkv,rows,d", [(8, 1, 1, 128), (224, 224, 2, 128), (444, 444, 1, 64), (8, 1, 16, 128)])
def test_values_of_zeros_alone(ops, hq, hkv, rows, d):
    """A long cache of zero values answers zeros and its log-sum-exp."""
    sealed = 4096
    g = torch.Generator(device=DEV).manual_seed(19)
    q = torch.randn(1, hq, rows, d, generator=g, device=DEV).to(torch.bfloat16)
    k = torch.randn(1, hkv, sealed, d, generator=g, device=DEV).to(ref.E4M3)
    scale = torch.full((1, hkv, sealed // 64), 2.0 ** -100, device=DEV)
    none = torch.zeros(1, hkv, 0, d, dtype=torch.bfloat16, device=DEV)
    cache = ops.Kv8Rows(k, torch.zeros_like(k), torch.ones_like(scale), scale, sealed, none, none, 64)
    out, lse = ops.kv8_tree_attention(q, cache, None, sealed, return_lse=True)
    x = torch.einsum("bhgrd,bhkd->bhgrk", q.double().view(1, hkv, -1, rows, d), k.double()) * d ** -0.5
    assert float(out.abs().max()) == 0
    assert float((lse.double() - torch.logsumexp(x, -1).view_as(lse)).abs().max()) <= 2e-4


def test_keys_that_are_the_values(ops):
    """One content in one place: sealed, compacted and read back."""
    g = torch.Generator().manual_seed(22)
    x = torch.randn(1, 96, 2, 64, generator=g).to(torch.bfloat16).to(DEV).permute(0, 2, 1, 3)[:, :, :, ::1]
    codes = torch.zeros(1, 2, 96, 64, device=DEV).to(ref.E4M3)
    scale = torch.zeros(1, 2, 3, device=DEV)
    for rows in (x, torch.stack([x, x], -1)[..., 0]):  # in place, and copied to be contiguous
        ops.kv8_seal(rows, rows, codes, codes, scale, scale)
        want, wscale = ref.seal(x.cpu(), 32)
        assert torch.equal(codes.cpu().double(), want) and torch.equal(scale.cpu().double(), wscale)
    none = torch.zeros(1, 2, 0, 64, dtype=torch.bfloat16, device=DEV)
    cache = ops.Kv8Rows(codes, codes, scale, scale, 96, none, none, 32)
    keep = torch.arange(0, 96, 2, dtype=torch.int32, device=DEV).expand(1, 2, 48).contiguous()
    oc, os = torch.zeros(1, 2, 32, 64, device=DEV).to(ref.E4M3), torch.zeros(1, 2, 1, device=DEV)
    ot = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    new, _ = ops.kv8_compact(cache, keep, out=ops.Kv8Rows(oc, oc, os, os, 32, ot, ot, 32))
    k, v = ops.kv8_read(new)
    old, _ = ops.kv8_read(cache)
    kept = old[:, :, ::2]
    assert torch.equal(k, v) and torch.equal(k[:, :, 32:], kept[:, :, 32:])
    assert float((k[:, :, :32].float() - kept[:, :, :32].float()).abs().max()) <= 2.0 ** -10 * float(os.max())


@pytest.mark.parametrize("hq,hkv,rows,sealed,tail", [(16, 2, 65, 1024, 65), (8, 1, 9, 320, 33)])
def test_many_rows_replayed_and_on_several_streams(ops, hq, hkv, rows, sealed, tail):
    """Captured once, replayed with other queries; and on three streams at once."""
    total = sealed + tail
    q, k, v = draw(2, hq, hkv, rows, total, 128, 23)
    cache = sealed_cache(ops, k, v, sealed, 64)
    vis = torch.ones(2, rows, total, dtype=torch.bool)
    vis[:, :, total - rows:] = torch.ones(rows, rows, dtype=torch.bool).tril()
    bits = pack(vis)
    inputs = [q, q.flip(2).contiguous(), -q]

    def call(x):
        out, lse = ops.kv8_tree_attention(x, cache, bits, 0, return_lse=True)
        return out, lse, ops.kv8_attention_mass(x, lse, cache, bits, 0, torch.zeros(2, hkv, total, device=DEV))

    want = [call(x) for x in inputs]
    x = q.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(x)
    for i in (1, 0, 2, 1):
        x.copy_(inputs[i])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want[i])), i
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[] for _ in inputs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(inputs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(3) for g in got[i] for a, b in zip(g, want[i]))
