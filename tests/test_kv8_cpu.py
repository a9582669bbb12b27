"""The 8-bit KV cache on the CPU: refusals of its operators before any launch,
and the cache's bookkeeping (sealing, rolling back, compaction, eviction) with
plain stand-ins for the kernels, against a list of the rows that should be
there."""
import ctypes
import math

import pytest
import torch

import kv8_reference as ref
from specfit_b200 import _native as N
from specfit_b200 import ops
from specfit_b200.runtime import kv8_cache as kc
from specfit_b200.runtime.kv_cache import compact_tree_cache_
from specfit_b200.runtime.qwen3_verifier import qwen3_moe_config
from specfit_b200.runtime.speculator import B200TreeSpeculator


def struct(**kw):
    base = dict(batch=1, num_kv_heads=2, head_dim=128, block_tokens=64, sealed=128, tail=8, k_codes=256, v_codes=256,
                code_batch_stride=0, code_head_stride=128 * 128, k_scale=256, v_scale=256, scale_batch_stride=0,
                scale_head_stride=2, k_tail=256, v_tail=256, tail_batch_stride=0, tail_head_stride=1024)
    base.update(kw)
    return N.Kv8RowsStruct(**base)


def addr(s):
    return ctypes.addressof(s)


# ------------------------------------------------------------ the C entries


def attention(rows, heads=8, q_len=3, words=1, prefix=133, scale=0.1, q=256, bits=256, out=256, ws=0, nbytes=0,
              q_stride=128):
    return N.lib.sf_kv8_tree_attention(q, 0, 0, q_stride, heads, q_len, addr(rows), bits, words, 0, prefix, scale, out,
                                       0, None, ws or None, nbytes, None)


@pytest.mark.parametrize("kw,what", [
    (dict(head_dim=120), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=144), "head_dim"),
    (dict(block_tokens=48), "block_tokens"), (dict(sealed=100), "sealed"), (dict(tail=-1), "sealed"),
    (dict(batch=0), "batch"), (dict(num_kv_heads=70000), "batch"), (dict(k_codes=None), "null"),
    (dict(k_codes=264), "aligned"), (dict(code_head_stride=8), "aligned"), (dict(k_tail=None), "null"),
    (dict(tail_head_stride=4), "aligned"), (dict(sealed=1 << 30), "sealed")])
def test_a_malformed_cache_is_refused(kw, what):
    assert attention(struct(**kw)) == N.SF_ERR_INVALID_ARGUMENT and what in N.last_error()
    if "v_" not in str(kw):
        s = struct(**kw)
        assert N.lib.sf_kv8_read(addr(s), 0, 1, 256, 256, 0, 0, None) == N.SF_ERR_INVALID_ARGUMENT


def test_malformed_calls_are_refused():
    s = struct()
    for kw, what in ((dict(heads=7), "num_heads"), (dict(q_len=-1), "lengths"), (dict(prefix=137), "lengths"),
                     (dict(prefix=-1), "lengths"), (dict(prefix=0, words=4), "tree_bits"), (dict(bits=None), "tree_bits"),
                     (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
                     (dict(scale=math.inf), "scale"), (dict(q=None), "null"), (dict(out=None), "null"),
                     (dict(q=264), "aligned"), (dict(q_stride=4), "aligned"), (dict(out=264), "aligned"),
                     (dict(q_len=1 << 19), "rows")):
        assert attention(s, **kw) == N.SF_ERR_INVALID_ARGUMENT, kw
        assert what in N.last_error(), (kw, N.last_error())
    assert attention(s, q_len=0, out=None) == N.SF_OK  # nothing to do
    need = N.lib.sf_kv8_attention_workspace_bytes(1, 8, 2, 128, 100, 4096, 8)
    big = struct(sealed=4096, code_head_stride=4096 * 128)
    assert need > 0 and attention(big, q_len=100, prefix=4104, bits=None, ws=256, nbytes=need - 1) == N.SF_ERR_WORKSPACE
    assert attention(big, q_len=100, prefix=4104, bits=None, ws=8, nbytes=need) == N.SF_ERR_INVALID_ARGUMENT
    assert N.lib.sf_kv8_attention_workspace_bytes(1, 7, 2, 128, 1, 64, 0) == 0
    # Sealing: blocks within the buffers, aligned rows.
    seal = lambda first, n, k=256, rs=128: N.lib.sf_kv8_seal(k, 256, 0, 0, rs, addr(s), first, n, None)
    for args in ((0, 3), (2, 1), (-1, 1), (0, -1), (0, 1, 264), (0, 1, 256, 12), (0, 1, None)):
        assert seal(*args) == N.SF_ERR_INVALID_ARGUMENT, args
    for args in (((1 << 63) - 1, 1), ((1 << 63) - 1, 2)):  # their sum has no 64 bits
        assert seal(*args) == N.SF_ERR_INVALID_ARGUMENT, args
    assert seal(2, 0) == N.SF_OK
    assert N.lib.sf_kv8_read(addr(s), 100, 37, 256, 256, 0, 0, None) == N.SF_ERR_INVALID_ARGUMENT
    assert N.lib.sf_kv8_read(addr(s), (1 << 63) - 1, 2, 256, 256, 0, 0, None) == N.SF_ERR_INVALID_ARGUMENT
    assert N.lib.sf_kv8_read(addr(s), 136, 0, None, None, 0, 0, None) == N.SF_OK
    # Mass and selection.
    mass = lambda **k: N.lib.sf_kv8_attention_mass(k.get("q", 256), 0, 0, 128, k.get("heads", 8), 3, k.get("lse", 256),
                                                   addr(s), 256, 1, 0, k.get("prefix", 133), k.get("scale", 0.1),
                                                   k.get("mass", 256), 0, 0, None, 0, None)
    for kw in (dict(heads=3), dict(prefix=200), dict(scale=0.0), dict(lse=None), dict(mass=None), dict(q=None)):
        assert mass(**kw) == N.SF_ERR_INVALID_ARGUMENT, kw
    keep = lambda length, budget, sinks, recent, m=256: N.lib.sf_kv_keep_heaviest(m, 0, 0, 1, 1, length, budget, sinks,
                                                                                 recent, 256, None)
    for args in ((10, 11, 0, 0), (10, 5, 3, 3), (10, 5, -1, 0), (10, -1, 0, 0), (1 << 30, 5, 0, 0), (10, 5, 0, 0, None),
                 (10, 5, 1 << 62, 1 << 62)):
        assert keep(*args) == N.SF_ERR_INVALID_ARGUMENT, args
    assert keep(10, 0, 0, 0) == N.SF_OK
    # Compaction: the target holds the kept rows, in buffers of its own.
    comp = lambda out, n, m=None, mo=None: N.lib.sf_kv8_compact(addr(s), 256, n, addr(out), m, 0, 0, mo, 0, 0, None)
    other = dict(k_codes=512, v_codes=512, k_tail=512, v_tail=512)
    for out, n in ((struct(sealed=64, tail=5, **other), 70), (struct(sealed=64, tail=6, **other), 137),
                   (struct(sealed=64, tail=6), 70), (struct(sealed=64, tail=6, block_tokens=32, **other), 70),
                   (struct(sealed=64, tail=6, num_kv_heads=1, **other), 70)):
        assert comp(out, n) == N.SF_ERR_INVALID_ARGUMENT
    assert comp(struct(sealed=64, tail=6, **other), 70, 256, 256) == N.SF_ERR_INVALID_ARGUMENT
    assert comp(struct(sealed=64, tail=6, **other), 70, 256, None) == N.SF_ERR_INVALID_ARGUMENT


def test_expanded_targets_are_refused():
    """Requests or heads that share memory may be read, not written."""
    other = dict(k_codes=512, v_codes=512, k_tail=512, v_tail=512)
    for kw in (dict(code_head_stride=0), dict(scale_head_stride=1), dict(code_head_stride=127 * 128),
               dict(batch=2, code_batch_stride=128 * 128, scale_batch_stride=4, tail_batch_stride=2048),
               dict(batch=2, code_batch_stride=256 * 128, scale_batch_stride=2, tail_batch_stride=2048)):
        s = struct(**kw)
        assert N.lib.sf_kv8_seal(256, 256, 0, 0, 128, addr(s), 0, 1, None) == N.SF_ERR_INVALID_ARGUMENT, kw
        assert "overlap" in N.last_error(), kw
    src = struct()
    for kw in (dict(code_head_stride=0), dict(tail_head_stride=0), dict(tail_head_stride=5 * 128)):
        out = struct(**{**other, "sealed": 64, "tail": 6, **kw})
        assert N.lib.sf_kv8_compact(addr(src), 256, 70, addr(out), None, 0, 0, None, 0, 0,
                                    None) == N.SF_ERR_INVALID_ARGUMENT, kw
        assert "overlap" in N.last_error(), kw
    out = struct(sealed=64, tail=6, **other)
    assert N.lib.sf_kv8_compact(addr(src), 256, 70, addr(out), 256, 0, 136, 512, 0, 69,
                                None) == N.SF_ERR_INVALID_ARGUMENT
    assert "overlap" in N.last_error()
    for hs in (0, 135):
        assert N.lib.sf_kv8_attention_mass(256, 0, 0, 128, 8, 3, 256, addr(src), 256, 1, 0, 133, 0.1, 256, 0, hs, None,
                                           0, None) == N.SF_ERR_INVALID_ARGUMENT
        assert "overlap" in N.last_error()
    two = struct(batch=2)  # read twice: allowed; written to one place: not
    assert attention(two) == N.SF_ERR_INVALID_ARGUMENT and "overlap" in N.last_error()


def test_python_entries_refuse_cpu_tensors_and_wrong_types():
    f8, bf = torch.float8_e4m3fn, torch.bfloat16
    codes, scale = torch.zeros(1, 2, 64, 64).to(f8), torch.zeros(1, 2, 1)
    tail = torch.zeros(1, 2, 3, 64, dtype=bf)
    with pytest.raises(ValueError, match="CUDA"):
        ops.Kv8Rows(codes, codes, scale, scale, 64, tail, tail, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_keep_heaviest(torch.zeros(1, 2, 8), 8, 4)
    with pytest.raises(TypeError):
        ops.kv8_seal(tail.float(), tail.float(), codes, codes, scale, scale)
    with pytest.raises(ValueError):
        ops.kv8_seal(tail, tail, codes, codes, scale, scale)


# ------------------------------------------------------- the cache's books


class PlainRows:
    def __init__(self, kcodes, vcodes, ks, vs, sealed, kt, vt, block):
        self.parts = ((kcodes, ks, kt), (vcodes, vs, vt))
        self.sealed, self.block = sealed, block

    def open(self, i):
        c, s, t = self.parts[i]
        return ref.open_rows(c.float(), s, self.sealed, t.float(), self.block)


@pytest.fixture
def plain(monkeypatch):
    """Plain stand-ins for the operators that the cache calls."""
    def seal(k, v, kcodes, vcodes, ks, vs, first_block=0, block=None):
        for x, codes, scale in ((k, kcodes, ks), (v, vcodes, vs)):
            c, s = ref.seal(x, block)
            codes[:, :, first_block * block: first_block * block + x.shape[2]] = c.to(ref.E4M3)
            scale[:, :, first_block: first_block + s.shape[2]] = s.float()

    def read(rows, first=0, count=None):
        out = [rows.open(i).to(torch.bfloat16) for i in (0, 1)]
        count = out[0].shape[2] - first if count is None else count
        return tuple(x[:, :, first: first + count] for x in out)

    def compact(rows, keep, mass=None, out=None, mass_out=None):
        n = keep.shape[2]
        for i in (0, 1):
            x = rows.open(i)
            x = x.gather(2, keep.long().unsqueeze(-1).expand(-1, -1, -1, x.shape[3])).to(torch.bfloat16)
            full = n // rows.block * rows.block
            c, s = ref.seal(x[:, :, :full], rows.block)
            codes, scale, tail = out.parts[i]
            codes[:, :, :full] = c.to(ref.E4M3)
            scale[:, :, : full // rows.block] = s.float()
            tail.copy_(x[:, :, full:])
        mass_out[:, :, :n] = mass.gather(2, keep.long())
        return out, mass_out

    monkeypatch.setattr(kc.ops, "kv8_seal", seal)
    monkeypatch.setattr(kc.ops, "kv8_read", read)
    monkeypatch.setattr(kc.ops, "kv8_compact", compact)
    monkeypatch.setattr(kc.ops, "Kv8Rows", PlainRows)
    monkeypatch.setattr(kc.ops, "kv_keep_heaviest",
                        lambda m, length, budget, sinks=0, recent=0: ref.keep_heaviest(m, length, budget, sinks, recent))


def rows_of(n, seed, h=2, d=16):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(1, h, n, d, generator=g).to(torch.bfloat16) for _ in range(2))


def cache(**kw):
    base = dict(config=qwen3_moe_config(2), capacity=96, block=32, tail_room=8)
    base.update(kw)
    return kc.Kv8Cache(**base)


def feed(c, n, seed):
    out = None
    for layer in range(2):
        k, v = rows_of(n, seed + layer)
        out = c.update(k, v, layer)
    return out


def rounded(x):
    c, s = ref.seal(x, 32)
    return (c * s.repeat_interleave(32, 2).unsqueeze(-1)).to(torch.bfloat16)


def test_blocks_are_sealed_when_the_next_pass_begins(plain):
    c = cache()
    k, v = rows_of(70, 1)
    got = feed(c, 70, 1)
    l = c.layers[1]
    assert (l.sealed, l.tail) == (0, 70) and c.get_seq_length() == 70
    kk, _ = rows_of(70, 2)
    assert torch.equal(got[0], kk)  # nothing rounded yet
    got = feed(c, 3, 5)
    assert (l.sealed, l.tail) == (64, 9) and c.get_seq_length() == 73
    assert torch.equal(got[0][:, :, :64], rounded(kk[:, :, :64])) and torch.equal(got[0][:, :, 64:70], kk[:, :, 64:])
    assert l._kt.shape[2] == 32 + 8  # the large tail of the first pass is gone
    for _ in range(10):  # past the reserved capacity
        got = feed(c, 30, 9)
    assert c.get_seq_length() == 373 and got[0].shape[2] == 373 and l.sealed % 32 == 0


def test_crop_in_the_tail_and_in_a_sealed_block(plain):
    c = cache()
    feed(c, 70, 1)
    got = feed(c, 6, 5)
    c.crop(70)
    assert c.get_seq_length() == 70 and c.layers[0].sealed == 64
    c.crop(-2)
    assert c.get_seq_length() == 68
    c.crop(100)
    assert c.get_seq_length() == 68
    c.crop(45)  # inside the second sealed block
    l = c.layers[1]
    assert (l.sealed, l.tail) == (32, 13)
    again = feed(c, 30, 11)
    assert torch.equal(again[0][:, :, :32], got[0][:, :, :32])
    assert torch.equal(again[0][:, :, 32:45], got[0][:, :, 32:45])
    c.crop(0)
    assert c.get_seq_length() == 0
    assert torch.equal(feed(c, 5, 3)[0], rows_of(5, 4)[0])


def test_tree_compaction_keeps_the_accepted_rows(plain):
    c = cache(budget=64, sinks=2, recent=8)
    feed(c, 70, 1)
    base = c.get_seq_length()
    got = feed(c, 6, 5)
    for i, l in enumerate(c.layers):
        l.mass[:, :, :76] = torch.arange(76.0) + i
    compact_tree_cache_(c, base_kv_length=base, verification_positions=(0, 2, 5), verification_node_count=6)
    assert c.get_seq_length() == 73
    l = c.layers[1]
    now = kc.ops.kv8_read(l.rows())
    assert torch.equal(now[0][:, :, 70:73], got[0][:, :, [70, 72, 75]])
    assert torch.equal(now[1][:, :, 70:73], got[1][:, :, [70, 72, 75]])
    assert l.mass[0, 0, 68:73].tolist() == [69, 70, 71, 73, 76]
    with pytest.raises(RuntimeError, match="unexpected length"):
        compact_tree_cache_(c, base_kv_length=base, verification_positions=(0,), verification_node_count=6)
    with pytest.raises(RuntimeError, match="sealed"):
        l.keep_tail_rows(10, (0,))


def test_eviction(plain):
    c = cache(budget=40, sinks=2, recent=8)
    assert c.evict() == 0
    feed(c, 90, 1)
    before = [kc.ops.kv8_read(l.rows()) for l in c.layers]
    g = torch.Generator().manual_seed(4)
    for l in c.layers:
        l.mass[:, :, :90] = torch.rand(1, 2, 90, generator=g)
    want = [ref.keep_heaviest(l.mass, 90, 40, 2, 8) for l in c.layers]
    weights = [l.mass.clone() for l in c.layers]
    assert c.evict() == 50
    assert c.get_seq_length() == 40 and c.next_position == 90 and c.dropped == 50
    for l, b, w, m in zip(c.layers, before, want, weights):
        assert (l.sealed, l.tail) == (32, 8)
        at = w.long().unsqueeze(-1).expand(-1, -1, -1, 16)
        now = kc.ops.kv8_read(l.rows())
        for i in (0, 1):
            kept = b[i].gather(2, at)
            assert torch.equal(now[i][:, :, 32:], kept[:, :, 32:])
            assert torch.equal(now[i][:, :, :32], rounded(kept[:, :, :32]))
        assert torch.equal(l.mass[:, :, :40], m.gather(2, w.long())) and float(l.mass[:, :, 40:].abs().max()) == 0
    feed(c, 3, 21)
    assert c.get_seq_length() == 43 and c.next_position == 93
    assert float(c.layers[0].mass[:, :, 40:43].abs().max()) == 0
    assert c.evict() == 3 and c.next_position == 93
    c.reset()
    assert c.get_seq_length() == 0 and c.next_position == 0


def test_refusals(plain):
    with pytest.raises(ValueError, match="block"):
        cache(block=16)
    with pytest.raises(ValueError, match="budget"):
        cache(budget=8, sinks=4, recent=8)
    with pytest.raises(ValueError, match="positive"):
        cache(capacity=0)
    with pytest.raises(RuntimeError, match="without a budget"):
        cache().evict()
    c = cache()
    with pytest.raises(TypeError, match="bf16"):
        c.update(torch.zeros(1, 2, 3, 16), torch.zeros(1, 2, 3, 16), 0)
    with pytest.raises(RuntimeError, match="static"):
        c.set_static(torch.zeros(()))
    feed(c, 5, 1)
    with pytest.raises(ValueError, match="batch or head"):
        c.update(*rows_of(3, 1, h=3), 0)
    for kw, what in ((dict(kv8=True), "lean"), (dict(kv8=True, lean=True, graphs=True), "eager"),
                     (dict(kv8_budget=64), "kv8_budget")):
        with pytest.raises(ValueError, match=what):
            B200TreeSpeculator.__init__(object.__new__(B200TreeSpeculator), None, None, cost_model=None,
                                        acceptance=None, **kw)


def test_batches(plain):
    c = cache(budget=64, sinks=0, recent=0)
    feed(c, 40, 1)
    feed(c, 2, 7)
    l = c.layers[0]
    one = kc.ops.kv8_read(l.rows())
    c.batch_repeat_interleave(3)
    three = kc.ops.kv8_read(l.rows())
    assert three[0].shape[0] == 3 and all(torch.equal(three[0][i], one[0][0]) for i in range(3))
    c.batch_select_indices(torch.tensor([2]))
    assert torch.equal(kc.ops.kv8_read(l.rows())[0], one[0]) and l.mass.shape[0] == 1
