"""Sealing and compaction write to memory of their own: what shares any is refused
before a launch, views that lie between each other are not (they go on to the
launch, which this machine has no device for)."""
import ctypes

import pytest
import torch

from specfit_b200 import _native as N

B, H, D, BLOCK = 2, 3, 64, 32
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are the host's")


def structure(codes, scales, tails, sealed, tail):
    """codes and scales: (K, V) tensors [B, H, ...]; as ``ops.Kv8Rows`` fills it."""
    p = lambda t: t.data_ptr()
    return N.Kv8RowsStruct(B, H, D, BLOCK, sealed, tail, p(codes[0]), p(codes[1]), codes[0].stride(0), codes[0].stride(1),
                           p(scales[0]), p(scales[1]), scales[0].stride(0), scales[0].stride(1), p(tails[0]), p(tails[1]),
                           tails[0].stride(0), tails[0].stride(1))


class Buffers:
    def __init__(self, tokens, tail):
        self.codes = [torch.zeros(B, H, tokens, D, dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.zeros(B, H, tokens // BLOCK) for _ in range(2)]
        self.tails = [torch.zeros(B, H, tail, D, dtype=torch.bfloat16) for _ in range(2)]

    def of(self, sealed, tail):
        return structure(self.codes, self.scales, self.tails, sealed, tail)


def compact(src, out, n, keep, mass=None, mass_out=None):
    m = (None, 0, 0, None, 0, 0) if mass is None else (mass.data_ptr(), mass.stride(0), mass.stride(1),
                                                       mass_out.data_ptr(), mass_out.stride(0), mass_out.stride(1))
    return N.lib.sf_kv8_compact(ctypes.addressof(src), keep.data_ptr(), n, ctypes.addressof(out), *m, None)


def refused(rc):
    if rc == N.SF_ERR_INVALID_ARGUMENT:
        assert "overlap" in N.last_error()
        return True
    assert rc == N.SF_ERR_CUDA  # the launch
    return False


def test_compaction_into_memory_of_its_own_is_not_refused():
    src, out = Buffers(128, 10), Buffers(64, 10)
    keep = torch.zeros(B, H, 70, dtype=torch.int32)
    mass, new = torch.zeros(B, H, 138), torch.zeros(B, H, 70)
    assert not refused(compact(src.of(128, 10), out.of(64, 6), 70, keep))
    assert not refused(compact(src.of(128, 10), out.of(64, 6), 70, keep, mass, new))


@pytest.mark.parametrize("what", ["codes", "scales", "tails"])
@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("other", [0, 1])
def test_a_target_inside_a_source_buffer_is_refused(what, kv, other):
    src, out = Buffers(192, 40), Buffers(64, 40)
    keep = torch.zeros(B, H, 70, dtype=torch.int32)
    theirs = getattr(src, what)[other]
    if what == "codes":
        view = theirs[:, :, 64:128]
    elif what == "scales":
        view = theirs[:, :, 2:4]
    else:
        view = theirs[:, :, 8:20]
    mine = getattr(out, what)
    # K and V share strides, so both get a view of that kind; only one lies in the source.
    spare = torch.zeros(theirs.shape, dtype=theirs.dtype)
    views = [spare[:, :, : view.shape[2]], spare[:, :, : view.shape[2]]]
    views[1 - kv] = torch.zeros(theirs.shape, dtype=theirs.dtype)[:, :, : view.shape[2]]
    views[kv] = view
    mine[:] = views
    assert refused(compact(src.of(192, 40), out.of(64, 6), 70, keep))


def test_targets_that_share_memory_with_each_other_or_other_inputs_are_refused():
    keep = torch.zeros(B, H, 70, dtype=torch.int32)
    mass = torch.zeros(B, H, 400)
    for change in ("kv", "mass", "keep"):
        src, out = Buffers(128, 10), Buffers(64, 10)
        new = torch.zeros(B, H, 70)
        k = keep
        if change == "kv":
            out.codes[1] = out.codes[0]
        elif change == "mass":
            new = mass[:, :, 100:170]
        else:
            k = new.view(torch.int32)
        assert refused(compact(src.of(128, 10), out.of(64, 6), 70, k, mass, new)), change


def test_views_between_each_other_are_not_refused():
    """Both halves of one buffer, head by head, and heads taken in turn."""
    keep = torch.zeros(B, H, 70, dtype=torch.int32)
    src, out = Buffers(128, 10), Buffers(64, 10)
    both = [torch.zeros(B, H, 192, D, dtype=torch.uint8) for _ in range(2)]
    src.codes, out.codes = [t[:, :, :128] for t in both], [t[:, :, 128:] for t in both]
    assert not refused(compact(src.of(128, 10), out.of(64, 6), 70, keep))
    out.codes = [t[:, :, 127:191] for t in both]
    assert refused(compact(src.of(128, 10), out.of(64, 6), 70, keep))
    two = [torch.zeros(B, 2 * H, 128, D, dtype=torch.uint8) for _ in range(2)]
    src.codes, out.codes = [t[:, ::2] for t in two], [t[:, 1::2] for t in two]
    assert not refused(compact(src.of(128, 10), out.of(64, 6), 70, keep))
    out.codes = [two[0][:, 1::2], two[1][:, :H]]
    out.codes[1] = torch.as_strided(two[1], out.codes[0].shape, out.codes[0].stride())
    assert refused(compact(src.of(128, 10), out.of(64, 6), 70, keep))


def seal(k, v, buffers, first, blocks):
    rows = buffers.of(buffers.codes[0].shape[2], 0)
    return N.lib.sf_kv8_seal(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), ctypes.addressof(rows),
                             first, blocks, None)


def test_sealing():
    k, v = (torch.zeros(B, H, 64, D, dtype=torch.bfloat16) for _ in range(2))
    assert not refused(seal(k, v, Buffers(128, 0), 1, 2))
    assert not refused(seal(k, k, Buffers(128, 0), 1, 2))  # read twice
    one = Buffers(128, 0)
    one.codes[1] = one.codes[0]
    assert refused(seal(k, v, one, 1, 2))
    one = Buffers(128, 0)
    one.scales[1] = one.scales[0]
    assert refused(seal(k, v, one, 1, 2))
    # Codes laid over the rows that they are made of, and beside them: a head's 64 tokens of
    # codes take the memory of its first 32 rows.
    wide = torch.zeros(B, H, 256, D, dtype=torch.bfloat16)
    stride = (H * 512 * D, 512 * D, D, 1)
    one = Buffers(128, 0)
    one.codes = [torch.as_strided(t, (B, H, 128, D), stride)
                 for t in (wide.view(torch.uint8), torch.zeros(B, H, 512, D, dtype=torch.uint8))]
    other = torch.zeros_like(wide)[:, :, :64]
    assert refused(seal(wide[:, :, :64], other, one, 0, 2))
    assert refused(seal(wide[:, :, 31:95], other, one, 0, 2))
    assert not refused(seal(wide[:, :, 32:96], other, one, 0, 2))


def test_keys_that_are_the_values_may_share_their_buffers():
    """One content, written twice: both sides must be one."""
    k, v = (torch.zeros(B, H, 64, D, dtype=torch.bfloat16) for _ in range(2))
    one = Buffers(128, 10)
    one.codes[1], one.scales[1], one.tails[1] = one.codes[0], one.scales[0], one.tails[0]
    assert not refused(seal(k, k, one, 0, 2))
    assert refused(seal(k, v, one, 0, 2))
    keep = torch.zeros(B, H, 70, dtype=torch.int32)
    out = Buffers(64, 10)
    out.codes[1], out.scales[1], out.tails[1] = out.codes[0], out.scales[0], out.tails[0]
    assert not refused(compact(one.of(128, 10), out.of(64, 6), 70, keep))
    one.tails[1] = torch.zeros_like(one.tails[0])
    assert refused(compact(one.of(128, 10), out.of(64, 6), 70, keep))
