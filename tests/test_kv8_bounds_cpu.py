"""The bounds that the 8-bit cache's attention is held to notice what is wrong: an
answer of zeros, a range of keys left out or counted twice, values in another
block's scale; and let pass what they were derived for.  The mistakes are planted in
the definition, on the CPU."""
import pytest
import torch

import kv8_bounds as kb


def case(rows=3, hq=4, hkv=2, total=4096, d=128, seed=1):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(1, hq, rows, d, generator=g).to(torch.bfloat16)
    k = torch.randn(1, hkv, total, d, generator=g).to(torch.bfloat16)
    v = torch.randn(1, hkv, total, d, generator=g).to(torch.bfloat16)
    v[:, :, ::3] *= 4
    vis = torch.ones(1, rows, total, dtype=torch.bool)
    return q, k, v, vis, kb.attention(q, k, v, vis, d ** -0.5)


def answer(want):
    return want["out"].transpose(1, 2).to(torch.bfloat16)


@pytest.mark.parametrize("total", [17, 529, 4096, 32768])
def test_the_rounded_definition_passes(total):
    q, k, v, vis, want = case(total=total)
    assert kb.off(answer(want), want) is None
    assert kb.lse_off(want["lse"].float(), want) is None


@pytest.mark.parametrize("total", [529, 4096, 32768])
def test_zeros_do_not_pass(total):
    *_, want = case(total=total)
    assert kb.off(torch.zeros_like(answer(want)), want) is not None


@pytest.mark.parametrize("total,length", [(529, 32), (4096, 128), (32768, 320)])
def test_a_range_of_keys_left_out_does_not_pass(total, length):
    """One of the key ranges that a long context is split into (a hundredth of it)."""
    q, k, v, vis, want = case(total=total)
    less = vis.clone()
    less[:, :, total // 2: total // 2 + length] = False
    wrong = kb.attention(q, k, v, less, 128 ** -0.5)
    assert kb.off(answer(wrong), want) is not None


def test_a_range_that_counts_twice_does_not_pass():
    q, k, v, vis, want = case()
    again = torch.cat([k, k[:, :, :128]], 2), torch.cat([v, v[:, :, :128]], 2)
    wrong = kb.attention(q, *again, torch.ones(1, 3, 4096 + 128, dtype=torch.bool), 128 ** -0.5)
    assert kb.off(answer(wrong), want) is not None


def test_a_block_in_another_scale_does_not_pass():
    q, k, v, vis, want = case()
    for at, factor in ((64, 0.0), (640, 0.5), (1280, 2.0)):
        other = v.clone()
        other[:, :, at: at + 64] *= factor
        assert kb.off(answer(kb.attention(q, k, other, vis, 128 ** -0.5)), want) is not None, (at, factor)


def test_probabilities_in_fp16_pass():
    q, k, v, vis, want = case(total=32768)
    x = torch.einsum("bhgrd,bhkd->bhgrk", q.double().view(1, 2, 2, 3, 128), k.double()) * 128 ** -0.5
    p = torch.softmax(x, -1)
    half = (p * 2.0 ** 7 / p.amax(-1, keepdim=True)).to(torch.float16).double() * p.amax(-1, keepdim=True) / 2.0 ** 7
    o = torch.einsum("bhgrk,bhkd->bhgrd", half, v.double()).reshape(1, 4, 3, 128).transpose(1, 2)
    assert kb.off(o.to(torch.bfloat16), want) is None


def test_rows_that_see_nothing():
    q, k, v, vis, _ = case(total=64)
    vis[:, 1] = False
    want = kb.attention(q, k, v, vis, 128 ** -0.5)
    out = answer(want)
    assert float(out[:, 1].abs().max()) == 0 and kb.off(out, want) is None
    out[:, 1, 0, 0] = 2.0 ** -20
    assert kb.off(out, want) is not None
