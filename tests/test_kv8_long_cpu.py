"""Long passes over an 8-bit cache: the calls that a pass is made of, on the CPU; and
importing the package where torch has no CUDA."""
import subprocess
import sys
import types
from pathlib import Path

import pytest
import torch

from specfit_b200.runtime import lean_forward as lf


class Layer:
    """Stands for a cache layer after ``end``: a view remembers where it ends."""

    def __init__(self, heads, length, scored):
        self._h, self.length, self.scored = heads, length, scored
        self.mass = object()

    def rows(self, end=None):
        return types.SimpleNamespace(length=self.length if end is None else end)


@pytest.fixture
def calls(monkeypatch):
    made = []

    def attention(q, rows, bits, prefix, out=None, return_lse=False):
        assert q.shape[1] // 2 * q.shape[2] < 1 << 20  # the operators' limit
        assert bits.shape[:2] == (q.shape[0], q.shape[2]) and out.shape[:2] == (q.shape[0], q.shape[2])
        made.append(("attention", q.storage_offset(), q.shape[2], rows.length, prefix, bits))
        return (out, "lse") if return_lse else out

    def mass(q, lse, rows, bits, prefix, m):
        assert lse == "lse"
        made.append(("mass", q.storage_offset(), q.shape[2], rows.length, prefix, bits))

    monkeypatch.setattr(lf.ops, "kv8_tree_attention", attention)
    monkeypatch.setattr(lf.ops, "kv8_attention_mass", mass)
    monkeypatch.setattr(lf, "_causal_bits", lambda n, dev: torch.zeros(n, 1, dtype=torch.int32))
    return made


def q_and_out(batch, heads, rows):
    # One element a row, expanded: nothing of the pass's true size.
    q = torch.empty(1, 1, rows, 1).expand(batch, heads, rows, 1)
    return q, torch.empty(1, rows, 1, 1).expand(batch, rows, heads, 1)


@pytest.mark.parametrize("rows,heads", [(1, 8), (16384, 16), (16385, 16), (131072, 16), (400000, 64), (300, 1 << 13)])
@pytest.mark.parametrize("scored", [False, True])
def test_a_causal_pass_of_any_length(calls, rows, heads, scored):
    q, out = q_and_out(2, heads, rows)
    layer = Layer(2, 37 + rows, scored)
    lf.attend_kv8(layer, q, None, out)
    at = 0
    for what, first, n, length, prefix, bits in calls:
        if what == "mass":
            assert (first, n, length, prefix) == last
            continue
        # Row r sees the 37 + r keys before it and itself: the call's keys end with its last row.
        assert first == at and prefix == 37 + at and length == 37 + at + n
        at += n
        last = (first, n, length, prefix)
    assert at == rows
    assert sum(c[0] == "mass" for c in calls) == (len(calls) // 2 if scored else 0)


def test_a_masked_pass_keeps_its_words(calls):
    q, out = q_and_out(1, 128, 40000)
    words = torch.arange(40000, dtype=torch.int32).view(1, 40000, 1)
    lf.attend_kv8(Layer(2, 50000, False), q, words, out)
    assert [c[3:5] for c in calls] == [(50000, 0)] * len(calls) and len(calls) > 1
    assert torch.equal(torch.cat([c[5] for c in calls], 1), words)


def test_the_package_imports_where_torch_has_no_cuda():
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "import specfit_b200.runtime\n"
            "from specfit_b200 import ops\n"
            "try:\n"
            "    ops.kv_keep_heaviest(torch.zeros(1, 1, 4), 4, 2)\n"
            "except ValueError as e:\n"
            "    assert 'CUDA' in str(e)\n"
            "else:\n"
            "    raise SystemExit('not refused')\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr
