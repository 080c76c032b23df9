"""Prompt attention over small values beside what its rows do not see: a NaN or
values past fp16 behind a prompt's last position or before its windows, and a
NaN key among its own positions.  The outputs are those without them.

Tolerance: values are exact in two fp16 parts, scores and weights as in
test_gpu_kv_scales; the norm of the difference stays under 1e-5 of the norm of
the output.  Scales rounded to 2^-20 for a neighbour's sake are off by 2e-4 and
up at these sizes."""
import math

import pytest
import torch

from test_gpu_kv import Filled, make_rows
from test_gpu_kv_scales import DEV, fill, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["nan", "large"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("small", [1e-3, 1e-4])
def test_prompt_beside_what_it_does_not_see(device, hd, what, small):
    """Small values, and behind the prompt's last position (in its own group of 16) or before its windows what no row
    sees: a NaN, or values past fp16."""
    f = Filled(8, 2, hd, [400], 64, seed=7)
    fill(f, torch.randn(400, 2, hd, generator=f.g, device=DEV), values(f, 400, (small,)))
    bad = torch.full((1, 2, hd), math.nan if what == "nan" else 4e5, device=DEV)
    q = f.q(150)
    want, _ = f.expected(q, [(0, 200, 150)])
    window = 80
    wantw, _ = f.expected(q, [(0, 200, 150)], window)
    for p in (350, 351, 118):   # rows 200 .. 349 see neither 350 nor, with a window of 80, 118 (121 is the first)
        f.kv.append(0, 0, 0, 0, bad.data_ptr(), bad.data_ptr(), 2 * hd, make_rows([(0, p, 1)]))
    got = f.attend(q, [(0, 200, 150)], window).double()
    f.kv.check()
    assert float((got - wantw).norm() / wantw.norm()) < 1e-5
    k, v = f.k[0][118:119].float(), f.v[0][118:119].float()
    f.kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), 2 * hd, make_rows([(0, 118, 1)]))
    got = f.attend(q, [(0, 200, 150)]).double()
    f.kv.check()
    again, _ = f.expected(q, [(0, 200, 150)])
    assert torch.equal(again, want)
    assert float((got - want).norm() / want.norm()) < 1e-5


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_small_values_beside_a_nan_key(device, hd):
    """A NaN among the keys of a prompt poisons the rows that see it; what the others read is not rounded for it."""
    f = Filled(8, 2, hd, [400], 64, seed=8)
    fill(f, torch.randn(400, 2, hd, generator=f.g, device=DEV), values(f, 400, (1e-4,)))
    q = f.q(150)
    want, _ = f.expected(q, [(0, 200, 150)])
    bad = torch.full((1, 2, hd), math.nan, device=DEV)
    f.kv.append(0, 0, 0, 0, bad.data_ptr(), bad.data_ptr(), 2 * hd, make_rows([(0, 300, 1)]))
    got = f.attend(q, [(0, 200, 150)]).double()
    f.kv.check()
    assert float((got[:100] - want[:100]).norm() / want[:100].norm()) < 1e-5
    assert torch.isnan(got[100:]).all()
