"""Attention over the 4-bit K/V cache where a head's blocks of 32 values have
very different magnitudes: an output depends on its own block's values only,
so its error is measured against those.

Tolerance, of each row and block.  With B = max_t sum_d |q_d k_td| * scale, a
score is off by at most B (2^-21 + (hd + 8) 2^-24), a weight by twice that and
2^-20 of itself, and by 2^-38 of the largest weight (2^-22 where a weight times
its block's scale passes 4, and 2^14 times that at most); rounding errors are of
either sign, so the norm of the difference stays under 1e-5 of the norm of the
values, and where scores are numbers near B, B 2^-24 more.  What is lost when a
small block is carried with a large one's power of two is 4e-4 and up.
"""
import math

import pytest
import torch

from test_gpu_kv import LAYOUTS, Filled, make_rows, stored

pytestmark = pytest.mark.gpu
DEV = "cuda"


def fill(f, k, v, pos=0):
    """Sequence 0 of `f` from position `pos` on."""
    n, w = k.shape[0], f.kv_heads * f.hd
    f.kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), w, make_rows([(0, pos, n)]))
    f.k[0][pos:pos + n], f.v[0][pos:pos + n] = stored(k), stored(v)


def check_blocks(f, q, entries, window=0):
    got = f.attend(q, entries, window).double()
    f.kv.check()
    want, _ = f.expected(q, entries, window)
    diff, size = (got - want).unflatten(-1, (-1, 32)), want.unflatten(-1, (-1, 32))
    rel = diff.norm(dim=(0, 3)) / size.norm(dim=(0, 3)).clamp(min=1e-30)   # of each head's blocks
    assert bool((rel < 1e-5 + f.b * 2 ** -24).all()), rel


def values(f, n, gains):
    """Random values, block b of every head times gains[b % len(gains)]."""
    v = torch.randn(n, f.kv_heads, f.hd, generator=f.g, device=DEV)
    for b in range(f.hd // 32):
        v[..., 32 * b:32 * b + 32] *= gains[b % len(gains)]
    return v


@pytest.mark.parametrize("heads,kv_heads,hd", [s for s in LAYOUTS if s[2] > 32])
@pytest.mark.parametrize("gains", [(128.0, 1e-2), (1e-2, 2e3), (1e3, 1e-2, 1.0), (4e5, 6e-3), (1.0, 1e-4), (1e-5, 30.0)])
def test_blocks_of_unlike_scale(device, heads, kv_heads, hd, gains):
    f = Filled(heads, kv_heads, hd, [900, 40], 32, seed=hd)
    fill(f, torch.randn(900, kv_heads, hd, generator=f.g, device=DEV), values(f, 900, gains))
    for pos in (20, 899):
        for gain in (0.1, 1.3):
            check_blocks(f, f.q(1, gain), [(0, pos, 1)])


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (16, 8, 128), (4, 1, 256), (6, 1, 96), (3, 3, 32)])
@pytest.mark.parametrize("at", [0, 3, 40, 300])
@pytest.mark.parametrize("big,small", [(1e4, 1e-2), (4e5, 1e-3), (50.0, 1e-5)])
def test_a_large_value_of_no_weight(device, heads, kv_heads, hd, at, big, small):
    """It leaves the values that have the weight as they are: in its own tile, and in those that come after."""
    n = 600
    f = Filled(heads, kv_heads, hd, [n], 64, seed=at)
    q = f.q(1)
    k = torch.randn(n, kv_heads, hd, generator=f.g, device=DEV)
    k[at] = -8 * q[0].view(kv_heads, f.group, hd)[:, 0]
    v = values(f, n, (small,))
    v[at] = big
    fill(f, k, v)
    qs = q.view(1, kv_heads, f.group, hd)[:, :, :1].expand(-1, -1, f.group, -1).reshape(1, heads, hd).contiguous()
    p = torch.softmax(torch.einsum("hd,khd->hk", qs[0].double(), f.k[0].repeat_interleave(f.group, 1)) / math.sqrt(hd), -1)
    assert float(p[:, at].max()) * big < 1e-9 * small
    check_blocks(f, qs, [(0, n - 1, 1)])


@pytest.mark.parametrize("hd", [64, 128])
def test_pairs_of_a_tile_do_not_share_a_scale(device, hd):
    """One head's weight lies on a huge value, another's on tiny ones of the same positions."""
    f = Filled(2, 1, hd, [64], 16, seed=5)
    k = torch.zeros(64, 1, hd, device=DEV)
    k[10, 0, 0], k[50, 0, 1] = 60.0, 60.0
    v = values(f, 64, (1e-3,))
    v[10] *= 3e8
    fill(f, k, v)
    q = torch.zeros(1, 2, hd, device=DEV)
    q[0, 0, 0], q[0, 1, 1] = 8.0, 8.0
    q[0, :, 2:] = torch.randn(2, hd - 2, device=DEV) * 0.1
    check_blocks(f, q, [(0, 63, 1)])


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (16, 8, 128), (6, 2, 128)])
@pytest.mark.parametrize("gains", [(128.0, 1e-2), (1e3, 1e-2, 1.0), (2e4, 1e-2), (1.0, 1e-4)])
def test_prompt_blocks_of_unlike_scale(device, heads, kv_heads, hd, gains):
    f = Filled(heads, kv_heads, hd, [700], 32, seed=hd)
    fill(f, torch.randn(700, kv_heads, hd, generator=f.g, device=DEV), values(f, 700, gains))
    check_blocks(f, f.q(300, 0.5), [(0, 400, 300)])
