"""The paged 4-bit K/V cache on the GPU against plain 64-bit implementations:
append (norm, rotation, Q4_0 blocks), read, and attention.

Tolerances.  q after norm and rotation is rounded once from 64 bits: half a
step of fp32, 2^-24 of the value.  Stored values are compared bit for bit.
Attention: with B = max_t sum_d |q_d k_td| * scale, a score is off by at most
B (2^-21 + (hd + 8) 2^-24) (q in two 11-bit parts, fp32 sums), a weight by
twice that plus 2^-21 (exponential and its rounding in two 11-bit parts), and
the sums over n positions by n 2^-24 of sum p |v|; all relative to
max |v|.  Each wrong digit of a code, a mask or a page would be off by 2^-4.
"""
import math

import pytest
import torch

from brewference_b200 import _native as N
from brewference_b200.api import ROPE_HALF, ROPE_INTERLEAVED, ROPE_NONE, KvCache, KvRope, KvRows

pytestmark = pytest.mark.gpu
EPS = 1e-6
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make_rows(entries, n_rows=None):
    """entries: (seq, pos, rows).  Returns KvRows and the arrays it points to."""
    seq, pos = i32([e[0] for e in entries]), i32([e[1] for e in entries])
    offs = [0]
    for e in entries:
        offs.append(offs[-1] + e[2])
    start = i32(offs)
    n_rows = offs[-1] if n_rows is None else n_rows
    r = KvRows(seq.data_ptr(), pos.data_ptr(), len(entries), n_rows, max([e[2] for e in entries] + [1]), start.data_ptr())
    r.keep = (seq, pos, start)
    return r


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def rotated(x, pos, mode, base, scale, w):
    """x [rows][heads][hd] in 64 bits."""
    x = x.double()
    hd = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    if mode == ROPE_NONE:
        return x
    a = pos.double()[:, None] * scale * base ** (-torch.arange(0, hd, 2, device=DEV).double() / hd)
    c, s = a.cos()[:, None], a.sin()[:, None]
    i0 = torch.arange(hd // 2, device=DEV) if mode == ROPE_HALF else torch.arange(0, hd, 2, device=DEV)
    i1 = i0 + (hd // 2 if mode == ROPE_HALF else 1)
    y = x.clone()
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def stored(x):
    """The values that Q4_0 blocks of fp32 x stand for (64 bits)."""
    b = x.float().unflatten(-1, (-1, 32))
    top = torch.gather(b, -1, b.abs().argmax(-1, keepdim=True))
    d = (top * -0.125).clamp(-65504, 65504)
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    q = torch.trunc(b * inv + 8.5).clamp(0, 15)
    return ((q - 8).double() * d.half().double()).flatten(-2)


class Filled:
    """A cache whose sequences hold random keys and values, and what they stand for."""

    def __init__(self, heads, kv_heads, hd, lens, page, seed=0, max_tokens=None, spare=0, vgain=1.0):
        g = gen(seed)
        self.heads, self.kv_heads, self.hd, self.group = heads, kv_heads, hd, heads // kv_heads
        per = [-(-n // page) for n in lens]
        self.kv = KvCache(1, heads, kv_heads, hd, len(lens), max_tokens or max(lens + [1]), page, sum(per) + spare or 1)
        for part in (3, 2, 1):   # pages of different sequences interleave
            for i, n in enumerate(lens):
                self.kv.reserve(i, -(-n // part))
        t = sum(lens)
        k = torch.randn(t, kv_heads, hd, generator=g, device=DEV) * torch.exp(torch.randn(kv_heads, hd, generator=g, device=DEV) / 2)
        v = torch.randn(t, kv_heads, hd, generator=g, device=DEV) * vgain
        if t:
            rows = make_rows([(i, 0, n) for i, n in enumerate(lens)])
            self.kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), kv_heads * hd, rows)
        self.k = list(torch.split(stored(k), lens))
        self.v = list(torch.split(stored(v), lens))
        self.ws = torch.zeros(self.kv.workspace_bytes(), dtype=torch.uint8, device=DEV)
        self.g = g

    def q(self, t, gain=1.3):
        return torch.randn(t, self.heads, self.hd, generator=self.g, device=DEV) * gain

    def attend(self, q, entries, window=0, scale=0.0, out=None, stream=0):
        out = torch.full_like(q, float("nan")) if out is None else out
        rows = make_rows(entries, q.shape[0])
        self.kv.attend(0, out.data_ptr(), self.heads * self.hd, q.data_ptr(), self.heads * self.hd, rows, window,
                       self.ws.data_ptr(), scale, stream)
        torch.cuda.synchronize()
        return out

    def expected(self, q, entries, window=0, scale=0.0):
        """(out, tolerance of each row's values) in 64 bits."""
        scale = scale or 1 / math.sqrt(self.hd)
        outs, tols = [], []
        at = 0
        self.b = 0.0
        for seq, pos, n in entries:
            k = self.k[seq][:pos + n].repeat_interleave(self.group, 1)
            v = self.v[seq][:pos + n].repeat_interleave(self.group, 1)
            qi = q[at:at + n].double()
            at += n
            x = torch.einsum("rhd,khd->hrk", qi, k) * scale
            t, last = torch.arange(pos + n, device=DEV), pos + torch.arange(n, device=DEV)[:, None]
            dead = (t > last) | ((t <= last - window) if window else torch.zeros_like(t > last))
            p = torch.softmax(x.masked_fill(dead, -math.inf), -1)
            outs.append(torch.einsum("hrk,khd->rhd", p, v))
            b = torch.einsum("rhd,khd->hrk", qi.abs(), k.abs()).amax() * scale if n and pos + n else 0.0
            self.b = max(self.b, float(b))
            ds = b * (2 ** -21 + (self.hd + 8) * 2 ** -24)
            tols.append(torch.full((n, 1, 1), float((2 * ds + 2 ** -20 + (pos + n + 64) * 2 ** -24) * v.abs().max())
                                   if n else 0.0, device=DEV))
        return torch.cat(outs), torch.cat(tols)

    def check(self, q, entries, window=0, scale=0.0):
        got = self.attend(q, entries, window, scale).double()
        self.kv.check()
        want, tol = self.expected(q, entries, window, scale)
        assert bool(((got - want).abs() <= tol).all()), ((got - want).abs() / tol).max()
        if want.numel():
            # Rounding errors are of either sign: far from adding up.  But scores near B are numbers with steps of
            # B 2^-23 in 32 bits (0.012 at B = 10^5, which q of 10^4 reaches), and half a step moves a weight by
            # B 2^-24 of itself: that much cannot be asked for.
            assert float((got - want).norm() / want.norm().clamp(min=1e-30)) < 1e-5 + self.b * 2 ** -24


# ---- append and read ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,hd,page,mode,norm", [
    (9, 3, 64, 64, ROPE_INTERLEAVED, False), (16, 8, 128, 32, ROPE_HALF, True), (4, 1, 256, 16, ROPE_HALF, True),
    (28, 4, 128, 128, ROPE_HALF, False), (3, 3, 32, 16, ROPE_INTERLEAVED, True), (5, 1, 96, 64, ROPE_HALF, True),
    (6, 2, 96, 16, ROPE_INTERLEAVED, False), (2, 2, 32, 32, ROPE_HALF, False), (8, 4, 256, 64, ROPE_INTERLEAVED, False),
    (7, 1, 64, 16, ROPE_NONE, True), (1, 1, 128, 64, ROPE_NONE, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_and_read(device, heads, kv_heads, hd, page, mode, norm, in_place):
    g = gen(heads * 131 + hd)
    entries = [(2, 5, 37), (0, 0, 1), (3, 90000, 0), (1, 16383, 19), (4, 0, 16)]
    t, extra, pad = sum(e[2] for e in entries), 3, 8
    kv = KvCache(2, heads, kv_heads, hd, 5, 20000, page, 2 * (20000 // page))
    for s, pos, n in entries:
        kv.reserve(s, pos + n if n else 0)
    ldq, ldkv = heads * hd + pad, kv_heads * hd + pad
    q = torch.randn(t + extra, ldq, generator=g, device=DEV)
    k = torch.randn(t + extra, ldkv, generator=g, device=DEV) * 2
    v = torch.randn(t + extra, ldkv, generator=g, device=DEV)
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    wq = 1 + torch.randn(hd, generator=g, device=DEV) / 4 if norm else None
    wk = 1 + torch.randn(hd, generator=g, device=DEV) / 4 if norm else None
    rope = KvRope(mode, 1e6, 0.25, wq.data_ptr() if norm else 0, wk.data_ptr() if norm else 0, EPS)
    out = q if in_place else torch.full_like(q, 7.0)
    rows = make_rows(entries, t + extra)
    kv.append(1, out.data_ptr(), q.data_ptr(), ldq, k.data_ptr(), v.data_ptr(), ldkv, rows, rope)
    kr, vr = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    kv.read(1, kr.data_ptr(), vr.data_ptr(), ldkv, rows)
    kv.check()
    pos = torch.cat([p + torch.arange(n, device=DEV) for _, p, n in entries])
    want_q = rotated(q0[:t, :heads * hd].view(t, heads, hd), pos, mode, 1e6, 0.25, wq)
    got_q = out[:t, :heads * hd].view(t, heads, hd).double()
    # half a step, and what 64 bits lose where the rotation cancels
    assert bool(((got_q - want_q).abs() <= want_q.abs() * 2 ** -24 * 1.0001 + 1e-13).all())
    want_k = stored(rotated(k0[:t, :kv_heads * hd].view(t, kv_heads, hd), pos, mode, 1e6, 0.25, wk))
    want_v = stored(v0[:t, :kv_heads * hd].view(t, kv_heads, hd))
    assert torch.equal(kr[:t, :kv_heads * hd].view(t, kv_heads, hd), want_k.float())
    assert torch.equal(vr[:t, :kv_heads * hd].view(t, kv_heads, hd), want_v.float())
    # what no entry has, and the padding of the rows, is as it was
    assert torch.equal(k, k0) and torch.equal(v, v0)
    assert bool((kr[t:] == 7).all()) and bool((vr[t:] == 7).all()) and bool((kr[:, kv_heads * hd:] == 7).all())
    keep = q0 if in_place else torch.full_like(q, 7.0)
    assert torch.equal(out[t:], keep[t:]) and torch.equal(out[:, heads * hd:], keep[:, heads * hd:])
    # layer 0 of the same pages was not touched
    kv.read(0, kr.data_ptr(), 0, ldkv, rows)
    torch.cuda.synchronize()
    assert float(kr[:t, :kv_heads * hd].abs().max()) == 0


def test_append_one_token_at_a_time_equals_at_once(device):
    """Neighbouring positions share words of the layout: each append leaves the others."""
    heads, hd, n = 2, 64, 45
    g = gen(5)
    k, v = torch.randn(n, heads, hd, generator=g, device=DEV), torch.randn(n, heads, hd, generator=g, device=DEV)
    a, b = KvCache(1, heads, heads, hd, 1, n, 16), KvCache(1, heads, heads, hd, 1, n, 16)
    a.reserve(0, n)
    b.reserve(0, n)
    rows = make_rows([(0, 0, n)])
    a.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), heads * hd, rows)
    order = torch.randperm(n).tolist()
    for i in order + order[:7]:
        one = make_rows([(0, i, 1)])
        b.append(0, 0, 0, 0, k[i].data_ptr(), v[i].data_ptr(), heads * hd, one)
    outs = []
    for c in (a, b):
        o = torch.empty(2, n, heads, hd, device=DEV)
        c.read(0, o[0].data_ptr(), o[1].data_ptr(), heads * hd, rows)
        c.check()
        outs.append(o)
    assert torch.equal(outs[0], outs[1])


def test_block_extremes(device):
    """Zero blocks, ties of magnitude, tiny and huge values, saturation, NaN."""
    hd = 64
    x = torch.zeros(8, 1, hd, device=DEV)
    x[1, 0, 3], x[1, 0, 9] = 2.0, -2.0                 # the first of equal magnitude decides
    x[2, 0, 3], x[2, 0, 9] = -2.0, 2.0
    x[3] = torch.linspace(-1e-6, 1e-6, hd, device=DEV)  # scales among fp16's subnormals
    x[4] = torch.linspace(-4e5, 5e5, hd, device=DEV)
    x[5, 0, 0], x[5, 0, 1] = 1e9, -3e5                 # past what fp16 scales hold
    x[6] = torch.linspace(-1e-30, 1e-30, hd, device=DEV)
    x[7] = torch.linspace(-7, 8, hd, device=DEV)
    kv = KvCache(1, 1, 1, hd, 1, 8, 16)
    kv.reserve(0, 8)
    rows = make_rows([(0, 0, 8)])
    kv.append(0, 0, 0, 0, x.data_ptr(), x.data_ptr(), hd, rows)
    k, v = torch.empty_like(x), torch.empty_like(x)
    kv.read(0, k.data_ptr(), v.data_ptr(), hd, rows)
    kv.check()
    want = stored(x).float()
    assert torch.equal(k, want) and torch.equal(v, want)
    assert torch.isfinite(k).all() and float(k[5].abs().max()) == 8 * 65504


# ---- attention ----------------------------------------------------------------------------------------------------------

LAYOUTS = [(9, 3, 64), (16, 8, 128), (4, 1, 256), (28, 4, 128), (2, 2, 32), (6, 1, 96), (12, 1, 64), (32, 2, 128), (8, 4, 256)]


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_attend_single_tokens(device, heads, kv_heads, hd, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 300, 513, 1500]
    f = Filled(heads, kv_heads, hd, lens, page, seed=heads + hd)
    f.check(f.q(len(lens)), [(i, n - 1, 1) for i, n in enumerate(lens)])


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 511, 4000])
def test_attend_windows(device, page, window):
    lens = [1, 16, 100, 130, 777, 1025]
    f = Filled(4, 1, 256, lens, page, seed=window) if page == 32 else Filled(8, 2, 64, lens, page, seed=window)
    f.check(f.q(len(lens)), [(i, n - 1, 1) for i, n in enumerate(lens)], window)
    f.check(f.q(33 + 1 + 40), [(4, 500, 33), (0, 0, 1), (5, 1025 - 40, 40)], window)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_attend_chunks(device, heads, kv_heads, hd):
    """Several rows a sequence: from the start, in the middle, ragged, empty entries, the same sequence twice."""
    lens = [200, 64, 1, 411, 90]
    f = Filled(heads, kv_heads, hd, lens, 32, seed=hd)
    entries = [(0, 0, 200), (3, 411 - 77, 77), (2, 0, 1), (1, 3, 0), (1, 30, 5), (4, 17, 3), (1, 30, 5), (3, 100, 2)]
    f.check(f.q(sum(e[2] for e in entries)), entries)


def test_attend_prompt_of_many_tiles(device):
    f = Filled(16, 8, 128, [1333], 64, seed=3)
    f.check(f.q(1333), [(0, 0, 1333)])


def test_attend_many_sequences(device):
    lens = [1 + (i * 37) % 211 for i in range(300)]
    f = Filled(4, 2, 64, lens, 16, seed=9)
    f.check(f.q(300), [(i, n - 1, 1) for i, n in enumerate(lens)])


def test_attend_long(device):
    """One sequence over every CTA of the device, and a short one beside it."""
    f = Filled(7, 1, 128, [40011, 5], 64, seed=4)
    f.check(f.q(2), [(0, 40010, 1), (1, 4, 1)])


def test_attend_without_row_start_and_with_strides(device):
    f = Filled(4, 2, 64, [50, 20, 70], 16, seed=6)
    ld = 4 * 64 + 12
    buf = torch.randn(3, ld, generator=f.g, device=DEV)
    out = torch.full((3, ld + 4), 5.0, device=DEV)
    seq, pos = i32([2, 0, 1]), i32([69, 49, 19])
    f.kv.attend(0, out.data_ptr(), ld + 4, buf.data_ptr(), ld, KvRows(seq.data_ptr(), pos.data_ptr(), 3), 0, f.ws.data_ptr(), 0.3)
    f.kv.check()
    want, tol = f.expected(buf[:, :256].reshape(3, 4, 64), [(2, 69, 1), (0, 49, 1), (1, 19, 1)], 0, 0.3)
    assert bool(((out[:, :256].reshape(3, 4, 64).double() - want).abs() <= tol).all())
    assert bool((out[:, 256:] == 5).all())


def test_attend_sees_nothing_behind_its_position(device):
    """NaN and infinities at later positions, in the same group and page, and before the window."""
    f = Filled(4, 2, 64, [100], 64, seed=8)
    bad = torch.full((1, 2, 64), float("nan"), device=DEV)
    inf = torch.full((1, 2, 64), float("inf"), device=DEV)
    for p in (41, 42, 47, 48, 63, 64, 99, 10, 0):
        x = bad if p % 2 else inf
        f.kv.append(0, 0, 0, 0, x.data_ptr(), x.data_ptr(), 128, make_rows([(0, p, 1)]))
    for pos, rows in ((40, 1), (38, 3), (25, 16)):
        f.check(f.q(rows), [(0, pos, rows)], window=15)   # sees 11 .. 40 at most
    # and the values that are NaN do come through where they are seen
    assert torch.isnan(f.attend(f.q(1), [(0, 41, 1)])).all()


def test_pages_of_a_released_sequence(device):
    """A page returns with what it held: a new owner sees only its own positions."""
    kv = KvCache(1, 2, 1, 64, 3, 64, 16, 4)
    assert kv.info()[1] == 4
    x = torch.full((64, 1, 64), float("nan"), device=DEV)
    kv.reserve(0, 50)
    assert kv.info()[1] == 0
    kv.reserve(0, 10)            # it only grows
    kv.append(0, 0, 0, 0, x.data_ptr(), x.data_ptr(), 64, make_rows([(0, 0, 64)]))
    with pytest.raises(N.IllegalStateException) as e:
        kv.reserve(1, 1)
    assert e.value.code == N.ERR_CONTEXT_FULL
    with pytest.raises(N.IllegalStateException):
        kv.reserve(1, 65)
    kv.release(0)
    kv.release(0)
    assert kv.info()[1] == 4
    kv.reserve(2, 20)
    y = torch.randn(18, 1, 64, device=DEV)
    kv.append(0, 0, 0, 0, y.data_ptr(), y.data_ptr(), 64, make_rows([(2, 0, 18)]))
    q, out = torch.randn(1, 2, 64, device=DEV), torch.empty(1, 2, 64, device=DEV)
    ws = torch.zeros(kv.workspace_bytes(), dtype=torch.uint8, device=DEV)
    kv.attend(0, out.data_ptr(), 128, q.data_ptr(), 128, make_rows([(2, 17, 1)]), 0, ws.data_ptr())
    kv.check()
    p = torch.softmax(torch.einsum("hd,kd->hk", q[0].double(), stored(y)[:, 0]) / 8, -1)
    assert float((out[0].double() - p @ stored(y)[:, 0]).abs().max()) < 1e-5 * 4
    # the released sequence has no positions
    kv.attend(0, out.data_ptr(), 128, q.data_ptr(), 128, make_rows([(0, 0, 1)]), 0, ws.data_ptr())
    with pytest.raises(N.IllegalStateException):
        kv.check()


@pytest.mark.parametrize("gain,vgain", [(1e4, 1.0), (1e-6, 1.0), (1.3, 1e-7), (1.3, 4e4), (0.0, 1.0), (30.0, 1e-3)])
def test_attend_magnitudes(device, gain, vgain):
    """Sharp and flat softmax, and values at both ends of the scales' range."""
    f = Filled(16, 8, 128, [700, 40], 64, seed=11, vgain=vgain)
    f.check(f.q(2, gain), [(0, 699, 1), (1, 39, 1)])
    f.check(f.q(90, gain), [(0, 610, 90)])


def test_attend_values_of_mixed_scale(device):
    """Value blocks from 1e-6 to 1e4 in one sequence, zero blocks among them, large ones late."""
    f = Filled(4, 1, 128, [600], 64, seed=12)
    v = torch.randn(600, 1, 128, generator=f.g, device=DEV) * torch.logspace(-6, 4, 600, device=DEV)[:, None, None]
    v[::7] = 0
    k = torch.randn(600, 1, 128, generator=f.g, device=DEV)
    f.kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), 128, make_rows([(0, 0, 600)]))
    f.k, f.v = [stored(k)], [stored(v)]
    for pos in (3, 99, 250, 599):
        f.check(f.q(1), [(0, pos, 1)])
    f.check(f.q(64), [(0, 500, 64)])


def test_bad_rows_are_skipped_and_told(device):
    """Each bad entry is refused by the kernels' own checks: nothing is read or written for it."""
    f = Filled(4, 2, 64, [40, 20], 16, seed=13)
    q = f.q(6)
    for bad in [(2, 0, 1), (-1, 0, 1), (0, -1, 1), (0, 48, 1), (1, 32, 1), (1, 2 ** 31 - 1, 1)]:
        for good in ([], [(0, 39, 1)]):
            entries = good + [bad]
            out = f.attend(q, entries)
            with pytest.raises(N.IllegalStateException):
                f.kv.check()
            f.kv.check()   # told once
            assert torch.isnan(out[len(good):]).all()
            if good:
                want, tol = f.expected(q[:1], good)
                assert bool(((out[:1].double() - want).abs() <= tol).all())
            k = torch.randn(6, 2, 64, device=DEV)
            q_out = torch.full_like(q, 3.0)
            rows = make_rows([bad], 6)
            f.kv.append(0, q_out.data_ptr(), q.data_ptr(), 256, k.data_ptr(), k.data_ptr(), 128, rows)
            with pytest.raises(N.IllegalStateException):
                f.kv.check()
            assert bool((q_out == 3).all())
            k_out = torch.full_like(k, 3.0)
            f.kv.read(0, k_out.data_ptr(), k_out.data_ptr(), 128, rows)
            with pytest.raises(N.IllegalStateException):
                f.kv.check()
            assert bool((k_out == 3).all())
    # row numbers outside the buffers, and more rows than max_rows
    seq, pos = i32([0]), i32([0])
    for start, n_rows, max_rows in (([0, 7], 6, 9), ([-1, 1], 6, 6), ([3, 2], 6, 6), ([0, 3], 6, 2), ([6, 8], 6, 6)):
        st = i32(start)
        out = torch.full_like(q, 3.0)
        f.kv.attend(0, out.data_ptr(), 256, q.data_ptr(), 256,
                    KvRows(seq.data_ptr(), pos.data_ptr(), 1, n_rows, max_rows, st.data_ptr()), 0, f.ws.data_ptr())
        with pytest.raises(N.IllegalStateException):
            f.kv.check()
        assert bool((out == 3).all())
    f.check(q[:1], [(1, 19, 1)])


def test_refusals(device):
    kv = KvCache(1, 4, 2, 64, 2, 64, 16)
    kv.reserve(0, 64)
    ws = torch.zeros(kv.workspace_bytes(), dtype=torch.uint8, device=DEV)
    x = torch.zeros(8, 256, device=DEV)
    p, w = x.data_ptr(), ws.data_ptr()
    rows = make_rows([(0, 0, 2)])
    s, t = rows.keep[0].data_ptr(), rows.keep[1].data_ptr()
    good_a = dict(layer=0, q_out_ptr=p, q_ptr=p, ldq=256, k_ptr=p, v_ptr=p, ldkv=128, rows=rows)
    for bad in (dict(layer=1), dict(layer=-1), dict(k_ptr=0), dict(v_ptr=0), dict(q_ptr=0), dict(q_out_ptr=0), dict(ldq=252),
                dict(ldq=257), dict(ldkv=124), dict(k_ptr=p + 4), dict(q_out_ptr=p + 8), dict(rows=KvRows(0, t, 1)),
                dict(rows=KvRows(s, 0, 1)), dict(rows=KvRows(s, t, -1)), dict(rows=KvRows(s, t, 2049)),
                dict(rows=KvRows(s, t, 1, 2, 1)), dict(rows=KvRows(s, t, 1, 1, 2)), dict(rows=KvRows(s + 2, t, 1)),
                dict(rope=KvRope(3)), dict(rope=KvRope(ROPE_HALF, 0.0)), dict(rope=KvRope(ROPE_HALF, math.inf)),
                dict(rope=KvRope(ROPE_HALF, 1e4, math.nan)), dict(rope=KvRope(ROPE_HALF, 1e4, 1.0, p, 0, -1.0))):
        with pytest.raises(N.IllegalArgumentException):
            kv.append(**{**good_a, **bad})
    good_t = dict(layer=0, out_ptr=p, ldo=256, q_ptr=p + 4096, ldq=256, rows=rows, window=0, workspace_ptr=w)
    for bad in (dict(layer=1), dict(out_ptr=0), dict(q_ptr=0), dict(ldo=252), dict(ldq=258), dict(window=-1),
                dict(scale=math.nan), dict(workspace_ptr=0), dict(workspace_ptr=w + 16), dict(out_ptr=p + 4)):
        with pytest.raises(N.IllegalArgumentException):
            kv.attend(**{**good_t, **bad})
    with pytest.raises(N.IllegalArgumentException):
        kv.read(0, 0, 0, 128, rows)
    with pytest.raises(N.IllegalArgumentException):
        kv.read(0, p, 0, 124, rows)
    for seq, n in ((2, 1), (-1, 1), (0, -1)):
        with pytest.raises(N.IllegalArgumentException):
            kv.reserve(seq, n)
    with pytest.raises(N.IllegalArgumentException):
        kv.release(2)
    none = KvRows(0, 0, 0)   # an empty call is no error
    kv.append(**{**good_a, "rows": none})
    kv.attend(**{**good_t, "rows": none})
    kv.check()


def test_graph_replay_with_growing_positions(device):
    """Append and attend captured once, replayed while the positions and inputs on the device change; two graphs, a
    workspace each, replayed on streams of their own."""
    heads, kvh, hd, n = 8, 2, 64, 3
    f = Filled(heads, kvh, hd, [60, 130, 5], 16, seed=21, max_tokens=400, spare=60)
    for i in range(n):
        f.kv.reserve(i, 200)
    rope = KvRope(ROPE_HALF, 1e4)
    pos = i32([60, 130, 5])
    seq = i32([0, 1, 2])
    rows = KvRows(seq.data_ptr(), pos.data_ptr(), n)
    q = torch.randn(n, heads, hd, device=DEV)
    k, v = torch.randn(n, kvh, hd, device=DEV), torch.randn(n, kvh, hd, device=DEV)
    qr = torch.empty_like(q)
    outs = [torch.empty_like(q), torch.empty_like(q)]
    spaces = [torch.zeros(f.kv.workspace_bytes(), dtype=torch.uint8, device=DEV) for _ in outs]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for o, w in zip(outs, spaces):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            st = torch.cuda.current_stream().cuda_stream
            if not graphs:
                f.kv.append(0, qr.data_ptr(), q.data_ptr(), heads * hd, k.data_ptr(), v.data_ptr(), kvh * hd, rows, rope, st)
            f.kv.attend(0, o.data_ptr(), heads * hd, qr.data_ptr(), heads * hd, rows, 0, w.data_ptr(), stream=st)
        graphs.append(gr)
    for step in range(5):
        with torch.cuda.stream(streams[0]):
            q.normal_()
            k.normal_()
            v.normal_()
            graphs[0].replay()
        streams[1].wait_stream(streams[0])
        with torch.cuda.stream(streams[1]):
            graphs[1].replay()
        with torch.cuda.stream(streams[0]):
            graphs[0].replay()   # the same rows again: the same bytes, beside the other graph
        torch.cuda.synchronize()
        f.kv.check()
        p = [int(x) for x in pos]
        qe = rotated(q, pos, ROPE_HALF, 1e4, 1.0, None)
        ke, ve = stored(rotated(k, pos, ROPE_HALF, 1e4, 1.0, None)), stored(v)
        for i in range(n):
            f.k[i], f.v[i] = torch.cat((f.k[i], ke[i:i + 1])), torch.cat((f.v[i], ve[i:i + 1]))
        want, tol = f.expected(qe.float(), [(i, p[i], 1) for i in range(n)])
        for o in outs:
            assert bool(((o.double() - want).abs() <= tol).all())
        pos += 1


def test_offsets_past_32_bits(device):
    """A pool of over 4 GiB: the last layer's last pages."""
    layers, kvh, hd, page = 40, 8, 128, 128
    n_pages = (9 << 29) // (layers * kvh * (page // 16) * 2304) + 1
    kv = KvCache(layers, 8, kvh, hd, 2, n_pages * page, page, n_pages)
    assert kv.info()[0] > 1 << 32
    kv.reserve(1, (n_pages - 1) * page)   # the pool's first pages
    kv.reserve(0, page)
    assert kv.info()[1] == 0
    g = gen(31)
    k = torch.randn(100, kvh, hd, generator=g, device=DEV)
    v = torch.randn(100, kvh, hd, generator=g, device=DEV)
    rows = make_rows([(0, 0, 100)])
    kv.append(layers - 1, 0, 0, 0, k.data_ptr(), v.data_ptr(), kvh * hd, rows)
    kr, vr = torch.empty_like(k), torch.empty_like(v)
    kv.read(layers - 1, kr.data_ptr(), vr.data_ptr(), kvh * hd, rows)
    q, out = torch.randn(1, 8, hd, generator=g, device=DEV), torch.empty(1, 8, hd, device=DEV)
    ws = torch.zeros(kv.workspace_bytes(), dtype=torch.uint8, device=DEV)
    kv.attend(layers - 1, out.data_ptr(), 8 * hd, q.data_ptr(), 8 * hd, make_rows([(0, 99, 1)]), 0, ws.data_ptr())
    kv.check()
    assert torch.equal(kr, stored(k).float()) and torch.equal(vr, stored(v).float())
    p = torch.softmax(torch.einsum("hd,khd->hk", q[0].double(), stored(k)) / math.sqrt(hd), -1)
    want = torch.einsum("hk,khd->hd", p, stored(v))
    assert float((out[0].double() - want).norm() / want.norm()) < 1e-5


def test_attend_is_deterministic(device):
    """Partial results join in a fixed order: the same call gives the same bits."""
    f = Filled(16, 8, 128, [5000, 333, 64, 2100], 64, seed=17)
    q = f.q(4)
    e = [(i, n - 1, 1) for i, n in enumerate([5000, 333, 64, 2100])]
    first = f.attend(q, e)
    for _ in range(5):
        assert torch.equal(first, f.attend(q, e))


# ---- prompts: many rows of a sequence ------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 2, 64), (3, 1, 128), (10, 2, 128), (7, 1, 64), (96, 1, 64), (128, 1, 128)])
@pytest.mark.parametrize("window", [0, 1, 63, 64, 65, 200, 5000])
def test_prompt_windows_and_groups(device, heads, kv_heads, hd, window):
    """Heads of a row in two tiles of pairs, rows of a tile that see different tiles of keys, pages of every size."""
    page = {0: 16, 1: 32, 63: 64, 64: 128}.get(window, 16)
    f = Filled(heads, kv_heads, hd, [391, 64, 129], page, seed=heads + window)
    entries = [(0, 391 - 150, 150), (1, 0, 64), (2, 128, 1), (2, 0, 129), (0, 5, 66)]
    f.check(f.q(sum(e[2] for e in entries)), entries, window)


def test_prompt_over_every_cta(device):
    """128 pairs whose keys all of the device's CTAs share; two of them beside short ones."""
    f = Filled(2, 1, 128, [38001, 90, 300], 64, seed=41)
    f.check(f.q(64), [(0, 38001 - 64, 64)])
    f.check(f.q(64 + 90 + 70), [(1, 0, 90), (0, 20000, 64), (2, 230, 70)])


def test_prompts_among_single_tokens(device):
    """More than 32 and more than 256 entries, one kernel's and the other's in turn, empty ones between."""
    lens = [1 + (i * 53) % 170 for i in range(300)]
    f = Filled(4, 2, 64, lens, 16, seed=42)
    entries = [(i, n - 1, 1) if i % 3 else (i, 0, n) if i % 2 else (i, n // 2, n - n // 2) for i, n in enumerate(lens)]
    entries[7] = (7, 3, 0)
    f.check(f.q(sum(e[2] for e in entries)), entries)
    f.check(f.q(sum(e[2] for e in entries)), entries, window=40)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kgain,vgain,qgain", [(4e4, 1.0, 1e-4), (1e-7, 4e5, 1e6), (1.0, 1e-7, 1.0), (4e5, 4e5, 1e-6)])
def test_prompt_magnitudes(device, hd, kgain, vgain, qgain):
    """Scales at both ends of fp16, tiles of large ones between tiles of small ones."""
    f = Filled(6, 2, hd, [330], 32, seed=43)
    k = torch.randn(330, 2, hd, generator=f.g, device=DEV)
    v = torch.randn(330, 2, hd, generator=f.g, device=DEV)
    k[100:150] *= kgain
    v[60:200] *= vgain
    f.kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), 2 * hd, make_rows([(0, 0, 330)]))
    f.k, f.v = [stored(k)], [stored(v)]
    f.check(f.q(130, qgain), [(0, 200, 130)])
    f.check(f.q(70, qgain), [(0, 100, 70)])


@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 64), (6, 1, 128)])
@pytest.mark.parametrize("window", [0, 50])
def test_prompt_rows_before_a_nan(device, heads, kv_heads, hd, window):
    """A value or key of a chunk that is NaN reaches the rows that see it and no others."""
    for what in "kv":
        f = Filled(heads, kv_heads, hd, [300], 64, seed=44)
        x = torch.randn(1, kv_heads, hd, generator=f.g, device=DEV)
        y = x.clone()
        (y if what == "v" else x)[:, 0, 32:64] = float("nan")
        f.kv.append(0, 0, 0, 0, x.data_ptr(), y.data_ptr(), kv_heads * hd, make_rows([(0, 210, 1)]))
        q = f.q(180)
        got = f.attend(q, [(0, 120, 180)], window)
        f.kv.check()
        want, tol = f.expected(q, [(0, 120, 180)], window)   # (with another key 210: right for the rows without it)
        row = torch.arange(120, 300, device=DEV)
        sees = (row >= 210) & ((row < 210 + window) if window else row >= 0)
        assert bool(((got[~sees].double() - want[~sees]).abs() <= tol[~sees]).all())
        g = heads // kv_heads
        part = slice(32, 64) if what == "v" else slice(None)
        assert torch.isnan(got[sees][:, :g, part]).all()


def test_prompt_nan_row_stays_alone(device):
    f = Filled(4, 2, 128, [200], 16, seed=45)
    q = f.q(150)
    q[70, 1, 5] = float("nan")
    got = f.attend(q, [(0, 50, 150)])
    f.kv.check()
    want, tol = f.expected(torch.nan_to_num(q), [(0, 50, 150)])
    bad = torch.zeros(150, 4, dtype=torch.bool, device=DEV)
    bad[70, 1] = True
    assert torch.isnan(got[bad]).all()
    assert bool(((got.double() - want).abs() <= tol)[~bad].all())


def test_prompt_strides_and_rows_behind(device):
    f = Filled(6, 2, 64, [150, 80], 32, seed=46)
    ld, n = 6 * 64 + 4, 100 + 80 + 9
    q = torch.randn(n, ld, generator=f.g, device=DEV)
    out = torch.full((n, ld + 8), 7.0, device=DEV)
    entries = [(0, 50, 100), (1, 0, 80)]
    f.kv.attend(0, out.data_ptr(), ld + 8, q.data_ptr(), ld, make_rows(entries, n), 0, f.ws.data_ptr(), -0.2)
    f.kv.check()
    want, tol = f.expected(q[:180, :384].reshape(180, 6, 64), entries, 0, -0.2)
    assert bool(((out[:180, :384].reshape(180, 6, 64).double() - want).abs() <= tol.abs()).all())
    assert bool((out[180:] == 7).all()) and bool((out[:, 384:] == 7).all())


def test_prompt_graphs_beside_each_other(device):
    """Two captured calls, a workspace each, replayed at once on their own streams; the same bits each time."""
    f = Filled(16, 4, 128, [900, 3000, 70], 64, seed=47)
    rows = [make_rows([(0, 300, 600), (2, 69, 1)]), make_rows([(1, 2800, 200), (2, 0, 70), (0, 899, 1)])]
    qs = [f.q(601), f.q(271)]
    outs = [torch.empty_like(q) for q in qs]
    spaces = [torch.zeros(f.kv.workspace_bytes(), dtype=torch.uint8, device=DEV) for _ in qs]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for r, q, o, w in zip(rows, qs, outs, spaces):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f.kv.attend(0, o.data_ptr(), 2048, q.data_ptr(), 2048, r, 0, w.data_ptr(),
                        stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(gr)
    first = None
    for _ in range(4):
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        f.kv.check()
        first = first or [o.clone() for o in outs]
        assert all(torch.equal(a, b) for a, b in zip(first, outs))
    for q, o, e in zip(qs, first, ([(0, 300, 600), (2, 69, 1)], [(1, 2800, 200), (2, 0, 70), (0, 899, 1)])):
        want, tol = f.expected(q, e)
        assert bool(((o.double() - want).abs() <= tol).all())


def test_prompt_bad_entries_between_good_ones(device):
    f = Filled(8, 2, 128, [200, 150], 16, seed=48)
    q = f.q(100 + 80 + 90)
    got = f.attend(q, [(0, 100, 100), (1, 100, 80), (1, 60, 90)])   # the second: behind what is reserved
    with pytest.raises(N.IllegalStateException):
        f.kv.check()
    for part, e in ((slice(0, 100), (0, 100, 100)), (slice(180, 270), (1, 60, 90))):
        want, tol = f.expected(q[part].contiguous(), [e])
        assert bool(((got[part].double() - want).abs() <= tol).all())
    assert torch.isnan(got[100:180]).all()


def test_prompt_of_few_rows_over_every_cta(device):
    """Two tiles of pairs whose keys all of the device's CTAs share, many parts to join."""
    f = Filled(2, 1, 64, [50003, 130], 32, seed=49)
    f.check(f.q(128), [(0, 50003 - 128, 128)])
    f.check(f.q(128 + 130), [(1, 0, 130), (0, 31000, 128)])


@pytest.mark.parametrize("rows", [15, 16, 17, 63, 64, 65])
def test_rows_on_both_sides_of_the_kernels_limits(device, rows):
    """4 heads a kv head: 64 pairs among many rows, 256 among few."""
    f = Filled(8, 2, 64, [300, 300, 300, 300], 16, seed=50)
    f.check(f.q(rows), [(0, 300 - rows, rows)])
    f.check(f.q(rows + 16 + 300), [(1, 100, rows), (2, 0, 16), (3, 0, 300)])


def test_pages_do_not_change_hands_in_a_captured_stream(device):
    """A replay would hand them out again: refused, and nothing is changed."""
    kv = KvCache(1, 2, 1, 64, 2, 64, 16)
    kv.reserve(0, 16)
    free = kv.info()[1]
    x = torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        x.add_(1)
        st = torch.cuda.current_stream().cuda_stream
        kv.reserve(0, 10, st)   # has them
        for call in (lambda: kv.reserve(1, 16, st), lambda: kv.reserve(0, 17, st), lambda: kv.release(0, st)):
            with pytest.raises(N.IllegalArgumentException):
                call()
    gr.replay()
    torch.cuda.synchronize()
    assert kv.info()[1] == free and bool((x == 1).all())
    kv.reserve(1, 16)
    assert kv.info()[1] == free - 1
