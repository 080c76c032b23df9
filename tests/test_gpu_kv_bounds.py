"""Where a sequence of the paged 4-bit K/V cache ends, and how many rows a
call may say an entry has."""
import pytest
import torch

from brewference_b200 import _native as N
from brewference_b200 import config as C
from brewference_b200.api import DeviceModel, KvCache, KvRows
from test_gpu_kv import DEV, Filled, i32, make_rows, stored
from test_gpu_model import small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 64])
def test_a_sequence_ends_at_max_tokens(device, page):
    """Not where its last page ends."""
    f = Filled(4, 2, 64, [100, 60], page, seed=1, max_tokens=100, spare=9)
    f.check(f.q(2), [(0, 99, 1), (1, 59, 1)])
    k = torch.randn(3, 2, 64, generator=f.g, device=DEV)
    for seq, pos, n in ((0, 100, 1), (0, 98, 3), (0, page * (99 // page + 1) - 1, 1)):
        rows = make_rows([(seq, pos, n)])
        f.kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 128, rows)
        with pytest.raises(N.IllegalStateException):
            f.kv.check()
        out = torch.full((3, 2, 64), 3.0, device=DEV)
        f.kv.read(0, out.data_ptr(), 0, 128, rows)
        with pytest.raises(N.IllegalStateException):
            f.kv.check()
        assert bool((out == 3).all())
        assert torch.isnan(f.attend(f.q(n), [(seq, pos, n)])).all()
        with pytest.raises(N.IllegalStateException):
            f.kv.check()
    # pages are given whole: what is reserved is usable up to the page's end, and no further
    end = min(100, page * (59 // page + 1))
    f.kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 128, make_rows([(1, end - 1, 1)]))
    f.kv.check()
    f.kv.reserve(1, 100)
    f.kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 128, make_rows([(1, 97, 3)]))
    f.kv.check()
    f.kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 128, make_rows([(1, 98, 3)]))
    with pytest.raises(N.IllegalStateException):
        f.kv.check()


def test_a_reservation_of_many_launches(device):
    """Pages past the 120 that one launch hands over, given in three steps."""
    kv = KvCache(1, 2, 1, 32, 2, 5003, 16, 0)
    k = torch.randn(5003, 1, 32, device=DEV)
    out = torch.empty_like(k)
    for n in (1900, 3900, 5003):
        kv.reserve(1, n)
        kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 32, make_rows([(1, 0, n)]))
        kv.read(0, out.data_ptr(), 0, 32, make_rows([(1, 0, n)]))
        kv.check()
        assert torch.equal(out[:n], stored(k[:n]).float())
    kv.append(0, 0, 0, 0, k.data_ptr(), k.data_ptr(), 32, make_rows([(1, 5003, 1)]))
    with pytest.raises(N.IllegalStateException):
        kv.check()


@pytest.mark.parametrize("qtype", [C.TYPE_F32, C.TYPE_Q4_0])
def test_a_models_sequence_ends_at_its_context(device, qtype):
    """Positions given on the device, past the 100 of the context."""
    dm = DeviceModel.synthesize(small(C.ARCH_QWEN3, seq_len=100), 3, max_batch=2)
    dm.set_kv_cache(qtype)
    tok, am = i32([5, 6]), i32([0, 0])

    def step(pos):
        p = i32(pos)
        torch.cuda.synchronize()
        N.check(N.lib().brew_model_forward_dev(dm.handle, tok.data_ptr(), p.data_ptr(), 2, None, am.data_ptr(), None))
        torch.cuda.synchronize()

    step([99, 99])
    dm.forward([1, 2], [0, 0])
    step([99, 100])
    with pytest.raises(N.IllegalStateException):   # told by the next call that checks
        dm.forward([1, 2], [0, 0])
    dm.forward([1, 2], [0, 0])
    dm.close()


@pytest.mark.parametrize("max_rows", [2 ** 31 - 1, 2 ** 31 - 3, 10 ** 6])
def test_max_rows_far_above_the_rows(device, max_rows):
    """Any bound at or above the entries' rows gives what the tight one gives."""
    f = Filled(4, 2, 64, [90, 70], 16, seed=2)
    entries = [(0, 20, 50), (1, 69, 1)]
    rows = make_rows(entries)
    loose = KvRows(rows.keep[0].data_ptr(), rows.keep[1].data_ptr(), 2, 51, max_rows, rows.keep[2].data_ptr())
    k, q = torch.randn(51, 2, 64, generator=f.g, device=DEV), f.q(51)
    outs = []
    for r in (rows, loose):
        o, kr, q2 = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
        f.kv.append(0, q2.data_ptr(), q.data_ptr(), 256, k.data_ptr(), k.data_ptr(), 128, r)
        f.kv.read(0, kr.data_ptr(), 0, 128, r)
        f.kv.attend(0, o.data_ptr(), 256, q.data_ptr(), 256, r, 0, f.ws.data_ptr())
        f.kv.check()
        outs.append((o, kr, q2))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("n_rows,max_rows,start", [(0, 0, [0, 2]), (4, 0, [0, 2]), (0, 5, [0, 1]), (1, 0, None)])
def test_rows_in_a_call_that_has_none_are_told(device, n_rows, max_rows, start):
    """Entries with rows where n_rows or max_rows says there are none: skipped and recorded, as any bad entry."""
    f = Filled(4, 2, 64, [40], 16, seed=3)
    seq, pos = i32([0]), i32([10])
    st = i32(start) if start else None
    x = torch.full((4, 4, 64), 3.0, device=DEV)
    y = x.clone()
    rows = KvRows(seq.data_ptr(), pos.data_ptr(), 1, n_rows, max_rows, st.data_ptr() if start else 0)
    for call in (lambda: f.kv.append(0, y.data_ptr(), x.data_ptr(), 256, x.data_ptr(), x.data_ptr(), 256, rows),
                 lambda: f.kv.read(0, y.data_ptr(), y.data_ptr(), 256, rows),
                 lambda: f.kv.attend(0, y.data_ptr(), 256, x.data_ptr(), 256, rows, 0, f.ws.data_ptr())):
        call()
        with pytest.raises(N.IllegalStateException):
            f.kv.check()
        assert torch.equal(x, y)


def test_entries_without_rows_are_no_error(device):
    f = Filled(4, 2, 64, [40, 7], 16, seed=3)
    rows = make_rows([(0, 10, 0), (1, 3, 0)])
    rows.c.max_rows = 0
    x = torch.full((4, 4, 64), 3.0, device=DEV)
    y = x.clone()
    f.kv.append(0, y.data_ptr(), x.data_ptr(), 256, x.data_ptr(), x.data_ptr(), 256, rows)
    f.kv.read(0, y.data_ptr(), y.data_ptr(), 256, rows)
    f.kv.attend(0, y.data_ptr(), 256, x.data_ptr(), 256, rows, 0, f.ws.data_ptr())
    f.kv.check()
    assert torch.equal(x, y)
    f.check(f.q(1), [(0, 39, 1)])
