"""Token log probabilities, entropy and top alternatives against 64 bits.

Tolerance.  With Y the largest |x - max| among logits of probability over
2^-40 and n = vocab / 32 + 64 additions at most on a value's way through a
sum: x - max is rounded (Y 2^-24), each exponential is off by that and 2^-22,
the sum by n 2^-24; log z by the same, and the result by half a step of each
of its two terms.  The entropy's second sum adds E|y| times those.
"""
import math

import pytest
import torch

from brewference_b200 import _native as N
from brewference_b200.api import MAX_TOP, Logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def score(x, tokens, top, ld=None, vocab=None, stream=0):
    rows, vocab = x.shape[0], vocab or x.shape[1]
    lp, ent = torch.full((rows,), 7.0, device=DEV), torch.full((rows,), 7.0, device=DEV)
    ids = torch.full((rows, top), -7, dtype=torch.int32, device=DEV)
    tops = torch.full((rows, top), 7.0, device=DEV)
    Logits.logprobs_device(x.data_ptr(), ld or x.stride(0), vocab, rows, tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), top,
                           ids.data_ptr() if top else 0, tops.data_ptr() if top else 0, stream)
    torch.cuda.synchronize()
    return lp, ent, ids, tops


def check(x, tokens, got):
    lp, ent, ids, tops = got
    xd = x.double()
    vocab = x.shape[1]
    top = xd.amax(-1, keepdim=True)
    logp = (xd - top) - torch.logsumexp(xd - top, -1, keepdim=True)   # logits of 10^38 leave no digit beside them
    y = (xd - xd.amax(-1, keepdim=True)).abs()
    near = torch.where(logp > -28, y, 0.0)
    n = vocab / 32 + 64
    rel = (near.amax(-1) * 2 + n + 8) * 2 ** -24      # of the sum z, so of log z in absolute terms
    want = torch.gather(logp, 1, tokens.long()[:, None])[:, 0]

    def close(a, b, tol):
        same = (a.double() == b) | ((a.double() - b).abs() <= tol)
        assert bool(same.all()), (a[~same][:4], b[~same][:4])

    close(lp, want, rel + want.abs().nan_to_num(0, 0, 0) * 2 ** -23)
    p = logp.exp()
    h = -torch.special.xlogy(p, p).sum(-1)
    close(ent, h, rel * (2 + (p * near).sum(-1)) + h * 2 ** -23)
    if ids.shape[1]:
        # exact: the largest values, equal ones by index
        order = torch.sort(x + 0.0, dim=-1, descending=True, stable=True)[1][:, :ids.shape[1]]
        assert torch.equal(ids.long(), order)
        w = torch.gather(logp, 1, order)
        close(tops, w, rel[:, None] + w.abs().nan_to_num(0, 0, 0) * 2 ** -23)


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 257, 1000, 4095, 4099, 32000, 49152, 151936, 262144])
@pytest.mark.parametrize("rows,top", [(1, 5), (3, 0), (7, 32), (1, 1)])
def test_scores(device, vocab, rows, top):
    g = torch.Generator(device=DEV)
    g.manual_seed(vocab * 7 + rows)
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 3
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV, dtype=torch.int32)
    check(x, tokens, score(x, tokens, min(top, vocab)))


@pytest.mark.parametrize("rows", [150, 601])
def test_many_rows(device, rows):
    x = torch.randn(rows, 5003, device=DEV) * 4
    tokens = torch.randint(0, 5003, (rows,), device=DEV, dtype=torch.int32)
    check(x, tokens, score(x, tokens, 20))


@pytest.mark.parametrize("vocab,off", [(1001, 0), (1001, 1), (4099, 3), (70001, 2)])
def test_strides_and_alignment(device, vocab, off):
    """Rows that start on any float, more columns than the vocabulary, values behind it that would win."""
    buf = torch.full((5, vocab + 13), 99.0, device=DEV)
    flat = buf.view(-1)[off:off + 4 * (vocab + 13)].view(4, vocab + 13)
    flat[:, :vocab] = torch.randn(4, vocab, device=DEV)
    x = flat[:, :vocab]
    tokens = torch.randint(0, vocab, (4,), device=DEV, dtype=torch.int32)
    check(x, tokens, score(flat, tokens, 9, vocab + 13, vocab))


@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "one high", "large", "zeros of both signs"])
def test_ties_and_orders(device, kind):
    for vocab in (700, 33333):
        i = torch.arange(vocab, device=DEV, dtype=torch.float32)
        x = {"equal": torch.zeros(vocab, device=DEV), "few values": (i * 7919 % 5), "rising": i * 1e-3, "falling": -i * 1e-3,
             "one high": torch.where(i == vocab - 2, 80.0, 0.0), "large": torch.randn(vocab, device=DEV) * 1e4,
             "zeros of both signs": torch.where(i % 3 == 0, -0.0, 0.0)}[kind].repeat(2, 1).contiguous()
        tokens = torch.tensor([vocab - 2, 0], dtype=torch.int32, device=DEV)
        check(x, tokens, score(x, tokens, 32))


def test_masked_rows(device):
    vocab = 9001
    x = torch.randn(6, vocab, device=DEV)
    x[0, 5:] = -math.inf                 # fewer tokens than alternatives
    x[1] = -math.inf                     # nothing is left
    x[2, torch.rand(vocab, device=DEV) < 0.9] = -math.inf
    x[3] = torch.finfo(torch.float32).min    # the type's lowest value is a value
    x[4, :] = torch.finfo(torch.float32).min
    x[4, 17] = 1.0
    tokens = torch.tensor([3, 4, int(torch.isfinite(x[2]).nonzero()[0]), 2, 17, 8], dtype=torch.int32, device=DEV)
    got = score(x, tokens, 12)
    keep = torch.tensor([0, 2, 3, 4, 5], device=DEV)
    check(x[keep], tokens[keep], tuple(t[keep] for t in got))
    lp, ent, ids, tops = got
    assert lp[1] == -math.inf and ent[1] == 0 and bool((tops[1] == -math.inf).all())
    assert ids[1].tolist() == list(range(12))
    # a masked token has the log probability -inf
    bad = score(x[:1], torch.tensor([77], dtype=torch.int32, device=DEV), 1)
    assert bad[0][0] == -math.inf


def test_nan_inf_and_tokens_outside(device):
    vocab = 3001
    x = torch.randn(4, vocab, device=DEV)
    x[0, 100] = math.nan
    x[1, 100] = math.inf
    tokens = torch.tensor([5, 5, -1, vocab], dtype=torch.int32, device=DEV)
    lp, ent, ids, tops = score(x, tokens, 3)
    assert torch.isnan(lp).all() and torch.isnan(ent[:2]).all() and torch.isfinite(ent[2:]).all()
    assert torch.isnan(tops[:2]).all() and 100 not in ids[0].tolist() and ids[1, 0] == 100
    assert torch.equal(ids[2].long(), torch.sort(x[2], dim=-1, descending=True, stable=True)[1][:3])


def test_outputs_asked_alone(device):
    x = torch.randn(3, 2222, device=DEV)
    tokens = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    full = score(x, tokens, 4)
    lp, ent = torch.full((3,), 7.0, device=DEV), torch.full((3,), 7.0, device=DEV)
    Logits.logprobs_device(x.data_ptr(), 2222, 2222, 3, tokens.data_ptr(), lp.data_ptr())
    Logits.logprobs_device(x.data_ptr(), 2222, 2222, 3, 0, 0, ent.data_ptr())
    ids, tops = torch.empty(3, 4, dtype=torch.int32, device=DEV), torch.empty(3, 4, device=DEV)
    Logits.logprobs_device(x.data_ptr(), 2222, 2222, 3, 0, 0, 0, 4, ids.data_ptr(), tops.data_ptr())
    Logits.logprobs_device(x.data_ptr(), 2222, 2222, 0, tokens.data_ptr(), lp.data_ptr())
    torch.cuda.synchronize()
    for a, b in zip((lp, ent, ids, tops), full):
        assert torch.equal(a, b)


def test_captured_and_on_another_stream(device):
    x = torch.randn(2, 60000, device=DEV)
    tokens = torch.tensor([7, 59999], dtype=torch.int32, device=DEV)
    lp, ent = torch.empty(2, device=DEV), torch.empty(2, device=DEV)
    ids, tops = torch.empty(2, 6, dtype=torch.int32, device=DEV), torch.empty(2, 6, device=DEV)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        Logits.logprobs_device(x.data_ptr(), 60000, 60000, 2, tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), 6,
                               ids.data_ptr(), tops.data_ptr(), torch.cuda.current_stream().cuda_stream)
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            x.normal_()
            gr.replay()
        torch.cuda.synchronize()
        check(x, tokens, (lp, ent, ids, tops))


def test_refused(device):
    assert MAX_TOP == 32
    x = torch.zeros(1, 10, device=DEV)
    with pytest.raises(N.IllegalArgumentException):
        Logits.logprobs_device(x.data_ptr(), 10, 10, 1, 0, 0, 0, 11, x.data_ptr(), x.data_ptr())
