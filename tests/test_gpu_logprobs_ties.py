"""Ties among the logits behind a row's last whole float4 and earlier ones:
the alternatives are the largest values, equal ones by index, whichever CTA,
warp and round of loads meets them."""
import pytest
import torch

from brewference_b200.api import Logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def top_ids(x, ld, vocab, rows, top):
    ids, lps = torch.empty(rows, top, dtype=torch.int32, device=DEV), torch.empty(rows, top, device=DEV)
    Logits.logprobs_device(x.data_ptr(), ld, vocab, rows, 0, 0, 0, top, ids.data_ptr(), lps.data_ptr())
    torch.cuda.synchronize()
    return ids.long()


def expected(x, top):
    return torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]


@pytest.mark.parametrize("rows", [300, 37])            # a CTA a row, eight
@pytest.mark.parametrize("vocab", [16385, 49153, 49155, 151937, 151938])
@pytest.mark.parametrize("top", [1, 5])
@pytest.mark.parametrize("pad", [0, 1, 3])             # rows start on every float of four
def test_last_logit_ties_an_earlier_one(device, rows, vocab, top, pad):
    """The largest values of a row are its last logit and, once more, one somewhere before it."""
    ld = (vocab + 3) // 4 * 4 + pad
    g = torch.Generator(device=DEV)
    g.manual_seed(vocab + rows + top)
    x = torch.rand(rows, ld, generator=g, device=DEV)
    high = torch.randint(0, vocab - 1, (rows, top - 1), generator=g, device=DEV)
    x.scatter_(1, high, 9.0 + torch.rand(rows, top - 1, generator=g, device=DEV))
    # the twin goes over the whole row, and over the last eighth of it in small steps
    at = torch.linspace(0, vocab - 2, rows, device=DEV).long() if rows > 100 else \
        torch.linspace(vocab - vocab // 8, vocab - 2, rows, device=DEV).long()
    x[:, vocab - 1] = 5.0
    x.scatter_(1, at[:, None], 5.0)
    x[:, vocab:] = 99.0
    got = top_ids(x, ld, vocab, rows, top)
    assert torch.equal(got, expected(x[:, :vocab], top))


@pytest.mark.parametrize("rows,vocab,early", [(300, 49153, 16390), (1, 151937, 149330), (300, 16385, 4096)])
def test_known_ties(device, rows, vocab, early):
    x = torch.zeros(rows, (vocab + 3) // 4 * 4, device=DEV)
    x[:, early] = x[:, vocab - 1] = 5.0
    assert bool((top_ids(x, x.shape[1], vocab, rows, 1) == early).all())


@pytest.mark.parametrize("vocab", [4099, 33335, 151938])
@pytest.mark.parametrize("rows", [300, 20, 1])
def test_coarse_logits(device, vocab, rows):
    """Logits of a few steps, as a bf16 model's: ties at the last alternative everywhere."""
    x = (torch.randn(rows, vocab, device=DEV) * 4).bfloat16().float()
    x[:, vocab - 3:] = torch.sort(x, dim=-1, descending=True)[0][:, 19:20]   # the last logits tie the 20th
    got = top_ids(x, vocab, vocab, rows, 20)
    assert torch.equal(got, expected(x, 20))
