"""Models on the paged 4-bit K/V cache (brew_model_set_kv_cache) and the
scoring of texts (brew_session_score).

The model is compared with a plain 64-bit forward whose K and V go through
the same 4-bit rounding.  Its fp32 activations are off by about 1e-6; a code
whose value lies that near a rounding border (8 borders a block: one of 6e4
values) comes out one higher or lower, which moves one of a vector's 64 to
256 cached values by an eighth of its block's largest and the logits by less
than 1e-2.  So: every step within 1e-2, and half of the steps within 1e-4,
where no code has changed."""
import math

import numpy as np
import pytest
import torch

from brewference_b200 import _native as N
from brewference_b200 import config as C
from brewference_b200.api import PREFILL_BATCHED, DeviceModel
from test_gpu_kv import stored
from test_gpu_model import small

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Plain:
    """TransformerGraph.forward in 64 bits on the model's own weights, K and V rounded to Q4_0 blocks."""

    def __init__(self, dm):
        self.c = c = dm.cfg
        shapes = c.matrix_shapes()
        self.w = {}
        for which, (rows, cols, _, layers) in shapes.items():
            t = dm.tensor(which)
            self.w[which] = [torch.from_numpy(t.dequantize_row(l * rows * cols, rows * cols)).to(DEV).double().view(rows, cols)
                             for l in range(layers)]
        self.k = [[] for _ in range(c.n_layers)]
        self.v = [[] for _ in range(c.n_layers)]

    def norm(self, x):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.c.eps)

    def rope(self, x, pos, base):
        hd = x.shape[-1]
        a = pos * base ** (-torch.arange(0, hd, 2, device=DEV).double() / hd)
        inter = self.c.arch in (C.ARCH_LLAMA, C.ARCH_SMOLLM3)
        i0 = torch.arange(0, hd, 2, device=DEV) if inter else torch.arange(hd // 2, device=DEV)
        i1 = i0 + (1 if inter else hd // 2)
        y = x.clone()
        y[:, i0] = x[:, i0] * a.cos() - x[:, i1] * a.sin()
        y[:, i1] = x[:, i0] * a.sin() + x[:, i1] * a.cos()
        return y

    def forward(self, tok, pos):
        c, w, hd = self.c, self.w, self.c.head_size
        gemma, qknorm = c.arch in (C.ARCH_GEMMA2, C.ARCH_GEMMA3), c.arch in (C.ARCH_QWEN3, C.ARCH_GEMMA3)
        x = w[C.W_EMBED][0][tok] * (math.sqrt(c.dim) if gemma else 1.0)
        for l in range(c.n_layers):
            every = 6 if c.arch == C.ARCH_GEMMA3 else 2
            local = gemma and (l + 1) % every != 0
            base = c.rope_base if c.rope_base > 0 else 1e4 if not gemma or local else 1e6
            h = self.norm(x)
            q, k, v = (w[i][l] @ h for i in (C.W_Q, C.W_K, C.W_V))
            q, k, v = q.view(-1, hd), k.view(-1, hd), v.view(-1, hd)
            if qknorm:
                q, k = self.norm(q), self.norm(k)
            if c.arch != C.ARCH_SMOLLM3 or (l + 1) % 4 != 0:
                q, k = self.rope(q, pos, base), self.rope(k, pos, base)
            del self.k[l][pos:], self.v[l][pos:]
            self.k[l].append(stored(k))
            self.v[l].append(stored(v))
            first = max(0, pos - c.sliding_window + 1) if local and c.sliding_window else 0
            ks, vs = torch.stack(self.k[l][first:]), torch.stack(self.v[l][first:])
            g = c.n_heads // c.n_kv_heads
            p = torch.softmax(torch.einsum("hd,thd->ht", q, ks.repeat_interleave(g, 1)) / math.sqrt(hd), -1)
            o = w[C.W_O][l] @ torch.einsum("ht,thd->hd", p, vs.repeat_interleave(g, 1)).reshape(-1)
            x = x + (self.norm(o) if gemma else o)
            h = self.norm(x)
            a, u = w[C.W_GATE][l] @ h, w[C.W_UP][l] @ h
            a = torch.nn.functional.gelu(a, approximate="tanh") if gemma else a * torch.sigmoid(a)
            o = w[C.W_DOWN][l] @ (a * u)
            x = x + (self.norm(o) if gemma else o)
        out = w[C.W_EMBED][0] if c.tied_embeddings else w[C.W_OUTPUT][0]
        return out @ self.norm(x)


def rel(a, b):
    a = torch.from_numpy(np.asarray(a)).to(DEV).double()
    return float((a - b).norm() / b.norm())


ARCHS = [C.ARCH_LLAMA, C.ARCH_QWEN3, C.ARCH_GEMMA3, C.ARCH_GEMMA2, C.ARCH_SMOLLM3]


@pytest.mark.parametrize("arch", ARCHS)
def test_forward_on_the_4bit_cache(device, arch):
    cfg = small(arch)
    dm = DeviceModel.synthesize(cfg, 5, max_batch=2)
    dm.set_kv_cache(C.TYPE_Q4_0)
    dm.set_kv_cache(C.TYPE_Q4_0)
    plain = Plain(dm)
    rng = np.random.default_rng(arch)
    toks = rng.integers(0, cfg.vocab_size, 40)
    errs = []
    for i, t in enumerate(toks):
        # the second sequence runs one token behind, at its own position
        lg, am = dm.forward([t, toks[max(i - 1, 0)]], [i, max(i - 1, 0)])
        want = plain.forward(int(t), i)
        errs.append(rel(lg[0], want))
        assert am[0] == int(np.argmax(lg[0]))
        if i > 0:
            errs.append(rel(lg[1], last))
        last = want
    assert max(errs) < 1e-2 and np.median(errs) < 1e-4, (max(errs), np.median(errs))
    dm.close()


@pytest.mark.parametrize("arch", [C.ARCH_LLAMA, C.ARCH_QWEN3, C.ARCH_GEMMA3])
def test_batched_prefill_on_the_4bit_cache(device, arch):
    kw = dict(dim=512, n_heads=8, n_kv_heads=4) if arch == C.ARCH_LLAMA else {}   # rows in multiples of 128
    cfg = small(arch, seq_len=900, **kw)
    rng = np.random.default_rng(7)
    prompt = rng.integers(0, cfg.vocab_size, 600)
    lgs = []
    for batched in (True, False):
        dm = DeviceModel.synthesize(cfg, 6)
        dm.set_kv_cache(C.TYPE_Q4_0)
        if batched:
            dm.set_prefill(PREFILL_BATCHED)
        dm.prefill(prompt)
        lg, _ = dm.forward([int(prompt[-1])], [600])
        lgs.append(lg[0])
        toks = dm.generate(prompt[:30].tolist(), 5)
        assert len(toks) == 5
        dm.close()
    want = torch.from_numpy(lgs[1]).to(DEV).double()
    assert rel(lgs[0], want) < 1e-2


def test_the_fp32_cache_is_given_back(device):
    cfg = small(C.ARCH_LLAMA, seq_len=4096, n_layers=8)
    dm = DeviceModel.synthesize(cfg, 1, max_batch=16)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    dm.set_kv_cache(C.TYPE_Q4_0)
    torch.cuda.synchronize()
    after = torch.cuda.mem_get_info()[0]
    fp32 = 2 * 4 * 16 * 8 * 4096 * cfg.kv_dim
    # 0.86 of it comes back, less the forward's other buffers and the attention's workspace
    assert after - before > 0.5 * fp32
    dm.reset()
    with pytest.raises(N.IllegalStateException):
        dm.set_kv_cache(C.TYPE_F32)
    with pytest.raises(N.IllegalStateException):
        dm.set_kv_cache(C.TYPE_Q8_0)
    with pytest.raises(N.IllegalArgumentException):   # the session is forgotten
        dm.decode(1)
    dm.close()


@pytest.mark.parametrize("qtype", [C.TYPE_F32, C.TYPE_Q4_0])
@pytest.mark.parametrize("arch", [C.ARCH_LLAMA, C.ARCH_QWEN3])
def test_score(device, arch, qtype):
    """The scores are those of the logits that forward returns for the same tokens."""
    cfg = small(arch)
    dm = DeviceModel.synthesize(cfg, 9)
    dm.set_kv_cache(qtype)
    toks = np.random.default_rng(3).integers(0, cfg.vocab_size, 33)
    lp, ent, ids, tops = dm.score(toks, 7)
    assert lp.shape == (32,) and ids.shape == (32, 7)
    dm.reset()
    for i in range(32):
        lg, am = dm.forward([toks[i]], [i])
        logp = torch.log_softmax(torch.from_numpy(lg[0]).double(), -1)
        # logits below 2^4 here, 4096 of them: (2 * 16 + 4096 / 32 + 72 + ...) 2^-24 < 2e-5
        assert abs(float(logp[toks[i + 1]]) - lp[i]) < 2e-5
        assert abs(float(-(logp.exp() * logp).sum()) - ent[i]) < 2e-5 * 10
        order = torch.sort(torch.from_numpy(lg[0]), descending=True, stable=True)[1][:7]
        assert ids[i].tolist() == order.tolist() and ids[i, 0] == am[0]
        assert np.abs(logp[order].numpy() - tops[i]).max() < 2e-5
    again = dm.score(toks, 0)
    # (the decode kernel of the fp32 cache does not repeat its last bits)
    assert np.abs(again[0] - lp).max() <= (0 if qtype == C.TYPE_Q4_0 else 2e-5) and again[2].shape == (32, 0)
    dm.close()


def test_score_shows_what_the_cache_costs(device):
    """The run a user makes of all of it: the same text under both caches."""
    cfg = small(C.ARCH_QWEN3)
    toks = np.random.default_rng(4).integers(0, cfg.vocab_size, 60)
    dm = DeviceModel.synthesize(cfg, 12)
    lp32 = dm.score(toks)[0]
    dm.set_kv_cache(C.TYPE_Q4_0)
    lp4 = dm.score(toks)[0]
    diff = np.abs(lp4 - lp32)
    assert diff[0] < 0.5 and diff.max() > 1e-4   # it is rounded, and it is the same model
    assert np.corrcoef(lp4, lp32)[0, 1] > 0.9
    dm.close()


def test_score_refusals(device):
    cfg = small(C.ARCH_LLAMA)
    dm = DeviceModel.synthesize(cfg, 2)
    for toks, top in (([1], 0), ([], 0), ([1, cfg.vocab_size], 0), ([1, -1], 0), ([1, 2], 33), ([1, 2], -1)):
        with pytest.raises(N.IllegalArgumentException):
            dm.score(toks, top)
    with pytest.raises(N.IllegalStateException) as e:
        dm.score([1] * (cfg.seq_len + 2))
    assert e.value.code == N.ERR_CONTEXT_FULL
    assert dm.score([1] * (cfg.seq_len + 1))[0].shape == (cfg.seq_len,)
    dm.close()
