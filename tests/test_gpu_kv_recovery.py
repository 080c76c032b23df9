"""A model on the 4-bit K/V cache after a step that did not end well: the
attention's arrival counters, raised as a bounded wait that gave up leaves
them, are put back by the call that reports the error, and by a reset."""
import numpy as np
import pytest
import torch

from brewference_b200 import _native as N
from brewference_b200 import config as C
from brewference_b200.api import PREFILL_BATCHED, DeviceModel
from test_gpu_kv import i32
from test_gpu_model import small

pytestmark = pytest.mark.gpu


def raise_counters(dm):
    N.check(N.lib().brew_selftest_raise_counters(dm.handle))


def fail_a_step(dm):
    """A position past the context, given on the device: told by the next call that checks."""
    tok, pos, am = i32([1]), i32([dm.cfg.seq_len]), i32([0])
    torch.cuda.synchronize()
    N.check(N.lib().brew_model_forward_dev(dm.handle, tok.data_ptr(), pos.data_ptr(), 1, None, am.data_ptr(), None))
    torch.cuda.synchronize()


@pytest.mark.parametrize("batched", [False, True])
def test_counters_are_put_back(device, batched):
    cfg = small(C.ARCH_QWEN3, seq_len=1024)
    prompt = np.random.default_rng(1).integers(0, cfg.vocab_size, 700)
    dm = DeviceModel.synthesize(cfg, 3)
    dm.set_kv_cache(C.TYPE_Q4_0)
    if batched:
        dm.set_prefill(PREFILL_BATCHED)
    dm.prefill(prompt)
    want = dm.forward([7], [700])[0]
    assert np.array_equal(dm.forward([7], [700])[0], want)   # the same bits each time
    raise_counters(dm)
    fail_a_step(dm)
    with pytest.raises(N.IllegalStateException):
        dm.forward([7], [700])
    assert np.array_equal(dm.forward([7], [700])[0], want)
    raise_counters(dm)
    dm.reset()
    dm.prefill(prompt)
    assert np.array_equal(dm.forward([7], [700])[0], want)
    dm.close()


def test_raise_counters_refusals(device):
    assert N.lib().brew_selftest_raise_counters(None) == N.ERR_INVALID_ARG
    dm = DeviceModel.synthesize(small(C.ARCH_QWEN3), 1)
    assert N.lib().brew_selftest_raise_counters(dm.handle) == N.ERR_INVALID_ARG
    dm.close()


def test_a_model_whose_cache_cannot_be_had_goes_on_as_it_was(device):
    """The device's memory is taken but for a part of what the pool needs."""
    cfg = small(C.ARCH_LLAMA, seq_len=16384, n_layers=8)
    dm = DeviceModel.synthesize(cfg, 1, max_batch=16)
    pool = 2 * 16 * 8 * 16384 * cfg.kv_dim * 18 // 32
    assert pool > 400 << 20
    want, kernels = dm.forward([3, 4], [0, 0])[0], dm.step_kernels(3)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = torch.empty(torch.cuda.mem_get_info()[0] - (pool // 2), dtype=torch.uint8, device="cuda")
    try:
        with pytest.raises(N.BrewError):
            dm.set_kv_cache(C.TYPE_Q4_0)
    finally:
        del taken
        torch.cuda.empty_cache()
    assert np.array_equal(dm.forward([3, 4], [0, 0])[0], want)
    assert dm.step_kernels(3) == kernels and dm.step_kernels(4) == kernels   # 4: captured only now
    dm.set_kv_cache(C.TYPE_Q4_0)
    dm.forward([3, 4], [0, 0])
    dm.close()
