"""The paged 4-bit K/V cache and the token scores without a GPU: index
arithmetic of the layout, and the refusals that come before any device work."""
import ctypes
import os
import subprocess

import pytest

from brewference_b200 import _native as N
from brewference_b200 import build as B
from brewference_b200.api import KvCache, KvRope, KvRows, Logits

HERE = os.path.dirname(os.path.abspath(__file__))


def test_layout_and_entry_checks(tmp_path):
    exe = str(tmp_path / "kv_layout_check")
    cuda = os.path.dirname(os.path.dirname(B.nvcc()))
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(cuda, "include"), "-I", B.CSRC,
                           os.path.join(HERE, "kv_layout_check.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout


@pytest.mark.parametrize("kw,exc", [
    (dict(head_size=48), N.IllegalStateException),          # not a built head size (unsupported)
    (dict(head_size=512), N.IllegalStateException),
    (dict(n_heads=7), N.IllegalArgumentException),          # heads that do not share evenly
    (dict(n_layers=0), N.IllegalArgumentException),
    (dict(n_kv_heads=0), N.IllegalArgumentException),
    (dict(max_seqs=0), N.IllegalArgumentException),
    (dict(max_seqs=2049), N.IllegalArgumentException),
    (dict(max_tokens=0), N.IllegalArgumentException),
    (dict(page_tokens=48), N.IllegalArgumentException),
    (dict(page_tokens=256), N.IllegalArgumentException),
    (dict(n_pages=-1), N.IllegalArgumentException),
    (dict(max_seqs=2048, max_tokens=1 << 30), N.IllegalArgumentException),   # 2^35 pages
])
def test_create_refusals(kw, exc):
    base = dict(n_layers=1, n_heads=8, n_kv_heads=4, head_size=64, max_seqs=2, max_tokens=100, page_tokens=16, n_pages=0)
    base.update(kw)
    with pytest.raises(exc):
        KvCache(**base)


def test_null_handles_are_refused():
    L = N.lib()
    rows = KvRows(16, 16, 1)
    assert L.brew_kv_reserve(None, 0, 1, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_release(None, 0, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_check(None) == N.ERR_INVALID_ARG
    assert L.brew_kv_info(None, None, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_workspace_bytes(None) == -1
    assert L.brew_kv_append_dev(None, 0, None, None, 0, None, None, 0, rows.ref, None, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_read_dev(None, 0, None, None, 0, rows.ref, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_attend_dev(None, 0, None, 0, None, 0, rows.ref, 0, 0.0, None, None) == N.ERR_INVALID_ARG
    assert L.brew_kv_free(None) == N.OK


@pytest.mark.parametrize("args", [
    dict(logits_ptr=0), dict(vocab=0), dict(rows=-1), dict(ld=99), dict(tokens_ptr=0), dict(logprob_ptr=0),
    dict(top=-1), dict(top=33), dict(vocab=5, top=6), dict(top_ids_ptr=0), dict(top_logprobs_ptr=0), dict(logits_ptr=4098),
    dict(tokens_ptr=0, logprob_ptr=0, entropy_ptr=0, top=0),
])
def test_logprobs_refusals(args):
    """Addresses are never read: the checks come first."""
    base = dict(logits_ptr=4096, ld=100, vocab=100, rows=2, tokens_ptr=4096, logprob_ptr=4096, entropy_ptr=4096, top=4,
                top_ids_ptr=4096, top_logprobs_ptr=4096)
    base.update(args)
    with pytest.raises(N.IllegalArgumentException):
        Logits.logprobs_device(**base)


def test_struct_sizes():
    assert ctypes.sizeof(N.KvConfig) == 32
    assert ctypes.sizeof(N.KvRowsC) == 40
    assert ctypes.sizeof(N.KvRopeC) == 48
    assert KvRope(1, 1e6).c.base == 1e6
