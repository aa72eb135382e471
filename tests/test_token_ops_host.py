"""CPU tests of the token operators' host side: packed arguments, refusals of the C ABI, no launches."""

import ctypes
import struct
import subprocess
import os

import pytest
import torch

from exponentially_weighted_signature_b200 import _lib, token_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _decay(batch=2, steps=100, heads=4, kv=2, dk=64, dv=64, dtype=1, scale=0.125):
    return token_ops._DECAY(batch, steps, heads, kv, dk, dv, dtype, scale, 16, 16, 16, *([0] * 9), 16, 0, 0, 16, 0, 16, 0, 0, 0, 0,
                            16, 16, 16, 0, 0, 0, 0)


def _vocab(rows=10, vocab=100, dim=16, dtype=1, hs=16, ws=16):
    return token_ops._VOCAB(rows, vocab, dim, dtype, 1, 16, 16, 16, hs, ws, -100, 16, 16, 16, 16, 16, 16, 0, 0, 0)


def test_packed_arguments_have_the_structs_sizes(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include "%s/include/ews_b200.h"\n#include <stdio.h>\nint main(void){printf("%%zu %%zu", sizeof(ews_decay_args), sizeof(ews_vocab_args));return 0;}' % ROOT)
    subprocess.run(["gcc", "-o", str(tmp_path / "s"), str(src)], check=True)
    sizes = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [len(_decay()), len(_vocab())] == [int(x) for x in sizes]


def test_decay_arguments_are_checked_before_the_device():
    lib = _lib.load()
    for bad, code in ((dict(heads=3), 1), (dict(kv=0), 1), (dict(dk=0), 1), (dict(dk=129), 2), (dict(dv=200), 2), (dict(dtype=7), 2), (dict(steps=-1), 1)):
        assert lib.ews_decay_work_size(_decay(**bad), 0) == 0
        assert lib.ews_decay_fwd(_decay(**bad), None) == code, bad
        assert lib.ews_decay_bwd(_decay(**bad), None) == code, bad
    assert lib.ews_decay_bwd(_decay(scale=0.0), None) == 1
    assert lib.ews_decay_fwd(_decay(batch=0), None) == 0
    assert lib.ews_decay_work_size(_decay(batch=0), 1) == 0
    assert lib.ews_decay_fwd(_decay(batch=1, heads=1, kv=1, steps=10000), None) == 3  # a split axis needs its workspace
    assert lib.ews_decay_step(_decay(), None, 1, 16, None) == 1  # fewer states than rows and no slots


def test_vocab_arguments_are_checked_before_the_device():
    lib = _lib.load()
    for bad, code in ((dict(vocab=0), 1), (dict(dim=0), 1), (dict(hs=8), 1), (dict(ws=8), 1), (dict(dtype=9), 2)):
        assert lib.ews_vocab_fwd(_vocab(**bad), None) == code, bad
        assert lib.ews_vocab_work_size(_vocab(**bad), 1) == 0
    assert lib.ews_vocab_fwd(_vocab(), None) == 3
    assert lib.ews_vocab_fwd(_vocab(rows=0), None) == 0
    assert lib.ews_vocab_work_size(_vocab(rows=0), 1) == 0
    # the backward's workspace is bounded by a piece of the vocabulary, not by it
    small, large = (lib.ews_vocab_work_size(_vocab(rows=8192, vocab=v, dim=1024, hs=1024, ws=1024), 1) for v in (20000, 2000000))
    assert large < 2 * small


def test_embedding_arguments_are_checked_before_the_device():
    lib = _lib.load()
    assert lib.ews_embed_fwd(16, 1, 16, 1, 4, 0, 8, 8, 1.0, 16, None, None) == 1
    assert lib.ews_embed_fwd(16, 1, 16, 1, 4, 10, 8, 7, 1.0, 16, None, None) == 1
    assert lib.ews_embed_fwd(16, 1, 16, 5, 4, 10, 8, 8, 1.0, 16, None, None) == 2
    assert lib.ews_embed_fwd(16, 1, 16, 1, 0, 10, 8, 8, 1.0, 16, None, None) == 0
    assert lib.ews_embed_work_size(256, 10, 8) == 0  # few positions take no sort and no workspace
    assert lib.ews_embed_work_size(1000, 10, 8) > 0
    assert lib.ews_embed_bwd(16, 1, 16, 1, 1000, 10, 8, 8, 1.0, -1, 16, None, 0, None, None) == 3


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError):
        token_ops.decayed_attention(q, q, q, torch.ones(2))
    with pytest.raises(RuntimeError):
        token_ops.token_embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4))
    with pytest.raises(RuntimeError):
        token_ops.vocab_loss(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64))


def test_index_error_code():
    assert b"out of range" in _lib.load().ews_error_string(_lib.EWS_ERR_INDEX)
    with pytest.raises(IndexError):
        _lib.check(_lib.EWS_ERR_INDEX, "x")
    assert struct.calcsize("@N") == ctypes.sizeof(ctypes.c_size_t)


def test_cached_workspace_sizes_are_the_librarys():
    lib = _lib.load()
    for backward in (0, 1):
        assert token_ops._decay_size(2, 5000, 4, 2, 64, 64, 1, backward) == lib.ews_decay_work_size(_decay(steps=5000), backward) > 0
        assert token_ops._vocab_size(10, 100, 16, 1, 16, 16, 0, backward) == lib.ews_vocab_work_size(_vocab(), backward) > 0
        # a weight that TMA cannot read as it lies is packed in the workspace
        assert token_ops._vocab_size(10, 100, 16, 1, 16, 16, 2, backward) > token_ops._vocab_size(10, 100, 16, 1, 16, 16, 0, backward)
    assert token_ops._embed_size(1000, 10, 8) == lib.ews_embed_work_size(1000, 10, 8) > 0
