"""CPU tests of the gated operators' and the distillation's host side: packed arguments, refusals of the C ABI, no launches."""

import subprocess
import os

import pytest
import torch

from exponentially_weighted_signature_b200 import _lib, gated_ops, recur_ops, token_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _recur(batch=2, steps=300, channels=64, dtype=1, x=16, rate=16, out=16, dx=16, carry=16):
    return recur_ops._RECUR(batch, steps, channels, dtype, x, 16, 16, *([0] * 6), rate, 0, 0, out, 0, carry, 16, 0, 0, 0, dx, 16, 16, 0, 0, 0, 0, 0)


def _gated(rows=200, dim=64, inner=128, dtype=1, act=0, xs=64, gs=64, us=64, x=16, kept=16, dout_stride=128, dx=16):
    return gated_ops._GATED(rows, dim, inner, dtype, act, x, 16, 16, xs, gs, us, 16, kept, 16, dout_stride, dx, 16, 16, 0, 0, 0)


def _distill(rows=10, vocab=100, dim=16, dtype=1, hs=16, ws=16, top=4, logits_dtype=0, inv_tau=1.0, ids=16, entries=16):
    v = token_ops._VOCAB(rows, vocab, dim, dtype, 0, 16, 16, 0, hs, ws, 0, 16, 16, 16, 16, 16, 16, 0, 0, 0)
    return v + token_ops._TOP(ids, 16, 0, top, logits_dtype, inv_tau, entries)


def test_packed_arguments_have_the_structs_sizes(tmp_path):
    src = tmp_path / "s.c"
    src.write_text('#include "%s/include/ews_b200.h"\n#include <stdio.h>\nint main(void){printf("%%zu %%zu %%zu", sizeof(ews_recur_args), '
                   'sizeof(ews_gated_args), sizeof(ews_distill_args));return 0;}' % ROOT)
    subprocess.run(["gcc", "-o", str(tmp_path / "s"), str(src)], check=True)
    sizes = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [len(_recur()), len(_gated()), len(_distill())] == [int(x) for x in sizes]


def test_recurrence_arguments_are_checked_before_the_device():
    lib = _lib.load()
    for bad, code in ((dict(batch=-1), 1), (dict(steps=-1), 1), (dict(channels=0), 1), (dict(dtype=5), 2)):
        assert lib.ews_recur_work_size(_recur(**bad), 0) == 0 and lib.ews_recur_carry_size(_recur(**bad)) == 0
        assert lib.ews_recur_fwd(_recur(**bad), None) == code and lib.ews_recur_bwd(_recur(**bad), None) == code, bad
        assert lib.ews_recur_step(_recur(**bad), None, 8, 16, None) == code
    for bad in (dict(x=0), dict(rate=0), dict(out=0)):
        assert lib.ews_recur_fwd(_recur(**bad), None) == 1
    assert lib.ews_recur_bwd(_recur(dx=0), None) == 1
    assert lib.ews_recur_bwd(_recur(carry=0), None) == 1  # several tiles need the forward's states
    assert lib.ews_recur_fwd(_recur(), None) == 3 and lib.ews_recur_bwd(_recur(), None) == 3
    assert lib.ews_recur_work_size(_recur(batch=0), 0) == 0 and lib.ews_recur_fwd(_recur(batch=0), None) == 0
    assert lib.ews_recur_work_size(_recur(steps=64), 0) == 0  # one tile waits for nobody
    assert lib.ews_recur_step(_recur(), None, 1, 16, None) == 1  # fewer states than rows and no slots
    assert lib.ews_recur_step(_recur(), 16, -1, 16, None) == 1 and lib.ews_recur_step(_recur(), 16, 8, None, None) == 1
    assert recur_ops._sizes(2, 300, 64, 1) == (lib.ews_recur_carry_size(_recur()), lib.ews_recur_work_size(_recur(), 0), lib.ews_recur_work_size(_recur(), 1))


def test_gated_arguments_are_checked_before_the_device():
    lib = _lib.load()
    for bad, code in ((dict(rows=-1), 1), (dict(dim=0), 1), (dict(inner=0), 1), (dict(xs=63), 1), (dict(gs=8), 1), (dict(us=8), 1),
                      (dict(dtype=4), 2), (dict(act=2), 2)):
        assert lib.ews_gated_work_size(_gated(**bad), 1) == 0
        assert lib.ews_gated_fwd(_gated(**bad), None) == code and lib.ews_gated_bwd(_gated(**bad), None) == code, bad
    assert lib.ews_gated_fwd(_gated(x=0), None) == 1
    assert lib.ews_gated_kept_size(_gated()) == gated_ops._kept_size(200, 64, 128, 1) == 3 * 2 * 200 * 128
    assert lib.ews_gated_bwd(_gated(kept=0), None) == 1 and lib.ews_gated_bwd(_gated(dout_stride=100), None) == 1
    assert lib.ews_gated_bwd(_gated(), None) == 3
    assert lib.ews_gated_fwd(_gated(dtype=0), None) == 3  # float32 is packed in planes
    assert lib.ews_gated_fwd(_gated(rows=0), None) == 0
    # operands that TMA cannot read as they lie are packed; few float32 rows are read as they lie
    assert lib.ews_gated_work_size(_gated(), 0) == 0 < lib.ews_gated_work_size(_gated(xs=65), 0)
    assert lib.ews_gated_work_size(_gated(rows=128), 0) == 0 < lib.ews_gated_work_size(_gated(rows=128, xs=65), 0)
    assert lib.ews_gated_work_size(_gated(rows=32, dtype=0), 0) == 0 < lib.ews_gated_work_size(_gated(rows=33, dtype=0), 0)
    size = gated_ops._size(200, 64, 128, 1, (64, 64, 64), (0, 0, 0), (1, 1, 1), 1)
    assert size == lib.ews_gated_work_size(_gated(), 1) > 0


def test_distillation_arguments_are_checked_before_the_device():
    lib = _lib.load()
    for bad, code in ((dict(vocab=0), 1), (dict(hs=8), 1), (dict(top=0), 1), (dict(inv_tau=0.0), 1), (dict(inv_tau=float("nan")), 1),
                      (dict(inv_tau=float("inf")), 1), (dict(top=129), 2), (dict(logits_dtype=3), 2), (dict(dtype=9), 2)):
        assert lib.ews_distill_work_size(_distill(**bad), 0) == 0
        assert lib.ews_distill_fwd(_distill(**bad), None) == code and lib.ews_distill_bwd(_distill(**bad), None) == code, bad
    assert lib.ews_distill_fwd(_distill(ids=0), None) == 1
    assert lib.ews_distill_fwd(_distill(entries=0), None) == 1 and lib.ews_distill_bwd(_distill(entries=0), None) == 1
    assert lib.ews_distill_fwd(_distill(), None) == 3 and lib.ews_distill_bwd(_distill(), None) == 3
    assert lib.ews_distill_fwd(_distill(rows=0), None) == 0
    assert lib.ews_distill_entries_size(10, 4) == 400 and lib.ews_distill_entries_size(0, 4) == 0
    for backward in (0, 1):
        assert token_ops._distill_size(10, 100, 16, 1, 16, 16, 0, 4, backward) == lib.ews_distill_work_size(_distill(), backward) > 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError):
        recur_ops.gated_recurrence(x, x, x, torch.ones(8))
    with pytest.raises(RuntimeError):
        recur_ops.gated_recurrence_step(x[0], x[0], x[0], torch.ones(8), torch.zeros(4, 8))
    with pytest.raises(RuntimeError):
        gated_ops.gated_linear(x, torch.zeros(3, 8), torch.zeros(3, 8))
    with pytest.raises(RuntimeError):
        token_ops.distill_loss(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))


def test_shapes_and_types_are_refused():
    x, r = torch.zeros(1, 4, 8), torch.ones(8)
    for call in (lambda: recur_ops.gated_recurrence(x, x, x[:, :3], r), lambda: recur_ops.gated_recurrence(x, x, x, r[:4]),
                 lambda: recur_ops.gated_recurrence(x[0], x[0], x[0], r), lambda: recur_ops.gated_recurrence(x, x, x, r, lengths=torch.zeros(1)),
                 lambda: recur_ops.gated_recurrence(x[..., :0], x[..., :0], x[..., :0], r[:0]),
                 lambda: gated_ops.gated_linear(x, torch.zeros(3, 7), torch.zeros(3, 7)),
                 lambda: gated_ops.gated_linear(x, torch.zeros(3, 8), torch.zeros(4, 8)),
                 lambda: gated_ops.gated_linear(x, torch.zeros(3, 8), torch.zeros(3, 8), activation="tanh"),
                 lambda: token_ops.distill_loss(x, torch.zeros(5, 8), torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, 4)),
                 lambda: token_ops.distill_loss(x, torch.zeros(5, 8), torch.zeros(1, 4, 2, dtype=torch.int64), torch.zeros(1, 4, 2), temperature=0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: recur_ops.gated_recurrence(x.half(), x.half(), x.half(), r), lambda: recur_ops.gated_recurrence(x, x, x.bfloat16(), r),
                 lambda: gated_ops.gated_linear(x, torch.zeros(3, 8), torch.zeros(3, 8).bfloat16()),
                 lambda: token_ops.distill_loss(x, torch.zeros(5, 8), torch.zeros(1, 4, 2), torch.zeros(1, 4, 2))):
        with pytest.raises(TypeError):
            call()


def test_a_gated_block_is_built_as_it_says():
    from exponentially_weighted_signature_b200 import GatedBlock, TokenModel

    block = GatedBlock(96)
    assert block.ff_gate.weight.shape == (256, 96) and block.inputs.weight.shape == (288, 96)
    assert torch.allclose(torch.exp(block.log_rate)[[0, -1]], torch.tensor([1.0, 2.0**-8]))
    assert [s.shape for s in TokenModel(20, 32, 2, ("gated", "decay"), gated_kwargs=dict(width=24)).states(3)] == [(3, 24), (3, 2, 16, 16)]
    with pytest.raises(ValueError):
        TokenModel(20, mixers=("gate",))


def test_narrow_rows_keep_one_plane():
    """A second plane of what the gradients' products read costs as much as its elements and its tiles do, however narrow the rows are."""
    from exponentially_weighted_signature_b200 import gated_ops, token_ops

    rows, many = 8192, 16384
    for dim in (1, 8, 16):
        stride = -(-dim // 8) * 8
        one = 2 * rows * many  # bytes of one plane of G, all of it in one piece
        size = token_ops._distill_size(rows, many, dim, 1, stride, stride, 0, 16, 1)
        assert one < size < 1.5 * one, dim
        for rows_, inner in ((rows, many), (many, rows)):
            size = gated_ops._size(rows_, dim, inner, 1, (stride, stride, stride), (0, 0, 0), (1, 1, 1), 1)
            assert 2 * one < size < 3 * one, dim
