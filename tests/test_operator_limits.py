"""Sizes beyond what a launch takes (a grid holds less than 2^32 threads): refused by the C entries
with their own message, and by the Python calls before anything is allocated.  No GPU needed."""
import ctypes as C

import pytest
import torch


def test_c_entries_stop_below_a_full_grid():
    from ugpg import _C
    lib, p = _C.lib, 0x1000  # never dereferenced on the host

    def gn(B, HW, Ch, G):
        d = _C.GroupNormDesc(p, 1, B, HW, Ch, G, None, None, 1e-5, 1, p, p)
        return lib.ugpg_group_norm_workspace(C.byref(d), 0)
    # one block of up to 1024 threads a group
    assert gn((1 << 22) - 1, 2049, 1, 1) > 0
    assert gn(1 << 22, 2049, 1, 1) == 0 and b"too large" in lib.ugpg_last_error()
    assert gn(1 << 20, 2049, 4, 4) == 0

    def maps(N, inner, V=40):
        d = _C.DistillDesc(p, 1, N, V, inner, V * inner, p, 1, p, 64, 3, None, None, 1.0, 1.0)
        return lib.ugpg_distill_workspace(C.byref(d), 0)
    # blocks of 64 pixels and 256 threads
    most = (1 << 30) - 64
    assert maps(1, most) > 0 and maps(2, most // 2) > 0
    for N, inner in ((1, most + 1), (1, (1 << 30) - 1), (2, most // 2 + 1)):
        assert maps(N, inner) == 0 and b"too large" in lib.ugpg_last_error()
        assert lib.ugpg_top_logits(p, 1, N, 40, inner, 40 * inner, 3, 1.0, p, p, p, None) == -1
        assert b"too large" in lib.ugpg_last_error()


def test_python_calls_name_their_limits():
    import ugpg

    def wide(*shape):  # one value, seen as many
        return torch.zeros((1,) * len(shape)).expand(shape)

    rows = wide((1 << 22) + 1, 7)
    with pytest.raises(ValueError, match="at most 4194304 rows"):
        ugpg.teacher_top_logits(rows, 3)
    top = (wide((1 << 22) + 1, 3), torch.zeros(1, 1, dtype=torch.int64).expand((1 << 22) + 1, 3), None)
    with pytest.raises(ValueError, match="at most 4194304 rows"):
        ugpg.distillation_loss(rows, top)
    with pytest.raises(ValueError, match="at most 1073741760 pixels"):
        ugpg.teacher_top_logits(wide(1 << 15, 7, 1 << 8, 1 << 7), 3)
    with pytest.raises(ValueError, match="4194304 or more"):
        ugpg.group_norm_act(wide(1 << 20, 2, 4), 4)
    with pytest.raises(ValueError, match="too many"):
        ugpg.group_norm_act(wide(1 << 21, 1, 1024), 1)
    # up to there the next check speaks
    for call in (lambda: ugpg.teacher_top_logits(wide(1 << 22, 7), 3),
                 lambda: ugpg.teacher_top_logits(wide(1 << 16, 7, 1 << 7, (1 << 7) - 1), 3),
                 lambda: ugpg.group_norm_act(wide((1 << 20) - 1, 2, 4), 4)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
