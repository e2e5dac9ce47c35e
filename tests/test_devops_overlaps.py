"""Buffers of the device operators that lie over one another, on the host only (as in test_devops.py)."""
import ctypes as C

import pytest
from test_devops import EINVAL, OK, dv, refused, reorder_of, select_of  # noqa: F401

X = 1 << 28  # logits: six rows of 500 f32; cum and done 24 bytes, the outputs 48


@pytest.mark.parametrize("over,code", [
    (dict(), OK),
    (dict(score=4096), EINVAL),                      # over cum, with more outputs than rows
    (dict(score=4096, n_out=3), OK),                 # in its place
    (dict(score=4100, n_out=3), EINVAL),
    (dict(parent=4096, n_out=3), EINVAL),
    (dict(token=4096 - 44), EINVAL),
    (dict(token=4096 - 48), OK),
    (dict(done=6144, parent=6144 + 20), EINVAL),
    (dict(done=6144, parent=6144 + 24), OK),
    (dict(parent=X + 6 * 2000 - 4), EINVAL),
    (dict(parent=X + 6 * 2000), OK),
    (dict(score=8192 + 44), EINVAL),                 # over parent
    (dict(score=12288), EINVAL),                     # over token
    (dict(token=8192 + 48), OK),
    (dict(score=4096, groups=0), OK),
])
def test_select_outputs(jd, dv, over, code):  # noqa: F811
    a = select_of(dv, **over)
    refused(jd, jd.lib().jdg_beam_select_check(C.byref(a)), code, "overlaps")


@pytest.mark.parametrize("dst,code", [
    (4096, EINVAL), (4096 + 28, EINVAL), (4096 + 32, OK), (4096 - 800, OK), (4096 - 799, EINVAL),
])
def test_reorder_parents(jd, dv, dst, code):  # noqa: F811
    a = reorder_of(dv, [(1 << 20, dst, 100, 100, 100)])  # two groups of four parents at 4096, eight rows of 100
    refused(jd, jd.lib().jdg_beam_reorder_check(C.byref(a)), code, "overlaps the parents")


@pytest.mark.gpu
def test_select_scores_in_place(jd, dv):  # noqa: F811
    """score = cum with n_out = beams, in C: the same as apart."""
    import torch
    torch.manual_seed(3)
    groups, beams, vocab = 40, 4, 3001
    logits, cum = torch.randn((groups * beams, vocab), device="cuda"), -torch.rand(groups * beams, device="cuda") * 4
    want = jd.beam_select(logits, cum, beams, beams)
    parent = torch.empty((groups, beams), dtype=torch.int32, device="cuda")
    token = torch.empty_like(parent)
    a = dv.JdgSelectArgs(logits.data_ptr(), 0, vocab, groups, beams, vocab, beams, cum.data_ptr(), None, 0,
                         parent.data_ptr(), token.data_ptr(), cum.data_ptr())
    n = jd.lib().jdg_beam_select_workspace(C.byref(a))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert jd.lib().jdg_beam_select(C.byref(a), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == OK
    assert torch.equal(parent, want[0]) and torch.equal(token, want[1]) and torch.equal(cum.view_as(want[2]), want[2])
