"""Calls of the training operators that their documentation allows, beside
the ordinary ones: the mode that changes between a workspace's query and the
call.  Bounds: tests/test_gpu_loss.py."""
import pytest
import torch

from hp_rms_norm_amd import abi
from test_gpu_loss import check_backward, check_forward, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "the gpu tests need a HIP device"
    import hp_rms_norm_amd
    return hp_rms_norm_amd


@pytest.mark.parametrize("rows,hidden,vocab", [(1, 64, 300), (17, 128, 5000), (100, 65, 9000)])
def test_the_mode_changes_between_a_workspace_and_its_call(ops, rows, hidden, vocab):
    h, w, t, dloss = make(rows, hidden, vocab, torch.bfloat16, rows)
    stream = torch.cuda.current_stream().cuda_stream
    previous = ops.set_batch_invariant(False)
    try:
        for mode in (False, True):
            ops.set_batch_invariant(mode)
            n = abi.linear_cross_entropy_workspace(rows, hidden, vocab, w.data_ptr(), hidden)
            m = abi.linear_cross_entropy_backward_workspace(rows, hidden, vocab, w.data_ptr(), hidden)
            ws = torch.empty(max(n, m), dtype=torch.uint8, device=DEV)
            ops.set_batch_invariant(not mode)
            loss, lse = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
            abi.linear_cross_entropy(loss.data_ptr(), lse.data_ptr(), h.data_ptr(), w.data_ptr(), t.data_ptr(),
                                     ws.data_ptr(), n, rows, hidden, vocab, hidden, hidden, -100, abi.DTYPE_BF16,
                                     stream)
            dh, dw = torch.empty_like(h), torch.empty_like(w)
            abi.linear_cross_entropy_backward(dh.data_ptr(), dw.data_ptr(), dloss.data_ptr(), h.data_ptr(),
                                              w.data_ptr(), t.data_ptr(), lse.data_ptr(), ws.data_ptr(), m, rows,
                                              hidden, vocab, hidden, hidden, hidden, hidden, -100, abi.DTYPE_BF16,
                                              stream)
            check_forward(loss, lse, h, w, t)
            check_backward(dh, dw, h, w, t, dloss)
            want = ops.linear_cross_entropy(h, w, t)
            assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    finally:
        ops.set_batch_invariant(previous)
