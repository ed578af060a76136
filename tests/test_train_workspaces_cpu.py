"""The workspaces that the training operators ask for, on the CPU."""
import pytest

from hp_rms_norm_amd import abi, ops


@pytest.mark.parametrize("rows", [1, 17, 100, 3000])
@pytest.mark.parametrize("hidden,vocab", [(64, 100), (4096, 131072), (1001, 7000)])
def test_loss_workspaces_serve_both_batch_invariant_modes(rows, hidden, vocab):
    """The mode may change between the query and the call."""
    sizes = []
    previous = ops.set_batch_invariant(False)
    try:
        for mode in (False, True):
            ops.set_batch_invariant(mode)
            sizes.append((abi.linear_cross_entropy_workspace(rows, hidden, vocab),
                          abi.linear_cross_entropy_backward_workspace(rows, hidden, vocab)))
    finally:
        ops.set_batch_invariant(previous)
    assert sizes[0] == sizes[1]
