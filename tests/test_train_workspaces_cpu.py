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


@pytest.mark.parametrize("rows", [16384, 100000, 1 << 22])
@pytest.mark.parametrize("vocab", [1 << 21, 1 << 23, (1 << 25) + 1, 1 << 28])
def test_forward_launches_stay_within_the_grid(rows, vocab):
    """A launch holds less than 2^32 work-items.  Its partial sums are what the
    workspace holds beyond index, target logits and packed rows: 8 bytes a
    row of the launch and a tile of 256 vocabulary entries; a workgroup of 512
    lanes takes 256 such rows."""
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    tiles = -(-vocab // 256)
    rest = 256 + 2 * up(4 * rows) + rows * 64 * 2
    size = abi.linear_cross_entropy_workspace(rows, 64, vocab)
    at_a_time, left = divmod(size - rest, tiles * 8)
    assert left == 0 and 0 < at_a_time <= rows
    assert tiles * -(-at_a_time // 256) * 512 < 1 << 32
