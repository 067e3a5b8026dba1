"""What the blocks of the adapters' cluster kernel take of a multiprocessor. No GPU: the library's own arithmetic."""
import ctypes

import pytest

MULTIPROCESSOR, OF_THE_SYSTEM, COLUMNS = 228 * 1024, 1024, 512     # shared memory, of which each block costs 1 KB more; tensor memory


def needs(width, rows):
    from tgo_b200.kernels.build import entry_points
    got = ctypes.c_int(0)
    columns = entry_points("adapters").tgo_low_rank_tile_needs(width, rows, ctypes.addressof(got))
    return columns, got.value


@pytest.mark.parametrize("rows", [64, 128])
def test_blocks_that_share_a_multiprocessor_all_have_tensor_memory(rows):
    """Blocks of a cluster wait for each other. If their shared memory let two of different clusters onto one multiprocessor
    whose tensor memory is too small for both, each cluster could have one block that waits for a column that the other's
    holds. So a block's share of the shared memory is at least its share of the columns."""
    for width in range(8, 513, 8):
        columns, shared = needs(width, rows)
        assert width <= columns <= COLUMNS and shared <= 227 * 1024
        assert (shared + OF_THE_SYSTEM) * COLUMNS >= columns * MULTIPROCESSOR, (width, columns, shared)
