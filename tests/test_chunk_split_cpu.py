"""CPU tests of the chunk attention's split rule."""

import pytest

from nvfp4_attn_kernel_b200.nvfp4_decode_kernel.chunk import chunk_split_heuristic


@pytest.mark.parametrize("heads_q,heads_kv", [(300, 2), (129, 1), (18, 2), (10, 4), (3, 8), (0, 2), (8, 0), (0, 0)])
def test_heads_that_the_library_refuses_are_left_to_it(heads_q, heads_kv):
    assert chunk_split_heuristic(1, 4, 4, heads_q, heads_kv, 16, sms=148) == 1


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 16, 32])
@pytest.mark.parametrize("rows,tokens,chunk,columns", [(0, 0, 0, 0), (1, 1, 1, 0), (1, 1, 1, 1), (4, 16, 4, 17), (1, 512, 512, 132),
                                                       (7, 3000, 777, 46), (65535, 65535, 1, 1024)])
def test_counts_are_within_the_tiles(group, rows, tokens, chunk, columns):
    splits = chunk_split_heuristic(rows, tokens, chunk, 2 * group, 2, columns, sms=148)
    assert 1 <= splits <= max(1, min(32, columns + -(-chunk // 128)))
