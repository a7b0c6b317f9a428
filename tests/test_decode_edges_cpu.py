"""Calls of the decode-step operators at the limits of their arguments, refused on the host."""

import ctypes

import pytest

from test_decode_ops_cpu import FAKE, cache, refused


@pytest.mark.parametrize("block_size,max_blocks,new_blocks,budget", [
    (2**31 - 1, 1, 1, 2**31 - 1),  # outputs: the loop over a row of `kept` stepped past 2^31
    (2**31 - 1, 0, 1, 2**31 - 500),
    (1, 2**31 - 1, 16, 16),  # lengths: so did the loops over a sequence's positions
    (2**31 - 8191, 1, 1, 16),
])
def test_evict_refuses_positions_near_the_end_of_32_bits(block_size, max_blocks, new_blocks, budget):
    c = cache(block_size=block_size, kv_heads=1)
    message = refused("int4gemv_paged_evict", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, FAKE, budget, 4,
                      1, max_blocks, new_blocks, None)
    assert message.startswith("paged_evict: batch = 1 with tables of") and message.endswith("out of range")
