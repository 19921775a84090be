"""Calls on 400-byte rows that run, unsplit, in each of the kernels (16, 32 or 128 heads or rows a workgroup), longer than
one span of 2048 entries or positions.  tests/test_fp4_kernels_cpu.py asks the library which they run in."""
from __future__ import annotations

KERNELS = (16, 32, 128)
# heads a workgroup -> tokens, heads, entries
LISTS = {16: (6, 40, 4300), 32: (110, 40, 4300), 128: (170, 128, 4300)}
# rows a workgroup -> new tokens, lengths, heads
CHUNKS = {16: ([1, 2, 1, 3], [4500, 2300, 2049, 4000], 20),
          32: ([5, 4, 6, 5, 5, 5, 5, 5], [4500, 2300, 2049, 4000, 2100, 40, 4097, 2048], 128),
          128: ([25, 20, 30, 25, 25, 25, 25, 25], [4500, 2300, 2049, 4000, 2100, 40, 4097, 2048], 128)}
BLOCK_SIZE = 64


def bound(lens):
    """What a block table of these sequences can hold."""
    return -(-max(lens) // BLOCK_SIZE) * BLOCK_SIZE
