"""What can be checked on the host of 4-bit products and of how they share an SM."""
import ctypes
import random

import pytest
import torch

from torchinferno_b200.kernels import ops


def room(rows, columns, features, experts=0, bits=4, codes=1):
    """{columns of tensor memory, bytes of shared memory} of a block of such a product."""
    found = (ctypes.c_int * 2)()
    at = ctypes.addressof(found)
    status = (ops.lib().tib_microscaled_room(rows, features, columns, experts, at) if bits == 4 else
              ops.lib().tib_block_scaled_tcgen05_room(codes, rows, features, columns, experts, at))
    assert status == 0, (rows, columns, features, experts, status)
    return tuple(found)


def shared(rows, columns, features, bits, codes):
    """How many blocks share a tile of such a product."""
    found = (ctypes.c_int * 4)()
    at = ctypes.addressof(found)
    status = (ops.lib().tib_microscaled_plan(rows, features, columns, 0, at) if bits == 4 else ops.lib().tib_block_scaled_plan(codes, rows, features, columns, 0, at))
    assert status == 0
    return found[1]


def test_blocks_that_fit_an_sm_together_find_their_columns():
    """512 columns and 228 KB an SM, 1 KB of that for each block itself.  A block of less shared memory than its columns' share can make another block wait that it
    waits for itself (csrc/tcgen05.cuh).  Of two blocks of 256 columns and more 56 columns' share may be left, 25 KB: less than the smallest block takes."""
    g = random.Random(5)
    seen = set()
    sizes = [(m, k, n, e) for m in (1, 8, 20, 33, 64, 128, 129, 300, 2000) for k in (16, 256, 300, 512, 768, 1000, 1300, 2048, 4096, 14336) for n in (64, 1024, 4096, 28672) for e in (0, 32)]
    sizes += [(int(2 ** g.uniform(0, 12)), int(2 ** g.uniform(0, 14)), int(2 ** g.uniform(0, 16)), g.choice([0, 0, 8, 200, 1024])) for _ in range(2000)]
    least = 228 * 1024
    for m, k, n, e in sizes:
        for bits, codes in ((4, 1), (8, 0), (8, 1)):
            columns, smem = room(m, k, n, e, bits, codes)
            seen.add((bits, columns))
            least = min(least, smem + 1024)
            assert columns in (32, 64, 128, 256, 512) and smem <= 227 * 1024, (m, k, n, e, bits)
            assert smem + 1024 >= (columns - (28 if columns >= 256 else 0)) * 228 * 1024 // 512, (m, k, n, e, bits, columns, smem)
            assert e or shared(m, k, n, bits, codes) == 1 or smem + 1024 > 30 * 1024      # (in clusters: beside 512 columns and 199 KB)
    assert {(4, 64), (4, 128), (4, 256), (4, 512), (8, 64), (8, 128), (8, 256), (8, 512)} <= seen and least > 56 * 228 * 1024 // 512


@pytest.mark.parametrize("sizes", [(0, 8, 8, 0), (8, 0, 8, 0), (8, 8, 0, 0), (8, 8, 8, -1)])
def test_no_room_for_no_product(sizes):
    m, n, k, e = sizes
    found = (ctypes.c_int * 2)()
    for status in (ops.lib().tib_microscaled_room(m, n, k, e, ctypes.addressof(found)), ops.lib().tib_block_scaled_tcgen05_room(1, m, n, k, e, ctypes.addressof(found)),
                   ops.lib().tib_microscaled_room(8, 8, 8, 0, 0), ops.lib().tib_block_scaled_tcgen05_room(1, 8, 8, 8, 0, 0)):
        assert status < 0
