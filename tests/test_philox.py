"""The masks' generator against the published answers of Philox4x32-10.

The generator in plain integers (Salmon, Moraes, Dror and Shaw 2011) is checked against its
authors' known answers; the reference that the mask tests use is then checked against it at counters
and keys whose words all differ, so that no two of them can be exchanged unseen.
"""

import numpy as np
import pytest

import low_rank_reference as ref

LOW = 0xFFFFFFFF


def philox(counter, key):
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ k0, b & LOW, (a >> 32) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return c0, c1, c2, c3


@pytest.mark.parametrize("counter, key, answer", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((LOW,) * 4, (LOW,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),  # digits of pi
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_known_answers(counter, key, answer):
    assert philox(counter, key) == answer


@pytest.mark.parametrize("row0", [0, 0x85A308D0])
@pytest.mark.parametrize("seed, offset", [(0x299F31D0A4093822, 0x0370734413198A2E), (2**64 - 1, 1)])
def test_the_mask_reference(seed, offset, row0):
    """Counter (column / 8, row, offset low, offset high), key (seed low, seed high); element
    column % 8 takes its 16 bits from the low half of the first word on."""
    got = ref.philox_halves(3, 20, seed, offset, row0)
    for row in range(3):
        for column in range(20):
            words = philox((column // 8, (row0 + row) & LOW, offset & LOW, offset >> 32),
                           (seed & LOW, seed >> 32))
            half = words[column % 8 // 2] >> 16 * (column % 2) & 0xFFFF
            assert got[row, column] == half
    assert got.dtype == np.int64
