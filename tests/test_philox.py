"""The generator that the dropout tests compare with: the published
known-answer vectors of Philox4x32-10, and the statistics of its words."""
import numpy as np

import philox


def test_known_answers():
    for counter, key, want in (
            ([0, 0, 0, 0], (0, 0), [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF),
             [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0),
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        got = philox.blocks([np.uint64(c) for c in counter], key)
        assert [int(x) for x in got] == want


def test_words_are_spread():
    w = philox.words(1 << 18, 12345, 7).astype(np.float64) / 2 ** 32
    # a mean of n uniform numbers is within 6 of its standard deviations
    assert abs(w.mean() - 0.5) < 6 * np.sqrt(1 / 12 / len(w))
    other = philox.words(1 << 18, 12345, 8).astype(np.float64) / 2 ** 32
    assert abs(np.corrcoef(w, other)[0, 1]) < 6 / np.sqrt(len(w))
