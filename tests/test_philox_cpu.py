"""Philox4x32-10 with all six of its input words against the published vectors of its authors (Random123, known answers of philox4x32 with ten
rounds), and the place that seed and offset have among those words."""
import pytest

from tests import attention_rule as R


def block(counter, key):
    """Four words from a counter of four and a key of two."""
    (a, b, c, d), (k, l) = counter, key
    for r in range(10):
        low, high = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (high >> 32) ^ b ^ ((k + r * 0x9E3779B9) % 2**32), high % 2**32, (low >> 32) ^ d ^ ((l + r * 0xBB67AE85) % 2**32), low % 2**32
    return [a, b, c, d]


@pytest.mark.parametrize("counter,key,words", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0], [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
], ids=["zeros", "ones", "pi"])
def test_published_vectors(counter, key, words):
    assert block(counter, key) == words


@pytest.mark.parametrize("seed,offset", [(0, 0), (1, 0), (1 << 32, 0), (0, 1), (0, 1 << 32), (0x0123456789ABCDEF, 0xFEDCBA98), (0x7FFFFFFF00000005, (5 << 32) - 2), (-1, 3), (7, 2**64 - 2)], ids=hex)
def test_low_words_come_first(seed, offset):
    """The oracle's words: 64 bits of the counter in words 0 and 1, 64 bits of the seed as the key, low words in front; the counter goes on from block to
    block over both words, and starts again behind 2^64 - 1."""
    want = []
    for i in range(4):
        at = (offset + i) % 2**64
        want += block([at % 2**32, at >> 32, 0, 0], [seed % 2**32, seed % 2**64 >> 32])
    assert R.philox_words(13, seed, offset).tolist() == want[:13]
    if seed % 2**32 != seed % 2**64 >> 32:
        assert R.philox_words(4, seed, offset).tolist() != R.philox_words(4, (seed % 2**32 << 32) | (seed % 2**64 >> 32), offset).tolist()
