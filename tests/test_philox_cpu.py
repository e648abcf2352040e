"""The generator behind dropout's masks, word by word: Philox4x32-10 against its published vectors, and the oracle's mask against it."""
import pytest

from tests import operator_ref as R


def words(counter, key):
    """Philox4x32-10 (Salmon et al. 2011) in whole numbers, its counter and key as 32-bit words in the published order."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


# (counter, key, words), as published with the generator
VECTORS = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
           ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]


@pytest.mark.parametrize("counter,key,want", VECTORS)
def test_published_vectors(counter, key, want):
    assert tuple(words(counter, key)) == want


@pytest.mark.parametrize("seed,offset", [(0, 0), (1, 0), (2 ** 32, 0), (0, 1), (0, 2 ** 32), (0xA4093822 | 0x299F31D0 << 32, 0x13198A2E | 0x03707344 << 32),
                                         (2 ** 64 - 1, 2 ** 64 - 1), (-7, -1)])
def test_the_oracles_mask_is_made_of_these_words(seed, offset):
    """Element e: word e % 4 of counter (e / 4 in two words, offset in two), key seed, low words first; kept from floor(p 2^32) on."""
    s, o = seed % 2 ** 64, offset % 2 ** 64
    draws = [v for q in range(25) for v in words((q, 0, o % 2 ** 32, o >> 32), (s % 2 ** 32, s >> 32))]
    for p in (.03, .25, .5, .9):
        assert R.keep(99, p, seed, offset).tolist() == [v >= int(p * 2 ** 32) for v in draws[:99]]
    # thresholds next to a word itself
    for e in (0, 1, 2, 3, 42, 97):
        assert bool(R.keep(99, draws[e] / 2 ** 32, seed, offset)[e]) and not bool(R.keep(99, (draws[e] + 1) / 2 ** 32, seed, offset)[e])
