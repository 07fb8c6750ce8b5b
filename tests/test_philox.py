"""The test oracle's Philox-4x32-10 against the known answers that its authors published (Salmon, Moraes, Dror, Shaw 2011)."""

import pytest

from tests.token_reference import philox_halves

# counter, key, result
KNOWN = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8))]


@pytest.mark.parametrize("counter,key,words", KNOWN)
def test_known_answers(counter, key, words):
    halves = philox_halves(key[1] << 32 | key[0], counter[3] << 32 | counter[2], 8).tolist()
    assert halves == [h for w in words for h in (w & 0xFFFF, w >> 16)]
