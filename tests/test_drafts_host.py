"""Drafts looked up in a row's own text (no GPU)."""

import random

import pytest

from qwenforge_amd.paged_engine import lookup_drafts


def _definition(tokens, n, longest):
    for k in range(min(longest, len(tokens) - 1), 0, -1):
        found = [i for i in range(len(tokens) - k) if tokens[i:i + k] == tokens[-k:]]
        if found:
            whole = [i for i in found if len(tokens) - i - k >= n]
            i = max(whole) if whole else min(found)
            return tokens[i + k:i + k + n]
    return []


def test_repeating_text_is_drafted_to_the_full_length():
    assert lookup_drafts([7] * 50, 4) == [7] * 4
    assert lookup_drafts([1, 2] * 20, 4) == [1, 2, 1, 2]
    assert lookup_drafts([1, 2, 3] * 4, 8) == [1, 2, 3, 1, 2, 3, 1, 2]
    assert lookup_drafts([7] * 5, 4) == [7, 7]           # no occurrence has more behind it
    # The last occurrence where it has enough behind it.
    assert lookup_drafts([1, 2, 3, 9, 9, 1, 2, 3, 4, 4, 1, 2, 3], 2) == [4, 4]


@pytest.mark.parametrize("longest", [0, 1, 2, 3, 5])
def test_against_the_definition(longest):
    rng = random.Random(longest)
    for _ in range(2000):
        tokens = [rng.randint(0, rng.choice([1, 3, 9])) for _ in range(rng.randint(0, 24))]
        n = rng.randint(0, 6)
        assert lookup_drafts(tokens, n, longest) == _definition(tokens, n, longest), (tokens, n)
    assert lookup_drafts((4, 5, 4), 2, longest) == ([5, 4] if longest else [])
