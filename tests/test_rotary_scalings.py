"""The frequencies of scaled rotary tables (no GPU)."""

import math

import pytest

from kohaku_tt_b200.rotary import rotary_frequencies


@pytest.mark.parametrize("dim,base,factor,original,fast,slow", [(128, 10000.0, 4.0, 4096, 32.0, 1.0), (128, 1e6, 4.0, 32768, 32.0, 1.0), (64, 5e5, 8.0, 8192, 4.0, 1.0)])
def test_parts_are_mixed_by_turns(built_lib, dim, base, factor, original, fast, slow):
    """A pair that makes r turns within the original context keeps the share (r - slow) / (fast - slow) of its frequency, 0 at
    least and 1 at most, and f / factor for the rest: linear in r, not in the pair's index."""
    got, scale = rotary_frequencies(dim, base, "parts", factor, original=original, fast=fast, slow=slow)
    mixed = 0
    for i, f in enumerate(got):
        plain = base ** (-2 * i / dim)
        keep = min(1.0, max(0.0, (original * plain / (2 * math.pi) - slow) / (fast - slow)))
        mixed += 0 < keep < 1
        assert math.isclose(f, plain * (keep + (1 - keep) / factor), rel_tol=1e-13)
    # (Frequencies fall by the same factor from pair to pair, so fast / slow spans that many of them, but for the ends.)
    assert mixed >= math.floor(math.log(fast / slow) / math.log(base) * dim / 2) >= 3 and math.isclose(scale, 0.1 * math.log(factor) + 1)
