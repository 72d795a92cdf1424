"""Frequencies scaled in bands, with the bounds that such models state: more than 4 turns within the original
context kept, fewer than 1 divided, a blend along the turns between."""
import math

import pytest


@pytest.mark.parametrize("rot,base,factor,original", [(128, 5e5, 8.0, 8192), (64, 1e4, 16.0, 4096), (128, 5e5, 32.0, 8192)])
def test_the_bands_end_at_four_turns_and_one(irx, rot, base, factor, original):
    plain = irx.rope_freqs(rot, base=base)
    want = []
    for f in plain:
        turns = original * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
        want.append(f * keep + f / factor * (1.0 - keep))
    got = irx.rope_freqs(rot, base=base, scaling="bands", factor=factor, original=original)
    assert got == pytest.approx(want, rel=1e-14)
    assert got == irx.rope_freqs(rot, base=base, scaling="bands", factor=factor, original=original, fast=4.0, slow=1.0)


def test_other_scalings_keep_their_bounds(irx):
    k = dict(scaling="yarn", factor=4.0, original=8192)
    assert irx.rope_freqs(128, **k) == irx.rope_freqs(128, fast=32.0, slow=1.0, **k)
    assert irx.rope_freqs(128, fast=16.0, **k) != irx.rope_freqs(128, **k)
    assert irx.rope_freqs(128, scaling="linear", factor=2.0) == irx.rope_freqs(128, scaling="linear", factor=2.0, fast=7.0)
