"""Frequencies stretched by parts where the ramp ends behind the last pair (long original contexts: every pair turns more than once)."""
import math

import numpy as np
import pytest

import mxnet_b200 as mx


@pytest.mark.parametrize('dim', [2, 64, 128])
@pytest.mark.parametrize('base', [1e4, 5e5])
@pytest.mark.parametrize('original', [8, 4096, 65536, 131072, 1048576, 10 ** 8])
@pytest.mark.parametrize('fast,slow', [(32.0, 1.0), (8.0, 0.5)])
def test_yarn_at_every_length(dim, base, original, fast, slow):
    factor = 4.0
    plain = mx.npx.rotary_inv_freq(dim=dim, base=base, dtype='float64').asnumpy()
    got = mx.npx.rotary_inv_freq(dim=dim, base=base, scaling='yarn', factor=factor, original_length=original, fast_turns=fast,
                                 slow_turns=slow, dtype='float64').asnumpy()
    turns, ratio = original * plain / (2 * math.pi), got / plain
    assert (ratio[turns > slow * (1 + 1e-9)] > 1 / factor).all()     # only pairs of so few turns are interpolated whole
    assert (ratio[turns >= fast * (1 + 1e-9) * base ** (2.0 / dim)] == 1).all()
    # the method's formula: a ramp between the whole pairs around the two real-valued ones, which may lie anywhere in 0 .. dim - 1
    at = [dim * np.log(original / (t * 2 * np.pi)) / (2 * np.log(base)) for t in (fast, slow)]
    low, high = max(np.floor(at[0]), 0), min(np.ceil(at[1]), dim - 1)
    ramp = np.clip((np.arange(dim // 2) - low) / max(high - low, 1e-3), 0, 1)
    np.testing.assert_allclose(got, plain / factor * ramp + plain * (1 - ramp), rtol=1e-12)
