"""Edges of the gradient norm, the clipping and the clipped Adam steps that need no GPU."""
from __future__ import annotations

import numpy as np

from oracle import adam_oracle as O


def test_rounding_keeps_what_is_not_finite():
    """The stochastic rounding to bfloat16 of NaN is NaN whatever the noise, of an infinity that infinity."""
    noise = np.arange(1 << 16, dtype=np.uint32)
    for bits in (0x7FFFFFFF, 0x7FC00000, 0x7F800001, 0xFFFFFFFF, 0xFFC00000):
        f = np.full(noise.size, bits, np.uint32).view(np.float32)
        assert np.isnan(O.bf16_bits_to_float(O.float_to_bf16_bits_sr(f, noise))).all()
    for sign in (1.0, -1.0):
        f = np.full(noise.size, sign * np.inf, np.float32)
        assert (O.bf16_bits_to_float(O.float_to_bf16_bits_sr(f, noise)) == sign * np.inf).all()
