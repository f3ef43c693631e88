"""The normal tail that bf16 results of K13's GELU are formed from."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np
from scipy.special import log_ndtr

SOURCE = Path(__file__).resolve().parent.parent / "mround_b200" / "csrc" / "linear_sm100.cu"


def test_tail_holds_its_stated_error():
    """The kernel's constants in 64 bits against log Phi.  The fit leaves 6.0e-7;
    rounding nine constants to float32 adds at most ln 2 times the sum of
    2^-24 |c| t^i, 4.4e-7 for their sum of magnitudes below 10.3, and 6.4e-7 is what
    both leave together."""
    body = re.search(r"float gelu_tail\(float z\) \{(.*?)\n\}", SOURCE.read_text(), re.S).group(1)
    first, *rest = re.findall(r"float p = fmaf\((\S+)f, t, (\S+)f\)|p = fmaf\(p, t, (\S+)f\)", body)
    coefficients = [float(c) for c in (*first[:2], *(r[2] for r in rest))]
    assert len(coefficients) == 9
    z = np.linspace(0.0, 13.2, 200001)
    t = 1.0 / (1.0 + 0.5 * z)
    exponent = np.polyval(np.float32(coefficients).astype(np.float64), t) - z * z / (2 * np.log(2))
    assert np.abs(t * np.exp2(exponent) / np.exp(log_ndtr(-z)) - 1).max() <= 6.5e-7
