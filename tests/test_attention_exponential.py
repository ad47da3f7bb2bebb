"""The polynomial for 2^f in attention.cu: the coefficients are those that fit_transcendentals.py derives, and its error is what the comment says."""
import os
import re
import sys

import numpy as np

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gevva_b200", "csrc")


def coefficients():
    with open(os.path.join(CSRC, "attention.cu")) as f:
        text = f.read()
    body = text[text.index("void exp2_by_polynomial("):]
    body = body[:body.index("\n}\n")]
    pairs = re.findall(r"two\((0\.\d+)f, (0\.\d+)f\)", body)
    assert len(pairs) == 5 and all(a == b for a, b in pairs)
    return np.array([float(a) for a, _ in pairs][::-1])


def test_coefficients_are_the_derived_ones(monkeypatch):
    monkeypatch.syspath_prepend(CSRC)
    from fit_transcendentals import exp2_minimax
    sys.modules.pop("fit_transcendentals")
    derived, worst = exp2_minimax()
    here = coefficients()
    assert (here == here.astype(np.float32)).all()
    assert (np.abs(here - derived) <= 2 * np.spacing(here.astype(np.float32))).all() and worst < 2.6e-6


def test_largest_error():
    """In 32 bits, every product and sum fused: one rounding each."""
    f = np.linspace(-0.5, 0.5, 2000001).astype(np.float32)
    c = coefficients()
    p = np.full_like(f, c[4])
    for a in c[3::-1]:
        p = (p.astype(np.float64) * f + a).astype(np.float32)
    assert np.abs(p / np.exp2(f.astype(np.float64)) - 1).max() < 2.7e-6 + 2.0 ** -24
