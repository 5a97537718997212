"""The norm's float32 levels (csrc/qs_norm.cu) are kept only where their error can not reach a border.

A level is the integer next to p * inv with p = t w and m = max |p| rounded to float32, inv = 127 / m by
__fdividef. Its documented error is 2 ulp (of a value whose ulp is at most 2^-23 of it). Where the remainder stays
below SURE the level has to be that of exact arithmetic; the same for the scale and its two neighbours.
"""

import re
from fractions import Fraction as F
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parent.parent / "quant-studio_b200" / "csrc" / "qs_norm.cu").read_text()


def constant(name):
    return F(float(np.float32(re.search(rf"\b{name} = ([0-9.e-]+)f", SOURCE).group(1))))


def test_levels():
    half_step, division = F(1, 1 << 24), 2 * F(1, 1 << 23)
    worst = (1 + half_step) * (1 + division) / (1 - half_step) - 1  # of p * inv, relative
    # levels reach 127 and the border behind it; the remainder is rounded once (below 1/2)
    assert F(1, 2) - constant("SURE") > F(255, 2) * worst + F(1, 1 << 26)


def test_scales():
    # ds: m, r / 127 and their product rounded; the exact one is rounded to float32 before float16
    half_step = F(1, 1 << 24)
    worst = (1 + half_step) ** 4 - 1
    near = np.float32(float(constant("NEAR")))
    low, high = F(float(np.float32(1) - near)), F(float(np.float32(1) + near))
    assert low * (1 + half_step) < 1 - worst and high * (1 - half_step) > 1 + worst


def test_constants_are_those_in_use():
    assert SOURCE.count("0.4999") == 1 and SOURCE.count("4e-7f") == 1
    assert len(re.findall(r"\bSURE\b", SOURCE)) >= 3 and len(re.findall(r"\bNEAR\b", SOURCE)) >= 3
