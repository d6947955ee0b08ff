"""The polynomial of the selective scan's softplus, with the coefficients that its source holds, against what it stands
for: 2 atanh(r) / r in r^2 on [0, 1 / 9], within what the comment beside it says."""

import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parents[1] / "boltz_lumi_amd" / "csrc" / "selective_scan.hip"


def test_polynomial():
    text = SOURCE.read_text()
    body = text[text.index("float step_of(float x)"):]
    body = body[:body.index("\n}")]
    first = re.search(r"float s = ([0-9.]+)f;", body)
    rest = re.findall(r"s = s \* q \+ ([0-9.]+)f;", body)
    assert first and len(rest) == 4
    q = np.linspace(1e-9, 1 / 9, 400_001)
    exact = 2 * np.arctanh(np.sqrt(q)) / np.sqrt(q)
    value = np.full_like(q, np.float32(first.group(1)))
    for c in rest:
        value = value * q + float(np.float32(c))
    stated = re.search(r"within ([0-9.e-]+) of it on \[0, 1 / 9\] \(([0-9.e-]+) relative", text)
    assert np.abs(value - exact).max() <= float(stated.group(1))
    assert np.abs(value / exact - 1).max() <= float(stated.group(2))
