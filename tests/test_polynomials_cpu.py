"""CPU: the polynomials the kernels evaluate in place of 2^x, from the
coefficients in their sources, against 2^x in higher precision."""
import re
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parent.parent / "infengine_b200" / "csrc"
NUMBER = r"([-+]?\d[\d.]*(?:e[-+]?\d+)?)"


def body(source, function):
    """The text of a function, from its name to the brace that ends its first line's column."""
    text = (CSRC / source).read_text()
    return re.search(r"\b" + function + r"\(.*?\n}\n", text, re.S).group(0)


def test_chunk_attention_polynomial():
    """No less exact than the hardware's ex2.approx (2^-22), so that a column's
    accuracy does not depend on which of the two its place gives it. fp32
    fused multiply-adds, as evaluated; one part in 16 for their roundings."""
    c = [np.float32(x) for x in re.findall(r"c\(" + NUMBER + r"f\)", body("paged_attention_tc.cu", "ex2_poly2"))]
    f = np.linspace(-0.5, 0.5, 400001).astype(np.float32)
    p = np.full_like(f, c[0])
    for x in c[1:]:  # (the product is exact in 64 bits)
        p = (p.astype(np.float64) * f.astype(np.float64) + np.float64(x)).astype(np.float32)
    off = np.abs(p.astype(np.float64) / np.exp2(f.astype(np.float64)) - 1).max()
    assert off <= 2.0 ** -22 * 17 / 16, np.log2(off)


def test_sampling_polynomial():
    """The coefficients as stored, in 50 digits: off by 2.8e-16 on [-1/2, 1/2];
    evaluated in 64 bits: 2^-53 of the last sum and as much of the one before
    it, of at most 0.35 beside 0.7 at its end, come on top."""
    from decimal import Decimal, localcontext
    text = body("sample.cu", "exp2_neg")
    c = re.findall(r"double p = " + NUMBER, text) + re.findall(r"p = fma\(p, f, " + NUMBER + r"\)", text)
    assert len(c) == 11
    with localcontext() as ctx:
        ctx.prec = 50
        ln2, stored, evaluated = Decimal(2).ln(), Decimal(0), Decimal(0)
        for i in range(-1500, 1501):
            f = i / 3000
            exact = (Decimal(f) * ln2).exp()
            p, y = Decimal(0), Decimal(0)
            for x in c:
                p = p * Decimal(f) + Decimal(float(x))
                y = Decimal(float(y * Decimal(f) + Decimal(float(x))))  # one rounding, as fma's
            stored, evaluated = max(stored, abs(p / exact - 1)), max(evaluated, abs(y / exact - 1))
    assert stored <= Decimal(2.8e-16) and evaluated <= Decimal(2.8e-16 + 2 ** -53 * 2), (stored, evaluated)
