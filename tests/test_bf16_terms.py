"""Float32 operands as sums of bf16 terms: the bounds that the kernels' comments state (csrc/bf16_terms.h), with
the same steps in numpy.  A term is what is left rounded to nearest, ties to even."""
import numpy as np
import pytest


def to_bf16(x):
    b = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + (b >> 16 & 1)) & 0xFFFF0000
    return b.astype(np.uint32).view(np.float32)


def split(x, n):
    terms, left = [], x.astype(np.float32)
    for _ in range(n):
        terms.append(to_bf16(left))
        left = left - terms[-1]
    return [t.astype(np.float64) for t in terms]


def values(seed, n=400_000):
    """All exponents' mantissas, the ends of a mantissa's range among them."""
    g = np.random.default_rng(seed)
    x = (g.uniform(1, 2, n) * 2.0 ** g.integers(-20, 20, n) * g.choice([-1, 1], n)).astype(np.float32)
    x[:6] = [1.0, 2.0 - 2.0 ** -23, 1.0 + 2.0 ** -8, 1.0 + 2.0 ** -8 + 2.0 ** -23, 1.0 + 2.0 ** -7 - 2.0 ** -23, 1.5]
    return x


@pytest.mark.parametrize("n,bound", [(1, 2.0 ** -8), (2, 2.0 ** -16), (3, 0.0)])
def test_terms_of_a_float(n, bound):
    x = values(1)
    off = np.abs(sum(split(x, n)) - x.astype(np.float64))
    assert (off <= bound * np.abs(x)).all()


@pytest.mark.parametrize("n,most,bound", [(3, 3, 2.0 ** -23), (2, 3, 2.0 ** -15), (2, 2, 3 * 2.0 ** -16)])
def test_pairs_of_terms(n, most, bound):
    """The pairs a + b < most of a product; what they leave out has either sign: its mean over 400,000 products is
    within 6 of a standard deviation, which is below the bound."""
    x, y = values(2), values(3)
    a, b = split(x, n), split(y, n)
    whole = x.astype(np.float64) * y.astype(np.float64)
    got = sum(a[i] * b[j] for i in range(n) for j in range(n) if i + j < most)
    off = (got - whole) / np.abs(whole)
    assert np.abs(off).max() <= bound * (1 + 2.0 ** -8)
    assert abs((off * np.sign(whole)).mean()) <= 6 * bound / len(x) ** 0.5
