"""Fits the polynomial of the ragged kernels' score cap (csrc/gqa_ragged_tile.cuh):
tanh(y) ~ y (c0 + c1 y^2 + c2 y^4 + c3 y^6) on |y| <= RANGE.

Method: Lawson's iteratively reweighted least squares on a Chebyshev grid, which makes the
absolute error near-equioscillating. The evaluation mirrors the kernel's float32 order
(square, three Horner FMAs, one product) and is compared with numpy's tanh in 64 bits.

    python tests/tanh_fit.py

tests/test_tanh_fit_host.py checks that the kernel's coefficients are this fit.
"""
import numpy as np

RANGE = 0.6


def fit(terms=4, most=RANGE, iters=400):
    y = (np.cos(np.linspace(0, np.pi, 4001)) * 0.5 + 0.5) * most
    y = y[y > 1e-3]
    a = y[:, None] ** (2 * np.arange(terms) + 1)
    w = np.ones_like(y) / len(y)
    for _ in range(iters):
        s = np.sqrt(w)
        c, *_ = np.linalg.lstsq(a * s[:, None], np.tanh(y) * s, rcond=None)
        w = w * np.abs(a @ c - np.tanh(y))
        w /= w.sum()
    return c


def kernel_tanh(y, c):
    y = y.astype(np.float32)
    z = y * y
    p = np.float32(c[-1])
    for ck in c[-2::-1]:
        p = p * z + np.float32(ck)
    return p * y


def max_error(c, most=RANGE):
    y = np.linspace(-most, most, 2_000_001).astype(np.float32)
    return float(np.abs(kernel_tanh(y, c) - np.tanh(y.astype(np.float64))).max())


if __name__ == "__main__":
    for terms in (3, 4, 5):
        for most in (0.4, 0.5, 0.6, 0.75, 1.0):
            c = fit(terms, most).astype(np.float32)
            print(terms, most, [float(x) for x in c], f"{max_error(c, most):.3e}")
