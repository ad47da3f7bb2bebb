"""Derives the polynomial coefficients hard-coded in gv_transcendentals.h and in attention.cu.

erf and exp are approximated by Chebyshev interpolants (converted to monomials in
a centred, scaled variable) so that the CPU oracle and the CUDA kernels evaluate
the very same fp32 fmaf chain and therefore agree bit for bit.  2^f of attention is the polynomial with the smallest largest
relative error, which no oracle repeats.  Run:

    python fit_transcendentals.py        # prints C initialisers + max errors
"""
import numpy as np
from numpy.polynomial import chebyshev as C
from scipy.special import erf


def cheb_mono(f, lo, hi, deg):
    c, h = (lo + hi) / 2.0, (hi - lo) / 2.0
    n = deg + 1
    k = np.arange(n)
    x = np.cos(np.pi * (k + 0.5) / n)
    return c, h, C.cheb2poly(C.chebfit(x, f(c + h * x), deg))


def horner32(mono, x):
    acc = np.full_like(x, np.float32(mono[-1]))
    for co in mono[-2::-1]:
        acc = (acc.astype(np.float64) * x.astype(np.float64)
               + np.float64(np.float32(co))).astype(np.float32)
    return acc


def fmt(mono, width):
    m = list(mono) + [0.0] * (width - len(mono))
    return "{" + ", ".join(f"{np.float32(v):.9e}f" for v in m) + "}"


def exp2_minimax(degree=4, rounds=2000):
    """Coefficients (of f^0 first) for 2^f on [-1/2, 1/2] with the smallest largest relative error, by iterated reweighted least squares
    (Lawson): each point's weight grows with its error.  The last place of a coefficient goes by the rounding of the least squares."""
    f = 0.5 * np.cos(np.pi * (np.arange(4001) + 0.5) / 4001)
    powers = np.vander(f, degree + 1, increasing=True) / np.exp2(f)[:, None]
    weight, best, least = np.ones_like(f), None, np.inf
    for _ in range(rounds):
        root = np.sqrt(weight)
        c = np.linalg.lstsq(powers * root[:, None], root, rcond=None)[0]
        off = np.abs(powers @ c - 1)
        if off.max() < least:
            best, least = c, off.max()
        weight = weight * off
        weight /= weight.sum()
    return best, least


def main():
    # erf on [0,4): eight intervals of width 0.5, degree 6 in u = a - centre
    worst = 0.0
    print("#define GV_ERF_TABLE_INIT {\\")
    for i in range(8):
        lo, hi = 0.5 * i, 0.5 * (i + 1)
        c, h, m = cheb_mono(erf, lo, hi, 6)
        m = m / (h ** np.arange(len(m)))  # monomial in (a - c)
        a = np.linspace(lo, hi, 100001)[:-1].astype(np.float32)
        u = (a - np.float32(c)).astype(np.float32)
        worst = max(worst, np.abs(horner32(m, u).astype(np.float64) - erf(a.astype(np.float64))).max())
        print("  " + fmt(m, 7)[:-1] + ", 0.0f},\\")
    print("}")
    print(f"// erf table max abs err {worst:.3e}")
    # exp on [-ln2/2, ln2/2]
    half = np.log(2.0) / 2
    c, h, m = cheb_mono(np.exp, -half, half, 6)
    r = np.linspace(-half, half, 400001).astype(np.float32)
    x = (r * np.float32(1 / h)).astype(np.float32)
    # fold 1/h into the coefficients so the kernel evaluates p(r) directly
    m2 = m / (h ** np.arange(len(m)))
    e = np.abs(horner32(m2, r).astype(np.float64) / np.exp(r.astype(np.float64)) - 1).max()
    print(f"// exp core max rel err {e:.3e}")
    print("GV_EXP_POLY =", fmt(m2, 7))
    # 2^f on [-1/2, 1/2], exp2_by_polynomial
    c, worst = exp2_minimax()
    print(f"// exp2 max rel err {worst:.3e}")
    print("exp2_by_polynomial =", fmt(c, 5))


if __name__ == "__main__":
    main()
