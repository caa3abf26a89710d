"""Generates nsrl_luts.h: the three 8-bit integer tables of the NSRL numeric core
and the quarter circle of the rotary positions.

The tables are defined mathematically (crates/nsrl-core/src/rsqrt_lut_8bit.rs
holds the same values):
  rsqrt[m-128] = round(32768 / sqrt(m / 128)), clamped to 32767, m in [128, 255]  (Q15)
  exp2[f]      = round(32768 * 2^(-f / 256)),  clamped to 32767, f in [0, 255]    (Q15)
  recip[m-128] = round(2^31 / m),                                 m in [128, 255]  (Q31)
and, for the rotary positions (no counterpart in the reference),
  quarter[i]   = round(2^30 * sin(2 pi i / 1024)),                i in [0, 256]    (Q30)
All are computed here with exact integer arithmetic (no floating point
decides a rounding), so the header is reproducible bit for bit.
"""
import os
from math import isqrt

HERE = os.path.dirname(os.path.abspath(__file__))
OUT = os.path.join(HERE, "nsrl_luts.h")


def rsqrt_table():
    out = []
    for m in range(128, 256):
        # largest r with (r - 1/2) <= sqrt(2^37 / m)  <=>  m * (2r - 1)^2 <= 2^39
        r = (isqrt((1 << 39) // m) + 1) // 2 + 2
        while m * (2 * r - 1) ** 2 > (1 << 39):
            r -= 1
        out.append(min(r, 32767))
    return out


def exp2_table():
    out = []
    for f in range(256):
        # largest r with (r - 1/2) <= 2^(15 - f/256)  <=>  (2r - 1)^256 <= 2^(4096 - f)
        # start just above the float estimate; the exact test decides, and the
        # assert checks that r + 1 fails it (r is the largest)
        r = min(32768, int(32768 * 2.0 ** (-f / 256)) + 3)
        while (2 * r - 1) ** 256 > 2 ** (4096 - f):
            r -= 1
        assert (2 * r + 1) ** 256 > 2 ** (4096 - f)
        out.append(min(r, 32767))
    return out


def recip_table():
    return [((1 << 31) + m // 2) // m for m in range(128, 256)]


def quarter_table():
    # sin by its Taylor series on integers scaled by 2^120: the angle is below
    # pi / 2, so 40 terms leave an error far below the distance of every entry
    # from a rounding border (above 2^-9)
    one = 1 << 120
    pi = 0  # 16 atan(1/5) - 4 atan(1/239)
    for coef, x in ((16, 5), (-4, 239)):
        term, k = one // x, 0
        while term:
            pi += (coef * term // (2 * k + 1)) * (-1 if k & 1 else 1)
            term //= x * x
            k += 1
    out = []
    for i in range(257):
        a = 2 * pi * i // 1024
        total, term = 0, a
        for k in range(1, 81, 2):
            total += term
            term = -(term * a >> 120) * a // ((k + 1) * (k + 2)) >> 120
        out.append(((total >> 89) + 1) >> 1)
    return out


def render() -> str:
    def rows(vals, per=12):
        return " \\\n".join("  " + ", ".join(str(v) for v in vals[i:i + per]) + ("," if i + per < len(vals) else "")
                             for i in range(0, len(vals), per))

    return (
        "// Generated by gen_luts.py -- do not edit.\n"
        "// Integer tables of the NSRL numeric core (see gen_luts.py for definitions).\n"
        "#pragma once\n\n"
        "// Q15 1/sqrt(m/128), m in [128, 255]\n"
        "#define NSRL_RSQRT_LUT_VALUES \\\n" + rows(rsqrt_table()) + "\n\n"
        "// Q15 2^(-f/256), f in [0, 255]\n"
        "#define NSRL_EXP2_LUT_VALUES \\\n" + rows(exp2_table()) + "\n\n"
        "// Q31 1/m, m in [128, 255]\n"
        "#define NSRL_RECIP_LUT_VALUES \\\n" + rows(recip_table(), 8) + "\n\n"
        "// Q30 sin(2 pi i / 1024), i in [0, 256]\n"
        "#define NSRL_QUARTER_LUT_VALUES \\\n" + rows(quarter_table(), 8) + "\n"
    )


def main():
    text = render()
    if not os.path.exists(OUT) or open(OUT).read() != text:
        with open(OUT, "w") as f:
            f.write(text)
    return OUT


if __name__ == "__main__":
    print(main())
