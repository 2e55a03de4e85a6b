"""The int8 quantiser's rounding, checked on the CPU over every operand it can meet: the
product x * fl(127 / m), rounded to 21 bits and then to a whole number, is the exactly
rounded 127 x / m (halves to even) for all 8-bit (BF16, E4M3) and 11-bit (FP16)
significands and every exponent difference at which the quotient can round to more than 0."""

import numpy as np
import pytest


@pytest.mark.parametrize("bits", [8, 11])
def test_quotient_is_exact(bits):
    one = np.float32(12582912)
    a = np.arange(1 << (bits - 1), 1 << bits, dtype=np.int64)
    for b in range(1 << (bits - 1), 1 << bits):
        c = np.float32(127) / np.float32(b)
        for s in range(9):
            x = (a * 2.0 ** -s).astype(np.float32)
            t = ((x * c).view(np.uint32) + np.uint32(4)) & np.uint32(0xFFFFFFF8)
            got = ((t.view(np.float32) + one) - one).astype(np.int64)
            num, den = 254 * a, b << s                       # twice the quotient
            q, rem = np.divmod(num, 2 * den)
            want = q + ((rem > den) | ((rem == den) & (q % 2 == 1)))
            assert np.array_equal(got[x <= b], want[x <= b]), (b, s)
