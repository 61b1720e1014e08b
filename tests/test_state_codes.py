"""The 8-bit states at the lower end of their range (oracle and kernel agree to the bit: tests/test_state_codes_gpu.py)."""

import numpy as np
import pytest

from oracle import learn as O

FIRST = {False: 1.25 * 2.0 ** -16, True: 1.125 * 2.0 ** -16}       # what code 1 stands for in a block whose largest is 1
PLACE = 1.125 * 2.0 ** -16                                          # below it m is 0


def roundings(y, root, steps=4000):
    """The values that a block of y, beside one of 1, is rounded to at each of the steps."""
    x = np.concatenate([[1.0], y]).astype(np.float32)
    return np.stack([O.decode(*O.encode(x, step, root), root)[1:] for step in range(steps)]), x[1:].astype(np.float64)


@pytest.mark.parametrize("root", [False, True])
def test_the_first_code(root):
    assert O.grid(root)[1] == FIRST[root]


@pytest.mark.parametrize("root", [False, True])
def test_the_mean_is_kept_down_to_the_first_code(root):
    """4,000 roundings to neighbours a share s apart scatter by s / 2 each, their mean by s / 2 / sqrt(4000); six of those."""
    y = FIRST[root] * np.exp(np.linspace(0, 6, 200))
    got, x = roundings(y, root)
    s = 2.0 ** -(4 if root else 3)
    assert (np.abs(got.mean(0) - x) <= 6 * x * s / 2 / np.sqrt(4000) + 1e-7 * x).all()


def test_first_moments_below_the_first_code():
    """Never more than the value in the mean, nothing at all one spacing below code 1 and further down."""
    got, x = roundings(-PLACE * np.linspace(1.0, 1.0 / 0.9, 60), False)
    # a share p of -FIRST scatters by FIRST / 2 each: six of the mean's
    assert (np.abs(got.mean(0)) <= np.abs(x) + 6 * FIRST[False] / 2 / np.sqrt(4000)).all() and (got <= 0).all()
    assert (np.unique(np.abs(got)) == np.array([0.0, FIRST[False]])).all()
    got, _ = roundings(PLACE * np.array([0.999, 0.5, 1e-3, 1e-20]), False)
    assert (got == 0).all()


def test_roots_below_the_first_code():
    """Raised to it every time: a step is divided by no less than the value's own root."""
    got, _ = roundings(PLACE * np.array([0.999, 0.5, 1e-3, 1e-20]), True)
    assert (got == FIRST[True]).all()


@pytest.mark.parametrize("root", [False, True])
def test_blocks_of_nothing(root):
    x = np.full(256, 2.0 ** -101, np.float32)
    codes, scale = O.encode(x, 3, root)
    assert scale[0] == 0 and (O.decode(codes, scale, root) == 0).all()
    assert (O.decode(*O.encode(x * 2, 3, root), root) == 2.0 ** -100).all()
