"""Which views of the adapter and balance calls count as overlapping: elements that two of them share, not address ranges that lie in one another
(csrc/tune_host.c on a stand-in for the CUDA shim, no GPU)."""
import random

import pytest

from picoforge_b200 import abi
from test_tuning_checks import AT, adapters, backward, balance, config, forward, lib, work  # noqa: F401

WIDE = 4096                                        # bytes between the rows of a buffer that holds several operands side by side


def test_columns_of_one_buffer_are_apart(lib, work):  # noqa: F811
    # k 32 (128 bytes), n 24 (96 bytes), 64 tokens: x, base, y and dy, dx as neighbouring columns
    at = AT["x"]
    same = dict(x=at, x_pitch=WIDE, base=at + 128, base_pitch=WIDE, y=at + 224, y_pitch=WIDE)
    assert forward(lib, work, **same) == abi.OK
    assert forward(lib, work, **dict(same, base=at + 224)) == abi.OK                       # base in place
    assert forward(lib, work, **dict(same, y=at + WIDE - 96)) == abi.OK                    # the last columns
    assert backward(lib, work, x=at, x_pitch=WIDE, dy=at + 128, dy_pitch=WIDE, dx=at + 224, dx_pitch=WIDE, base=at + 352, base_pitch=WIDE) == abi.OK
    assert balance(lib, work, back=True, logits=at, pitch=WIDE, grad=at + 64, grad_pitch=WIDE) == abi.OK
    assert balance(lib, work, back=True, logits=at + 64, pitch=WIDE, grad=at, grad_pitch=WIDE) == abi.OK


@pytest.mark.parametrize("change", [
    {"y": AT["x"] + 124}, {"y": AT["x"] + WIDE - 92}, {"base": AT["x"] + 128, "y": AT["x"] + 220}, {"base": AT["x"] + 128, "y": AT["x"] + 132},
    {"base": AT["x"] + 224, "y": AT["x"] + 224 + WIDE}, {"y": AT["x"] + 128, "y_pitch": 2 * WIDE}, {"slots": AT["x"] + 128, "y": AT["x"] + 128}])
def test_shared_elements_are_refused(lib, work, change):  # noqa: F811
    assert forward(lib, work, **(dict(x=AT["x"], x_pitch=WIDE, base=None, y_pitch=WIDE, base_pitch=WIDE) | change)) == abi.INVALID_ARGUMENT
    assert balance(lib, work, back=True, logits=AT["x"], pitch=WIDE, grad=AT["x"] + 60, grad_pitch=WIDE) == abi.INVALID_ARGUMENT


def test_against_every_byte(lib, work):  # noqa: F811
    """Two views of few rows laid anywhere: taken if no byte of y is one of x (same pitch, or a view of one row), never taken if one is."""
    rng = random.Random(1)
    taken = 0
    for _ in range(3000):
        tokens, k, n = rng.choice([1, 2, 3, 5]), rng.randint(1, 6), rng.randint(1, 6)
        xp = 4 * rng.randint(k, 14)
        yp = xp if xp >= 4 * n and rng.random() < 0.8 else 4 * rng.randint(n, 14)
        x = AT["x"] + (1 << 20)
        y = x + 4 * rng.randint(-60, 60)

        def cells(at, width, pitch):
            return {at + r * pitch + c * 4 for r in range(tokens) for c in range(width)}
        shared = bool(cells(x, k, xp) & cells(y, n, yp))
        st = forward(lib, work, adapters(k=k, n=n), x=x, x_pitch=xp, y=y, y_pitch=yp, base=None, tokens=tokens)
        if shared:
            assert st == abi.INVALID_ARGUMENT
        elif xp == yp or tokens == 1:
            assert st == abi.OK
            taken += 1
    assert taken > 500
