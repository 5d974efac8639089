"""Seqs, Prefixes and Rope without a GPU: numbers that 32 bits do not hold, or that are not whole, never reach the
library, where they would be others."""
import numpy as np
import pytest

import exn_hip as X

BAD = [[2 ** 32 + 1], np.array([2 ** 31]), np.array([-2 ** 31 - 1]), np.array([2 ** 63], np.uint64), [0.5], [np.nan], [np.inf],
       ["1"], [1j]]


@pytest.fixture
def calls(monkeypatch):
    made = []

    def call(name, *a):
        made.append(name)
        raise X.ExnError(X.ENODEV, "noted")

    monkeypatch.setattr(X, "call", call)
    return made


class Plan:
    seqs, h = 1, None


MAKE = {"seqs": lambda a: X.Seqs(X.Context.__new__(X.Context), a), "of": lambda a: X.Prefixes(X.Context.__new__(X.Context), Plan, a, [3]),
        "blocks": lambda a: X.Prefixes(X.Context.__new__(X.Context), Plan, [0], a),
        "axis": lambda a: X.Rope(X.Context.__new__(X.Context), [0.5], axis=a)}


@pytest.fixture(autouse=True)
def no_handle(monkeypatch):
    monkeypatch.setattr(X.Context, "h", None, raising=False)


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("make", MAKE)
def test_refused(calls, make, bad):
    with pytest.raises(X.ExnError) as e:
        MAKE[make](bad)
    assert e.value.code == X.EINVAL and not calls


@pytest.mark.parametrize("good", [[0], (0,), np.array([0], np.int64), np.array([0.0]), np.array([[0]], np.uint8), [False]], ids=str)
@pytest.mark.parametrize("make", MAKE)
def test_taken(calls, make, good):
    with pytest.raises(X.ExnError) as e:
        MAKE[make](good)
    assert e.value.code == X.ENODEV and len(calls) == 1
