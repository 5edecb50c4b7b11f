"""examples/long_chat.py: it runs in pieces of any size, and eviction keeps to its budget."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_pieces_of_a_prompt():
    """However a prompt is cut, every query row hands out a weight of one in each layer and head
    (each weight is off by a few 2^-21 of itself, and a sum of 1000 terms by 1000 times 2^-24)."""
    from long_chat import run
    a = run(prompt=200, piece=200, budget=4000, steps=1)
    b = run(prompt=200, piece=33, budget=4000, steps=1)
    assert a["status"] == b["status"] == 0
    assert np.array_equal(a["seen"], b["seen"]) and np.array_equal(a["held"], a["seen"])
    for r in (a, b):
        given = r["seen"] * r["layers"] * r["heads"]
        assert np.all(np.abs(r["received"] - given) <= 2.0 ** -13 * given)


def test_eviction_keeps_to_its_budget():
    from long_chat import run
    r = run(chats=3, prompt=300, piece=64, budget=160, steps=24)
    assert r["status"] == 0
    assert np.array_equal(r["seen"], [300 + 24, 283 + 24, 266 + 24])
    assert np.all(r["held"] <= 160 + 16) and np.all(r["held"] >= 160)
    assert np.all(np.isfinite(r["received"])) and np.all(r["received"] > 0)
