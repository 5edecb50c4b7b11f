"""The decode loop of examples/shared_prompt_decode.py, end to end."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def stack():
    import shared_prompt_decode as e
    from diskmule_b200 import CudaContext
    ctx = CudaContext(0)
    st = e.Stack(ctx, max_sequences=8)
    yield e, st
    st.close()
    ctx.close()


def test_loop_runs_and_gives_every_page_back(stack):
    e, st = stack
    first = e.run(prompt=100, samples=5, steps=6, stack=st)
    again = e.run(prompt=100, samples=5, steps=6, stack=st)
    assert first["status"] == 0 and first["tokens"].shape == (6, 5)
    # the same pages, the same sums: the same tokens
    assert np.array_equal(first["tokens"], again["tokens"]) and np.array_equal(first["after"], again["after"])


def test_decode_continues_the_prompt(stack):
    """The token after a prompt of n tokens is the one that decoding its last token over the
    first n - 1 gives, to the rounding of one attention output: compared on the hidden state's
    logits, not on an argmax that a tie could turn."""
    e, st = stack
    r = np.random.RandomState(5)
    tokens = torch.tensor(r.randint(0, st.embed.shape[0], 90), device="cuda")
    logits = {}
    whole = st.tokens_of

    def record(x):
        logits["last"] = (st._norm(x).bfloat16() @ st.embed.T).float()
        return whole(x)
    st.tokens_of = record
    try:
        st.prompt(0, tokens)
        want = logits["last"]
        st.prompt(1, tokens[:-1])
        row = e.ints([1])
        st.step(row, tokens[-1:], 0, 90)
        got = logits["last"]
        every = e.ints([0, 1])
        st.cache.free(every.data_ptr(), 2, stream=st.stream)
    finally:
        st.tokens_of = whole
    # bf16 activations (2^-9 each) through a few layers
    assert (got - want).norm() <= 0.02 * want.norm()
    assert st.cache.status() == 0
