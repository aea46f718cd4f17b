"""The generator's stream from any word on: the same words, and no work beyond the generator's own."""

import numpy as np
import pytest

from quabla_b200 import random as qr


@pytest.mark.parametrize("key", [0, 5, 0xDEADBEEFCAFEBABE, 2**64 - 1])
@pytest.mark.parametrize("first", [0, 1, 1000, 2**32 - 5, 2**63 - 20])
def test_words_from_a_later_one_on(key, first):
    mask = 2**64 - 1
    want = [qr._mix_scalar((key + (first + i + 1) * qr._GAMMA) & mask) for i in range(40)]
    assert [int(w) for w in qr._stream(key, 40, first)] == want
    assert [int(w) for w in qr._stream(key, 30, first + 10)] == want[10:]


def test_a_word_takes_the_generators_passes_and_no_more(monkeypatch):
    # Two for the state, eight for the output function (three shifts, three exclusive ors, two products).
    passes = []

    class Counted(np.ndarray):
        def __array_ufunc__(self, ufunc, method, *inputs, **kwargs):
            passes.append(ufunc.__name__)
            plain = [i.view(np.ndarray) if isinstance(i, Counted) else i for i in inputs]
            return getattr(ufunc, method)(*plain, **kwargs).view(Counted)

    arange = np.arange
    monkeypatch.setattr(np, "arange", lambda *a, **k: arange(*a, **k).view(Counted))
    for first in (0, 7):
        passes.clear()
        qr._stream(11, 100, first)
        assert len(passes) == 10, passes
