"""CudaServe.generate's steps on the CPU: what each is given, with a step that only notes it."""
from __future__ import annotations

import numpy as np
import pytest

from llaccel_b200.cuda_backend import CudaServe


class Noted(CudaServe):
    def __init__(self, max_rows=8):
        self.max_seqs, self.max_rows, self.steps, self.freed = 4, max_rows, [], []
        self.model = type("Model", (), {"_validate": staticmethod(lambda p, n: list(p))})

    def step(self, slots, tokens, **how):
        self.steps.append((list(slots), [list(t) for t in tokens], how))
        return {"next": np.arange(len(slots)) + 100}

    def free(self, slots):
        self.freed.append(list(slots))


def test_settings_stay_with_their_prompts():
    """Prompts that are through at different steps: the arrays follow the sequences that are left."""
    s = Noted()
    out = s.generate([[1], [2] * 5, [3] * 9], 2, rng=np.random.default_rng(0), chunk=3, temperature=[0.1, 0.2, 0.3], top_k=[4, 5, 6], min_p=0.5,
                     top_p=None)
    assert [len(o) for o in out] == [2, 2, 2]
    assert [slots for slots, _, _ in s.steps] == [[0, 1, 2], [0, 1, 2], [1, 2], [2]]
    for slots, _, how in s.steps:
        assert how["temperature"].tolist() == [[0.1, 0.2, 0.3][i] for i in slots]
        assert how["top_k"].tolist() == [[4, 5, 6][i] for i in slots] and how["min_p"].tolist() == [0.5] * len(slots)
        assert len(how["random"]) == len(slots) and "top_p" not in how


def test_prompts_go_in_by_chunks():
    s = Noted(max_rows=4)
    s.generate([[1, 2, 3, 4, 5], [6, 7]], 1)
    assert [(slots, feed) for slots, feed, _ in s.steps] == [([0, 1], [[1, 2, 3], [6]]), ([0, 1], [[4, 5], [7]])]
    assert all(how == {} for _, _, how in s.steps) and s.freed == [[0, 1], [0, 1]]


@pytest.mark.parametrize("how,words", [(dict(chunk=-1), "chunk"), (dict(temperature=0.5), "random numbers"),
                                       (dict(rng=np.random.default_rng(0), top_k=[1, 2, 3]), "broadcast")])
def test_refused_before_any_slot_is_freed(how, words):
    s = Noted()
    with pytest.raises(ValueError, match=words):
        s.generate([[1, 2], [3]], 2, **how)
    assert s.freed == [] and s.steps == []
