"""A conversation's last pick after sampling inside the engine (imi_cuda_sample_states, imi_cuda_sampled)."""
import numpy as np
import pytest

import nunchi_b200 as nb
from test_gpu_serve_engine import engine, read  # noqa: F401

pytestmark = pytest.mark.gpu


def test_the_last_pick_s_value_is_its_word_s_score(engine):  # noqa: F811
    states = read(engine, 4)
    top = [s.argmax() for s in states]
    assert [s.logits.max() for s in states] == [v for _, v in top]
    nb.sample_states(states, [0.1, 0.5, 0.9, 0.99], temperature=3.0)
    for s in states:
        i, v = s.argmax()
        assert v == s.logits[i]
    nb.sampled(states, 3, np.full((3, 4), 0.6, np.float32), temperature=[2.0, 0.0, 1.0, 3.0])
    for s in states:
        i, v = s.argmax()
        assert v == s.logits[i]
    assert states[1].argmax()[0] == int(states[1].logits.argmax())
