"""Log probabilities and draws are of the rows that the LAST step left: a step with fewer rows than one before it leaves no more than its own."""
import numpy as np
import pytest

from test_gpu_karusun import CONFIGS, build, make_weights, tokens_for
from test_gpu_logprobs_engine import TOL, logp

pytestmark = pytest.mark.gpu


def test_a_large_step_and_a_smaller_one():
    cfg = CONFIGS["odd"]
    m = build(cfg, make_weights(cfg, 61), "float32")

    def has(n, lg):
        tok = m.sample(n, 0.0)
        assert (tok == lg[:n].argmax(-1)).all()
        lp = m.logprobs(n, tok, 2)[0]
        assert np.abs(lp - logp(lg[:n])[np.arange(n), tok]).max() < TOL

    def refused(n):
        for call in (lambda: m.logprobs(n, [0] * n, 1), lambda: m.sample(n, 0.0)):
            with pytest.raises(ValueError, match=f"no logits for {n} rows"):
                call()

    refused(1)                                             # no step yet
    s = m.admit()
    lg = m.step([s], [6], tokens_for(cfg, 6, 62), list(range(6)))
    has(6, lg), has(4, lg), refused(7)
    lg = m.step([s], [4], tokens_for(cfg, 4, 63), [1, 3])
    has(2, lg), has(1, lg), refused(3), refused(6)
    for k in range(3):                                     # single tokens: eager, captured, replayed
        lg = m.step([s], [1], tokens_for(cfg, 1, 64 + k), [0])
        has(1, lg), refused(2)
    m.step([s], [2], tokens_for(cfg, 2, 70), [])           # nothing wanted
    refused(1)
    lg = m.step([s], [3], tokens_for(cfg, 3, 71), [0, 1, 2])
    with pytest.raises(ValueError):
        m.step([s + 100], [1], [0], [0])                   # refused before anything ran: the rows are still those of the step before
    has(3, lg), refused(4)
    m.close()
