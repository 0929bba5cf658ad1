"""Requests that ask for log probabilities, on a model without a GPU; refusals of the engine's call through the C ABI."""
import numpy as np
import pytest

from test_karusun_host import FakeModel
from wf_bitnet.scheduler import Request, SamplingParams, Scheduler


class WithLogprobs(FakeModel):
    """Its logit rows are one-hot; log probabilities by definition, in 64 bits."""

    def logprobs(self, n, tokens, top=0, temperature=1.0):
        assert n == len(tokens) and temperature == 1.0
        self.asked.append(top)
        lp = self._last[:n].astype(np.float64) - np.log(np.exp(self._last[:n].astype(np.float64)).sum(-1, keepdims=True))
        ids = np.argsort(-lp, axis=-1, kind="stable")[:, :top].astype(np.int32)
        return lp[np.arange(n), tokens], -(np.exp(lp) * lp).sum(-1), np.take_along_axis(lp, ids, -1), ids

    def __init__(self, **kw):
        super().__init__(**kw)
        self.asked = []


def test_only_requests_that_ask_get_them_and_each_its_number():
    m = WithLogprobs(slots=3, pages=20)
    s = Scheduler(m, max_prefill_chunk=5)
    for rid, n, temp in (("none", None, 0.0), ("zero", 0, 0.0), ("three", 3, 0.0)):
        s.add(Request(rid, [2] * 4, max_new_tokens=3, sampling=SamplingParams(temp), logprobs=n))
    done = {r.rid: r for r in s.run()}
    assert done["none"].token_logprobs == [] and done["none"].top_logprobs == []
    hit = 1.0 - np.log(np.e + m.vocab - 1)
    for rid, n in (("zero", 0), ("three", 3)):
        r = done[rid]
        assert len(r.token_logprobs) == len(r.entropies) == len(r.top_logprobs) == 3
        assert np.allclose(r.token_logprobs, hit) and [len(t) for t in r.top_logprobs] == [n] * 3
    for t, alt in zip(done["three"].output, done["three"].top_logprobs):
        assert alt[0][0] == t and np.isclose(alt[0][1], hit) and [i for i, _ in alt[1:]] == [i for i in range(m.vocab) if i != t][:2]
    assert max(m.asked) == 3
    quiet = WithLogprobs(slots=1, pages=20)
    s = Scheduler(quiet)
    s.add(Request("q", [1], max_new_tokens=2))
    s.run()
    assert quiet.asked == []                               # nobody asked: the model is not called


def test_requests_that_cannot_be_served_are_refused():
    for n in (-1, 12, 65):
        with pytest.raises(ValueError):
            Scheduler(WithLogprobs()).add(Request("r", [1], logprobs=n))
    with pytest.raises(NotImplementedError):
        Scheduler(FakeModel()).add(Request("r", [1], logprobs=0))


def test_the_engines_call_refuses_what_it_has_no_rows_for():
    from wf_bitnet import _lib
    L = _lib.seq_lib()
    assert L.wf_seq_logprobs(None, 1, None, 0, 1.0, None, None, None, None) == _lib.WF_ERR_INVALID
    assert b"no logits" in L.wf_last_error()


def test_command_line_takes_the_option(capsys, monkeypatch):
    import json

    from wf_bitnet import cli
    m = WithLogprobs(slots=4, pages=50)
    m.close = lambda: None
    monkeypatch.setattr(cli, "load_model", lambda *a: m)
    assert cli.main(["generate", "--model", "x", "--prompt-ids", "1,2", "--max-new-tokens", "2", "--logprobs", "2"]) == 0
    (line,) = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert len(line["logprobs"]) == len(line["entropy"]) == len(line["output_ids"]) == 2 and [len(t) for t in line["top_logprobs"]] == [2, 2]
    assert line["top_logprobs"][0][0][0] == line["output_ids"][0]
    assert cli.main(["generate", "--model", "x", "--prompt-ids", "1,2", "--max-new-tokens", "2"]) == 0
    assert set(json.loads(capsys.readouterr().out)) == {"id", "prompt_tokens", "output_ids"}
