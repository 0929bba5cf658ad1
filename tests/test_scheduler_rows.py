"""Requests of different sampling parameters in one batch: the scheduler draws equal ones together, each from its own row."""
from test_karusun_host import FakeModel
from wf_bitnet.scheduler import Request, SamplingParams, Scheduler, execute


def test_the_rows_left_for_sampling_stand_in_the_order_they_were_asked_for():
    m = FakeModel(slots=3, pages=20)
    a, b, c = m.admit(), m.admit(), m.admit()
    rows = execute(m, [(a, [1, 2]), (b, [5]), (c, [7, 3])], [(2, 1), (0, 1), (1, 0)])
    assert rows.argmax(-1).tolist() == m._last.argmax(-1).tolist() == [4, 3, 5]


def test_every_request_draws_from_its_own_row():
    m = FakeModel(slots=4, pages=40)
    s = Scheduler(m)
    for i, temp in enumerate((0.9, 0.0, 0.5, 0.0)):              # sorted by their parameters the batch's rows stand otherwise
        s.add(Request(f"r{i}", [i + 1] * (2 + i), max_new_tokens=4, sampling=SamplingParams(temp)))
    done = s.run()
    assert len(done) == 4
    for r in done:                                               # the fake model's next token is a function of position and token, whatever the temperature
        seq = list(r.prompt)
        for t in r.output:
            assert t == (len(seq) - 1 + seq[-1]) % m.vocab, r.rid
            seq.append(t)
