"""Log probabilities of a served model: the engine's rows of the last step, requests of the scheduler, the BitNet engine's rows."""
import numpy as np
import pytest

from test_gpu_karusun import CONFIGS, build, make_weights, tokens_for

pytestmark = pytest.mark.gpu


def logp(rows):
    x = rows.astype(np.float64)
    x = x - x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


# float sums of a few hundred terms and differences of logits below 100: some hundred half steps of 2^-24 of at most 100
TOL = 100 * 200 * 2.0**-24


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_of_the_last_step(dtype):
    cfg = CONFIGS["odd"]
    m = build(cfg, make_weights(cfg, 61), dtype)
    s = m.admit()
    lg = m.step([s], [6], tokens_for(cfg, 6, 62), list(range(6)))
    ref = logp(lg)
    tok = m.sample(6, 0.0)
    lp, ent, tlp, tid = m.logprobs(6, tok, 5)
    order = np.argsort(-lg, axis=-1, kind="stable")[:, :5]
    assert (tid == order).all() and (tid[:, 0] == tok).all()
    assert np.abs(lp - ref[np.arange(6), tok]).max() < TOL and np.abs(tlp - np.take_along_axis(ref, order, -1)).max() < TOL
    assert np.abs(ent + (np.exp(ref) * ref).sum(-1)).max() < TOL
    lp2, _, tlp2, tid2 = m.logprobs(3, [0, cfg["vocab"] - 1, cfg["vocab"]], 0, 0.5)      # fewer rows, no alternatives, another temperature, no such token
    half = logp(2 * lg)
    assert np.abs(lp2[:2] - half[[0, 1], [0, -1]]).max() < TOL and np.isnan(lp2[2]) and tlp2.shape == tid2.shape == (3, 0)
    for bad in (lambda: m.logprobs(6, tok[:5], 0), lambda: m.logprobs(6, tok, -1), lambda: m.logprobs(6, tok, 65), lambda: m.logprobs(6, tok, cfg["vocab"] + 1),
                lambda: m.logprobs(6, tok, 1, 0.0), lambda: m.logprobs(0, [], 1)):
        with pytest.raises(ValueError):
            bad()
    m.close()


def test_scheduled_requests_get_the_distribution_they_were_drawn_from():
    from wf_bitnet.scheduler import Request, SamplingParams, Scheduler
    cfg = CONFIGS["mixed"]
    m = build(cfg, make_weights(cfg, 71), "float32", max_tokens=96, slots=2, page_size=4, max_step_tokens=16)
    sched = Scheduler(m, max_prefill_chunk=6)
    kinds = [(None, 0.0), (4, 0.0), (1, 0.8), (0, 0.0)]
    for i, (n, temp) in enumerate(kinds):
        sched.add(Request(f"r{i}", tokens_for(cfg, 5 + 3 * i, 80 + i), max_new_tokens=6, sampling=SamplingParams(temp, seed=i), logprobs=n))
    seen = []                                              # (rows, drawn) of every step
    draw = sched._draw
    sched._draw = lambda lg, owners: seen.append((lg.copy(), [r.rid for r in owners])) or draw(lg, owners)
    done = {r.rid: r for r in sched.run()}
    at = {rid: 0 for rid in done}
    for lg, rids in seen:
        ref = logp(lg)
        for k, rid in enumerate(rids):
            r, i = done[rid], at[rid]
            at[rid] += 1
            if r.logprobs is None:
                continue
            assert abs(r.token_logprobs[i] - ref[k, r.output[i]]) < TOL and abs(r.entropies[i] + (np.exp(ref[k]) * ref[k]).sum()) < TOL
            want = np.argsort(-lg[k], kind="stable")[:r.logprobs]
            assert [t for t, _ in r.top_logprobs[i]] == want.tolist() and np.abs(np.array([p for _, p in r.top_logprobs[i]]) - ref[k, want]).max(initial=0) < TOL
    assert all(at[f"r{i}"] == 6 for i in range(4)) and done["r0"].token_logprobs == []
    m.close()


def test_bitnet_rows():
    from sglang.srt.models.bitnet import BitNetForCausalLM
    from wf_bitnet.scheduler import Request, Scheduler
    m = BitNetForCausalLM({"hidden_size": 256, "num_hidden_layers": 1, "num_attention_heads": 2, "num_key_value_heads": 1, "intermediate_size": 384, "vocab_size": 512,
                           "rms_norm_eps": 1e-5, "rope_theta": 500000.0}, max_batch=1, max_seq=64, page_size=16)
    m.engine.init_synthetic(3)
    s = Scheduler(m)
    s.add(Request("r", [3, 14, 15], max_new_tokens=4, logprobs=2))
    (r,) = s.run()
    assert len(r.output) == len(r.token_logprobs) == 4 and all(alt[0][0] == t and alt[0][1] == lp for t, lp, alt in zip(r.output, r.token_logprobs, r.top_logprobs))
    assert all(0 < e <= np.log(512) + 1e-5 for e in r.entropies)
    m.close()
