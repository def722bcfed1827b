"""Prompts scored end to end: lengths -> tables of the passes -> model -> log-probabilities (`LLM.score`, `/v1/score`)."""
import json
import math
from types import SimpleNamespace

import pytest
import torch

from xllm_b200 import LLM
from xllm_b200.api import scoring
from xllm_b200.api.embedding import hidden_states
from xllm_b200.engine.fault import DeviceWatchdog
from xllm_b200.engine.llm_engine import EngineConfig, LLMEngine
from xllm_b200.ops import _lib

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def engine(device, dtype=None, model="tiny", **kw):
    return LLMEngine(EngineConfig(**{**dict(model=model, device=device, dtype=dtype or ("float32" if device == "cpu" else "bfloat16"),
                                            num_blocks=64, enable_graph=False, max_seqs_per_batch=8, max_tokens_per_batch=256), **kw}))


def prompts(*lengths, vocab=32000, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lengths]


def plain(eng, ids, temperature=1.0):
    """Log-softmax in 64 bits of every place, from one pass over the prompt alone."""
    x = eng.model.logits(hidden_states(eng, ids)).double().cpu() / temperature
    return torch.log_softmax(x, dim=-1)


def compare(eng, lists, scores, n_top, tol, temperature=1.0):
    for ids, s in zip(lists, scores):
        assert len(s.logprobs) == len(s.entropies) == len(ids)
        if not ids:
            continue
        assert s.logprobs[0] is None and s.entropies[0] is None
        lp = plain(eng, ids, temperature)
        for i in range(1, len(ids)):
            row = lp[i - 1]
            assert abs(s.logprobs[i] - float(row[ids[i]])) <= tol
            assert abs(s.entropies[i] + float((row.exp() * row).sum())) <= tol * (1 + math.log(len(row)))
            if n_top:
                assert len(s.top_logprobs[i]) == n_top
                for t, v in s.top_logprobs[i]:
                    assert abs(v - float(row[t])) <= tol
                assert abs(s.top_logprobs[i][0][1] - float(row.max())) <= tol
                values = [v for _, v in s.top_logprobs[i]]
                assert values == sorted(values, reverse=True)
        assert (s.top_logprobs is None) == (n_top == 0)


# fp32 on the CPU: the passes differ in the order of sums over 256-wide states, some 1e-6 of scores of a few units.  bf16: a score is a
# sum over 256 products of states that differ by bf16 steps (2^-9 relative, some 20 independent ones on the way), and rounds to bf16 once
# more in the plain form: 2^-9 of scores up to 4, so up to 0.04 in all.
TOL = {"cpu": 2e-4, "cuda:0": 0.05}


def test_watchdog_reads_the_error_word(monkeypatch):
    """A wait that expired in head_logprobs is a finding like one in a product; a library without it is none."""
    class Library:
        xllm_fmha_error_status = xllm_talk_error_status = xllm_gemm_error_status = xllm_gemm_few_error_status = lambda self: 0
        xllm_head_logprobs_error_status = lambda self: 1

    found, eng = [], SimpleNamespace(device=torch.device("cuda", 0), ps=SimpleNamespace(comm=None))
    monkeypatch.setattr(_lib, "load", lambda *a: Library())
    dog = DeviceWatchdog.for_engine(eng, found.append)
    assert not dog.check() and found == ["head_logprobs: a bounded wait expired (status 1)"]
    monkeypatch.delattr(Library, "xllm_head_logprobs_error_status")
    assert DeviceWatchdog.for_engine(eng).check()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_top", [0, 4])
def test_packed_prompts(device, n_top):
    eng = engine(device)
    lists = prompts(5, 1, 33, 16, 0, 17, 2, 90)
    compare(eng, lists, scoring.score_token_lists(eng, lists, n_top), n_top, TOL[device])
    compare(eng, lists, scoring.score_token_lists(eng, lists, n_top, temperature=0.7), n_top, TOL[device] / 0.7, 0.7)


@pytest.mark.parametrize("device", DEVICES)
def test_long_prompt_in_portions(device):
    """A prompt longer than a pass: later portions read the cache of the earlier ones, at any alignment of portions and blocks."""
    lists = prompts(130, 7, 40, 41)
    want = engine(device, max_tokens_per_batch=256)
    for limit in (40, 48):
        eng = engine(device, max_tokens_per_batch=limit)
        scores = scoring.score_token_lists(eng, lists, 2)
        compare(want, lists, scores, 2, TOL[device])


@pytest.mark.parametrize("device", DEVICES)
def test_models_with_state(device):
    """Layers with a recurrent state: a prompt a pass, on the scratch slot."""
    from xllm_b200.models import ModelArgs
    a = ModelArgs(model_type="qwen3_next", vocab_size=512, hidden_size=256, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                  head_dim=64, intermediate_size=512, qk_norm=True, rope_theta=1e6, partial_rotary_factor=0.25, max_position_embeddings=512,
                  tie_word_embeddings=False,
                  extra=dict(linear_num_value_heads=4, linear_num_key_heads=2, linear_key_head_dim=64, linear_value_head_dim=64,
                             linear_conv_kernel_dim=4, full_attention_interval=4))
    eng = LLMEngine(EngineConfig(model="qwen3_next", device=device, dtype="float32" if device == "cpu" else "bfloat16", num_blocks=64,
                                 enable_graph=False, max_seqs_per_batch=4, max_tokens_per_batch=32, random_weights=True), model_args=a)
    lists = prompts(9, 70, 3, vocab=512)
    compare(eng, lists, scoring.score_token_lists(eng, lists, 0), 0, TOL[device])


def test_passes():
    assert scoring._passes([3, 0, 4, 2, 10, 5], 8, False) == [[[(0, 0, 3), (2, 0, 4)]], [[(4, 0, 8)], [(4, 8, 2)]], [[(3, 0, 2), (5, 0, 5)]]]
    assert scoring._passes([3, 0, 20], 8, True) == [[[(0, 0, 3)]], [[(2, 0, 20)]]]
    assert scoring._passes([0], 8, False) == []


def test_llm_and_refusals():
    llm = LLM("tiny", devices="cpu", dtype="float32", num_blocks=64, enable_graph=False, max_model_len=128)
    lists = prompts(12, 4)
    outs = llm.score(lists, top_logprobs=3)
    compare(llm.engine, lists, outs, 3, TOL["cpu"])
    assert outs[0].usage.num_prompt_tokens == 12 and outs[0].prompt_token_ids == lists[0]
    assert math.isclose(outs[1].total_logprob, sum(outs[1].logprobs[1:]))
    assert llm.score(lists[0])[0].logprobs == llm.score([lists[0]])[0].logprobs
    assert llm.score([[]])[0].logprobs == []
    from xllm_b200.api import c_bridge
    got = json.loads(c_bridge.call(llm, "score", json.dumps({"prompts": lists, "top_logprobs": 1})))
    assert got[1]["logprobs"][1:] == outs[1].logprobs[1:] and got[1]["top_logprobs"][1][0] == list(outs[1].top_logprobs[1][0])
    for bad in (dict(top_logprobs=129), dict(top_logprobs=-1), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(temperature=1e-50), dict(temperature=float("inf"))):
        with pytest.raises(ValueError):
            llm.score(lists, **bad)
    for bad in ([[1, 2, 32000]], [[-1]], [[1] * 129]):
        with pytest.raises(ValueError):
            llm.score(bad)
    llm.sleep(1)
    with pytest.raises(RuntimeError):
        llm.score(lists)


def test_serving_is_left_alone():
    """Requests in flight keep their tokens while prompts are scored between their steps."""
    eng = engine("cpu")
    lists = prompts(20, 31)
    for i, p in enumerate(lists):
        eng.add_request(f"r{i}", p, max_tokens=8, ignore_eos=True)
    want = {}
    eng.run_until_done(on_event=lambda e: want.setdefault(e.request_id, []).append(e.token))
    for i, p in enumerate(lists):
        eng.add_request(f"s{i}", p, max_tokens=8, ignore_eos=True)
    got = {}
    while eng.has_unfinished():
        for e in eng.step():
            got.setdefault(e.request_id, []).append(e.token)
        scoring.score_token_lists(eng, prompts(9, 30), 1)
    assert [got[f"s{i}"] for i in range(2)] == [want[f"r{i}"] for i in range(2)]


def test_route(tmp_path):
    import threading

    from test_server_cpu import _post, _tokenizer
    from xllm_b200.api.server import ApiServer
    eng = engine("cpu")
    srv = ApiServer(eng, _tokenizer(tmp_path), model_name="tiny", host="127.0.0.1", port=0)
    t = threading.Thread(target=srv.serve_forever, args=(10,), daemon=True)
    t.start()
    try:
        status, data = _post(srv.port, "/v1/score", {"prompt": ["hello world", [5, 6, 7, 8]], "logprobs": 2})
        obj = json.loads(data)
        assert status == 200 and obj["object"] == "score" and [c["index"] for c in obj["choices"]] == [0, 1]
        lp = obj["choices"][1]["logprobs"]
        want = scoring.score_token_lists(eng, [[5, 6, 7, 8]], 2)[0]
        assert lp["token_ids"] == [5, 6, 7, 8] and lp["token_logprobs"][0] is None and len(lp["tokens"]) == 4
        assert all(abs(a - b) < 1e-4 for a, b in zip(lp["token_logprobs"][1:], want.logprobs[1:]))
        assert [a["token_id"] for a in lp["top_logprobs"][2]] == [t for t, _ in want.top_logprobs[2]]
        assert obj["usage"]["prompt_tokens"] == 4 + len(obj["choices"][0]["logprobs"]["token_ids"])
        assert _post(srv.port, "/v1/score", {"prompt": [5, 6, 7]})[0] == 200
        for bad in ({}, {"prompt": []}, {"prompt": 7}, {"prompt": [[1, "x"]]}, {"prompt": "a", "logprobs": 500}, {"prompt": [[99999999]]}):
            assert _post(srv.port, "/v1/score", bad)[0] == 400
    finally:
        srv.shutdown()
        t.join(timeout=5)


def state_args(model):
    from xllm_b200.models import ModelArgs
    if model == "rwkv7":
        return ModelArgs(model_type="rwkv7", vocab_size=512, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=4,
                         head_dim=16, intermediate_size=128, max_position_embeddings=512, tie_word_embeddings=False, extra={})
    return ModelArgs(model_type="qwen3_next", vocab_size=512, hidden_size=256, num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                     head_dim=64, intermediate_size=512, qk_norm=True, rope_theta=1e6, partial_rotary_factor=0.25, max_position_embeddings=512,
                     tie_word_embeddings=False,
                     extra=dict(linear_num_value_heads=4, linear_num_key_heads=2, linear_key_head_dim=64, linear_value_head_dim=64,
                                linear_conv_kernel_dim=4, full_attention_interval=4))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("model", ["qwen3_next", "rwkv7"])
@pytest.mark.parametrize("outside", ["score", "embed"])
def test_full_pool_of_states_is_left_alone(device, model, outside):
    """As many requests in flight as the pool has states: each keeps its own, bit by bit, while prompts are scored or embedded between
    the steps, and with it its tokens (on the CPU, where a step's sums have one order)."""
    from xllm_b200.api.embedding import embed_token_lists
    eng = LLMEngine(EngineConfig(model=model, device=device, dtype="float32" if device == "cpu" else "bfloat16", num_blocks=64, enable_graph=False, max_seqs_per_batch=2,
                                 max_tokens_per_batch=64, random_weights=True), model_args=state_args(model))
    assert eng.model.state.n_slots == 3
    lists = prompts(9, 14, 5, vocab=512)

    def tokens(tag, between):
        for i, p in enumerate(lists):
            eng.add_request(f"{tag}{i}", p, max_tokens=12, ignore_eos=True)
        got = {}
        while eng.has_unfinished():
            for e in eng.step():
                got.setdefault(e.request_id[1:], []).append(e.token)
            between()
        return got
    want = tokens("r", lambda: None)
    pool, most = eng.model.state, []

    def states():
        return [t[:, :pool.n_slots].clone() for t in vars(pool).values() if torch.is_tensor(t)]

    def between():
        most.append(len(pool.owner))
        before = states()
        if outside == "score":
            scoring.score_token_lists(eng, prompts(7, 30, vocab=512, seed=8), 1)
        else:
            embed_token_lists(eng, prompts(7, 30, vocab=512, seed=8))
        assert len(before) > 1 and all(torch.equal(a, b) for a, b in zip(before, states()))
    got = tokens("s", between)
    assert max(most) == pool.n_slots and (device != "cpu" or got == want)


def test_an_expired_wait_gives_no_scores(monkeypatch):
    """What head_logprobs returns when a wait of it has expired is not handed out, and the watchdog still hears of it."""
    class Library:
        words = [0, 7, 0, 0]
        xllm_head_logprobs_error_status = lambda self: self.words.pop(0)

    eng = engine("cpu")
    monkeypatch.setattr(scoring.score, "head_supported", lambda h, w: True)
    monkeypatch.setattr(scoring.score, "head_logprobs", lambda h, w, ids, temperature=None: (h[:, 0] * math.nan,) * 2)
    monkeypatch.setattr(_lib, "load", lambda *a: Library())
    scoring.score_token_lists(eng, prompts(4))
    with pytest.raises(RuntimeError, match="wait"):
        scoring.score_token_lists(eng, prompts(4))
    assert scoring.score.error_status() == 7 and scoring.score.error_status() == 0


@pytest.mark.parametrize("device", DEVICES)
def test_alternatives_change_no_score(device):
    """A token's log-probability and its entropy have the same bits whether alternatives are asked for or not; the alternatives are those of
    the logits as they are sampled from, on the GPU rounded to bf16: 2^-8 of a logit, and as much of the sum's logarithm."""
    eng = engine(device)
    hidden = hidden_states(eng, prompts(300)[0])
    ids = torch.tensor(prompts(300, seed=5)[0], device=hidden.device)
    logits = eng.model.logits(hidden)
    for temperature in (None, 0.6):
        want, _ = scoring._score_rows(eng.model, hidden, ids, 0, temperature)
        got, _ = scoring._score_rows(eng.model, hidden, ids, 5, temperature)
        assert want[2] is None and want[3] is None
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        exact = torch.log_softmax((hidden.double() @ eng.model.lm_head.weight[:logits.shape[1]].double().T) / (temperature or 1.0), dim=1)
        off = float(logits.abs().max()) / (temperature or 1.0) * (2.0 ** -7 if device != "cpu" else 1e-5)
        listed = exact.gather(1, got[2].long())
        assert float((got[3] - listed).abs().max()) <= off and float((listed - exact.topk(5, dim=1).values).abs().max()) <= 2 * off


def test_generation_goes_on_between_passes(tmp_path, monkeypatch):
    """A request of many passes shares the loop with the requests that generate: a step of theirs behind every pass."""
    from test_server_cpu import _tokenizer
    from xllm_b200.api.server import ApiServer
    eng = engine("cpu", max_tokens_per_batch=32)
    lists = prompts(20, 25, 70, 1, 30)
    want = scoring.score_token_lists(eng, lists, 1)
    srv = ApiServer(eng, _tokenizer(tmp_path), model_name="tiny", host="127.0.0.1", port=0)
    log, answers = [], []
    forward, step = scoring._forward, eng.step
    monkeypatch.setattr(scoring, "_forward", lambda *a: (log.append("pass"), forward(*a))[1])
    monkeypatch.setattr(eng, "step", lambda *a: (log.append("step"), step(*a))[1])
    monkeypatch.setattr(srv, "_json", lambda http_id, status, obj: answers.append((http_id, status, obj)))
    try:
        eng.add_request("r", prompts(5)[0], max_tokens=40, ignore_eos=True)
        srv._score(SimpleNamespace(id=1), {"prompt": lists, "logprobs": 1})
        srv._score(SimpleNamespace(id=2), {"prompt": lists[2]})
        rounds = 0
        while srv._busy():
            srv._after_poll()
            rounds += 1
            assert rounds < 200
        assert log.count("pass") == 6 + 3 and ("pass", "pass") not in zip(log, log[1:]), log
        assert [(i, status) for i, status, _ in answers] == [(1, 200), (2, 200)]
        for c, s in zip(answers[0][2]["choices"], want):
            assert c["logprobs"]["token_logprobs"] == s.logprobs and c["logprobs"]["entropies"] == s.entropies
        # between two passes the engine may go to sleep: the request ends with an error, the loop goes on
        srv._score(SimpleNamespace(id=3), {"prompt": lists})
        srv._after_poll()
        eng.sleep(1)
        srv._after_poll()
        assert not srv._busy() and answers[-1][:2] == (3, 500) and "asleep" in json.dumps(answers[-1][2])
    finally:
        srv.shutdown()
        srv.http.stop()


@pytest.mark.parametrize("number", ["1e999", "-1e999", "NaN"])
@pytest.mark.parametrize("name", ["logprobs", "temperature"])
def test_numbers_without_an_integer(tmp_path, monkeypatch, name, number):
    """What JSON may hold and no 64 bits do is the caller's mistake, not the server's."""
    from test_server_cpu import _tokenizer
    from xllm_b200.api.server import ApiServer
    srv = ApiServer(engine("cpu"), _tokenizer(tmp_path), model_name="tiny", host="127.0.0.1", port=0)
    answers = []
    monkeypatch.setattr(srv, "_json", lambda http_id, status, obj: answers.append(status))
    try:
        srv._score(SimpleNamespace(id=1), {"prompt": [5, 6], **json.loads('{"%s": %s}' % (name, number))})
        assert answers == [400]
    finally:
        srv.shutdown()
        srv.http.stop()
