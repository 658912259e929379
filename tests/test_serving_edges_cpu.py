"""Completion requests at the edges of what the server accepts, on the CPU."""
import json

import pytest
import torch


@pytest.fixture(scope="module")
def srv(tmp_path_factory):
    from distrain_b200.config import ModelConfig
    from distrain_b200.models.params import ParamLayout, init_flat
    from distrain_b200.serve import CompletionServer
    from distrain_b200.utils.checkpoint import save_safetensors
    cfg = ModelConfig(hidden_dim=32, num_layers=2, num_heads=4, num_kv_heads=2, ffn_hidden_dim=64, vocab_size=260,
                      max_seq_len=128, rope_theta=10000.0)
    L = ParamLayout(cfg)
    path = str(tmp_path_factory.mktemp("ckpt") / "m.safetensors")
    save_safetensors(L.to_state_dict(init_flat(L, seed=3)), path)
    return CompletionServer(path, "cpu", tokenizer="bytes", max_tokens_cap=16, max_n=3)


def _post(srv, body, route="/v1/completions"):
    base = {"prompt": [1, 2, 3], "messages": [{"role": "user", "content": "hi"}], "max_tokens": 4}
    text = json.dumps(dict(base, **body)) if isinstance(body, dict) else body
    return srv.handle_request("POST", route, text.encode())


@pytest.mark.parametrize("route", ["/v1/completions", "/v1/chat/completions"])
@pytest.mark.parametrize("body", [
    # beyond fp32, where the product with a count of zero is NaN for every other token
    {"presence_penalty": 1e39}, {"frequency_penalty": 1e39}, {"frequency_penalty": -1e39}, {"logit_bias": {"7": 1e39}},
    {"logit_bias": {"7": -1e300}}, {"repetition_penalty": 1e39},
    # zero in fp32, or a reciprocal beyond it
    {"repetition_penalty": 1e-50}, {"repetition_penalty": 1e-39},
    # beyond doubles
    {"presence_penalty": 10 ** 400}, {"frequency_penalty": 10 ** 400}, {"logit_bias": {"7": 10 ** 400}},
    {"allowed_token_ids": [float("inf")]}, {"allowed_token_ids": [float("nan")]}, {"allowed_token_ids": [10 ** 400]},
    {"presence_penalty": float("nan")}, {"logit_bias": {"7": float("nan")}},
    # not a token id
    {"allowed_token_ids": [1.7]}, {"logit_bias": {"1.7": 1}}])
def test_options_past_the_edge_of_fp32_are_refused(srv, route, body):
    st, out = _post(srv, body, route)
    assert st == 400 and out["error"]["type"] == "invalid_request_error", out


@pytest.mark.parametrize("body", [
    {"presence_penalty": 1e9}, {"presence_penalty": -1e9}, {"frequency_penalty": 1e9}, {"frequency_penalty": -1e9},
    {"repetition_penalty": 1e9}, {"repetition_penalty": 1e-9}, {"logit_bias": {"7": 1e9}}, {"logit_bias": {"7": -1e9}},
    {"presence_penalty": 1e9, "frequency_penalty": 1e9, "repetition_penalty": 1e9, "logit_bias": {"7": 1e9}},
    {"allowed_token_ids": [1.0, 2]}])
@pytest.mark.parametrize("temperature", [0, 1.0])
def test_options_at_their_limits_work(srv, body, temperature):
    from distrain_b200.serve import LogitOptions
    st, out = _post(srv, dict(body, temperature=temperature))
    assert st == 200 and len(out["choices"][0]["token_ids"]) == 4, out
    o = LogitOptions.from_request(body, 260)
    z = o.apply(torch.linspace(-20, 20, 260), [1, 2, 2, 3, 7], 2)
    assert not torch.isnan(z).any() and (z < float("inf")).all()
    if "allowed_token_ids" in body:
        assert o.allowed == [1, 2]


def test_options_made_in_python_are_checked_too():
    from distrain_b200.serve import LogitOptions
    for kw in (dict(presence=1e39), dict(frequency=float("inf")), dict(repetition=0.0), dict(bias={3: float("nan")})):
        with pytest.raises(ValueError):
            LogitOptions(**kw)


def test_n_of_a_client_that_writes_floats(srv):
    st, out = _post(srv, {"n": 2.0})
    assert st == 200 and [c["index"] for c in out["choices"]] == [0, 1]
    assert len(_post(srv, {"n": 1.0}, "/v1/chat/completions")[1]["choices"]) == 1
    for bad in (1.5, 0.0, 4.0, float("inf"), float("nan")):
        assert _post(srv, {"n": bad})[0] == 400


# ───────────────────────── buffers that share memory ─────────────────────────
def test_spans_meet_where_a_byte_is_in_both():
    """The launchers' test of buffers against the sets of their bytes; nothing is read there."""
    import ctypes
    import random
    from distrain_b200.ops._lib import lib
    f = lib().dt_spans_meet
    f.argtypes, f.restype = [ctypes.c_void_p] + [ctypes.c_longlong] * 3 + [ctypes.c_void_p] + [ctypes.c_longlong] * 3, ctypes.c_int
    rng, base, hits = random.Random(0), 1 << 40, 0
    for _ in range(20000):
        spans, sets = [], []
        for _ in range(2):
            at, rows, nbytes = rng.randint(0, 60), rng.randint(1, 6), rng.randint(1, 12)
            stride = rng.choice([0, nbytes, nbytes + rng.randint(0, 20), rng.randint(1, 12)])
            spans += [base + at, rows, nbytes, stride]
            sets.append({at + r * stride + i for r in range(rows) for i in range(nbytes)})
        want = bool(sets[0] & sets[1])
        hits += want
        assert f(*spans) == want, spans
    assert 4000 < hits < 16000
    assert f(base, 0, 4, 4, base, 1, 4, 4) == 0 and f(base, 1, 0, 0, base, 1, 4, 4) == 0 and f(0, 1, 8, 8, 0, 1, 8, 8) == 0
    for _ in range(20000):  # rows of one stride, as views of one buffer have
        stride, spans, sets = rng.randint(6, 20), [], []
        for _ in range(2):
            at, rows, nbytes = rng.randint(0, 90), rng.randint(1, 6), rng.randint(1, stride)
            spans += [base + at, rows, nbytes, stride]
            sets.append({at + r * stride + i for r in range(rows) for i in range(nbytes)})
        assert f(*spans) == bool(sets[0] & sets[1]), spans
    far = 1 << 33  # spans past 32 bits
    assert f(base, 2, 4, far, base + far, 1, 4, 4) == 1 and f(base, 2, 4, far, base + far + 4, 1, 4, 4) == 0


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-46, 9e-31, 1e39, 1.1e30, float("inf"), float("nan")])
def test_attention_scales_past_the_edge_of_fp32_are_refused(scale):
    from distrain_b200.ops import paged
    from test_paged_cpu import _Plan, _i
    plan = _Plan(6, 3, 0, 4, 2, 32, 16)
    plan.cu_q, plan.tables = _i(4), _i(3, 5)
    b16 = lambda *s: torch.zeros(*s).bfloat16()  # noqa: E731
    a = (b16(6, 128), b16(3, 2, 16, 32), b16(3, 2, 16, 32), b16(6, 128), plan)
    with pytest.raises(ValueError, match="scale"):
        paged.paged_attention(*a, scale=scale)
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_attention(*a, scale=1e-30)


@pytest.mark.parametrize("body", [{"allowed_token_ids": "12"}, {"allowed_token_ids": {"5": 1}}, {"allowed_token_ids": [True]},
                                  {"allowed_token_ids": 7}, {"logit_bias": "7"}])
def test_fields_of_another_kind_are_refused(srv, body):
    assert _post(srv, body)[0] == 400
