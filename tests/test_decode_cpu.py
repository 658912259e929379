"""The host side of generation over the paged cache: what it refuses before anything reaches a GPU."""
from types import SimpleNamespace

import pytest
import torch


def _decoder(**kw):
    """A decoder without buffers; whatever comes after the checks fails for want of an attribute."""
    from distrain_b200.models.decode import PagedDecoder
    dec = PagedDecoder.__new__(PagedDecoder)
    dec.eng, dec.dev = SimpleNamespace(V=100), torch.device("cpu")
    dec.max_prompt, dec.max_new, dec.max_batch, dec.n, dec.length = 8, 4, 2, 2, 0
    dec.__dict__.update(kw)
    return dec


@pytest.mark.parametrize("bad", [100, -1, 2 ** 31 - 1, 10 ** 12])
def test_ids_outside_the_vocabulary_are_refused(bad):
    """An id past the embedding's rows would be read out of range on the GPU."""
    dec = _decoder()
    with pytest.raises(ValueError, match="vocabulary"):
        dec.prefill([1, 2, bad])
    with pytest.raises(ValueError, match="vocabulary"):
        dec.step([99, bad])
    with pytest.raises(AttributeError):  # ids of the vocabulary pass
        dec.prefill([0, 99])


class FakeDecoder:
    """Logits of a fixed table instead of a model: the token after t is drawn from row t. Takes part in
    ``sample_cached`` without a GPU."""

    def __init__(self, V=50, max_prompt=16, max_batch=4, report=None, seed=0):
        self.eng, self.dev, self.max_prompt, self.max_batch = SimpleNamespace(V=V), torch.device("cpu"), max_prompt, max_batch
        self.z = torch.randn(V, V, generator=torch.Generator().manual_seed(seed))
        self.report, self.checked, self.n = report, 0, 0

    def prefill(self, ids):
        return self.z[ids[-1]:ids[-1] + 1]

    def branch(self, n):
        assert 1 <= n <= self.max_batch
        self.n = n

    def step(self, tokens):
        assert len(tokens) == self.n
        return self.z[torch.tensor(tokens)]

    def check(self):
        self.checked += 1
        if self.report:
            raise RuntimeError(self.report)


def test_what_the_gpu_reports_fails_the_request():
    from distrain_b200.serve import sample_cached
    dec = FakeDecoder()
    assert len(sample_cached(dec, [1, 2], 2, 5)[0][0]) == 5 and dec.checked == 1
    for tokens in (1, 5):
        with pytest.raises(RuntimeError, match="gave up"):
            sample_cached(FakeDecoder(report="gave up"), [1, 2], 1, tokens)
    first = sample_cached(dec, [1, 2], 1, 1)[0][0][0]
    with pytest.raises(RuntimeError, match="gave up"):  # an answer that stops is checked too
        sample_cached(FakeDecoder(report="gave up"), [1, 2], 1, 5, stop_token=first)


def test_a_request_that_ends_in_an_exception_is_checked_too():
    """The report must not be left for the next request to find."""
    from distrain_b200.serve import sample_cached
    dec = FakeDecoder()
    dec.z[:] = float("nan")
    with pytest.raises(RuntimeError, match="nan"):
        sample_cached(dec, [1, 2], 1, 3, temperature=1.0)
    assert dec.checked == 1


def test_a_prompt_that_fails_leaves_nothing_to_continue():
    """The pages of the prompt before are overwritten by then."""
    dec = _decoder(prompt_len=5)
    with pytest.raises(AttributeError):  # fails behind the checks
        dec.prefill([1, 2])
    with pytest.raises(RuntimeError, match="prefill"):
        dec.branch(1)
    with pytest.raises(ValueError, match="tokens"):
        dec.step([1, 2])
    dec = _decoder(prompt_len=5)
    with pytest.raises(ValueError):  # a refused prompt changes nothing
        dec.prefill([])
    assert (dec.prompt_len, dec.n) == (5, 2)


def test_answers_whose_buffers_fail_cannot_be_stepped():
    dec = _decoder(prompt_len=5)
    with pytest.raises(AttributeError):
        dec.branch(1)
    with pytest.raises(ValueError, match="tokens"):
        dec.step([1])


def _plain_process(logits, out, *, history, lens, prompt_lens, repetition, presence, frequency, bias_ids=None,
                   bias_vals=None, bias_lens=None, mask=None):
    """The processor's formula, one row after another on the CPU."""
    for b in range(logits.shape[0]):
        z = logits[b].clone()
        h = history[b, :int(lens[b])].long()
        seen = torch.bincount(h, minlength=z.numel()) > 0
        count = torch.bincount(h[int(prompt_lens[b]):], minlength=z.numel())
        z = torch.where(seen, torch.where(z > 0, z / repetition[b], z * repetition[b]), z)
        z = z - frequency[b] * count - presence[b] * (count > 0)
        if bias_ids is not None:
            for e in range(int(bias_lens[b])):
                z[int(bias_ids[b, e])] += bias_vals[b, e]
        if mask is not None:
            v = torch.arange(z.numel())
            z[(mask[b].long()[v // 32] >> (v % 32)) & 1 == 0] = float("-inf")
        out[b] = z


class _FakeLM:
    """The fake decoder's logits for ``sample``."""

    def __init__(self, dec):
        self.dec = dec

    def next_logits(self, seq):
        return self.dec.z[seq[-1]]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("options", [None, dict(presence=0.7, frequency=0.3, repetition=1.8, bias={3: 1.5, 40: -2.0}),
                                     dict(repetition=2.5, allowed=list(range(0, 50, 3)))])
@pytest.mark.parametrize("prompt", [5, 40])  # 40: longer than the decoder has room for
def test_answers_follow_sample(monkeypatch, temperature, options, prompt):
    """Answer i is what ``sample`` draws with seed + i, penalties on the whole prompt among the rest."""
    from distrain_b200.ops import sampling
    from distrain_b200.serve import LogitOptions, sample, sample_cached
    monkeypatch.setattr(sampling, "process_logits", _plain_process)
    dec = FakeDecoder(seed=4)
    ids = torch.randint(0, 50, (prompt,), generator=torch.Generator().manual_seed(1)).tolist()
    o = None if options is None else LogitOptions(**options)
    got = sample_cached(dec, ids, 4, 12, temperature, 7, options=o)
    sd = {"x": torch.zeros(1)}
    want = [sample(sd, None, ids, 12, temperature, 7 + i, lm=_FakeLM(dec), options=o) for i in range(4)]
    assert got == want
    if temperature:
        assert len({tuple(a) for a, _ in got}) > 1
    stop = got[0][0][3]
    got = sample_cached(dec, ids, 4, 12, temperature, 7, stop_token=stop, options=o)
    assert got == [sample(sd, None, ids, 12, temperature, 7 + i, stop_token=stop, lm=_FakeLM(dec), options=o) for i in range(4)]


def test_every_call_runs_on_the_decoders_device(monkeypatch):
    """The current device is a thread's own: a decoder on another one makes it current around all it launches."""
    from distrain_b200 import ops, serve
    from distrain_b200.models import decode, engine
    from distrain_b200.ops import sampling
    current, seen = [0], []

    class Device:  # stands in for torch.cuda.device
        def __init__(self, dev):
            self.index = torch.device(dev).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before
    monkeypatch.setattr(torch.cuda, "device", Device)

    def note(*a, **kw):
        seen.append(current[0])
        raise KeyError("seen")
    dec = _decoder(dev=torch.device("cuda", 1), prompt_len=3, rows=128, eng=SimpleNamespace(V=100, H=8))
    dec._buffers = dec._ints = note
    monkeypatch.setattr(ops, "device_error", note)
    for call in (lambda: dec.step([1, 2]), lambda: dec.prefill([1]), dec.check):
        with pytest.raises(KeyError):
            call()
    monkeypatch.setattr(torch, "full", note)
    with pytest.raises(KeyError):
        dec.prompt_len = 3
        dec.prompt_pages = dec.answer_pages = 1
        dec.P = 16
        dec.branch(1)
    monkeypatch.undo()
    assert seen == [1] * 4 and current == [0]

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(engine, "TrainEngine", note)
    from distrain_b200.config import ModelConfig
    cfg = ModelConfig(hidden_dim=32, num_layers=1, num_heads=4, num_kv_heads=2, ffn_hidden_dim=64, vocab_size=64, max_seq_len=32)
    from distrain_b200.models.params import ParamLayout, init_flat
    L = ParamLayout(cfg)
    with pytest.raises(KeyError):
        serve.load_decoder(L.to_state_dict(init_flat(L, seed=1)), cfg, "cuda:1", 8, 8)
    fake = FakeDecoder()

    def processor(logits, out, **kw):
        seen.append(current[0])
        out.copy_(logits)
    monkeypatch.setattr(sampling, "process_logits", processor)
    monkeypatch.setattr(decode, "on_device", lambda dev: Device("cuda:2"))
    serve.sample_cached(fake, [1], 1, 2, options=serve.LogitOptions(presence=1.0))
    assert seen[4:] == [1, 2, 2] and current == [0]
