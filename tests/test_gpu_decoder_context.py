"""The decode loop over a context: store -> attention -> projections -> log probabilities, as a program uses them together.

The CPU restatement runs the same model in float64 mat-vecs and the oracle's FP32 row operations, with keys and values taken
through the block quantisation.  Bar: the mat-vecs of both sides differ by about 1e-7 relative, so now and then a key or
value component falls on the other side of a rounding border of its 8-bit code: one step is 1/127 of its block's largest
value, at most 1/127 of that token's value row in norm, and a row has a weight of about 1 / tokens; a handful of such steps in 20 to
60 tokens stays below 5 / (127 * 20) = 2e-3 of a head's output, 1e-3 of the logits behind two layers and eight heads.
"""
import numpy as np
import pytest

import kv_reference as ref
import oracle
from nntrain_amd import GGML_Q4_K, GGML_Q5_K, GGML_Q6_K, GgufReader, HipExecutionLane, NotSupportedError, Rotary
from nntrain_amd.decoder import DecoderDescriptor, QuantizedDecoder
from test_gpu_decoder import EMB, EPS, HEADS, HW, KV, LAYERS, VOCAB, _kv, _model

pytestmark = pytest.mark.gpu

BAR = 1e-3


@pytest.fixture(scope="module")
def lane():
    with HipExecutionLane(0) as ln:
        yield ln


class CpuContext:
    def __init__(self, host, window=0, sinks=0):
        self.host, self.window, self.sinks = host, window, sinks
        self.k = [np.zeros((0, KV, HW), np.float32) for _ in range(LAYERS)]
        self.v = [np.zeros((0, KV, HW), np.float32) for _ in range(LAYERS)]

    def _weights(self, name):
        typ, raw, out_w, in_w = self.host[name]
        return oracle.dequantize(typ, raw).reshape(out_w, in_w).astype(np.float64)

    def _project(self, name, x):
        return (x.astype(np.float64) @ self._weights(name).T).astype(np.float32)

    def step(self, tokens):
        """Logits after each of `tokens`, which enter the context together."""
        start, n = self.k[0].shape[0], len(tokens)
        inv = Rotary.frequencies(HW)
        at = np.arange(start, start + n)
        hidden = self._weights("token_embd.weight")[tokens].astype(np.float32)
        norm = lambda x, name: oracle.rms_norm(x, self.host[name], n, EMB, EPS).reshape(n, EMB)     # noqa: E731
        for i in range(LAYERS):
            p = f"blk.{i}."
            x = norm(hidden, p + "attn_norm.weight")
            q, k, v = (self._project(p + f"attn_{s}.weight", x).reshape(n, -1, HW) for s in "qkv")
            q, k = (ref.rotate(y, at, inv, HW, pairs=True) for y in (q, k))
            self.k[i], self.v[i] = np.concatenate([self.k[i], k]), np.concatenate([self.v[i], v])
            ctx, _ = ref.attend(q, ref.cached(self.k[i]), ref.cached(self.v[i]), start, self.window, self.sinks)
            hidden = hidden + self._project(p + "attn_output.weight", ctx.reshape(n, -1).astype(np.float32))
            x = norm(hidden, p + "ffn_norm.weight")
            act = oracle.silu_multiply(self._project(p + "ffn_gate.weight", x).ravel(), self._project(p + "ffn_up.weight", x).ravel())
            hidden = hidden + self._project(p + "ffn_down.weight", act.reshape(n, -1))
        return self._project("output.weight", norm(hidden, "output_norm.weight"))


def _decoder(lane, path, **kw):
    with GgufReader(path) as reader:
        return QuantizedDecoder(lane, reader, **{"context_length": 100, **kw})


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 3)])
def test_tokens_one_by_one(lane, tmp_path, window, sinks):
    path, host = _model(tmp_path, "m.gguf")
    tokens = list(np.random.default_rng(1).integers(0, VOCAB, 24))
    options = dict(attention_window=window, attention_sinks=sinks)
    with _decoder(lane, path, **options) as fused, _decoder(lane, path, fused=False, **options) as plain:
        cpu, eager = CpuContext(host, window, sinks), []
        for t in tokens:
            got = lane.read(fused.forward_token(int(t)), count=VOCAB)
            other = lane.read(plain.forward_token(int(t)), count=VOCAB)
            assert np.array_equal(got.view(np.uint32), other.view(np.uint32))
            want = cpu.step([t])[0]
            assert oracle.rel_l2(got, want) <= BAR
            assert fused.most_probable() == int(np.argmax(got))
            eager.append(got)
        assert fused.position == len(tokens) and list(fused.cache.read_lengths()) == [len(tokens)]
        # the graph serves every position
        fused.capture_graph()
        fused.reset()
        for t, e in zip(tokens, eager):
            lane.synchronize()
            assert np.array_equal(lane.read(fused.forward_token(int(t)), count=VOCAB).view(np.uint32), e.view(np.uint32))


@pytest.mark.parametrize("types", [(GGML_Q4_K,) * 3, (GGML_Q4_K, GGML_Q5_K, GGML_Q6_K)])
@pytest.mark.parametrize("fused", [True, False])
def test_prompts_in_pieces_then_tokens(lane, tmp_path, types, fused):
    path, host = _model(tmp_path, "p.gguf", qkv_types=types)
    tokens = list(np.random.default_rng(2).integers(0, VOCAB, 75))
    with _decoder(lane, path, fused=fused) as dec:
        cpu = CpuContext(host)
        got = lane.read(dec.prefill(tokens[:70], rows=33), count=VOCAB)
        for at in (0, 33, 66):
            want = cpu.step(tokens[at:min(at + 33, 70)])[-1]
        assert oracle.rel_l2(got, want) <= BAR
        for t in tokens[70:]:
            got = lane.read(dec.forward_token(int(t)), count=VOCAB)
            assert oracle.rel_l2(got, cpu.step([t])[0]) <= BAR


def test_scores_of_a_text(lane, tmp_path):
    path, host = _model(tmp_path, "s.gguf")
    tokens = list(np.random.default_rng(3).integers(0, VOCAB, 65))
    with _decoder(lane, path) as dec:
        log_probs, entropies = dec.score(tokens, rows=32)
        cpu = CpuContext(host)
        logits = np.concatenate([cpu.step(tokens[at:at + 32]) for at in (0, 32, 64)])
        want, want_entropy = ref.log_probs(logits)
        assert log_probs.shape == entropies.shape == (64,) and dec.position == 65
        # a relative error of BAR in logits of size s moves a log probability by at most 2 BAR max |logit|
        slack = 2 * BAR * np.abs(logits).max()
        assert np.abs(log_probs - want[np.arange(64), tokens[1:]]).max() <= slack
        assert np.abs(entropies - want_entropy[:64]).max() <= slack * (1 + np.abs(want).max())
        # (token by token the values differ: a block's scale then knows nothing of the tokens behind the query)


def test_generation_from_a_prompt(lane, tmp_path):
    path, _ = _model(tmp_path, "g.gguf")
    prompt = [5, 9, 200, 17, 3]
    with _decoder(lane, path, context_length=16) as dec:
        seen = []
        tokens, timing = dec.generate(prompt, 6, on_token=seen.append)
        assert tokens == seen and timing.generated_tokens == 6 and timing.first_token_milliseconds > 0
        dec.reset()
        lane.read(dec.prefill(prompt), count=VOCAB)
        want = [dec.most_probable()]
        while len(want) < 6:
            want.append(int(np.argmax(lane.read(dec.forward_token(want[-1]), count=VOCAB))))
        assert tokens == want
        dec.reset()
        assert dec.generate(5, 2)[0][0] == int(np.argmax(_first(lane, path, 5)))
        with pytest.raises(ValueError):
            dec.generate(prompt, 15)                                    # 2 + 5 + 14 tokens into 16


def _first(lane, path, token):
    with _decoder(lane, path, context_length=4) as dec:
        return lane.read(dec.forward_token(token), count=VOCAB)


def test_limits_and_refusals(lane, tmp_path):
    path, _ = _model(tmp_path, "l.gguf")
    before = lane.counters()["allocated_bytes"]
    with _decoder(lane, path, context_length=3) as dec:
        dec.prefill([1, 2])
        dec.forward_token(3)
        for call in (lambda: dec.forward_token(4), lambda: dec.prefill([1]), lambda: dec.score([1, 2]), lambda: dec.prefill([])):
            with pytest.raises(ValueError):
                call()
        dec.reset()
        with pytest.raises(IndexError):
            dec.prefill([VOCAB])
        with pytest.raises(ValueError):
            dec.score([1])
    assert lane.counters()["allocated_bytes"] == before
    with GgufReader(path) as reader, QuantizedDecoder(lane, reader) as dec:
        for call in (dec.reset, dec.most_probable, lambda: dec.prefill([1]), lambda: dec.score([1, 2])):
            with pytest.raises(ValueError):
                call()
    with GgufReader(path) as reader, pytest.raises(ValueError):
        QuantizedDecoder(lane, reader, context_length=-1)
    with GgufReader(path) as reader:
        d = DecoderDescriptor.inspect(reader)
        assert (d.rotary_base, d.rotary_width, d.rotary_pairs, d.sliding_window, d.rotary_scaling) == (10000.0, 0, True, 0, "none")


def test_pieces_of_no_tokens_are_refused(lane, tmp_path):
    path, _ = _model(tmp_path, "p.gguf")
    with _decoder(lane, path, context_length=8) as dec:
        for call in (lambda: dec.prefill([1, 2], rows=0), lambda: dec.prefill([1, 2], rows=-1), lambda: dec.score([1, 2], rows=0)):
            with pytest.raises(ValueError):
                call()
        assert dec.position == 0


def test_metadata_of_positions(lane, tmp_path):
    from gguf_writer import write_gguf
    path, _ = _model(tmp_path, "a.gguf")
    with GgufReader(path) as reader:
        kvs = [_kv(k, v) for k, v in reader.metadata.items() if k.startswith("llama") or k == "general.architecture"]
        tensors = [(t.name, t.shape, t.type, bytes(reader.read_tensor_bytes(t))) for t in reader.tensors]
    more = [_kv("llama.rope.freq_base", 500000.0), _kv("llama.rope.dimension_count", 32), _kv("llama.attention.sliding_window", 7)]
    path = write_gguf(tmp_path / "b.gguf", tensors, kvs + more)
    with _decoder(lane, path) as dec:
        assert (dec._rotary.width, dec.attention_window) == (32, 7)
        assert np.array_equal(lane.read(dec._rotary.inv_freq), Rotary.frequencies(32, 500000.0))
    path = write_gguf(tmp_path / "c.gguf", tensors, kvs + [_kv("llama.rope.scaling.type", "yarn")])
    with GgufReader(path) as reader:
        QuantizedDecoder(lane, reader).dispose()
        with pytest.raises(NotSupportedError):
            QuantizedDecoder(lane, reader, context_length=8)


@pytest.mark.parametrize("types", [(GGML_Q4_K,) * 3, (GGML_Q4_K, GGML_Q5_K, GGML_Q6_K)])
def test_scores_are_those_of_token_by_token_decoding(lane, tmp_path, types):
    """By default a token's log probability depends on the tokens before it alone: as if each had entered the context by itself."""
    path, host = _model(tmp_path, "t.gguf", qkv_types=types)
    tokens = list(np.random.default_rng(4).integers(0, VOCAB, 70))
    with _decoder(lane, path) as dec:
        log_probs, entropies = dec.score(tokens[:66])
        cpu = CpuContext(host)
        logits = np.concatenate([cpu.step([t]) for t in tokens[:66]])
        want, want_entropy = ref.log_probs(logits)
        slack = 2 * BAR * np.abs(logits).max()                          # (as above)
        assert log_probs.shape == (65,) and dec.position == 66 and list(dec.cache.read_lengths()) == [66]
        assert np.abs(log_probs - want[np.arange(65), tokens[1:66]]).max() <= slack
        assert np.abs(entropies - want_entropy[:65]).max() <= slack * (1 + np.abs(want).max())
        for t in tokens[66:]:                                           # what the context holds serves the tokens behind it
            assert oracle.rel_l2(lane.read(dec.forward_token(int(t)), count=VOCAB), cpu.step([t])[0]) <= BAR


def test_scores_do_not_depend_on_the_tokens_behind(lane, tmp_path):
    path, host = _model(tmp_path, "u.gguf")
    rng = np.random.default_rng(5)
    tokens, other = rng.integers(0, VOCAB, 64).tolist(), rng.integers(0, VOCAB, 24).tolist()
    with _decoder(lane, path) as dec:
        first, _ = dec.score(tokens)
        dec.reset()
        second, _ = dec.score(tokens[:40] + other)
    logits = np.concatenate([CpuContext(host).step(tokens)])
    assert np.abs(first[:39] - second[:39]).max() <= 2 * BAR * np.abs(logits).max()


def test_a_score_that_fails_leaves_the_context_as_it_was(lane, tmp_path, monkeypatch):
    path, _ = _model(tmp_path, "v.gguf")
    with _decoder(lane, path) as dec:
        dec.prefill([1, 2, 3])
        before = lane.read(dec.forward_token(4), count=VOCAB)
        dec.cache.set_lengths([3])
        dec.position = 3
        calls, attention = [], dec.cache.attention

        def failing(*args, **kw):
            calls.append(args)
            if len(calls) == 6:                                         # the second layer's second token
                raise RuntimeError("stop")
            return attention(*args, **kw)
        monkeypatch.setattr(dec.cache, "attention", failing)
        with pytest.raises(RuntimeError):
            dec.score([7, 8, 9, 10])
        monkeypatch.undo()
        assert dec.position == 3 and list(dec.cache.read_lengths()) == [3]
        assert np.array_equal(before, lane.read(dec.forward_token(4), count=VOCAB))


def test_an_architecture_that_turns_halves_of_a_head(lane, tmp_path, monkeypatch):
    from gguf_writer import write_gguf
    path, host = _model(tmp_path, "h.gguf")
    with GgufReader(path) as reader:
        kvs = [_kv(k.replace("llama.", "qwen2."), "qwen2" if k == "general.architecture" else v) for k, v in reader.metadata.items()
               if k.startswith("llama") or k == "general.architecture"]
        tensors = [(t.name, t.shape, t.type, bytes(reader.read_tensor_bytes(t))) for t in reader.tensors]
    path = write_gguf(tmp_path / "i.gguf", tensors, kvs)
    rotate = ref.rotate
    monkeypatch.setattr(ref, "rotate", lambda x, at, inv, width, pairs: rotate(x, at, inv, width, pairs=False))
    tokens = [int(t) for t in np.random.default_rng(6).integers(0, VOCAB, 12)]
    with _decoder(lane, path) as dec:
        cpu = CpuContext(host)
        for t in tokens:
            assert oracle.rel_l2(lane.read(dec.forward_token(t), count=VOCAB), cpu.step([t])[0]) <= BAR


def test_scores_of_more_rows_than_a_call_takes_are_refused_before_any_work(lane, tmp_path):
    path, _ = _model(tmp_path, "w.gguf")
    with _decoder(lane, path, context_length=66000) as dec:
        launches = lane.counters()["kernel_launches"]
        with pytest.raises(ValueError):
            dec.score([1] * 65540, rows=65537)
        assert dec.position == 0 and lane.counters()["kernel_launches"] == launches
        assert dec.score([1, 2, 3], rows=65537)[0].shape == (2,)
