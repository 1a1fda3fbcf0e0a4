"""What the decode loop reads from a GGUF file's metadata, and when it says that it cannot keep a context (no GPU)."""
import struct

import pytest

from gguf_writer import write_gguf
from nntrain_amd import GgufReader, NotSupportedError
from nntrain_amd.decoder import DecoderDescriptor, QuantizedDecoder


def _value(value):
    """GGUF type and bytes of a metadata value."""
    if isinstance(value, bool):
        return 7, struct.pack("<?", value)
    if isinstance(value, str):
        return 8, struct.pack("<Q", len(value)) + value.encode()
    if isinstance(value, float):
        return 6, struct.pack("<f", value)
    if isinstance(value, list):
        kind, _ = _value(value[0])
        return 9, struct.pack("<IQ", kind, len(value)) + b"".join(_value(v)[1] for v in value)
    return (5, struct.pack("<i", value)) if value < 0 else (4, struct.pack("<I", value))


def _inspect(tmp_path, arch="llama", **more):
    values = {"block_count": 1, "embedding_length": 64, "feed_forward_length": 64, "attention.head_count": 2, "attention.head_count_kv": 1,
              "attention.layer_norm_rms_epsilon": 1e-5, **{k.replace("__", "."): v for k, v in more.items()}}
    kvs = [("general.architecture", *_value(arch))] + [(f"{arch}.{k}", *_value(v)) for k, v in values.items()]
    path = write_gguf(tmp_path / "m.gguf", [("token_embd.weight", (64, 32), 0, bytes(4 * 64 * 32))], kvs)
    with GgufReader(path) as reader:
        return DecoderDescriptor.inspect(reader)


def _refuses(descriptor, **kw):
    """Whether the loop refuses to keep a context, before it touches a lane."""
    def never(*args):
        raise AssertionError("reached")
    try:
        QuantizedDecoder.from_weights(None, descriptor, never, never, True, **kw)
    except NotSupportedError:
        return True
    except AssertionError:
        return False


@pytest.mark.parametrize("more", [{"attention__sliding_window": [512, 0, 512]}, {"rope__freq_base": [1e4, 1e6]}, {"rope__dimension_count": "32"},
                                  {"attention__sliding_window": -1}])
def test_metadata_that_only_a_context_needs_does_not_stop_a_loop_without_one(tmp_path, more):
    d = _inspect(tmp_path, **more)
    assert d.layer_count == 1 and d.context_refusal
    assert not _refuses(d) and _refuses(d, context_length=8)


def test_metadata_of_a_plain_file(tmp_path):
    d = _inspect(tmp_path, rope__freq_base=5e5, rope__dimension_count=16, attention__sliding_window=7)
    assert (d.rotary_base, d.rotary_width, d.sliding_window, d.context_refusal) == (5e5, 16, 7, "")
    assert not _refuses(d) and not _refuses(d, context_length=8)


@pytest.mark.parametrize("arch,pairs", [("llama", True), ("qwen2", False)])
def test_pairing_follows_a_table_of_architectures(tmp_path, arch, pairs):
    d = _inspect(tmp_path, arch)
    assert d.rotary_pairs == pairs and not _refuses(d, context_length=8)


@pytest.mark.parametrize("arch,more", [("another", {}), ("qwen2", {"attention__sliding_window": 512}), ("llama", {"rope__scale_linear": 4.0}),
                                       ("llama", {"rope__scaling__factor": 4.0}), ("llama", {"attention__sliding_window_pattern": [True, False]}),
                                       ("llama", {"attention__sliding_window_pattern": 6}), ("llama", {"attn_logit_softcapping": 50.0}),
                                       ("llama", {"attention__causal": False}), ("llama", {"attention__scale": 0.25})])
def test_attention_that_the_loop_does_not_carry_out_is_refused_with_a_context(tmp_path, arch, more):
    d = _inspect(tmp_path, arch, **more)
    assert not _refuses(d) and _refuses(d, context_length=8)


def test_metadata_that_asks_for_nothing_is_no_reason_to_refuse(tmp_path):
    d = _inspect(tmp_path, rope__scale_linear=1.0, rope__scaling__factor=1.0, attention__causal=True, attn_logit_softcapping=0.0)
    assert not d.context_refusal and not _refuses(d, context_length=8)
    d = _inspect(tmp_path, rope__scaling__type="none", rope__scaling__factor=8.0)
    assert not _refuses(d, context_length=8)


def test_a_descriptor_that_states_its_pairing_is_taken_at_its_word():
    d = DecoderDescriptor("another", 1, 64, 64, 2, 1, 32, 1e-5, 32, rotary_pairs=True)
    assert not _refuses(d, context_length=8)
