"""A decode loop over a GGUF file's quantized projections, shaped like the reference's per-token path.

The reference's ForwardTokenDevice (NNtrain.Core/Modules/Qwen35QuantizedModel.cs:451-513) walks the layers as
    n = RMSNorm(hidden) -> attention(n) -> hidden += attention; m = RMSNorm(hidden) ->
    hidden += W_down(SiLU(W_gate m) * W_up m)                                  -> ... -> logits = W_out RMSNorm(hidden)
with one launch per operation.  This module runs the same sequence of projections from a llama-style GGUF file
(token_embd, blk.N.attn_norm / attn_q / attn_k / attn_v / attn_output / ffn_norm / ffn_gate / ffn_up / ffn_down,
output_norm, output) on one lane, either that way (`fused=False`) or with the launches this library fuses
(`fused=True`: q|k|v and gate|up stacked, the norms and the SiLU product folded into the projections that consume them,
the residual adds folded into the o and down projections, the value heads read by the o projection itself, SiLU(gate) * up
left by the stacked gate|up projection): four launches per layer instead of twelve, same bits.

Without a context (`context_length=0`) every token is decoded as the first token of its own sequence, where causal
attention is exact without a cache: the single key has softmax weight 1, so each query head receives its group's value
head (qwen35_gpu.first_token_attention).  All the projections of a real decode step run, with their real shapes, which is
what the per-token timing is about.  With `context_length=N` the decoder keeps one sequence of up to N tokens: keys and
values go into an 8-bit cache (kv_cache.QuantizedKvCache) with rotary positions from the file's metadata, and every token
attends to those before it (six launches per layer in the fused form); `prefill` takes a prompt many rows at a time, `score`
gives the log probabilities of a text, `reset` starts over.

Timing follows QwenGgufCommand.WriteGeneration (NNtrain.Cli/QwenGgufCommand.cs:119-157): first-token latency and the
decode rate over the tokens after the first.
"""
from __future__ import annotations

import time
from dataclasses import dataclass

import numpy as np

from . import qwen35_gpu
from .gguf import GgufReader, InvalidDataError
from .kv_cache import QuantizedKvCache, Rotary, Rows
from .lane import HipBuffer, HipExecutionLane
from .loader import GgufTensorDirectory, HipGgufLoader, NotSupportedError
from .native import POST_SILU_PAIR
from .quantized_matrix import PRE_RMS_NORM, PRE_SILU_MULTIPLY, HipQuantizedMatrix


# Which components of a head turn together: neighbours (True) or those half the rotary width apart (False).  Files of other
# architectures may hold the same tensors and pair them either way, so none is assumed for them.
_NEIGHBOURS_TURN = {"llama": True, "qwen2": False}

# Metadata of attention that this loop does not carry out, and the value at which it asks for nothing.
_NEUTRAL = {"rope.scale_linear": 1, "attention.scale": None, "attn_logit_softcapping": 0, "attention.max_alibi_bias": 0, "attention.clamp_kqv": 0,
            "attention.causal": True, "attention.sliding_window_pattern": None}


@dataclass(frozen=True)
class DecoderDescriptor:
    """The metadata a llama-style GGUF file gives for this loop (Qwen35Gguf.Inspect keeps the same fields,
    NNtrain.Core/Serialization/Qwen35Gguf.cs:40-108)."""
    architecture: str
    layer_count: int
    embedding_length: int
    feed_forward_length: int
    head_count: int
    kv_head_count: int
    head_width: int
    rms_epsilon: float
    vocabulary: int
    # what attention over a context needs besides (llama.cpp's keys and their defaults)
    rotary_base: float = 10000.0
    rotary_width: int = 0           # 0: head_width
    rotary_pairs: bool = False      # neighbouring components turn together, else halves of the head
    sliding_window: int = 0         # 0: none
    rotary_scaling: str = "none"
    context_refusal: str = ""       # what the file asks of attention over a context and this loop does not do; empty: nothing

    @staticmethod
    def inspect(reader: GgufReader) -> "DecoderDescriptor":
        md = reader.metadata
        arch = md.get("general.architecture")
        if not isinstance(arch, str) or not arch:
            raise InvalidDataError("GGUF metadata 'general.architecture' is missing.")

        def need(key: str, kind=int):
            value = md.get(f"{arch}.{key}")
            if value is None or isinstance(value, (str, list)):
                raise InvalidDataError(f"GGUF metadata '{arch}.{key}' is missing.")
            return kind(value)

        emb, heads = need("embedding_length"), need("attention.head_count")
        kv = md.get(f"{arch}.attention.head_count_kv")
        kv = heads if kv is None else int(kv)
        head_width = md.get(f"{arch}.attention.key_length")
        head_width = emb // heads if head_width is None else int(head_width)
        token = reader.get_tensor("token_embd.weight")
        if len(token.shape) != 2:
            raise InvalidDataError("GGUF tensor 'token_embd.weight' is not a matrix.")
        refusals: list[str] = []            # (a loop without a context runs whatever these say)
        if arch not in _NEIGHBOURS_TURN:
            refusals.append(f"Rotary positions of architecture '{arch}' are not known.")
        refusals += [f"GGUF metadata '{arch}.{key}' is not supported with a context." for key, neutral in _NEUTRAL.items()
                     if md.get(f"{arch}.{key}", neutral) != neutral]
        if f"{arch}.rope.scaling.type" not in md and md.get(f"{arch}.rope.scaling.factor", 1) != 1:
            refusals.append("Rotary scaling is not supported.")             # (a factor alone scales positions)
        if arch != "llama" and md.get(f"{arch}.attention.sliding_window", 0) != 0:
            refusals.append(f"Which layers of architecture '{arch}' have a sliding window is not known.")

        def number(key: str, default, kind=int):
            value = md.get(f"{arch}.{key}")
            if value is None:
                return default
            if isinstance(value, (str, list)) or not 0 <= value < (2**31 if kind is int else float("inf")):
                refusals.append(f"GGUF metadata '{arch}.{key}' is not one finite number from 0 on.")
                return default
            return kind(value)

        d = DecoderDescriptor(arch, need("block_count"), emb, need("feed_forward_length"), heads, kv, head_width,
                              need("attention.layer_norm_rms_epsilon", float), int(token.shape[1]),
                              number("rope.freq_base", 10000.0, float), number("rope.dimension_count", 0),
                              _NEIGHBOURS_TURN.get(arch, False), number("attention.sliding_window", 0),
                              str(md.get(f"{arch}.rope.scaling.type", "none")), " ".join(refusals))
        if min(d.layer_count, d.embedding_length, d.feed_forward_length, d.head_count, d.kv_head_count, d.head_width) <= 0:
            raise InvalidDataError("GGUF decoder dimensions must be positive.")
        if d.head_count % d.kv_head_count != 0:
            raise InvalidDataError("attention.head_count must be a multiple of attention.head_count_kv.")
        if not np.isfinite(d.rms_epsilon) or d.rms_epsilon < 0:
            raise InvalidDataError("attention.layer_norm_rms_epsilon must be finite and not negative.")
        return d


@dataclass
class GenerationTiming:
    """QwenGgufCommand.GenerationTiming (QwenGgufCommand.cs:165-169)."""
    generated_tokens: int
    total_milliseconds: float
    first_token_milliseconds: float | None
    decode_tokens_per_second: float | None


class _Layer:
    __slots__ = ("attn_norm", "ffn_norm", "q", "k", "v", "o", "gate", "up", "down", "qkv", "gate_up")


class QuantizedDecoder:
    """Weights of one GGUF file resident on one lane, and the per-token loop over them."""

    def __init__(self, lane: HipExecutionLane, reader: GgufReader, fused: bool = True, chunk_bytes: int = 64 << 20,
                 context_length: int = 0, attention_window: int | None = None, attention_sinks: int = 0):
        descriptor = DecoderDescriptor.inspect(reader)
        directory = GgufTensorDirectory(reader)
        loader = HipGgufLoader(lane, reader, chunk_bytes)
        self._build(lane, descriptor, fused,
                    matrix=lambda name, in_w, out_w: loader.load_matrix(directory.matrix(name, in_w, out_w)),
                    dense=lambda name, width: loader.load_dense(directory.dense(name, width)),
                    has_output="output.weight" in directory, finish=directory.reject_unexpected,
                    context=(context_length, attention_window, attention_sinks))
        self.quantized_bytes, self.dense_bytes = loader.quantized_bytes, loader.dense_bytes

    @classmethod
    def from_weights(cls, lane: HipExecutionLane, descriptor: DecoderDescriptor, matrix, dense, has_output: bool,
                     fused: bool = True, context_length: int = 0, attention_window: int | None = None,
                     attention_sinks: int = 0) -> "QuantizedDecoder":
        """The same loop over weights that are already on the lane: matrix(name, in_w, out_w) returns a
        HipQuantizedMatrix whose payload is resident, dense(name, width) an FP32 HipBuffer; the decoder owns both."""
        self = cls.__new__(cls)
        self._build(lane, descriptor, fused, matrix, dense, has_output, finish=lambda: None,
                    context=(context_length, attention_window, attention_sinks))
        self.quantized_bytes = sum(m.storage_bytes for m in self._owned if isinstance(m, HipQuantizedMatrix))
        self.dense_bytes = sum(b.nbytes for b in self._owned if isinstance(b, HipBuffer))
        return self

    def _build(self, lane, descriptor, fused, matrix, dense, has_output, finish, context) -> None:
        self.context_length, window, self.attention_sinks = context
        self.attention_window = descriptor.sliding_window if window is None else window
        if self.context_length < 0 or self.attention_window < 0 or self.attention_sinks < 0:
            raise ValueError("context_length, attention_window and attention_sinks must not be negative.")
        if self.context_length > 0 and descriptor.rotary_scaling != "none":
            raise NotSupportedError(f"Rotary scaling '{descriptor.rotary_scaling}' is not supported.")
        if self.context_length > 0 and descriptor.context_refusal:
            raise NotSupportedError(descriptor.context_refusal)
        self.cache: QuantizedKvCache | None = None
        self.position = 0           # tokens of the context so far
        self.lane = lane
        self.fused = fused
        self.descriptor = d = descriptor
        q_width, kv_width = d.head_count * d.head_width, d.kv_head_count * d.head_width
        self._owned: list = []

        def own(item):
            self._owned.append(item)
            return item

        def stack(parts):
            """One matrix from projections of the same vector; the parts are freed, the stack replaces them."""
            whole = own(HipQuantizedMatrix.stacked(lane, parts))
            for m in parts:
                self._owned.remove(m)
                m.dispose()
            return whole

        try:
            self.embedding = own(matrix("token_embd.weight", d.embedding_length, d.vocabulary))
            self.layers: list[_Layer] = []
            for i in range(d.layer_count):
                p, L = f"blk.{i}.", _Layer()
                L.attn_norm = own(dense(p + "attn_norm.weight", d.embedding_length))
                L.q = own(matrix(p + "attn_q.weight", d.embedding_length, q_width))
                L.k = own(matrix(p + "attn_k.weight", d.embedding_length, kv_width))
                L.v = own(matrix(p + "attn_v.weight", d.embedding_length, kv_width))
                L.o = own(matrix(p + "attn_output.weight", q_width, d.embedding_length))
                L.ffn_norm = own(dense(p + "ffn_norm.weight", d.embedding_length))
                L.gate = own(matrix(p + "ffn_gate.weight", d.embedding_length, d.feed_forward_length))
                L.up = own(matrix(p + "ffn_up.weight", d.embedding_length, d.feed_forward_length))
                L.down = own(matrix(p + "ffn_down.weight", d.feed_forward_length, d.embedding_length))
                L.qkv = L.gate_up = None
                if fused:
                    # projections of the same vector become one launch when their storage types agree
                    if L.q.ggml_type == L.k.ggml_type == L.v.ggml_type:
                        L.qkv = stack([L.q, L.k, L.v])
                        L.q = L.k = L.v = None
                    if L.gate.ggml_type == L.up.ggml_type:
                        L.gate_up = stack([L.gate, L.up])
                        L.gate = L.up = None
                self.layers.append(L)
            self.output_norm = own(dense("output_norm.weight", d.embedding_length))
            # a file without output.weight ties the head to the embedding, as llama.cpp does
            self.output = own(matrix("output.weight", d.embedding_length, d.vocabulary)) if has_output else self.embedding
            finish()
        except BaseException:
            self.dispose()
            raise

        # activations: allocated once, so a token step allocates nothing (and can be captured in a graph)
        alloc = lane.allocate
        self._hidden = [alloc(d.embedding_length), alloc(d.embedding_length)]
        self._cur = 0
        self._norm = alloc(d.embedding_length)
        self._qkv = alloc(q_width + 2 * kv_width)
        self._ctx = alloc(q_width)
        self._attn = alloc(d.embedding_length)
        self._gate_up = alloc(2 * d.feed_forward_length)
        self._act = alloc(d.feed_forward_length)
        self._down = alloc(d.embedding_length)
        self.logits = alloc(d.vocabulary)
        self._owned += self._hidden + [self._norm, self._qkv, self._ctx, self._attn, self._gate_up, self._act, self._down,
                                       self.logits]
        self._graph = None
        self._graph_start = 0
        self._prompt: dict[str, HipBuffer] = {}
        if self.context_length > 0:
            try:
                self.cache = own(QuantizedKvCache(lane, d.layer_count, 1, d.kv_head_count, d.head_width, self.context_length))
                width = d.rotary_width or d.head_width
                if not 2 <= width <= d.head_width or width % 2 != 0 or not d.rotary_base > 0:
                    raise InvalidDataError("rope.dimension_count must be even and within a head, rope.freq_base positive.")
                self._rotary = Rotary(own(lane.upload_raw(Rotary.frequencies(width, d.rotary_base))), width, d.rotary_pairs)
                self._next = own(lane.allocate_bytes(4)), own(lane.allocate(1)), own(lane.allocate(1))
            except BaseException:
                self.dispose()
                raise

    # ---------------------------------------------------------------------------------------------- one token
    def _attend(self, layer: int, q: HipBuffer, k: HipBuffer, v: HipBuffer) -> None:
        """The attention of one token into _ctx: over the context, or as the first token of a sequence."""
        d = self.descriptor
        if self.cache is None:
            qwen35_gpu.first_token_attention(self.lane, v, d.head_count, d.kv_head_count, d.head_width, out=self._ctx)
            return
        self.cache.store(layer, k, v, 1, rotary=self._rotary, q=q, heads=d.head_count)
        self.cache.attention(layer, q, d.head_count, 1, window=self.attention_window, sinks=self.attention_sinks, out=self._ctx)

    def _layers_and_head(self) -> None:
        d, lane = self.descriptor, self.lane
        q_width, kv_width, ffn, eps = d.head_count * d.head_width, d.kv_head_count * d.head_width, d.feed_forward_length, d.rms_epsilon
        q_view = self._qkv.view(0, 4 * q_width)
        k_view = self._qkv.view(4 * q_width, 4 * kv_width)
        v_view = self._qkv.view(4 * (q_width + kv_width), 4 * kv_width)
        gate_view, up_view = self._gate_up.view(0, 4 * ffn), self._gate_up.view(4 * ffn, 4 * ffn)
        for i, L in enumerate(self.layers):
            cur, nxt = self._hidden[self._cur], self._hidden[self._cur ^ 1]
            if self.fused and L.qkv is not None and L.gate_up is not None:
                # Four launches.  The o projection reads the value heads itself (what first-token attention would have
                # copied) and adds the residual stream; the stacked gate | up projection leaves SiLU(gate) * up, so the
                # down projection reads one vector and nobody forms the product twice.  Every value has the bits of the
                # one-launch-per-operation sequence.  (With a context: the store and the attention in between.)
                L.qkv.forward_fused(lane, cur, pre_op=PRE_RMS_NORM, norm_weight=L.attn_norm, epsilon=eps, out=self._qkv)
                if self.cache is None:
                    L.o.forward_fused(lane, v_view, addend=cur, out=nxt, x_head_width=d.head_width,
                                      x_head_group=d.head_count // d.kv_head_count)
                else:
                    self._attend(i, q_view, k_view, v_view)
                    L.o.forward_fused(lane, self._ctx, addend=cur, out=nxt)
                L.gate_up.forward_fused(lane, nxt, pre_op=PRE_RMS_NORM, norm_weight=L.ffn_norm, epsilon=eps, out=self._act,
                                        post_op=POST_SILU_PAIR)
                L.down.forward_fused(lane, self._act, addend=nxt, out=nxt)
                self._cur ^= 1
            elif self.fused:
                if L.qkv is not None:
                    L.qkv.forward_fused(lane, cur, pre_op=PRE_RMS_NORM, norm_weight=L.attn_norm, epsilon=eps, out=self._qkv)
                else:
                    L.q.forward_fused(lane, cur, pre_op=PRE_RMS_NORM, norm_weight=L.attn_norm, epsilon=eps, x_out=self._norm, out=q_view)
                    L.k.forward(lane, self._norm, None, out=k_view)
                    L.v.forward(lane, self._norm, None, out=v_view)
                self._attend(i, q_view, k_view, v_view)
                L.o.forward(lane, self._ctx, None, out=self._attn)
                if L.gate_up is not None:
                    L.gate_up.forward_fused(lane, cur, pre_op=PRE_RMS_NORM, x2=self._attn, norm_weight=L.ffn_norm, epsilon=eps,
                                            sum_out=nxt, out=self._gate_up)
                else:
                    L.gate.forward_fused(lane, cur, pre_op=PRE_RMS_NORM, x2=self._attn, norm_weight=L.ffn_norm, epsilon=eps,
                                         x_out=self._norm, sum_out=nxt, out=gate_view)
                    L.up.forward(lane, self._norm, None, out=up_view)
                L.down.forward_fused(lane, gate_view, pre_op=PRE_SILU_MULTIPLY, x2=up_view, addend=nxt, out=nxt)
                self._cur ^= 1
            else:
                qwen35_gpu.rms_norm(lane, cur, L.attn_norm, 1, d.embedding_length, eps, out=self._norm)
                L.q.forward(lane, self._norm, None, out=q_view)
                L.k.forward(lane, self._norm, None, out=k_view)
                L.v.forward(lane, self._norm, None, out=v_view)
                self._attend(i, q_view, k_view, v_view)
                L.o.forward(lane, self._ctx, None, out=self._attn)
                qwen35_gpu.add_residual_and_rms_norm(lane, cur, self._attn, L.ffn_norm, d.embedding_length, eps, out=self._norm)
                L.gate.forward(lane, self._norm, None, out=gate_view)
                L.up.forward(lane, self._norm, None, out=up_view)
                qwen35_gpu.silu_multiply(lane, gate_view, up_view, ffn, out=self._act)
                L.down.forward(lane, self._act, None, out=self._down)
                qwen35_gpu.add_in_place(lane, cur, self._down, d.embedding_length)
        hidden = self._hidden[self._cur]
        if self.fused:
            self.output.forward_fused(lane, hidden, pre_op=PRE_RMS_NORM, norm_weight=self.output_norm, epsilon=eps, out=self.logits)
        else:
            qwen35_gpu.rms_norm(lane, hidden, self.output_norm, 1, d.embedding_length, eps, out=self._norm)
            self.output.forward(lane, self._norm, None, out=self.logits)
        if self.cache is not None:
            self.cache.advance(1)

    def forward_token(self, token_id: int) -> HipBuffer:
        """Logits after `token_id`, decoded as the next token of the context (without one: as the first token of a
        sequence); the buffer is reused by the next call."""
        if not 0 <= token_id < self.descriptor.vocabulary:
            raise IndexError(f"Embedding index {token_id} is outside the vocabulary.")
        self._room(1)
        if self._graph is not None:
            self._cur = self._graph_start
            self.embedding.dequantize(self.lane, row=token_id, out=self._hidden[self._cur])
            self.lane.graph_launch(self._graph)
            self._cur = self._graph_end
        else:
            self.embedding.dequantize(self.lane, row=token_id, out=self._hidden[self._cur])
            self._layers_and_head()
        if self.cache is not None:
            self.position += 1
        return self.logits

    # ---------------------------------------------------------------------------------------------- context
    def _room(self, tokens: int) -> None:
        if self.cache is not None and self.position + tokens > self.context_length:
            raise ValueError(f"The context holds {self.context_length} tokens; {self.position} are in it and {tokens} were to follow.")

    def reset(self) -> None:
        """Forgets the context."""
        self._context().reset()
        self.position = 0

    def _context(self) -> QuantizedKvCache:
        if self.cache is None:
            raise ValueError("The decoder has no context: give it a context_length.")
        return self.cache

    def _prompt_buffers(self, rows: int, head_rows: int) -> dict[str, HipBuffer]:
        d = self.descriptor
        q_width, kv_width = d.head_count * d.head_width, d.kv_head_count * d.head_width
        need = {"hidden": rows * d.embedding_length, "norm": rows * d.embedding_length, "qkv": rows * (q_width + 2 * kv_width),
                "ctx": rows * q_width, "attn": rows * d.embedding_length, "gate": rows * d.feed_forward_length,
                "up": rows * d.feed_forward_length, "act": rows * d.feed_forward_length, "logits": head_rows * d.vocabulary,
                "targets": head_rows, "log_probs": head_rows, "entropy": head_rows}
        for name, elements in need.items():
            have = self._prompt.get(name)
            if elements and (have is None or have.nbytes < 4 * elements):
                if have is not None:
                    self._owned.remove(have)
                    have.dispose()
                self._prompt[name] = self.lane.allocate(elements)
                self._owned.append(self._prompt[name])
        return self._prompt

    def _prompt_layers(self, tokens, buf: dict[str, HipBuffer], together: int) -> None:
        """The layers over `tokens`, all rows at once; buf["hidden"] receives the last layer's output.  `together` tokens enter a
        layer's cache at a time and attend before the next ones do."""
        try:
            self._all_prompt_layers(tokens, buf, together)
        except BaseException:
            if len(tokens) > together:
                self.lane.fill_u32(self.cache.lengths, self.position, 1)
            raise
        self.position += len(tokens)

    def _all_prompt_layers(self, tokens, buf: dict[str, HipBuffer], together: int) -> None:
        d, lane, n = self.descriptor, self.lane, len(tokens)
        emb, ffn, eps = d.embedding_length, d.feed_forward_length, d.rms_epsilon
        q_width, kv_width = d.head_count * d.head_width, d.kv_head_count * d.head_width
        row = q_width + 2 * kv_width
        hidden, norm, qkv, ctx, attn = (buf[k] for k in ("hidden", "norm", "qkv", "ctx", "attn"))
        for i, token in enumerate(tokens):
            self.embedding.dequantize(lane, row=int(token), out=hidden.view(4 * i * emb, 4 * emb))
        for i, L in enumerate(self.layers):
            qwen35_gpu.rms_norm(lane, hidden, L.attn_norm, n, emb, eps, out=norm)
            if L.qkv is not None:
                L.qkv.forward(lane, norm, None, rows=n, out=qkv)
                places = (0, row), (q_width, row), (q_width + kv_width, row)            # offset and stride of q, k and v
            else:
                places = (0, q_width), (n * q_width, kv_width), (n * (q_width + kv_width), kv_width)
                for m, (at, width) in zip((L.q, L.k, L.v), places):
                    m.forward(lane, norm, None, rows=n, out=qkv.view(4 * at, 4 * n * width))
            if i > 0 and n > together:
                lane.fill_u32(self.cache.lengths, self.position, 1)                     # the layer before moved it
            for first in range(0, n, together):
                now = min(together, n - first)
                q, k, v = (Rows(qkv, stride, 0, at + first * stride) for at, stride in places)
                self.cache.store(i, k, v, now, rotary=self._rotary, q=q, heads=d.head_count)
                self.cache.attention(i, q, d.head_count, now, window=self.attention_window, sinks=self.attention_sinks,
                                     out=Rows(ctx, q_width, 0, first * q_width))
                if n > together:
                    self.cache.advance(now)
            L.o.forward(lane, ctx, None, rows=n, out=attn)
            qwen35_gpu.add_in_place(lane, hidden, attn, n * emb)
            qwen35_gpu.rms_norm(lane, hidden, L.ffn_norm, n, emb, eps, out=norm)
            gate, up = (L.gate, L.up) if L.gate_up is None else self._halves(L.gate_up, ffn)
            gate.forward(lane, norm, None, rows=n, out=buf["gate"])
            up.forward(lane, norm, None, rows=n, out=buf["up"])
            qwen35_gpu.silu_multiply(lane, buf["gate"], buf["up"], n * ffn, out=buf["act"])
            L.down.forward(lane, buf["act"], None, rows=n, out=attn)
            qwen35_gpu.add_in_place(lane, hidden, attn, n * emb)
        if n <= together:
            self.cache.advance(n)

    def _halves(self, stacked: HipQuantizedMatrix, rows: int) -> tuple[HipQuantizedMatrix, HipQuantizedMatrix]:
        """The two projections of a stack, as matrices over windows of its payload."""
        payload, size = stacked.device_payload(self.lane), stacked.storage_bytes // 2
        return tuple(HipQuantizedMatrix.from_device(self.lane, payload.view(at, size), stacked.ggml_type, rows, stacked.input_width)
                     for at in (0, size))

    def _tokens(self, tokens, least: int, rows: int) -> list[int]:
        if rows < 1:
            raise ValueError("rows must be positive.")
        ids = [int(t) for t in tokens]
        if len(ids) < least:
            raise ValueError(f"at least {least} token(s) are needed.")
        if any(not 0 <= t < self.descriptor.vocabulary for t in ids):
            raise IndexError("A token is outside the vocabulary.")
        self._context()
        return ids

    def prefill(self, tokens, rows: int = 512) -> HipBuffer:
        """Takes `tokens` into the context, `rows` at a time, and returns the logits after the last one (the buffer that
        forward_token returns).  The tokens of a piece enter the 8-bit cache together, so the scale of a block covers all of
        them when the first attends: what the context holds depends on `rows` as far as block scales do (rows=1: as
        forward_token leaves it)."""
        ids = self._tokens(tokens, 1, rows)
        self._room(len(ids))
        d, lane = self.descriptor, self.lane
        for at in range(0, len(ids), rows):
            part = ids[at:at + rows]
            buf = self._prompt_buffers(len(part), 0)
            self._prompt_layers(part, buf, len(part))
        last = buf["hidden"].view(4 * (len(part) - 1) * d.embedding_length, 4 * d.embedding_length)
        qwen35_gpu.rms_norm(lane, last, self.output_norm, 1, d.embedding_length, d.rms_epsilon, out=self._norm)
        self.output.forward(lane, self._norm, None, out=self.logits)
        return self.logits

    def score(self, tokens, rows: int = 1) -> tuple[np.ndarray, np.ndarray]:
        """Natural log probability of every token but the first, given those before it, and the entropy of the distribution
        it was drawn from; the tokens are taken into the context.  The projections take many tokens at a time; the cache takes
        `rows`.  With rows=1 nothing behind a token has any influence on what precedes it.  With more, which is quicker, the
        scale of a cache block covers the tokens of the piece behind a query too, the one whose probability is asked for among
        them: results then depend on `rows` as far as 8-bit rounding goes, and entirely where a later token is many times larger
        than those before it, or not finite."""
        ids = self._tokens(tokens, 2, rows)
        self._room(len(ids))
        d, lane = self.descriptor, self.lane
        log_probs, entropies = [], []
        if min(rows, len(ids)) > 65535:
            raise ValueError("rows must be at most 65535.")             # (what one call of token_log_probs takes)
        batch = max(rows, 128 // rows * rows)
        for at in range(0, len(ids), batch):
            part, targets = ids[at:at + batch], ids[at + 1:at + 1 + batch]
            n = len(targets)
            buf = self._prompt_buffers(len(part), n)
            self._prompt_layers(part, buf, rows)
            if n == 0:
                break
            qwen35_gpu.rms_norm(lane, buf["hidden"], self.output_norm, n, d.embedding_length, d.rms_epsilon, out=buf["norm"])
            self.output.forward(lane, buf["norm"], None, rows=n, out=buf["logits"])
            lane.write(buf["targets"], np.asarray(targets, np.int32))
            qwen35_gpu.token_log_probs(lane, buf["logits"], n, d.vocabulary, buf["targets"], out=buf["log_probs"], entropy=buf["entropy"])
            log_probs.append(lane.read(buf["log_probs"], count=n))
            entropies.append(lane.read(buf["entropy"], count=n))
        return np.concatenate(log_probs), np.concatenate(entropies)

    def most_probable(self) -> int:
        """The token with the largest logit after the last step (the first of equal ones), found on the device."""
        ids, top, entropy = self._next_buffers()
        qwen35_gpu.token_log_probs(self.lane, self.logits, 1, self.descriptor.vocabulary, top=1, entropy=entropy, top_ids=ids, top_log_probs=top)
        return int(self.lane.read(ids, np.int32, 1)[0])

    def _next_buffers(self) -> tuple[HipBuffer, HipBuffer, HipBuffer]:
        self._context()
        return self._next

    def capture_graph(self) -> None:
        """Records the layers and the head of a token step into a HIP graph that forward_token then replays (the
        embedding lookup stays outside: its source row changes with the token).  One eager step must have run."""
        if self._graph is not None:
            return
        self._graph_start = self._cur
        self.lane.graph_begin()
        try:
            self._layers_and_head()
        finally:
            graph = self.lane.graph_end()
        self._graph, self._graph_end = graph, self._cur

    # ---------------------------------------------------------------------------------------------- generation
    def generate(self, first_token, max_new_tokens: int, on_token=None) -> tuple[list[int], GenerationTiming]:
        """Greedy decoding, one token per step; first tie wins, as the reference's device ArgMax does.  With a context
        `first_token` may be a prompt (a sequence of tokens), every step sees the tokens before it and the argmax runs on the
        device.  Without one each step sees only its own token and the argmax runs on the host over the downloaded logits."""
        if max_new_tokens < 0:
            raise ValueError("max_new_tokens must not be negative.")
        if self.cache is not None:
            return self._generate_in_context(first_token, max_new_tokens, on_token)
        tokens: list[int] = []
        first = last = None
        started = time.perf_counter()
        token = first_token
        for _ in range(max_new_tokens):
            logits = self.lane.read(self.forward_token(token), count=self.descriptor.vocabulary)
            token = int(np.argmax(logits))
            last = (time.perf_counter() - started) * 1e3
            first = last if first is None else first
            tokens.append(token)
            if on_token is not None:
                on_token(token)
        total = (time.perf_counter() - started) * 1e3
        rate = (len(tokens) - 1) * 1000.0 / (last - first) if len(tokens) > 1 and last > first else None
        return tokens, GenerationTiming(len(tokens), total, first, rate)

    def _generate_in_context(self, prompt, max_new_tokens: int, on_token) -> tuple[list[int], GenerationTiming]:
        ids = [int(prompt)] if np.ndim(prompt) == 0 else [int(t) for t in prompt]
        self._room(len(ids) + max(0, max_new_tokens - 1))
        tokens: list[int] = []
        first = last = None
        started = time.perf_counter()
        for _ in range(max_new_tokens):
            if tokens or len(ids) == 1:
                self.forward_token(tokens[-1] if tokens else ids[0])
            else:
                self.prefill(ids)
            tokens.append(self.most_probable())
            last = (time.perf_counter() - started) * 1e3
            first = last if first is None else first
            if on_token is not None:
                on_token(tokens[-1])
        total = (time.perf_counter() - started) * 1e3
        rate = (len(tokens) - 1) * 1000.0 / (last - first) if len(tokens) > 1 and last > first else None
        return tokens, GenerationTiming(len(tokens), total, first, rate)

    def dispose(self) -> None:
        if getattr(self, "_graph", None) is not None and not self.lane.disposed:
            self.lane.graph_destroy(self._graph)
        self._graph = None
        for item in reversed(getattr(self, "_owned", [])):
            item.dispose()
        self._owned = []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()


__all__ = ["DecoderDescriptor", "GenerationTiming", "QuantizedDecoder", "NotSupportedError"]
