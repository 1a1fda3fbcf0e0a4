"""Cases of the 8-bit key/value cache, of attention over it and of token log probabilities, for timing and comparison.

`own` false: the plain form in elementary torch operations.  `own` true: the framework's operators.  Three operators:
  store   rotary positions of new queries and keys, block quantisation of keys and values into the cache, and the 8-bit
          values read back (a block is 64 consecutive tokens of one head; scale = max |x| / 127)
  attend  attention of new tokens over the cache: causal, grouped queries, optional sliding window with first tokens kept
  score   log probabilities of given tokens, the entropy of the distribution and its top alternatives, from logits
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64
_lane = None


# ------------------------------------------------------------------------------------------------------------- cases
def _store(name, sequences, heads, kv_heads, width, tokens, before, chunk=0):
    return {"name": name, "op": "store", "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "width": width,
            "tokens": tokens, "before": before, "chunk": chunk}


def _attend(name, sequences, heads, kv_heads, width, tokens, before, window=0, sinks=0, ragged=False):
    return {"name": name, "op": "attend", "sequences": sequences, "heads": heads, "kv_heads": kv_heads, "width": width,
            "tokens": tokens, "before": before, "window": window, "sinks": sinks, "ragged": ragged}


def _score(name, rows, vocabulary, top, spread):
    return {"name": name, "op": "score", "rows": rows, "vocabulary": vocabulary, "top": top, "spread": spread}


def listed():
    return [
        # one token of a small model, early in a conversation: latency alone
        _store("store_token_small", 1, 4, 2, 64, 1, 100),
        # one decode step of 32 sequences of different lengths
        _store("store_step_batch", 32, 32, 16, 128, 1, 4096),
        # a prompt of odd length, taken in two pieces, as a chunked prefill stores it
        _store("store_prompt", 1, 40, 8, 128, 4093, 0, chunk=2500),
        # one token over a short history: latency alone
        _attend("attend_token_small", 1, 4, 2, 64, 1, 100),
        # one token of one sequence at the end of a long document
        _attend("attend_token_long", 1, 40, 8, 128, 1, 131000),
        # one decode step of 32 sequences of different lengths
        _attend("attend_step_batch", 32, 32, 16, 128, 1, 8191, ragged=True),
        # a decode step of layers with a sliding window that keep the first four tokens
        _attend("attend_step_window", 16, 40, 8, 128, 1, 20000, window=4096, sinks=4, ragged=True),
        # a whole prompt of odd length against itself
        _attend("attend_prompt", 1, 40, 8, 128, 4093, 0),
        # a chunk of a prompt behind a cached part, window and first tokens, sequences of different lengths in a padded batch
        _attend("attend_chunk_window", 2, 32, 16, 128, 509, 7000, window=1024, sinks=4, ragged=True),
        # the next token of one sequence: its most probable alternative alone (greedy decoding)
        _score("score_token", 1, 32000, 1, 3.0),
        # a decode step of 32 sequences with twenty alternatives
        _score("score_step_batch", 32, 262144, 20, 2.0),
        # the log probabilities of a prompt's tokens, with five alternatives
        _score("score_prompt", 512, 262144, 5, 2.5),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the ranges above: head layouts, lengths, batch sizes, windows, vocabularies."""
    op = rng.choice(["store", "attend", "attend", "score"])
    if op == "score":
        rows, vocabulary = _log_uniform(rng, 1, 512), _log_uniform(rng, 1000, 262144)
        return _without_name(_score("", rows, vocabulary, rng.choice([0, 1, 3, 5, 20, 32]), rng.choice([1.0, 2.5, 6.0])))
    kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8])
    width = rng.choice([64, 80, 96, 128, 128, 256])
    if op == "store":
        if rng.random() < 0.5:
            return _without_name(_store("", _log_uniform(rng, 1, 48), kv_heads * group, kv_heads, width, 1, _log_uniform(rng, 1, 60000)))
        most = 4093 * 56 * 128 // ((group + 2) * kv_heads * width)
        tokens = _log_uniform(rng, 2, max(3, min(4093, most)))
        chunk = rng.choice([0, 0, max(1, tokens // 2 + 1)])
        sequences = max(1, min(4, most // tokens))
        return _without_name(_store("", rng.randint(1, sequences), kv_heads * group, kv_heads, width, tokens, 0, chunk))
    window, sinks = rng.choice([(0, 0), (0, 0), (512, 4), (1024, 0), (4096, 64)])
    if rng.random() < 0.6:                                      # a decode step, or a few tokens at once
        tokens = rng.choice([1, 1, 1, 2, 5])
        before = _log_uniform(rng, 1, 131000)
        most = 32 * 8192 * 16 * 128 // (before * kv_heads * width)
        sequences = max(1, min(48, most))
        return _without_name(_attend("", rng.randint(1, sequences), kv_heads * group, kv_heads, width, tokens, before, window, sinks,
                                     rng.random() < 0.5))
    before = rng.choice([0, 0, _log_uniform(rng, 1, 30000)])   # a prompt, or a chunk behind a cached part
    tokens = _log_uniform(rng, 6, 4093)
    sequences = rng.choice([1, 1, 2]) if tokens < 1000 and before < 8000 else 1
    while sequences * kv_heads * group * width * tokens * (before + tokens // 2 + 1) > 40 * 128 * 4093 * 2047:
        tokens, before = max(6, tokens // 2), before // 2
    return _without_name(_attend("", sequences, kv_heads * group, kv_heads, width, tokens, before, window, sinks, rng.random() < 0.5))


def _without_name(case):
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """Tokens before the call and tokens of the call, for each sequence."""
    rng = np.random.default_rng([seed, 7])
    B, n, before = case["sequences"], case["tokens"], case["before"]
    if case["op"] == "store":
        start = rng.integers(before // 2, before + 1, B) if n == 1 else np.zeros(B, dtype=np.int64)
        return start.astype(np.int32), np.full(B, n, dtype=np.int32)
    if not case["ragged"]:
        return np.full(B, before, dtype=np.int32), np.full(B, n, dtype=np.int32)
    start = rng.integers(before // 2, before + 1, B)
    counts = rng.integers(max(1, n // 2), n + 1, B)
    counts[0] = n
    return start.astype(np.int32), counts.astype(np.int32)


def _visible(case, start, counts):
    """Pairs of a query token and a key it sees, and the keys that some query of the call sees, over all sequences."""
    pairs = keys = 0
    for s, c in zip(start.tolist(), counts.tolist()):
        p = np.arange(s, s + c)
        w = case["window"] or 1 << 40
        first = np.maximum(0, p - w + 1)
        pairs += int((p + 1 - first + np.minimum(first, case["sinks"])).sum())
        keys += int(s + c - first[0] + min(first[0], case["sinks"]))
    return pairs, keys


def _quantise(x):
    """[..., 64 tokens, width] -> codes (int8) and scales (FP32), one scale over the last two axes."""
    scale = (x.abs().amax((-2, -1)).double() / 127.0).float()
    codes = (x.double() / scale.double().clamp_min(1e-300)[..., None, None]).round().clamp(-127, 127)
    return codes.to(torch.int8), scale


def _rotate(x, start, inv_freq):
    """x [B, n, heads, width] at positions start[b] + i: halves (j, j + width / 2) turn by position * inv_freq[j]."""
    position = start[:, None].double() + torch.arange(x.shape[1], device=x.device)
    angle = position[..., None, None] * inv_freq.double()
    cos, sin = angle.cos(), angle.sin()
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).float()


def _inv_freq(width):
    return (10000.0 ** (-torch.arange(0, width, 2, dtype=torch.float64) / width)).float().cuda()


def _randn(seed, part, *shape):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed * 8 + part), device="cuda")


def _keys_values(seed, B, n, kv_heads, width):
    """Keys with channels of very different size, as projections give them, and values."""
    channel = (0.6 * _randn(seed, 3, kv_heads, width)).exp()
    return _randn(seed, 1, B, n, kv_heads, width) * channel, _randn(seed, 2, B, n, kv_heads, width)


def _store_inputs(case, seed):
    B, n, kv, D = case["sequences"], case["tokens"], case["kv_heads"], case["width"]
    start, _ = _lengths(case, seed)
    k, v = _keys_values(seed, B, n, kv, D)
    early = _keys_values(seed + (1 << 31), B, BLOCK - 1, kv, D)   # tokens of the open block that are there already
    return start, _randn(seed, 0, B, n, case["heads"], D), k, v, early


def _attend_inputs(case, seed):
    B, kv, D = case["sequences"], case["kv_heads"], case["width"]
    start, counts = _lengths(case, seed)
    k, v = _keys_values(seed, B, int((start + counts).max()), kv, D)
    total = torch.from_numpy(start + counts).cuda()
    there = (torch.arange(k.shape[1], device="cuda") < total[:, None])[..., None, None]
    q = _randn(seed, 0, B, case["tokens"], case["heads"], D) * 1.2
    return start, counts, q, k.mul_(there), v.mul_(there)


def _score_inputs(case, seed):
    logits = _randn(seed, 0, case["rows"], case["vocabulary"]) * case["spread"]
    targets = torch.randint(0, case["vocabulary"], (case["rows"],), dtype=torch.int32, device="cuda",
                            generator=torch.Generator("cuda").manual_seed(seed * 8 + 1))
    likely = torch.arange(case["rows"], device="cuda") % 2 == 0   # every other text token is one the model finds likely
    at = targets.long()[:, None]
    logits.scatter_add_(1, at, (likely * 4.0 * case["spread"])[:, None].float())
    return logits, targets


def _blocks(x):
    """[B, n, heads, width] -> [B, heads, blocks, 64, width], the last block filled up with zeros."""
    B, n, heads, width = x.shape
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, -n % BLOCK))
    return x.reshape(B, -1, BLOCK, heads, width).permute(0, 3, 1, 2, 4)


# ------------------------------------------------------------------------------------------------------------- states
def _own_lane():
    global _lane
    if _lane is None:
        import nntrain_amd as nn
        _lane = nn.HipExecutionLane(torch.cuda.current_device())
    return _lane


def _wrap(x):
    return _own_lane().wrap(x.data_ptr(), x.numel() * x.element_size())


def prepare(case, seed):
    if case["op"] == "score":
        logits, targets = _score_inputs(case, seed)
        state = {"case": case, "logits": logits, "targets": targets}
        if own:
            rows, top = case["rows"], case["top"]
            state["out"] = {"log_probs": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda")}
            if top:
                state["out"] |= {"top_ids": torch.empty(rows, top, dtype=torch.int32, device="cuda"),
                                 "top_log_probs": torch.empty(rows, top, device="cuda")}
            state["buffers"] = {k: _wrap(x) for k, x in state["out"].items()}
            state["in"] = _wrap(logits), _wrap(targets)
            torch.cuda.synchronize()
        return state
    B, n, H, kv, D = (case[k] for k in ("sequences", "tokens", "heads", "kv_heads", "width"))
    if case["op"] == "store":
        start, q, k, v, (ek, ev) = _store_inputs(case, seed)
        inv_freq = _inv_freq(D)
        starts = torch.from_numpy(start).cuda()
        state = {"case": case, "q": q, "k": k, "v": v, "inv_freq": inv_freq, "start": starts}
        if n == 1:      # what is kept of the open block's tokens: rotated keys and values
            there = (torch.arange(BLOCK - 1, device="cuda") < (starts % BLOCK)[:, None])[..., None, None]
            state["open"] = [torch.nn.functional.pad(x * there, (0, 0, 0, 0, 0, 1)) for x in (_rotate(ek, starts - starts % BLOCK, inv_freq), ev)]
        if own:
            import nntrain_amd as nn
            cache = state["cache"] = nn.QuantizedKvCache(_own_lane(), 1, B, kv, D, int(start.max()) + n)
            rotary = state["rotary"] = nn.Rotary(_wrap(inv_freq), D)
            first = (start // BLOCK * BLOCK).astype(np.int32) if n == 1 else np.zeros(B, dtype=np.int32)
            state["first"] = _own_lane().upload_raw(first)
            if n == 1:
                open_tokens = _own_lane().upload_raw((start - first).astype(np.int32))
                cache.set_lengths(first)
                torch.cuda.synchronize()
                cache.store(0, _wrap(ek), _wrap(ev), BLOCK - 1, counts=open_tokens, rotary=rotary)
            cache.set_lengths(start)
            m = BLOCK if n == 1 else n
            state["out"] = {"q": torch.empty_like(q), "k": torch.empty(B, m, kv, D, device="cuda"), "v": torch.empty(B, m, kv, D, device="cuda")}
            state["buffers"] = {name: _wrap(x) for name, x in {**state["out"], "q_in": q, "k_in": k, "v_in": v}.items()}
            _own_lane().synchronize()
            torch.cuda.synchronize()
        return state
    start, counts, q, k, v = _attend_inputs(case, seed)
    state = {"case": case, "q": q, "start": torch.from_numpy(start).cuda(), "counts": torch.from_numpy(counts).cuda()}
    if own:
        import nntrain_amd as nn
        cache = state["cache"] = nn.QuantizedKvCache(_own_lane(), 1, B, kv, D, k.shape[1])
        cache.set_lengths(np.zeros(B, dtype=np.int32))
        total = _own_lane().upload_raw((start + counts).astype(np.int32))
        torch.cuda.synchronize()
        cache.store(0, _wrap(k), _wrap(v), k.shape[1], counts=total)
        cache.set_lengths(start)
        state["out"] = torch.zeros_like(q)
        state["buffers"] = _wrap(q), _wrap(state["out"])
        state["count_buffer"] = _own_lane().upload_raw(counts)
        _own_lane().synchronize()
        torch.cuda.synchronize()
    else:
        state["k"], state["v"] = _quantise(_blocks(k)), _quantise(_blocks(v))
    return state


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_store(state):
    case, start, inv_freq = state["case"], state["start"], state["inv_freq"]
    q, k, v = _rotate(state["q"], start, inv_freq), _rotate(state["k"], start, inv_freq), state["v"]
    if case["tokens"] == 1:
        here = (torch.arange(BLOCK, device="cuda") == (start % BLOCK)[:, None])[..., None, None]
        k, v = torch.where(here, k, state["open"][0]), torch.where(here, v, state["open"][1])
    out = {"q": q}
    for name, x in (("k", k), ("v", v)):
        codes, scale = _quantise(_blocks(x))
        values = codes.float() * scale[..., None, None]
        out[name] = values.permute(0, 2, 3, 1, 4).reshape(x.shape[0], -1, *x.shape[2:])[:, :x.shape[1]].contiguous()
    return out


def _plain_attend(state):
    case, start, counts = state["case"], state["start"].long(), state["counts"].long()
    B, n, H, kv, D = (case[k] for k in ("sequences", "tokens", "heads", "kv_heads", "width"))
    k, v = ((codes.float() * scale[..., None, None]).flatten(2, 3) for codes, scale in (state["k"], state["v"]))
    q = state["q"].reshape(B, n, kv, H // kv, D).permute(0, 2, 1, 3, 4).reshape(B, kv, -1, D)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(D)).reshape(B, kv, n, H // kv, -1)
    p, t = start[:, None, None] + torch.arange(n, device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
    seen = t <= p
    if case["window"]:
        seen &= (t > p - case["window"]) | (t < case["sinks"])
    s = s.masked_fill_(~seen[:, None, :, None], -math.inf)
    e = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.reshape(B, kv, -1, k.shape[2]), v).reshape(B, kv, n, -1, D) / e.sum(-1, keepdim=True)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, H, D)
    return o * (torch.arange(n, device="cuda") < counts[:, None])[..., None, None]   # rows behind a sequence stay zero


def _plain_score(state):
    x, targets, top = state["logits"], state["targets"].long(), state["case"]["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(-1, dtype=torch.float64)
    log_total = total.log()
    out = {"log_probs": (d.gather(1, targets[:, None])[:, 0].double() - log_total).float(),
           "entropy": (log_total - (d * e).sum(-1, dtype=torch.float64) / total).float()}
    if top:
        value, index = torch.sort(x, dim=-1, descending=True, stable=True)   # (equal logits keep the order of their indexes)
        out["top_ids"] = index[:, :top].int()
        out["top_log_probs"] = ((value[:, :top] - m).double() - log_total[:, None]).float()
    return out


# ------------------------------------------------------------------------------------------------------------- the framework
def _own_store(state):
    case, cache, b = state["case"], state["cache"], state["buffers"]
    B, n, H, kv, D = (case[k] for k in ("sequences", "tokens", "heads", "kv_heads", "width"))
    import nntrain_amd as nn
    if n == 1 or not case["chunk"]:
        cache.store(0, b["k_in"], b["v_in"], n, q=b["q_in"], q_out=b["q"], heads=H, rotary=state["rotary"])
    else:
        cache.lane.fill_u32(cache.lengths, 0, B)
        for first in range(0, n, case["chunk"]):
            now = min(case["chunk"], n - first)
            part = lambda name, h: nn.Rows(b[name], h * D, n * h * D, first * h * D)  # noqa: E731
            cache.store(0, part("k_in", kv), part("v_in", kv), now, q=part("q_in", H), q_out=part("q", H), heads=H, rotary=state["rotary"])
            cache.advance(now)
    cache.read(0, BLOCK if n == 1 else n, first=state["first"], k_out=b["k"], v_out=b["v"])
    return state["out"]


def _own_attend(state):
    case, (q, out) = state["case"], state["buffers"]
    state["cache"].attention(0, q, case["heads"], case["tokens"], window=case["window"], sinks=case["sinks"],
                             counts=state["count_buffer"] if case["ragged"] else None, out=out)
    return state["out"]


def _own_score(state):
    from nntrain_amd import qwen35_gpu
    case, (logits, targets), b = state["case"], state["in"], state["buffers"]
    qwen35_gpu.token_log_probs(_own_lane(), logits, case["rows"], case["vocabulary"], targets, top=case["top"], out=b["log_probs"],
                               entropy=b["entropy"], top_ids=b.get("top_ids"), top_log_probs=b.get("top_log_probs"))
    return state["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "score": _own_score}[op](state)
    return {"store": _plain_store, "attend": _plain_attend, "score": _plain_score}[op](state)


# ------------------------------------------------------------------------------------------------------------- work, exact values
def work(case):
    if case["op"] == "score":
        rows, V, top = case["rows"], case["vocabulary"], case["top"]
        return {"bytes": 4.0 * rows * V + rows * (12 + 8 * top), "flops": 6.0 * rows * V}
    B, n, H, kv, D = (case[k] for k in ("sequences", "tokens", "heads", "kv_heads", "width"))
    if case["op"] == "store":
        back = BLOCK if n == 1 else n
        # queries in and out, keys and values in and as codes, codes and their values read back
        return {"bytes": float(B * D * (8 * H * n + 2 * kv * n * 5 + 2 * kv * back * 5)), "flops": float(B * n * D * (3 * H + 7 * kv))}
    start, counts = _lengths(case, 0)
    pairs, keys = _visible(case, start, counts)
    return {"bytes": float(2 * kv * D * keys + 8 * H * D * int(counts.sum())), "flops": 4.0 * H * D * pairs}


def _exact_rotation(x, start, inv_freq):
    width = x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(x.shape[0]):
        turn = torch.outer(torch.arange(x.shape[1], device=x.device).double() + float(start[b]), inv_freq.double())[:, None]
        z = torch.complex(x[b, ..., : width // 2].double(), x[b, ..., width // 2:].double()) * torch.polar(torch.ones_like(turn), turn)
        out[b] = torch.cat((z.real, z.imag), -1)
    return out


def _exact_values(x):
    """What 8 bits keep of x [64 tokens, heads, width] (64-bit values of FP32 numbers): one scale for each head."""
    step = (x.abs().amax((0, 2), keepdim=True) / 127).float().double()
    return torch.where(step > 0, torch.round(x / step.clamp_min(1e-300)).clamp(-127, 127) * step, torch.zeros_like(x))


def exact(case, seed):
    if case["op"] == "score":
        logits, targets = _score_inputs(case, seed)
        out = {"log_probs": [], "entropy": []} | ({"top_ids": [], "top_log_probs": []} if case["top"] else {})
        for r in range(case["rows"]):
            lp = torch.log_softmax(logits[r].double(), 0)
            out["log_probs"].append(lp[int(targets[r])])
            out["entropy"].append(-(lp.exp() * lp).sum())
            if case["top"]:
                value, index = torch.sort(logits[r], dim=-1, descending=True, stable=True)
                out["top_ids"].append(index[:case["top"]].int())
                out["top_log_probs"].append(lp[index[:case["top"]]])
        return {k: torch.stack(x) for k, x in out.items()}
    if case["op"] == "store":
        start, q, k, v, (ek, ev) = _store_inputs(case, seed)
        inv_freq = _inv_freq(case["width"])
        out = {"q": _exact_rotation(q, start, inv_freq)}
        k = _exact_rotation(k, start, inv_freq).float().double()
        early = {"k": _exact_rotation(ek, start // BLOCK * BLOCK, inv_freq).float().double(), "v": ev.double()}
        for name, x in (("k", k), ("v", v.double())):
            if case["tokens"] == 1:
                values = torch.zeros(x.shape[0], BLOCK, *x.shape[2:], dtype=torch.float64, device="cuda")
                for b in range(x.shape[0]):
                    n = int(start[b]) % BLOCK
                    values[b, :n + 1] = _exact_values(torch.cat((early[name][b, :n], x[b])))
            else:
                values = torch.empty_like(x)
                for b in range(x.shape[0]):
                    for t in range(0, x.shape[1], BLOCK):
                        values[b, t:t + BLOCK] = _exact_values(x[b, t:t + BLOCK])
            out[name] = values
        return out
    start, counts, q, k, v = _attend_inputs(case, seed)
    H, kv, D, n = case["heads"], case["kv_heads"], case["width"], case["tokens"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(q.shape[0]):
        total, c = int(start[b] + counts[b]), int(counts[b])
        kb, vb = (torch.cat([_exact_values(x[b, t:t + BLOCK].double()) for t in range(0, total, BLOCK)])[:total] for x in (k, v))
        p, t = torch.arange(c, device="cuda")[:, None] + int(start[b]), torch.arange(total, device="cuda")[None]
        hidden = t > p
        if case["window"]:
            hidden |= (t <= p - case["window"]) & (t >= case["sinks"])
        for h in range(H):
            s = (q[b, :c, h].double() @ kb[:, h * kv // H].t().contiguous()) / D ** 0.5
            out[b, :c, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vb[:, h * kv // H]
    return out
