"""Attention and what feeds it, as cases to time and compare.

Between the q|k|v projection and the output projection of a transformer layer
stand three operators. A case is one of three kinds:

  rope    the rotary embedding of the new tokens' queries and keys at their
          positions, and the write of keys and values into a paged cache
  prompt  causal attention over whole prompts, packed one after the other
  paged   attention of the new tokens of many sequences over their paged cache

Activations are fp32, as the projections leave them; a cache holds f32, f16 or
bf16. `heads` and `kv_heads` are those of queries and of keys; `new` lists how
many tokens each sequence brings, `length` how many it then has.
"""
import importlib
import math

import torch

own = False

GGML = {"f32": 0, "f16": 1, "bf16": 30}
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1e6


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def listed():
    def prompt(name, new, heads, kv_heads, dim):
        return {"name": name, "kind": "prompt", "new": _text(new), "heads": heads, "kv_heads": kv_heads, "dim": dim}

    def paged(name, new, length, heads, kv_heads, dim, cache, page):
        return {"name": name, "kind": "paged", "new": _text(new), "length": _text(length), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page}

    def rope(name, new, length, heads, kv_heads, dim, cache, page, interleaved):
        return {"name": name, "kind": "rope", "new": _text(new), "length": _text(length), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page, "interleaved": interleaved}

    many = [1 + (977 * i * i + 4001 * i) % 8191 for i in range(64)]
    return [
        # A short question to a model of 1.5 B weights: what counts is latency.
        prompt("prompt_1_5b_37", [37], 12, 2, 128),
        # Prompts of several users in one pass, 0.5 B, ragged down to one token.
        prompt("prompt_0_5b_packed", [1, 611, 17, 1024, 333, 64, 2, 450], 14, 2, 64),
        # A long document, 7 B.
        prompt("prompt_7b_8192", [8192], 28, 4, 128),
        # One session that decodes, 0.5 B: the smallest call of a decode loop.
        paged("decode_0_5b_x1_f16", [1], [777], 14, 2, 64, "f16", 16),
        # One session far into a long document, 7 B: few rows, a long axis.
        paged("decode_7b_x1_long_f16", [1], [32749], 28, 4, 128, "f16", 64),
        # Sixty-four sessions of all lengths that decode together, 7 B.
        paged("decode_7b_x64_f16", [1] * 64, many, 28, 4, 128, "f16", 64),
        # Eight sessions over a cache of full precision, 1.5 B; one of them idle.
        paged("decode_1_5b_x8_f32", [1, 1, 1, 1, 0, 1, 1, 1], [2048, 31, 1500, 4001, 0, 1, 96, 3333], 12, 2, 128, "f32", 32),
        # Prompts in the largest chunks that a projection call takes, beside
        # sessions that decode, 7 B.
        paged("chunk_7b_mixed_bf16", [32, 1, 32, 1, 1, 13], [4129, 900, 32, 2047, 6000, 7001], 28, 4, 128, "bf16", 16),
        # A later part of a long prompt in one large chunk, 7 B.
        paged("chunk_7b_512_f16", [512], [16100], 28, 4, 128, "f16", 128),
        # One token of each of sixty-four sessions, far positions, 7 B.
        rope("rope_decode_7b_x64", [1] * 64, [16 * n + 1 for n in many], 28, 4, 128, "f16", 64, False),
        # One token of one session, 0.5 B, pairs side by side.
        rope("rope_decode_0_5b_x1", [1], [778], 14, 2, 64, "f32", 16, True),
        # Whole prompts on their way into the cache, 7 B.
        rope("rope_prompt_7b", [2048, 1, 1500, 547], [2048, 4000, 1500, 1571], 28, 4, 128, "bf16", 64, False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["prompt", "prompt", "paged", "paged", "paged", "paged", "rope", "rope"])
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (28, 4, 128), (16, 16, 64), (8, 1, 128),
                                       (32, 8, 128), (15, 5, 96), (16, 4, 80), (20, 4, 40)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim}
    if kind == "prompt":
        longest = spread(1, 5000)
        return {**case, "new": _text([longest] + [rng.randint(1, longest) for _ in range(rng.randint(0, max(0, min(7, 6000 // longest - 1))))])}
    case |= {"cache": rng.choice(["f32", "f16", "f16", "bf16"]), "page": rng.choice([1, 8, 16, 16, 32, 48, 64, 128, 256])}
    if kind == "paged" and rng.random() < 0.5:
        count, longest = spread(1, 64), spread(16, 8000)
        lengths = [rng.randint(1, longest) for _ in range(count)]
        new = [0 if rng.random() < 0.05 else 1 for _ in lengths]
        new[0] = 1
        return {**case, "new": _text(new), "length": _text(lengths)}
    if kind == "paged":
        count, longest, most = spread(1, 6), spread(32, 12000), spread(2, 512)
    else:
        count, longest, most = spread(1, 64), spread(16, 100000), spread(1, 64)
    new = [rng.randint(1, most) for _ in range(count)]
    return {**case, "new": _text(new), "length": _text([n + rng.randint(0, longest) for n in new])} | (
        {"interleaved": rng.random() < 0.5} if kind == "rope" else {})


# ---- inputs --------------------------------------------------------------------------


def _generator(seed, *what):
    g = torch.Generator(device="cuda")
    number = int(seed) & 0x7FFFFFFF
    for w in what:
        number = (number * 1000003 + int(w) + 12345) & 0x7FFFFFFFFFFF
    g.manual_seed(number)
    return g


def _heads(tokens, heads, dim, g, wide):
    """Normal values, a few channels of each head far larger"""
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda")
    outlier = torch.rand(heads, dim, generator=g, device="cuda") < 0.03
    return torch.where(outlier, x * wide, x)


def _int(numbers):
    return torch.tensor(numbers, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    new, heads, kv_heads, dim = _numbers(case["new"]), case["heads"], case["kv_heads"], case["dim"]
    tokens, g = sum(new), _generator(seed, 1)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    state = {"case": case, "tokens": tokens, "starts": _int(starts), "longest_new": max(new),
             "q": _heads(tokens, heads, dim, g, 2.0), "out": torch.zeros(tokens, heads, dim, device="cuda")}
    if case["kind"] != "paged":
        state["k"] = _heads(tokens, kv_heads, dim, g, 3.0)
        state["v"] = torch.randn(tokens, kv_heads, dim, generator=g, device="cuda")
    if case["kind"] == "prompt":
        return state
    length, page, kind = _numbers(case["length"]), case["page"], TORCH[case["cache"]]
    state |= {"lengths": _int(length), "longest": max(length), "status": _int([1])}
    columns = max(1, -(-max(length) // page))
    # the pages that this call touches are the sequences' own, in any order;
    # of a write's earlier pages only the numbers matter
    first = [0 if case["kind"] == "paged" else (n - m) // page for n, m in zip(length, new)]
    touched = [max(0, -(-n // page) - f) for n, f in zip(length, first)]
    pages = sum(touched) + 1
    free = (torch.randperm(pages - 1, generator=_generator(seed, 2), device="cuda") + 1).int()
    state["table"] = torch.zeros(len(new), columns, dtype=torch.int32, device="cuda")
    for row, f, n in zip(state["table"], first, touched):
        row[f:f + n], free = free[:n], free[n:]
    if case["kind"] == "rope":
        state["keys"] = torch.zeros(pages, kv_heads, page, dim, device="cuda", dtype=kind)
        state["k_out"] = torch.zeros(tokens, kv_heads, dim, device="cuda")
        state["frequencies"] = THETA ** (-2 * torch.arange(dim // 2, device="cuda", dtype=torch.float64) / dim)
        state["values"] = torch.zeros_like(state["keys"])
    else:
        state["keys"] = _heads(pages * page, kv_heads, dim, g, 3.0).reshape(pages, page, kv_heads, dim).transpose(1, 2).to(kind).contiguous()
        state["values"] = torch.randn(pages, kv_heads, page, dim, generator=g, device="cuda").to(kind)
    return state


# ---- one pass ------------------------------------------------------------------------


def _own(state):
    qmv = importlib.import_module("my-inference-engine_amd")
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    heads, kv_heads, dim, tokens = case["heads"], case["kv_heads"], case["dim"], state["tokens"]
    if case["kind"] == "prompt":
        sequences = qmv.make_sequences(state["starts"].data_ptr(), state["starts"].numel() - 1)
        qmv.device_attention_prompt(state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(), tokens, heads, kv_heads,
                                    dim, 1 / math.sqrt(dim), sequences, state["out"].data_ptr(), stream)
        return state["out"]
    keys, values, table = state["keys"], state["values"], state["table"]
    sequences = qmv.make_sequences(state["starts"].data_ptr(), table.shape[0], state["lengths"].data_ptr(), table.data_ptr(), table.shape[1])
    cache = qmv.make_paged_cache(keys.data_ptr(), values.data_ptr(), GGML[case["cache"]], kv_heads, dim, case["page"], keys.shape[0])
    if case["kind"] == "paged":
        qmv.device_attention_paged(state["q"].data_ptr(), tokens, heads, 1 / math.sqrt(dim), sequences, cache, state["out"].data_ptr(),
                                   stream, d_status=state["status"].data_ptr())
        return state["out"], state["status"]
    qmv.device_rope_append(state["q"].data_ptr(), heads, state["k"].data_ptr(), state["v"].data_ptr(), kv_heads, dim, tokens,
                           state["frequencies"].data_ptr(), dim, sequences, state["out"].data_ptr(), state["k_out"].data_ptr(), cache,
                           interleaved=case["interleaved"], d_status=state["status"].data_ptr(), stream=stream)
    return state["out"], state["k_out"], keys, values, state["status"]


def _places(state):
    """Each token's sequence and its number among the sequence's new ones"""
    token = torch.arange(state["tokens"], device="cuda")
    sequence = torch.searchsorted(state["starts"].long(), token, right=True) - 1
    return sequence, token - state["starts"][sequence]


def _rotated(x, cos, sin, interleaved):
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _rope(state):
    case, page = state["case"], state["case"]["page"]
    sequence, number = _places(state)
    position = state["lengths"][sequence] - (state["starts"][sequence + 1] - state["starts"][sequence]) + number
    angle = position.double()[:, None] * state["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q = _rotated(state["q"], cos, sin, case["interleaved"])
    k = _rotated(state["k"], cos, sin, case["interleaved"])
    at = state["table"][sequence, position // page].long()
    state["keys"][at, :, position % page] = k.to(state["keys"].dtype)
    state["values"][at, :, position % page] = state["v"].to(state["values"].dtype)
    return q, k, state["keys"], state["values"], state["status"]


def _attention(q, k, v, seen):
    """q [S, Hk, G, n, D], k and v [S, Hk, L, D], seen [S, n, L]: softmax(q k^T / sqrt(D)) v where seen; zeros where nothing is"""
    s, hk, g, n, d = q.shape
    seen = seen[:, None, None]
    scores = torch.matmul(q.reshape(s, hk, g * n, d), k.transpose(2, 3).contiguous()).reshape(s, hk, g, n, -1)
    scores = (scores * (1 / math.sqrt(d))).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = weights.sum(-1, keepdim=True)
    o = torch.matmul(weights.reshape(s, hk, g * n, -1), v).reshape(s, hk, g, n, d)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _attend(state):
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    starts, sequence, number = state["starts"].long(), *_places(state)
    new = starts[1:] - starts[:-1]
    n = torch.arange(state["longest_new"], device="cuda")
    rows = torch.minimum(starts[:-1, None] + n, starts[1:, None] - 1).clamp_(min=0)
    q = state["q"][rows].reshape(len(new), len(n), kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    if case["kind"] == "prompt":
        length, j = new, n
        k, v = (state[x][rows].transpose(1, 2).contiguous() for x in ("k", "v"))
    else:
        length, j, page = state["lengths"].long(), torch.arange(state["longest"], device="cuda"), case["page"]
        at = state["table"].long()[:, j // page]
        k, v = (state[x][at, :, j % page].transpose(1, 2).float() for x in ("keys", "values"))
    seen = j <= (length - new)[:, None, None] + n[:, None]
    v = v.masked_fill((j >= length[:, None])[:, None, :, None], 0)
    o = _attention(q.contiguous(), k, v.contiguous(), seen)
    return o.permute(0, 3, 1, 2, 4)[sequence, number].reshape(state["tokens"], heads, dim)


def run(state):
    if own:
        return _own(state)
    if state["case"]["kind"] == "rope":
        return _rope(state)
    out = _attend(state)
    return out if state["case"]["kind"] == "prompt" else (out, state["status"])


# ---- what a pass cannot do without -------------------------------------------------------


def work(case):
    new, heads, kv_heads, dim = _numbers(case["new"]), case["heads"], case["kv_heads"], case["dim"]
    tokens = sum(new)
    if case["kind"] == "prompt":
        return {"bytes": 4 * tokens * 2 * (heads + kv_heads) * dim, "flops": 4 * dim * heads * sum(n * (n + 1) // 2 for n in new)}
    length, size = _numbers(case["length"]), SIZE[case["cache"]]
    if case["kind"] == "rope":
        return {"bytes": tokens * dim * (4 * (2 * heads + 3 * kv_heads) + 2 * size * kv_heads), "flops": 3 * tokens * dim * (heads + kv_heads)}
    seen = sum(m * n - m * (m - 1) // 2 for n, m in zip(length, new))
    return {"bytes": 8 * tokens * heads * dim + 2 * size * kv_heads * dim * sum(n for n, m in zip(length, new) if m),
            "flops": 4 * dim * heads * seen}


# ---- the same in 64 bits, one sequence and head after the other --------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    new, heads, kv_heads, dim = _numbers(case["new"]), case["heads"], case["kv_heads"], case["dim"]
    length = _numbers(case["length"]) if "length" in case else new
    page = case.get("page")
    if case["kind"] == "rope":
        # multiplication by exp(i angle) of the pairs as complex numbers
        interleaved, keys, values = case["interleaved"], state["keys"].double(), state["values"].double()
        position = torch.tensor([n - m + i for n, m in zip(length, new) for i in range(m)], dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), position[:, None, None] * state["frequencies"])

        def turned(x):
            x = x.double()
            pairs = x.unflatten(-1, (dim // 2, 2)) if interleaved else x.unflatten(-1, (2, dim // 2)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            return (y if interleaved else y.transpose(-1, -2)).flatten(-2)

        q, k = turned(state["q"]), turned(state["k"])
        table, t = state["table"].tolist(), 0
        for row, n, m in zip(table, length, new):
            for p in range(n - m, n):
                keys[row[p // page], :, p % page] = k[t]
                values[row[p // page], :, p % page] = state["v"][t].double()
                t += 1
        return q, k, keys, values, None
    out = torch.zeros(state["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    t = 0
    for s, (n, m) in enumerate(zip(length, new)):
        if m == 0:
            continue
        if case["kind"] == "paged":
            used = state["table"][s, :-(-n // page)].long()
        for h in range(heads):
            c = h // (heads // kv_heads)
            if case["kind"] == "prompt":
                k, v = state["k"][t:t + n, c].double(), state["v"][t:t + n, c].double()
            else:
                k, v = (state[x][used, c].reshape(-1, dim)[:n].double() for x in ("keys", "values"))
            for i in range(0, m, 2048):
                q = state["q"][t + i:t + min(m, i + 2048), h].double()
                last = n - m + i + torch.arange(len(q), device="cuda")
                scores = torch.mm(q, k.t()) / math.sqrt(dim)
                scores[torch.arange(n, device="cuda") > last[:, None]] = -math.inf
                out[t + i:t + i + len(q), h] = torch.mm(torch.softmax(scores, -1), v)
        t += m
    return out if case["kind"] == "prompt" else (out, None)
