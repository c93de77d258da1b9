"""Timed cases of the packed attention, the cached attention and the linears with low-rank adapters.

Each case runs an operator once, either through chess_transformer_b200.ops (`own`) or in its plain form: elementary
torch operations in fp32, rounded once at the end. `exact` computes the same from the definitions in fp64.

  packed  softmax(scale q k^T) v over sequences packed one behind the other, grouped heads, causal or not; with keys
          longer than the queries, the queries are a sequence's last tokens
  cached  the same for one query token a sequence over a cache [sequences, capacity, kv heads, width] with lengths
  linear  x W^T + bias + residual, plus (x down_a^T) up_a^T for each row's request's adapter a (fp16)
  int8    the same beside the int8 linear: x and W int8 with a scale a row, the adapters fp16
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one board's 70 tokens through Fry's 24 query and 12 key/value heads of 32: the smallest call
        {"name": "packed one board", "op": "packed", "sequences": 1, "longest": 70, "queries": 0, "ragged": False, "heads": 24, "kv_heads": 12,
         "width": 32, "causal": False, "dtype": "fp16"},
        # the leaf batch of 256 boards
        {"name": "packed 256 boards", "op": "packed", "sequences": 256, "longest": 70, "queries": 0, "ragged": False, "heads": 24, "kv_heads": 12,
         "width": 32, "causal": False, "dtype": "fp16"},
        # prompts of a serving batch, from empty ones to 2048 tokens
        {"name": "packed ragged prompts", "op": "packed", "sequences": 16, "longest": 2048, "queries": 0, "ragged": True, "heads": 32, "kv_heads": 8,
         "width": 128, "causal": True, "dtype": "bf16"},
        # one long prompt
        {"name": "packed long prompt", "op": "packed", "sequences": 1, "longest": 8192, "queries": 0, "ragged": False, "heads": 32, "kv_heads": 4,
         "width": 128, "causal": True, "dtype": "bf16"},
        # the next 512 tokens of prompts whose earlier keys are there already, the microbench configuration's 12 heads of 64
        {"name": "packed later chunk", "op": "packed", "sequences": 8, "longest": 4096, "queries": 512, "ragged": True, "heads": 12, "kv_heads": 12,
         "width": 64, "causal": True, "dtype": "fp16"},
        # one long conversation's next token
        {"name": "cached one long", "op": "cached", "sequences": 1, "capacity": 32768, "ragged": False, "heads": 32, "kv_heads": 4, "width": 128,
         "dtype": "bf16"},
        # a batch of short and middling ones
        {"name": "cached ragged", "op": "cached", "sequences": 64, "capacity": 2048, "ragged": True, "heads": 24, "kv_heads": 12, "width": 64,
         "dtype": "fp16"},
        # a full serving batch
        {"name": "cached full batch", "op": "cached", "sequences": 64, "capacity": 8192, "ragged": True, "heads": 32, "kv_heads": 8, "width": 128,
         "dtype": "bf16"},
        # the next token of 16 requests, each with an adapter of its own
        {"name": "linear one token each", "op": "linear", "requests": 16, "longest": 1, "adapters": 16, "rank": 16, "K": 2048, "N": 2048,
         "residual": False},
        # the prompts of 24 requests
        {"name": "linear prompts", "op": "linear", "requests": 24, "longest": 1024, "adapters": 12, "rank": 32, "K": 2048, "N": 2048, "residual": True},
        # the projection of 64 boards (dq 24: 1440 columns), a request a board, 8 adapters
        {"name": "int8 64 boards", "op": "int8", "requests": 64, "longest": 70, "adapters": 8, "rank": 16, "K": 768, "N": 1440, "residual": False},
        # the projection of 256 boards (dq 16: 1152 columns)
        {"name": "int8 256 boards", "op": "int8", "requests": 256, "longest": 70, "adapters": 32, "rank": 8, "K": 768, "N": 1152, "residual": True},
    ]


def _between(rng, low, high):
    """A whole number spread over the logarithm of its range."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "cached", "linear", "int8"])
    if op in ("packed", "cached"):
        kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8] if kv_heads <= 4 else [1, 2, 3, 4])
        width = rng.choice([8, 16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
        case = {"op": op, "heads": heads, "kv_heads": kv_heads, "width": width, "dtype": rng.choice(["fp16", "bf16"])}
        if op == "cached":
            capacity = _between(rng, 1, 16384)
            most = min(64, 64 * 8192 * 8 * 128 // (capacity * kv_heads * width))
            return {**case, "sequences": _between(rng, 1, most), "capacity": capacity, "ragged": rng.random() < 0.7}
        longest = _between(rng, 1, min(8192, math.isqrt(2 ** 30 // heads)))
        queries = 0 if rng.random() < 0.7 else _between(rng, 1, longest)
        # at most half the padded scores of the largest listed case, since here some see all of them
        most = max(1, min(256, 2 ** 30 // (heads * longest * (queries or longest)), 2 ** 28 // (kv_heads * width * longest)))
        return {**case, "sequences": _between(rng, 1, most), "longest": longest, "queries": queries, "ragged": rng.random() < 0.7,
                "causal": rng.random() < 0.7}
    requests, longest = _between(rng, 1, 96), rng.choice([1, 1, 70, _between(rng, 1, 1000)])
    K, N = 16 * _between(rng, 4, 128), 8 * _between(rng, 2, 256)
    return {"op": op, "requests": min(requests, max(1, 24576 // longest)), "longest": longest, "adapters": _between(rng, 1, 48),
            "rank": rng.choice([8, 16, 24, 32, 64]), "K": K, "N": N, "residual": rng.random() < 0.5}


def _lengths(count, longest, ragged, least, salt):
    """The case's own lengths: all alike, or spread over their logarithm, the longest first and an empty one (or `least`) second."""
    if not ragged:
        return [longest] * count
    rng = random.Random(f"{count} {longest} {salt}")
    return [longest if i == 0 else least if i == 1 else max(least, _between(rng, 1, longest)) for i in range(count)]


def _packed_lengths(case):
    keys = _lengths(case["sequences"], case["longest"], case["ragged"], case["queries"], "packed")
    return [case["queries"] or n for n in keys], keys


def _cached_lengths(case):
    # a full batch's contexts are mostly long: half the capacity and up, one of them empty
    full = _lengths(case["sequences"], case["capacity"], case["ragged"], 0, "cached")
    return [n if i < 2 or not case["ragged"] or i % 4 == 0 else max(n, case["capacity"] // 2 + (n * 7 + i) % (case["capacity"] // 2 + 1))
            for i, n in enumerate(full)]


def _request_lengths(case):
    return _lengths(case["requests"], case["longest"], case["longest"] not in (1, 70), 0, "requests")


def _offsets(lengths, device):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device=device, dtype=dtype)  # noqa: E731
    state = dict(case)
    if case["op"] == "packed":
        dtype = DTYPES[case["dtype"]]
        queries, keys = _packed_lengths(case)
        state |= {"q": normal(sum(queries), case["heads"], case["width"], dtype=dtype), "k": normal(sum(keys), case["kv_heads"], case["width"], dtype=dtype),
                  "v": normal(sum(keys), case["kv_heads"], case["width"], dtype=dtype), "q_offsets": _offsets(queries, device),
                  "k_offsets": _offsets(keys, device), "max_q": max(queries), "max_k": max(keys)}
    elif case["op"] == "cached":
        dtype = DTYPES[case["dtype"]]
        cache = (case["sequences"], case["capacity"], case["kv_heads"], case["width"])
        state |= {"q": normal(case["sequences"], case["heads"], case["width"], dtype=dtype), "k": normal(*cache, dtype=dtype),
                  "v": normal(*cache, dtype=dtype), "lengths": torch.tensor(_cached_lengths(case), dtype=torch.int32, device=device)}
    else:
        K, N, A, R = case["K"], case["N"], case["adapters"], case["rank"]
        lengths = _request_lengths(case)
        M = sum(lengths)
        rng = random.Random(seed)
        # a request in sixteen has no adapter
        ids = [-1 if i % 16 == 15 else rng.randrange(A) for i in range(case["requests"])]
        half = lambda t: t.to(torch.float16)  # noqa: E731
        state |= {"offsets": _offsets(lengths, device), "ids": torch.tensor(ids, dtype=torch.int32, device=device),
                  "down": half(normal(A, R, K) / math.sqrt(K)), "up": half(normal(A, N, R) * (0.25 / math.sqrt(R))), "bias": half(normal(N) * 0.02),
                  "added": half(normal(M, N)) if case["residual"] else None}
        if case["op"] == "linear":
            state |= {"x": half(normal(M, K)), "weight": half(normal(N, K) / math.sqrt(K))}
        else:  # normed rows and N(0, 1/K) weights, both quantised by the row's largest value
            for name, real in (("x", normal(M, K)), ("weight", normal(N, K) / math.sqrt(K))):
                scale = (real.abs().amax(1) / 127).clamp(min=1e-20)
                state |= {name: (real / scale[:, None]).round().to(torch.int8), name + "_scale": scale}
    return state


def _softmax_product(scores, seen, v):
    """Rows of softmax(scores, where seen) v; a row that sees nothing is 0."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total == 0, 1.0, total)


def _plain_packed(s):
    q, k, v, q_offsets, k_offsets = s["q"], s["k"], s["v"], s["q_offsets"].long(), s["k_offsets"].long()
    S, H, KV, D, mq, mk = s["sequences"], s["heads"], s["kv_heads"], s["width"], s["max_q"], s["max_k"]
    i, j = torch.arange(mq, device=q.device), torch.arange(mk, device=q.device)
    nq, nk = q_offsets.diff()[:, None], k_offsets.diff()[:, None]
    rows = torch.where(i < nq, q_offsets[:-1, None] + i, q.shape[0])  # padded places take the row behind the last one
    columns = torch.where(j < nk, k_offsets[:-1, None] + j, k.shape[0])
    pad = lambda t: torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, 1))  # noqa: E731
    wide_q = pad(q)[rows].view(S, mq, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(S, KV, H // KV * mq, D)
    wide_k, wide_v = pad(k)[columns].transpose(1, 2), pad(v)[columns].transpose(1, 2)
    scores = (wide_q @ wide_k.transpose(2, 3)).view(S, KV, H // KV, mq, mk) * (1 / math.sqrt(D))
    seen = (j < nk)[:, None, :].expand(S, mq, mk)
    if s["causal"]:
        seen = seen & (j <= (i[None, :] + nk - nq)[:, :, None])
    out = _softmax_product(scores, seen[:, None, None], wide_v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(S, mq, H, D)
    packed = torch.zeros(q.shape[0] + 1, H, D, device=q.device, dtype=q.dtype)
    packed[rows] = out.to(q.dtype)
    return packed[:-1]


def _plain_cached(s):
    q, k, v = s["q"].float(), s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    S, H, KV, D = s["sequences"], s["heads"], s["kv_heads"], s["width"]
    scores = (q.view(S, KV, H // KV, D) @ k.transpose(2, 3)) * (1 / math.sqrt(D))
    seen = torch.arange(s["capacity"], device=q.device) < s["lengths"][:, None]
    return _softmax_product(scores, seen[:, None, None], v).view(S, H, D).to(s["q"].dtype)


def _plain_linear(s):
    x, A, R, N = s["x"].float(), s["adapters"], s["rank"], s["N"]
    out = x @ s["weight"].float().T
    if s["op"] == "int8":
        out = out * s["x_scale"][:, None] * s["weight_scale"]
        x = x * s["x_scale"][:, None]
    out = out + s["bias"].float()
    request = torch.searchsorted(s["offsets"][1:], torch.arange(x.shape[0], device=x.device, dtype=torch.int32), right=True)
    mine = s["ids"][request][:, None] == torch.arange(A, device=x.device)
    low = (x @ s["down"].float().view(A * R, -1).T).view(-1, A, R) * mine[:, :, None]
    out = out + low.view(-1, A * R) @ s["up"].float().transpose(1, 2).reshape(A * R, N)
    if s["added"] is not None:
        out = out + s["added"].float()
    return out.half()


def run(state):
    s = state
    if own:
        from chess_transformer_b200 import ops
        if s["op"] == "packed":
            return ops.packed_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["causal"])
        if s["op"] == "cached":
            return ops.cached_attention(s["q"], s["k"], s["v"], s["lengths"])
        if s["op"] == "linear":
            return ops.adapter_linear(s["x"], s["weight"], s["bias"], s["added"], s["down"], s["up"], s["offsets"], s["ids"])
        return ops.int8_adapter_linear(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], s["added"], s["down"], s["up"], s["offsets"],
                                       s["ids"])
    return {"packed": _plain_packed, "cached": _plain_cached}.get(s["op"], _plain_linear)(s)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "int8"):
        x, weight = s["x"].double(), s["weight"].double()
        if case["op"] == "int8":
            x, weight = x * s["x_scale"].double()[:, None], weight * s["weight_scale"].double()[:, None]
        out = x @ weight.T + s["bias"].double()
        first = 0
        for length, a in zip(_request_lengths(case), s["ids"].tolist()):
            if a >= 0:
                out[first:first + length] += (x[first:first + length] @ s["down"][a].double().T) @ s["up"][a].double().T
            first += length
        return out if s["added"] is None else out + s["added"].double()
    group, scale = case["heads"] // case["kv_heads"], case["width"] ** -0.5
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "cached":
        queries, keys = [1] * case["sequences"], _cached_lengths(case)
    else:
        queries, keys = _packed_lengths(case)
    q0 = k0 = 0
    for n, (nq, nk) in enumerate(zip(queries, keys)):
        k, v = (t[n, :nk] if case["op"] == "cached" else t[k0:k0 + nk] for t in (s["k"], s["v"]))
        for h in range(case["kv_heads"]):
            key, value = k[:, h].double(), v[:, h].double()
            for head in range(h * group, (h + 1) * group):
                scores = s["q"][q0:q0 + nq, head].double() @ key.T * scale
                if case.get("causal"):
                    scores += torch.full((nq, nk), -math.inf, dtype=torch.float64, device="cuda").triu(1 + nk - nq)
                if nk:
                    out[q0:q0 + nq, head] = torch.softmax(scores, -1) @ value
        q0, k0 = q0 + nq, k0 + nk
    return out


def work(case):
    if case["op"] in ("linear", "int8"):
        M, K, N, A, R = sum(_request_lengths(case)), case["K"], case["N"], case["adapters"], case["rank"]
        element = 2 if case["op"] == "linear" else 1
        read = element * (M * K + N * K) + 2 * min(A, case["requests"]) * R * (K + N) + 2 * N + (2 * M * N if case["residual"] else 0)
        scales = 0 if case["op"] == "linear" else 4 * (M + N)
        return {"bytes": read + scales + 2 * M * N, "flops": 2 * M * K * N + 2 * M * R * (K + N)}
    H, KV, D = case["heads"], case["kv_heads"], case["width"]
    if case["op"] == "cached":
        keys, queries = sum(_cached_lengths(case)), case["sequences"]
        pairs = keys
    else:
        nq, nk = _packed_lengths(case)
        keys, queries = sum(nk), sum(nq)
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(nq, nk))
    return {"bytes": 2 * D * (2 * KV * keys + 2 * H * queries), "flops": 4 * D * H * pairs}
