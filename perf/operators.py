"""Workloads of the operators between a decoder layer's projections, and their plain forms.

A case is one call that a serving process makes in every decoder layer:

* ``rotary``  `rotary_positions`: queries and keys, views of the projections' output, are turned by
              their tokens' positions;
* ``append``  `kv4_append`: the new tokens' keys are turned on the way and laid with the values into
              the pages of a 4-bit cache, and their queries are turned; `kv4_read` then reads the
              tokens back, as a program does that shares a prefix or moves it to another cache;
* ``attend``  `kv4_attention`: attention of the new tokens' queries over their sequences' pages.

Head counts are those of the shipped weave tables' models (8 query heads and 1 key head on one of
eight ranks, 6 and 1, 16 and 2 on one of four, 64 and 8 whole) and generic ones.

A page holds `page` tokens of every key head, 4 bits a value (the eight magnitudes 0, 0.5, 1, 1.5, 2,
3, 4, 6 and a sign) with one power of two for 32 channels.  Of one head, in bytes:
    keys    [page][D / 2]             low nibble first
    values  [page / 4][16][4][D / 32] four tokens side by side for each sixteenth of the channels
    scales of the keys, then of the values: [D / 32][page], exponent + 127, 255: not a number
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = ((8, 1), (8, 1), (6, 1), (16, 2), (64, 8), (48, 8), (32, 8), (28, 4), (12, 12))
BASE = 500000.0
MOST_TURNED = 16384 * 72 * 128       # values of the largest listed rotary
MOST_APPENDED = 8192 * 80 * 128      # values of the largest listed append
MOST_CACHED = 256 * 4096 * 8 * 128   # values of the largest listed cache
MOST_SCORES = 8192 * 8192 * 8        # scores of the largest listed prompt


def listed():
    return [
        # 64 sequences decoding on one of eight ranks: one new token each
        {"name": "rotary_decode", "op": "rotary", "tokens": 64, "q_heads": 8, "kv_heads": 1, "D": 128, "turned": 128,
         "interleaved": False, "scaling": "none", "dtype": "bf16"},
        # a long prompt, all heads on this GPU, frequencies stretched for long contexts
        {"name": "rotary_prompt", "op": "rotary", "tokens": 16384, "q_heads": 64, "kv_heads": 8, "D": 128,
         "turned": 128, "interleaved": False, "scaling": "bands", "dtype": "bf16"},
        # full precision, odd count of tokens, neighbouring channels turned together, a third of each head
        {"name": "rotary_partial", "op": "rotary", "tokens": 1001, "q_heads": 12, "kv_heads": 12, "D": 96, "turned": 32,
         "interleaved": True, "scaling": "linear", "dtype": "fp32"},
        # 64 sequences decoding: their tokens go to the end of their pages
        {"name": "append_decode", "op": "append", "tokens": 64, "q_heads": 8, "kv_heads": 1, "D": 128, "turned": 128,
         "interleaved": False, "scaling": "none", "dtype": "bf16", "page": 64, "padded": 0},
        # a prompt of 8192 tokens, all heads on this GPU
        {"name": "append_prompt", "op": "append", "tokens": 8192, "q_heads": 64, "kv_heads": 8, "D": 128, "turned": 128,
         "interleaved": False, "scaling": "bands", "dtype": "bf16", "page": 64, "padded": 0},
        # a ragged fp16 step padded to the captured graph's size, heads of 64 turned by half
        {"name": "append_padded", "op": "append", "tokens": 1003, "q_heads": 28, "kv_heads": 4, "D": 64, "turned": 32,
         "interleaved": True, "scaling": "none", "dtype": "fp16", "page": 16, "padded": 117},
        # one user's short chat: the time of a call counts
        {"name": "attend_one_short", "op": "attend", "seqs": 1, "context": 700, "queries": 1, "q_heads": 8,
         "kv_heads": 1, "D": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
        # 64 sequences of ragged lengths decoding on one of eight ranks
        {"name": "attend_decode", "op": "attend", "seqs": 64, "context": 8192, "queries": 1, "q_heads": 8,
         "kv_heads": 1, "D": 128, "page": 64, "ragged": True, "window": 0, "dtype": "bf16"},
        # one very long document
        {"name": "attend_one_long", "op": "attend", "seqs": 1, "context": 131071, "queries": 1, "q_heads": 8,
         "kv_heads": 1, "D": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
        # a full batch decoding, all heads on this GPU
        {"name": "attend_decode_all", "op": "attend", "seqs": 256, "context": 4096, "queries": 1, "q_heads": 64,
         "kv_heads": 8, "D": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
        # four drafted tokens verified at once behind a sliding window, six heads to a key head, fp16
        {"name": "attend_drafted", "op": "attend", "seqs": 37, "context": 6000, "queries": 4, "q_heads": 6,
         "kv_heads": 1, "D": 128, "page": 16, "ragged": True, "window": 4096, "dtype": "fp16"},
        # a prompt's own attention, causal
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "context": 8192, "queries": 8192, "q_heads": 8,
         "kv_heads": 1, "D": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    """Spread over the logarithm; a third of the larger values are rounded to a multiple of 16."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n > 64 and rng.random() < 0.33:
        n = (n + 15) // 16 * 16
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(("rotary", "append", "attend", "attend", "attend"))
    q_heads, kv_heads = rng.choice(HEADS)
    if op != "attend":
        D = rng.choice((128, 128, 64, 96, 80, 256) if op == "rotary" else (128, 128, 64, 256))
        case = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "D": D, "turned": rng.choice((D, D, D // 2, 32)),
                "interleaved": rng.random() < 0.4, "scaling": rng.choice(("none", "linear", "bands", "yarn")),
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
        if op == "rotary":
            most = MOST_TURNED * 2 // ((q_heads + kv_heads) * D * DTYPES[case["dtype"]].itemsize)
            return dict(case, tokens=min(_log_int(rng, 1, 16384), most))
        most = MOST_APPENDED * 2 // ((q_heads + 2 * kv_heads) * D * DTYPES[case["dtype"]].itemsize)
        tokens = min(_log_int(rng, 1, 8192), most)
        return dict(case, tokens=tokens, page=rng.choice((16, 32, 64, 128)),
                    padded=rng.randint(0, tokens // 2) if rng.random() < 0.4 else 0)
    D = rng.choice((128, 128, 128, 64, 256))
    kind = rng.choice(("decode", "decode", "drafted", "chunk"))
    seqs = _log_int(rng, 1, 256 if kind == "decode" else 64 if kind == "drafted" else 8)
    context = min(_log_int(rng, 16, 131072), max(16, MOST_CACHED // (seqs * kv_heads * D)))
    queries = {"decode": 1, "drafted": rng.randint(2, 8), "chunk": _log_int(rng, 16, 8192)}[kind]
    queries = max(1, min(queries, context, MOST_SCORES // (seqs * context * q_heads)))
    return {"op": op, "seqs": seqs, "context": context, "queries": queries, "q_heads": q_heads, "kv_heads": kv_heads,
            "D": D, "page": rng.choice((16, 32, 64, 128)), "ragged": rng.random() < 0.6,
            "window": _log_int(rng, 8, context) if rng.random() < 0.25 else 0, "dtype": rng.choice(("bf16", "bf16", "fp16"))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _table(case, length):
    """cos and sin of the positions, [length, turned] in fp32 from 64 bits: what a model keeps."""
    inv, factor = _frequencies(case)
    angle = torch.arange(length, dtype=torch.float64, device=DEV)[:, None] * inv
    return (torch.cat((angle.cos(), angle.sin()), 1) * factor).float()


def _frequencies(case):
    """Radians a position for each pair of channels, and what cos and sin are multiplied by."""
    n = case["turned"] // 2
    inv = BASE ** (-torch.arange(n, dtype=torch.float64, device=DEV) / n)
    kind = case["scaling"]
    if kind == "linear":
        return inv / 4.0, 1.0
    if kind == "bands":     # long waves are stretched by 8, short ones kept, a slope between
        turns = 8192 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * keep + inv / 8.0 * (1 - keep), 1.0
    if kind == "yarn":      # the slope runs over the pairs' numbers, cos and sin are enlarged
        at = lambda t: n * math.log(4096 / (t * 2 * math.pi)) / math.log(BASE)  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), 2 * n - 1)
        keep = 1 - ((torch.arange(n, dtype=torch.float64, device=DEV) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return inv * keep + inv / 16.0 * (1 - keep), 0.1 * math.log(16.0) + 1.0
    return inv, 1.0


def _lengths(case):
    """Cached tokens of each sequence, its new ones among them, and its new ones: by the case alone."""
    n, q, r = case["context"], case["queries"], random.Random(case["context"] * 1009 + case["seqs"])
    if not case["ragged"]:
        return [n] * case["seqs"], [q] * case["seqs"]
    lengths = [max(1, round(n * r.random() ** 1.5)) for _ in range(case["seqs"] - 1)] + [n]
    return lengths, [min(length, max(1, round(q * r.uniform(0.3, 1.0)))) for length in lengths]


def _page_bytes(case):
    return case["page"] * (case["D"] + case["D"] // 16)


def _slots(tokens, pages, page, g):
    """Places of consecutive tokens in pages taken in any order."""
    order = torch.randperm(pages, generator=g, device=DEV)
    at = torch.arange(tokens, device=DEV)
    return order[at // page] * page + at % page


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, D, Hq, Hk = DTYPES[case["dtype"]], case["D"], case["q_heads"], case["kv_heads"]
    state = {"case": case}
    if case["op"] != "attend":
        T = case["tokens"]
        # what the projections wrote: queries, keys and values of a token side by side
        qkv = _normal((T, (Hq + 2 * Hk) * D), g, dtype)
        state["q"], state["k"], state["v"] = (x.view(T, -1, D) for x in qkv.split((Hq * D, Hk * D, Hk * D), 1))
        state["table"] = _table(case, 32768)
        state["positions"] = torch.randint(0, 32768, (T,), generator=g, device=DEV) if T <= 256 else \
            torch.arange(T, device=DEV) + int(torch.randint(0, 32768 - T + 1, (1,), generator=g, device=DEV))
        state["q_out"] = torch.empty((T, Hq, D), dtype=dtype, device=DEV)
        state["k_out"] = torch.empty((T, Hk, D), dtype=dtype, device=DEV)
        if case["op"] == "append":
            pages = -(-T // case["page"]) + 3
            state["slots"] = _slots(T, pages, case["page"], g)
            if case["padded"]:
                state["slots"][T - case["padded"]:] = -1
            # memory as the allocator gave it
            state["pages"] = torch.randint(0, 256, (pages, Hk, _page_bytes(case)), generator=g, device=DEV, dtype=torch.uint8)
            state["v_out"] = torch.empty((T, Hk, D), dtype=dtype, device=DEV)
        return state
    lengths, news = _lengths(case)
    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    width = max(counts)
    # pages are taken in any order; places of the table behind a sequence's end hold nothing
    order = torch.randperm(sum(counts) + 5, generator=g, device=DEV, dtype=torch.int64).int()
    inside = torch.arange(width, device=DEV)[None, :] < torch.tensor(counts, device=DEV)[:, None]
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
    table[inside] = order[:sum(counts)]
    channels = 0.5 + 1.5 * torch.rand(D, generator=g, device=DEV) ** 2    # some channels of the keys are larger
    pages = torch.empty((sum(counts) + 5, Hk, _page_bytes(case)), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (Hk * page * D))
    for first in range(0, len(pages), step):
        n = min(step, len(pages) - first)
        k, v = _normal((n, Hk, page, D), g) * channels, _normal((n, Hk, page, D), g)
        pages[first:first + n] = _page_of(k, v)
    # what lies behind the sequences' ends was never written
    ends = torch.tensor(lengths, device=DEV)[:, None] - torch.arange(width, device=DEV)[None, :] * page
    behind = torch.arange(page, device=DEV) >= ends[inside][:, None]
    scales = pages[:, :, -(D // 16) * page:].view(len(pages), Hk, -1, page)
    at = order[:sum(counts)].long()
    scales[at] = torch.where(behind[:, None, None, :], torch.full_like(scales[at], 255), scales[at])
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    qkv = _normal((starts[-1], (Hq + 2 * Hk) * D), g, dtype)
    state.update(q=qkv[:, :Hq * D].view(-1, Hq, D), pages=pages, table=table, scale=D ** -0.5, most=max(news),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                 starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                 out=torch.empty((starts[-1], Hq, D), dtype=dtype, device=DEV))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from tokenweave_amd import ops
    case = state["case"]
    if case["op"] == "attend":
        ops.kv4_attention(state["out"], state["q"], state["pages"], state["table"], state["lengths"], state["scale"],
                          state["starts"], state["most"], case["window"])
        return state["out"]
    if case["op"] == "rotary":
        ops.rotary_positions(state["q"], state["k"], state["positions"], state["table"], case["interleaved"],
                             q_out=state["q_out"], k_out=state["k_out"])
        return state["q_out"], state["k_out"]
    ops.kv4_append(state["pages"], state["k"], state["v"], state["slots"], state["positions"], state["table"],
                   case["interleaved"], q=state["q"], q_out=state["q_out"])
    ops.kv4_read(state["k_out"], state["v_out"], state["pages"], state["slots"])
    return state["q_out"], state["k_out"], state["v_out"]


def _run_plain(state):
    case = state["case"]
    if case["op"] == "attend":
        return _attend(state)
    q, k = (_turned(state[x], state) for x in "qk")
    if case["op"] == "rotary":
        return q, k
    _append(state["pages"], k, state["v"], state["slots"], case["page"])
    return (q, *_read(state, k.dtype))


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _turned(x, state):
    """y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin for each pair of the turned channels."""
    case, n = state["case"], state["case"]["turned"]
    cos, sin = state["table"][state["positions"]][:, None, :].chunk(2, -1)
    f = x.float()
    y = f.clone()
    pairs = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    x1, x2 = f[..., pairs[0]], f[..., pairs[1]]
    y[..., pairs[0]] = x1 * cos - x2 * sin
    y[..., pairs[1]] = x2 * cos + x1 * sin
    return y.to(x.dtype)


def _encode(x):
    """Codes [..., D] and scale bytes [..., D / 32] of fp32 values: a block's power of two is the
    smallest that keeps its largest magnitude within 7, in [-23, 13]; ties go to the even code."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    most = x.abs().amax(-1)
    e = (((most.view(torch.int32) + 0x1FFFFF) >> 23) - 129).clamp(-23, 13)
    a = x.abs() * ((127 - e) << 23).view(torch.float32)[..., None]
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    code = code + 8 * torch.signbit(x).byte()
    return code.flatten(-2), torch.where(most.isfinite(), e + 127, torch.full_like(e, 255)).byte()


def _bytes(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _page_of(k, v):
    """Bytes of pages from their keys and values [n, heads, page, D]."""
    n, H, P, D = k.shape
    (kc, ks), (vc, vs) = _encode(k), _encode(v)
    values = _bytes(vc).view(n, H, P // 4, 4, 16, D // 32).transpose(3, 4)
    return torch.cat((_bytes(kc).flatten(2), values.flatten(2), ks.transpose(2, 3).flatten(2),
                      vs.transpose(2, 3).flatten(2)), 2)


def _places(slots, H, P, D):
    """Offsets of a slot's bytes in the pages: keys and values [T, H, D / 2], scales [T, H, D / 32]."""
    dev = slots.device
    base = (slots // P)[:, None, None] * H + torch.arange(H, device=dev)[None, :, None]
    base, t = base * (P * (D + D // 16)), (slots % P)[:, None, None]
    i, group = torch.arange(D // 2, device=dev), torch.arange(D // 32, device=dev)
    w = D // 32
    keys = base + t * (D // 2) + i
    values = base + P * D // 2 + t // 4 * (2 * D) + i // w * (4 * w) + t % 4 * w + i % w
    return keys, values, base + P * D + group * P + t, base + P * D + w * P + group * P + t


def _append(pages, k, v, slots, page):
    live = slots >= 0
    H, D = k.shape[1:]
    keys, values, ks, vs = _places(slots[live], H, page, D)
    flat = pages.view(-1)
    code, scale = _encode(k[live].float())
    flat[keys], flat[ks] = _bytes(code), scale
    code, scale = _encode(v[live].float())
    flat[values], flat[vs] = _bytes(code), scale


def _values(codes, scales):
    """fp32 values of code bytes [..., D / 2] and scale bytes [..., D / 32]."""
    half = torch.tensor((0, 0.5, 1, 1.5, 2, 3, 4, 6), device=codes.device)
    nibble = torch.cat((half, -half))
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack((nibble[byte & 15], nibble[byte >> 4]), 1)
    s = (scales.int() << 23).view(torch.float32)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (pairs[codes.int()].flatten(-2).unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _read(state, dtype):
    """Keys and values of the slots; zeros for a slot below zero."""
    slots, (T, H, D) = state["slots"], state["k"].shape
    live = slots >= 0
    keys, values, ks, vs = _places(slots.clamp(min=0), H, state["case"]["page"], D)
    flat = state["pages"].view(-1)
    found = [torch.where(live[:, None, None], _values(flat[c], flat[s]), torch.zeros((), device=flat.device))
             for c, s in ((keys, ks), (values, vs))]
    return [x.to(dtype) for x in found]


def _attend(state):
    """softmax(scale q k^T) v for every query head over the tokens that a query may see: those of its
    sequence up to itself, and of them the last `window` where there is one."""
    case, q, table = state["case"], state["q"], state["table"]
    B, Hq, Hk, D, P = case["seqs"], case["q_heads"], case["kv_heads"], case["D"], case["page"]
    G, mq, L = Hq // Hk, state["most"], state["table"].shape[1] * P
    lengths, first = state["lengths"].long(), state["starts"][:-1].long()
    news = state["starts"][1:].long() - first
    taken = state["pages"][table.clamp(min=0).long()].transpose(1, 2)           # [B, Hk, pages, bytes]
    codes, scales = taken[..., :P * D], taken[..., P * D:].unflatten(-1, (2, D // 32, P))
    keys = _values(codes[..., :P * D // 2].unflatten(-1, (P, D // 2)), scales[..., 0, :, :].transpose(-1, -2))
    rows = torch.arange(mq, device=q.device)
    live = rows[None, :] < news[:, None]
    at = torch.where(live, first[:, None] + rows, 0)                            # [B, mq]
    x = q[at].float().unflatten(2, (Hk, G)).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * mq, D)
    s = x @ keys.reshape(B, Hk, L, D).transpose(2, 3) * state["scale"]
    del keys
    t = torch.arange(L, device=q.device)
    last = lengths[:, None] - news[:, None] + rows                              # position of each query
    sees = (t <= last[..., None]) & live[..., None]
    if case["window"]:
        sees &= t > last[..., None] - case["window"]
    sees = sees[:, None, None]
    s = torch.where(sees, s.view(B, Hk, G, mq, L), torch.full((), -math.inf, device=q.device))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    values = codes[..., P * D // 2:].unflatten(-1, (P // 4, 16, 4, D // 32)).transpose(-2, -3)
    values = _values(values.reshape(B, Hk, -1, P, D // 2), scales[..., 1, :, :].transpose(-1, -2)).reshape(B, Hk, L, D)
    values = torch.where((t < lengths[:, None])[:, None, :, None], values, torch.zeros((), device=q.device))
    o = (p.view(B, Hk, G * mq, L) @ values).view(B, Hk, G, mq, D) / torch.where(total > 0, total, 1.0)
    out = torch.zeros_like(state["out"])
    out[at[live]] = o.permute(0, 3, 1, 2, 4).reshape(B, mq, Hq, D)[live].to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(state)
    out = [_exact_turned(state[x], state) for x in "qk"]
    if case["op"] == "rotary":
        return tuple(out)
    slots, dtype = state["slots"].tolist(), state["k"].dtype
    live = torch.tensor([s >= 0 for s in slots], device=DEV)
    # what the keys' type holds of the turned keys is what the cache is given
    k, v = (_exact_grid(x.double()) * live[:, None, None] for x in (out[1].to(dtype), state["v"]))
    return out[0], k, v


def _exact_turned(x, state):
    """Each pair as a complex number, times e^(i position frequency)."""
    case, n = state["case"], state["case"]["turned"]
    inv, factor = _frequencies(case)
    turn = torch.polar(torch.full((), factor, dtype=torch.float64, device=DEV),
                       state["positions"].double()[:, None, None] * inv)
    head, tail = x[..., :n].double(), x[..., n:].double()
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], n // 2, 2).contiguous()) * turn
        return torch.cat((torch.view_as_real(z).flatten(-2), tail), -1)
    z = torch.complex(head[..., :n // 2].contiguous(), head[..., n // 2:].contiguous()) * turn
    return torch.cat((z.real, z.imag, tail), -1)


def _exact_grid(x):
    """The nearest of the 15 values of each block of 32, of equally near ones the even code's."""
    grid = torch.tensor((0, 0.5, 1, 1.5, 2, 3, 4, 6), dtype=torch.float64, device=DEV)
    even = torch.tensor((0, 1, 0, 1, 0, 1, 0, 1), dtype=torch.float64, device=DEV) * 1e-12
    b = x.unflatten(-1, (-1, 32))
    most = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(most > 0, most, 1e-30) / 7.0) - 1e-15).clamp(-23, 13)
    near = ((b.abs() / 2.0 ** e)[..., None] - grid).abs() + even
    return (grid[near.argmin(-1)] * torch.sign(b) * 2.0 ** e).flatten(-2)


def _exact_tokens(state, b, n):
    """Keys and values [heads, n, D] of the first n tokens of a sequence: a page's parts one by one."""
    case = state["case"]
    P, half, groups = case["page"], case["D"] // 2, case["D"] // 32
    parts = state["pages"][state["table"][b, :-(-n // P)].long()].split((P * half, P * half, P * groups, P * groups), 2)
    rows = (parts[0].unflatten(2, (P, half)),
            torch.cat([parts[1].unflatten(2, (-1, 16, 4, groups))[:, :, :, :, i].flatten(-2)[:, :, :, None]
                       for i in range(4)], 3).flatten(2, 3))
    found = []
    for row, scale in zip(rows, parts[2:]):
        c = torch.empty((*row.shape[:-1], 2 * half), dtype=torch.float64, device=DEV)
        c[..., 0::2], c[..., 1::2] = (row % 16).double(), (row // 16).double()
        sign, c = 1 - 2 * (c // 8), c % 8
        size = torch.where(c < 2, c / 2, (1 + c % 2 / 2) * 2.0 ** (c // 2 - 1))
        s = 2.0 ** (scale.double().unflatten(2, (groups, P)).transpose(2, 3) - 127)
        found.append((sign * size * s.repeat_interleave(32, -1)).transpose(0, 1).flatten(1, 2)[:, :n])
    return found


def _exact_attend(state):
    case, q = state["case"], state["q"]
    G, D = case["q_heads"] // case["kv_heads"], case["D"]
    lengths, news = _lengths(case)
    out, first = [], 0
    for b, (n, m) in enumerate(zip(lengths, news)):
        k, v = _exact_tokens(state, b, n)
        x = q[first:first + m].double().view(m, -1, G, D).permute(1, 2, 0, 3)     # [Hk, G, m, D]
        first += m
        ago = (n - m + torch.arange(m, device=DEV))[:, None] - torch.arange(n, device=DEV)
        hidden = (ago < 0) | (ago >= case["window"] if case["window"] else torch.zeros_like(ago, dtype=torch.bool))
        o = torch.empty_like(x)
        for h in range(case["kv_heads"]):
            for j in range(G):
                s = (x[h, j] @ k[h].T * state["scale"]).masked_fill_(hidden, -math.inf)
                o[h, j] = torch.softmax(s, -1) @ v[h]
        out.append(o.permute(2, 0, 1, 3).reshape(m, -1, D))
    return torch.cat(out)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    D, Hq, Hk, size = case["D"], case["q_heads"], case["kv_heads"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "attend":
        lengths, news = _lengths(case)
        seen = pairs = 0
        for n, m in zip(lengths, news):
            w = case["window"] or n
            seen += min(n, m + w - 1)
            # query i sees min(w, n - m + i + 1) tokens
            full = min(m, max(0, m - (w - (n - m + 1))))
            a = m - full
            pairs += full * w + a * (n - m + 1) + a * (a - 1) // 2
        cache = seen * Hk * 2 * (D // 2 + D // 32)
        return {"bytes": cache + 2 * sum(news) * Hq * D * size, "flops": 4.0 * pairs * Hq * D}
    T = case["tokens"]
    table = T * (case["turned"] * 4 + 8)
    if case["op"] == "rotary":
        return {"bytes": 2 * T * (Hq + Hk) * D * size + table, "flops": 0}
    # queries in and out; keys and values in, to the pages, from them, and out; slots twice
    kept = (T - case["padded"]) * 2 * Hk * (D // 2 + D // 32)
    return {"bytes": 2 * T * Hq * D * size + 4 * T * Hk * D * size + 2 * kept + table + 16 * T, "flops": 0}
