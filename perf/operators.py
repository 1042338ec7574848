"""The operators around a KV cache held in 4 bits, measured: what they are
given, their plain forms, and the calls that a user makes.

The cache is the StreamingLLM ring (``sink`` first tokens, then a circular
window) of one decoder layer, for ``b`` sequences and ``hkv`` KV heads of
``d`` values, in groups of ``group`` consecutive values that share a scale
``s`` and a zero point ``z`` (0..15): a value is ``s (c - z)`` with ``c`` in
4 bits.  ``s`` is a fp16 number of 7 significant bits (its low four bits are
zero), so ``s (c - z)`` is a fp16 number exactly; ``z`` sits in those four
bits of the group's 16-bit word.  ``s`` is the smallest such number that is at
least ``(max(x, 0) - min(x, 0)) / 15`` over the group, ``z = rint(-min(x, 0) /
s)``, ``c = rint(x / s) + z`` within 0..15 and with ``|s (c - z)|`` at most the
largest finite fp16 number; a group that holds a NaN or an infinity gets the
scale NaN.

Storage of a layer: ``codes`` uint8 ``[2, b, hkv, cap, d / 2]`` and ``params``
int16 ``[2, b, hkv, cap, d / group]`` (0: keys, 1: values; ``cap``: sink +
window rounded up to 64 slots).  A row of codes is ``d / 4`` 16-bit halfwords
of four values, low bits first.  The 8-value block ``j`` of a row is the two
halfwords of its even and its odd values; with ``c = j % 4``, ``i = j // 4``
and ``n = d / 32`` they stand at halfwords ``2 (c n + i)`` and the next one in
a row of keys, and at ``2 c n + i`` and ``(2 c + 1) n + i`` in one of values.

Kinds of cases:

* ``rope``: RMS norm of every query and key head and its rotation, from the
  fused projection's output to q, k and v;
* ``store``: a chunk quantised into the ring, then the whole ring read back in
  logical order;
* ``decode``: attention of one query token for each sequence over the ring;
* ``prefill``: attention of a prompt chunk over the ring and over its own keys
  and values, causal, with the sink + window mask.
"""

import math

import torch

own = False

EPS = 1e-6
THETA = 1e6
F16_MAX = 65504.0


def listed():
    """Head counts and sizes are those of the decoder's default configuration
    (32 query and 8 KV heads of 128, 4 + 4092 slots, prompt chunks of 2048),
    and odd ones."""
    return [
        # one sequence's next token: what a decode step runs before its attention
        _case("rope", "rope_step", b=1, t=1, hq=32, hkv=8, d=128),
        # a prompt chunk of the default size
        _case("rope", "rope_chunk", b=1, t=2048, hq=32, hkv=8, d=128),
        # small heads, an odd number of tokens, a batch with its own positions
        _case("rope", "rope_odd", b=3, t=333, hq=15, hkv=5, d=64, ragged=True),
        # 32 sequences' next token into short rings
        _case("store", "store_step", b=32, t=1, hkv=8, d=128, group=32, window=60, count=100),
        # a prompt chunk into the default ring that has wrapped
        _case("store", "store_chunk", b=1, t=2048, hkv=8, d=128, group=64, window=4092, count=4219),
        # one conversation: the latency of a decode step
        _case("decode", "decode_one", b=1, hq=32, hkv=8, d=128, group=64, window=4092, count=8192),
        # a served batch
        _case("decode", "decode_batch", b=32, hq=32, hkv=8, d=128, group=64, window=4092, count=4101),
        # one long context in a wide ring
        _case("decode", "decode_long", b=1, hq=32, hkv=8, d=128, group=32, window=131068, count=200000),
        # a batch of sequences of different lengths, one of them empty; odd heads
        _case("decode", "decode_ragged", b=7, hq=15, hkv=5, d=64, group=32, window=1001, count=1500, ragged=True),
        # the fifth chunk of a prompt, the window full
        _case("prefill", "prefill_chunk", b=1, t=2048, hq=32, hkv=8, d=128, group=64, window=4092, count=8192),
        # a few new tokens after a long conversation (a follow-up question)
        _case("prefill", "prefill_short", b=1, t=33, hq=32, hkv=8, d=128, group=64, window=4092, count=5000),
        # sequences of different lengths, small heads, an odd chunk
        _case("prefill", "prefill_ragged", b=3, t=301, hq=15, hkv=5, d=64, group=32, window=1001, count=1400, ragged=True),
    ]


def _case(kind, name=None, *, b, hkv, d, hq=0, t=1, group=0, sink=4, window=0, count=0, ragged=False):
    case = {"kind": kind, "b": b, "t": t, "hq": hq, "hkv": hkv, "d": d, "group": group, "sink": sink,
            "window": window, "count": count, "ragged": ragged}
    return case if name is None else {"name": name, **case}


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["rope", "store", "decode", "prefill"])
    d = rng.choice([64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= d])
    hkv = rng.choice([1, 2, 4, 5, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 7, 8])
    sink = rng.choice([0, 1, 4, 4, 17])
    ragged = rng.random() < 0.4
    if kind == "rope":
        b = log(1, 32)
        return _case(kind, b=b, t=log(1, max(1, 2048 // b)), hq=min(hq, 32), hkv=hkv, d=d, ragged=ragged)
    if kind == "store":
        b = log(1, 32)
        window = log(8, max(9, 32768 // (b * hkv)))
        return _case(kind, b=b, t=log(1, 2048 // b), hkv=hkv, d=d, group=group, sink=sink, window=window,
                     count=log(1, 3 * window) - 1)
    if kind == "decode":
        b = log(1, 64)
        window = log(8, 1048000 // (b * hkv))
        window = min(window, 131068)
        return _case(kind, b=b, hq=hq, hkv=hkv, d=d, group=group, sink=sink, window=window,
                     count=log(1, 3 * window), ragged=ragged)
    b = log(1, 4)
    window = log(8, 4092)
    return _case(kind, b=b, t=log(1, 2048 // b), hq=min(hq, 32 // hkv * hkv), hkv=hkv, d=d, group=group, sink=sink,
                 window=window, count=log(1, 3 * window) - 1, ragged=ragged)


# ------------------------------------------------------------------- inputs --
def _cap(case):
    return (case["sink"] + case["window"] + 63) // 64 * 64


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    state = {"case": case}
    if case["kind"] == "rope":
        first = torch.randint(0, 60000, (b if case["ragged"] else 1,), generator=g, device=dev)
        pos = first[:, None] + torch.arange(t, device=dev)
        inv = THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = pos.double()[..., None] * inv
        cos, sin = angle.cos().float(), angle.sin().float()
        cos, sin = torch.cat([cos, cos], -1), torch.cat([sin, sin], -1)
        state["qkv"] = (normal(b, t, (hq + 2 * hkv) * d) * 2).half()
        state["q_norm"] = (1 + 0.3 * normal(d)).half()
        state["k_norm"] = (1 + 0.3 * normal(d)).half()
        state["cos"], state["sin"] = (cos, sin) if case["ragged"] else (cos[0].contiguous(), sin[0].contiguous())
        return state
    # a ring that was written before: keys with a few wide channels, as rotated keys have, and plain values
    cap = _cap(case)
    wide = torch.where(torch.rand(2, hkv, 1, d, generator=g, device=dev) < 0.04, 6.0, 1.0)
    wide[1] = 1.0
    codes = torch.empty(2, b, hkv, cap, d // 2, dtype=torch.uint8, device=dev)
    params = torch.empty(2, b, hkv, cap, d // case["group"], dtype=torch.int16, device=dev)
    for i in range(b):  # a sequence at a time: the values need not fit the card all at once
        codes[:, i], params[:, i] = _pack((normal(2, hkv, cap, d) * wide).half(), case["group"])
    state["codes"], state["params"] = codes, params
    state["count"] = case["count"]
    if case["ragged"]:
        counts = torch.randint(0, case["count"] + 1, (b,), generator=g, device=dev)
        if b > 1:
            counts[b // 2] = 0
        counts[0] = case["count"]
        state["count"] = counts
    if case["kind"] in ("store", "prefill"):
        state["k_new"] = (normal(b, t, hkv, d) * wide[0].transpose(0, 1)).half()
        state["v_new"] = normal(b, t, hkv, d).half()
    if case["kind"] == "decode":
        state["q"] = normal(b, hq, d).half()
    elif case["kind"] == "prefill":
        state["q"] = normal(b, t, hq, d).half()
    return state


# ------------------------------------------------------------------ one pass --
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    return {"rope": _rope, "store": _store, "decode": _decode, "prefill": _prefill}[kind](state)


def _own(kind, state):
    from qextract_infer_b200 import _C

    case = state["case"]
    if kind == "rope":
        return _C.qk_norm_rope(state["qkv"], case["hq"], case["hkv"], state["q_norm"], state["k_norm"], EPS,
                               state["cos"], state["sin"])
    ring = (state["codes"], state["params"], state["count"], case["sink"], case["window"])
    if kind == "store":
        _C.ring_append_q4(state["k_new"], state["v_new"], *ring)
        codes, params, count, sink, window = ring
        return _C.ring_gather_q4(codes, params, count + case["t"], sink, window)
    if kind == "decode":
        return _C.decode_attention_q4(state["q"], *ring)
    return _C.prefill_attention_q4(state["q"], state["k_new"], state["v_new"], *ring)


# --------------------------------------------------------------- plain forms --
def _rope(state):
    case = state["case"]
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))
    x = state["qkv"].view(b, t, hq + 2 * hkv, d)
    cos, sin = state["cos"], state["sin"]
    cos, sin = (c.unsqueeze(-2) for c in (cos, sin))

    def heads(y, w):
        y = y.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        turned = torch.cat([-y[..., d // 2:], y[..., : d // 2]], -1)
        return (y * cos + turned * sin).half()

    return (heads(x[:, :, :hq], state["q_norm"]), heads(x[:, :, hq:hq + hkv], state["k_norm"]),
            x[:, :, hq + hkv:].contiguous())


def _places(d, which, device):
    """The value (0..d-1) that stands at each 4-bit place of a row."""
    n = d // 32
    j = torch.arange(d // 8, device=device)
    c, i = j % 4, j // 4
    even = 2 * (c * n + i) if which == 0 else 2 * c * n + i
    odd = even + 1 if which == 0 else even + n
    value = torch.empty(d // 4, 4, dtype=torch.int64, device=device)
    four = 2 * torch.arange(4, device=device)
    value[even] = 8 * j[:, None] + four
    value[odd] = 8 * j[:, None] + four + 1
    return value.reshape(-1)


def _quantise(x, group):
    """(c, z, s) of ``x`` ``[..., d]``: c like x, z and s ``[..., d / group]``."""
    x = x.double().unflatten(-1, (-1, group))
    fine = x.isfinite().all(-1)
    y = torch.where(fine[..., None], x, 0.0)
    lo, hi = y.amin(-1).clamp(max=0), y.amax(-1).clamp(min=0)
    least = (hi - lo) / 15
    # the smallest number of 7 significant bits (and of fp16's range) that is at least `least`
    step = torch.exp2(torch.floor(torch.log2(least.clamp(min=2.0 ** -14))) - 6)
    s = torch.ceil(least / step) * step
    part = torch.where(s > 0, s, 1.0)
    z = torch.round(-lo / part)
    k = torch.round(y / part[..., None])
    k = (k + z[..., None]).clamp(0, 15) - z[..., None]
    k = torch.where((k * s[..., None]).abs() > F16_MAX, k - k.sign(), k)
    c = k + z[..., None]
    return c.flatten(-2), z, torch.where(fine, s, math.nan)


def _pack(x, group):
    """codes and params of ``x`` ``[2, ..., d]``."""
    d = x.size(-1)
    c, z, s = _quantise(x, group)
    c, z = c.to(torch.int16), z.to(torch.int16)
    word = (s.half().view(torch.int16) & -16) | z
    word = torch.where(s.isnan(), 0x7E00, word)
    nibbles = torch.stack([c[w][..., _places(d, w, x.device)] for w in (0, 1)])
    return (nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)).to(torch.uint8), word.to(torch.int16)


def _values(codes, params):
    """``[2, ..., slots, d]`` in 32 bits."""
    d = codes.size(-1) * 2
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    c = torch.empty_like(nibbles)
    c[0][..., _places(d, 0, codes.device)] = nibbles[0]
    c[1][..., _places(d, 1, codes.device)] = nibbles[1]
    s = (params & -16).view(torch.float16).float().unsqueeze(-1)
    z = (params & 15).float().unsqueeze(-1)
    return (s * (c.float().unflatten(-1, (params.size(-1), -1)) - z)).flatten(-2)


def _ring_positions(count, sink, window, slots):
    """The position that each of ``slots`` holds after ``count`` tokens (``[b]`` or a number), -1 where there is none:
    position ``p`` stands in slot ``p``, or ``sink + (p - sink) % window`` from ``sink`` on."""
    count = torch.as_tensor(count, device="cuda").reshape(-1, 1)
    i = torch.arange(slots, device="cuda").expand(count.size(0), -1)
    newest = count - 1 - sink
    ring = newest - (newest - (i - sink)) % window
    pos = torch.where(i < sink, i, torch.where(ring >= 0, ring + sink, -1))
    return torch.where((pos < count) & (i < sink + window), pos, -1)


def _store(state):
    case = state["case"]
    sink, window, count, t = case["sink"], case["window"], case["count"], case["t"]
    codes, params = state["codes"], state["params"]
    pos = count + torch.arange(t, device="cuda")
    keep = (pos < sink) | (pos >= count + t - window)  # what a later token of the chunk does not replace
    pos = pos[keep]
    slots = torch.where(pos < sink, pos, sink + (pos - sink) % window)
    new = torch.stack([state["k_new"], state["v_new"]])[:, :, keep].transpose(2, 3)
    codes[:, :, :, slots], params[:, :, :, slots] = _pack(new, case["group"])
    held = _ring_positions(count + t, sink, window, codes.size(3))[0]
    order = torch.argsort(torch.where(held < 0, 1 << 40, held))[: int(min(count + t, sink) + max(0, min(count + t - sink, window)))]
    k, v = _values(codes[:, :, :, order], params[:, :, :, order]).half().transpose(2, 3).contiguous()
    return k, v


def _decode(state):
    case = state["case"]
    q = state["q"].float()
    k, v = _values(state["codes"], state["params"])
    held = _ring_positions(state["count"], case["sink"], case["window"], k.size(2)) >= 0
    q = q.unflatten(1, (case["hkv"], -1))
    s = q @ k.transpose(-1, -2) / math.sqrt(case["d"])
    s = s.masked_fill(~held[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top.isfinite(), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = p @ v / torch.where(total > 0, total, 1.0)
    return out.flatten(1, 2).half()


def _prefill(state):
    case = state["case"]
    sink, window, t = case["sink"], case["window"], case["t"]
    k, v = _values(state["codes"], state["params"])
    first = torch.as_tensor(state["count"], device="cuda").reshape(-1, 1)
    if first.size(0) == 1:
        first = first.expand(case["b"], 1)
    at = first + torch.arange(t, device="cuda")  # the chunk's positions
    old = _ring_positions(first, sink, window, k.size(2))
    k = torch.cat([k, state["k_new"].float().transpose(1, 2)], 2)
    v = torch.cat([v, state["v_new"].float().transpose(1, 2)], 2)
    pos = torch.cat([old, at], 1)
    seen = (pos[:, None] >= 0) & (pos[:, None] <= at[:, :, None])
    seen &= (pos[:, None] < sink) | (pos[:, None] > at[:, :, None] - window)
    q = state["q"].float().transpose(1, 2).unflatten(1, (case["hkv"], -1))
    s = q @ k.unsqueeze(2).transpose(-1, -2) / math.sqrt(case["d"])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = p @ v.unsqueeze(2) / p.sum(-1, keepdim=True)
    return out.flatten(1, 2).transpose(1, 2).half().contiguous()


# ------------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "decode": _exact_attention,
            "prefill": _exact_attention}[case["kind"]](case, state)


def _exact_rope(case, state):
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))
    x = state["qkv"].double().view(b, t, hq + 2 * hkv, d)
    cos, sin = (state[n].double().view(-1, t, 1, d) for n in ("cos", "sin"))
    w = torch.cat([state["q_norm"].double().expand(hq, d), state["k_norm"].double().expand(hkv, d)])
    y = x[:, :, : hq + hkv]
    y = y / (y.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w
    a, c = y[..., : d // 2], y[..., d // 2:]
    y = torch.cat([a * cos[..., : d // 2] - c * sin[..., : d // 2], c * cos[..., d // 2:] + a * sin[..., d // 2:]], -1)
    return y[:, :, :hq], y[:, :, hq:], x[:, :, hq + hkv:]


def _exact_read(codes, params, which):
    """One of keys (0) and values (1) in 64 bits, block by block of 8 values."""
    d, groups = codes.size(-1) * 2, params.size(-1)
    n = d // 32
    half = codes[which].to(torch.int64)
    half = half[..., 0::2] + 256 * half[..., 1::2]
    out = torch.empty(*half.shape[:-1], d, dtype=torch.float64, device=codes.device)
    for j in range(d // 8):
        c, i = j % 4, j // 4
        places = (2 * (c * n + i), 2 * (c * n + i) + 1) if which == 0 else (2 * c * n + i, (2 * c + 1) * n + i)
        word = params[which, ..., 8 * j * groups // d].to(torch.int64) & 0xFFFF
        z = word % 16
        bits = word - z
        power, part = bits // 1024, bits % 1024
        s = torch.where(power > 0, (1024 + part).double() * torch.exp2(power.double() - 25), part.double() * 2.0 ** -24)
        s = torch.where(power == 31, math.nan, s)
        for e in range(8):
            out[..., 8 * j + e] = s * ((half[..., places[e % 2]] >> (4 * (e // 2))) % 16 - z)
    return out


def _exact_quantised(x, group):
    """What the values of ``x`` ``[..., d]`` become in the cache."""
    x = x.double().unflatten(-1, (-1, group))
    fine = x.isfinite().all(-1, keepdim=True)
    y = torch.where(fine, x, 0.0)
    span = (y.amax(-1, keepdim=True).clamp(min=0) - y.amin(-1, keepdim=True).clamp(max=0))
    part, power = torch.frexp(span / 15)  # span / 15 = part 2^power, part in [1/2, 1)
    low = (power - 7).clamp(min=-20)
    s = torch.ceil(torch.ldexp(span / 15, -low)) * torch.exp2(low.double())
    z = torch.where(s > 0, torch.round(-y.amin(-1, keepdim=True).clamp(max=0) / s), 0.0)
    k = torch.where(s > 0, torch.round(y / s), 0.0)
    k = torch.minimum(torch.maximum(k, -z), 15 - z)
    k = torch.where((k * s).abs() > F16_MAX, k - k.sign(), k)
    return torch.where(fine, k * s, math.nan).flatten(-2)


def _exact_store(case, state):
    sink, window, count, t = case["sink"], case["window"], case["count"], case["t"]
    end = count + t
    positions = list(range(min(end, sink))) + list(range(max(sink, end - window), end))
    pos = torch.tensor(positions, device="cuda")
    slots = torch.where(pos < sink, pos, sink + (pos - sink) % window)
    outs = []
    for which, new in ((0, state["k_new"]), (1, state["v_new"])):
        old = _exact_read(state["codes"], state["params"], which)[:, :, slots].transpose(1, 2)
        fresh = _exact_quantised(new, case["group"])
        out = old.clone()
        is_new = pos >= count
        out[:, is_new] = fresh[:, pos[is_new] - count]
        outs.append(out)
    return tuple(outs)


def _exact_attention(case, state):
    b, t, hq, hkv, d, sink, window = (case[n] for n in ("b", "t", "hq", "hkv", "d", "sink", "window"))
    counts = state["count"].tolist() if case["ragged"] else [case["count"]] * b
    new = case["kind"] == "prefill"
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    q_all = state["q"].double().view(b, t, hq, d)
    for n in range(b):
        one = slice(n, n + 1)
        k, v = (_exact_read(state["codes"][:, one], state["params"][:, one], w)[0] for w in (0, 1))
        count = counts[n]
        positions = list(range(min(count, sink))) + list(range(max(sink, count - window), count))
        pos = torch.tensor(positions, dtype=torch.int64, device="cuda")
        slots = torch.where(pos < sink, pos, sink + (pos - sink) % window)
        k, v = k[:, slots], v[:, slots]
        at = torch.arange(t, device="cuda") + (count if new else count - 1)
        if new:
            k = torch.cat([k, state["k_new"][n].double().transpose(0, 1)], 1)
            v = torch.cat([v, state["v_new"][n].double().transpose(0, 1)], 1)
            pos = torch.cat([pos, at])
        if not pos.numel():
            continue
        gone = (pos > at[:, None]) | ((pos >= sink) & (pos <= at[:, None] - window))
        for h in range(hq):
            kv = h * hkv // hq
            s = q_all[n, :, h] @ k[kv].T / math.sqrt(d)
            out[n, :, h] = torch.softmax(torch.where(gone, -math.inf, s), -1) @ v[kv]
    return out if new else out[:, 0]


# ---------------------------------------------------------------- what it costs --
def work(case):
    b, t, hq, hkv, d = (case[n] for n in ("b", "t", "hq", "hkv", "d"))
    if case["kind"] == "rope":
        rows = (b if case["ragged"] else 1) * t
        return {"bytes": 2 * b * t * (hq + 2 * hkv) * d * 2 + rows * d * 8 + 4 * d, "flops": 8 * b * t * (hq + hkv) * d}
    sink, window, count = case["sink"], case["window"], case["count"]
    row = 2 * (d // 2 + 2 * (d // case["group"]))  # bytes of one slot and KV head, keys and values

    def held(n):
        return min(n, sink) + max(0, min(n - sink, window))

    # lengths of a ragged batch are spread evenly from none to `count`; one of them is `count`
    counts = [count] * b if not case["ragged"] else [count * i // max(1, b - 1) for i in range(b)] if b > 1 else [count]
    ring = sum(held(c) for c in counts) * hkv * row
    if case["kind"] == "store":
        new = 2 * b * t * hkv * d * 2
        kept = max(0, min(sink - count, t)) + min(max(0, min(t, count + t - sink)), window)
        values = b * held(count + t) * hkv
        old = values * row - b * kept * hkv * row
        return {"bytes": new + b * kept * hkv * row + old + values * 4 * d, "flops": 8 * b * t * hkv * d}
    if case["kind"] == "decode":
        return {"bytes": 2 * b * hq * d * 2 + ring, "flops": 4 * hq * d * sum(held(c) for c in counts)}
    pairs = sum(min(p + 1, sink) + max(0, min(p - sink + 1, window)) for c in counts for p in range(c, c + t))
    return {"bytes": 2 * b * t * hq * d * 2 + 2 * b * t * hkv * d * 2 + ring, "flops": 4 * hq * d * pairs}
