"""The operators by which each request of a served batch brings its own adapter
and its own sampling settings, measured: what they are given, their plain forms,
and the calls that a user makes.

Kinds of cases:

* ``lora``: low-rank adapters beside a shared projection.  Sequence ``i`` has
  adapter ``a = adapters[i]`` of ``n`` (none where that is -1) and ``t`` tokens;
  ``out = y + scales[a] (x A[a]) B[a]`` with ``y`` the shared projection's
  output, ``A`` ``[n, k, p r]`` and ``B`` ``[n, r, sum(splits)]``: the
  projection's columns are ``p`` blocks (the parts of a fused projection) of
  widths ``splits``, block ``j`` taking ranks ``j r .. (j + 1) r - 1`` of ``A``;
* ``head``: the logits of a batch's last hidden states, whole;
* ``sample``: one token for each row of logits from one number ``u`` in [0, 1).
  Tokens stand in the order of their logits, the largest first, equal ones by
  their index; the weight of a token is ``exp((l - max l) / temperature)``.
  The first ``top_k`` stay (0: all), of these the shortest run from the front
  that has at least ``top_p`` of their weight (1: all), of these the ones whose
  weight is at least ``min_p``; the token drawn is the first at which the
  running sum of the weights that stay exceeds ``u`` times their sum.
  Temperature 0 takes the first token.  Beside the tokens stand the logarithms of
  their probabilities among the tokens that stay.
"""

import math

import numpy as np
import torch

own = False


def listed():
    """Sizes are those of the decoder's default configuration (hidden 4096, 32 + 8 + 8 heads of 128, 2 x 12288 of the
    MLP, 151936 tokens, chunks of 2048, rank 16), of the smaller projection that the benchmark runs (2560 x 9728), and
    odd ones."""
    return [
        # one conversation's next token through the fused q|k|v projection
        _lora("lora_one", b=1, t=1, k=4096, splits=(4096, 1024, 1024), r=16, n=4),
        # a served batch, every request with another adapter, through the fused gate|up projection
        _lora("lora_batch", b=32, t=1, k=4096, splits=(12288, 12288), r=16, n=32),
        # a prompt chunk of the default size through the MLP's second projection, a wide adapter
        _lora("lora_chunk", b=1, t=2048, k=12288, splits=(4096,), r=64, n=2),
        # three prompts of odd length, two of them with the same adapter
        _lora("lora_prompts", b=3, t=333, k=2560, splits=(9728,), r=8, n=2),
        # a batch in which a few adapters are shared and every fourth request has none; odd sizes
        _lora("lora_shared", b=50, t=1, k=2560, splits=(1000, 328), r=32, n=5, bare=4),
        # one conversation's logits
        _head("head_one", b=1, k=4096, v=151936),
        # a served batch's
        _head("head_batch", b=32, k=4096, v=151936),
        # a quarter of the vocabulary, as one of four ranks holds it, an odd batch
        _head("head_slice", b=5, k=4096, v=37984),
        # one conversation
        _sample("sample_one", b=1, v=151936, temperature=0.8, top_k=0, top_p=0.95, min_p=0.0),
        # a served batch with usual settings
        _sample("sample_batch", b=32, v=151936, temperature=0.7, top_k=50, top_p=0.9, min_p=0.02),
        # every request with its own settings: greedy ones, hot ones without any limit, ...
        _sample("sample_mixed", b=32, v=151936, mixed=True),
        # a small vocabulary of odd size
        _sample("sample_odd", b=7, v=32003, temperature=1.3, top_k=1000, top_p=0.99, min_p=0.0),
    ]


def _lora(name=None, *, b, t, k, splits, r, n, bare=0):
    """``bare``: every ``bare``-th sequence has no adapter (0: all have one)"""
    case = {"kind": "lora", "b": b, "t": t, "k": k, "r": r, "n": n, "bare": bare,
            "splits": "+".join(str(s) for s in splits)}
    return case if name is None else {"name": name, **case}


def _head(name=None, *, b, k, v):
    case = {"kind": "head", "b": b, "k": k, "v": v}
    return case if name is None else {"name": name, **case}


def _sample(name=None, *, b, v, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    case = {"kind": "sample", "b": b, "v": v, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "mixed": mixed}
    return case if name is None else {"name": name, **case}


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))

    kind = rng.choice(["lora", "lora", "head", "sample", "sample"])
    if kind == "lora":
        b = log(1, 64)
        t = 1 if rng.random() < 0.5 else log(1, max(1, 2048 // b))
        parts = rng.choice([1, 1, 2, 3])
        splits = [8 * log(4, 12288 // parts // 8) for _ in range(parts)]
        return _lora(b=b, t=t, k=8 * log(8, 12288 // 8), splits=splits, r=rng.choice([8, 16, 16, 24, 32, 64]),
                     n=log(1, 32), bare=rng.choice([0, 0, 2, 3, 5]))
    if kind == "head":
        return _head(b=log(1, 32), k=64 * log(1, 64), v=8 * log(64, 151936 // 8))
    b = log(1, 64)
    return _sample(b=b, v=log(100, min(262144, 32 * 151936 // b)), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.6]),
                   top_k=rng.choice([0, 0, 1, 40, log(2, 2000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.999]),
                   min_p=rng.choice([0.0, 0.0, 0.05, 0.3]), mixed=rng.random() < 0.3)


def _splits(case):
    return [int(s) for s in case["splits"].split("+")]


def _adapters(case):
    """The adapter of each sequence, before they are mixed: each adapter in turn, so that any seed has as many of them."""
    ids, given = [], 0
    for i in range(case["b"]):
        if case["bare"] and i % case["bare"] == case["bare"] - 1:
            ids.append(-1)
        else:
            ids.append(given % case["n"])
            given += 1
    return ids


# ------------------------------------------------------------------- inputs --
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    state = {"case": case}
    if case["kind"] == "lora":
        b, t, k, r, n = (case[x] for x in ("b", "t", "k", "r", "n"))
        splits = _splits(case)
        lead = (b,) if t == 1 else (b, t)
        state["x"] = normal(*lead, k).half()
        state["y"] = normal(*lead, sum(splits)).half()
        state["lora_A"] = (normal(n, k, r * len(splits)) / math.sqrt(k)).half()
        state["lora_B"] = (normal(n, r, sum(splits)) * 0.3).half()
        state["scales"] = 0.5 + 2 * torch.rand(n, generator=g, device=dev)
        ids = torch.tensor(_adapters(case), device=dev)
        state["adapters"] = ids[torch.randperm(b, generator=g, device=dev)]
        return state
    if case["kind"] == "head":
        state["h"] = normal(case["b"], case["k"]).half()
        weight = torch.empty(case["k"], case["v"], dtype=torch.float16, device=dev)
        for part in weight.split(512):
            part.copy_(normal(*part.shape) * (4 / math.sqrt(case["k"])))
        state["weight"] = weight
        return state
    # logits as a head gives them: a broad heap, and a few tokens that stand out
    b, v = case["b"], case["v"]
    logits = 2.5 * normal(b, v)
    peaks = torch.randint(0, v, (b, 20), generator=g, device=dev)
    # (where two of a row fall on one token, as they do in small vocabularies, the larger one counts: a plain
    # scatter leaves open which, and the logits were not the seed's alone)
    logits.scatter_reduce_(1, peaks, 9 + 3 * normal(b, 20), "amax", include_self=False)
    state["logits"] = logits.half()
    state["u"] = torch.rand(b, generator=g, device=dev)
    if case["mixed"]:
        def pick(values, dtype):
            values = torch.tensor(values, dtype=dtype, device=dev)
            return values[torch.randint(0, len(values), (b,), generator=g, device=dev)]

        state["temperature"] = pick([0.0, 0.2, 0.7, 1.0, 1.0, 2.0], torch.float32)
        state["top_k"] = pick([0, 0, 0, 1, 20, 400, 20000], torch.int64)
        state["top_p"] = pick([1.0, 1.0, 0.95, 0.8, 0.3], torch.float32)
        state["min_p"] = pick([0.0, 0.0, 0.01, 0.1], torch.float32)
    else:
        for name in ("temperature", "top_p", "min_p"):
            state[name] = torch.full((b,), case[name], dtype=torch.float32, device=dev)
        state["top_k"] = torch.full((b,), case["top_k"], dtype=torch.int64, device=dev)
    return state


# ------------------------------------------------------------------ one pass --
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    return {"lora": _plain_lora, "head": _plain_head, "sample": _plain_sample}[kind](state)


def _own(kind, state):
    from qextract_infer_b200 import _C

    if kind == "lora":
        return _C.multi_lora_add(state["y"], state["x"], state["lora_A"], state["lora_B"], state["adapters"],
                                 state["scales"], splits=_splits(state["case"]))
    if kind == "head":
        return _C.lm_head_logits(state["h"], state["weight"])
    return _C.sample_logits(state["logits"], state["u"], state["temperature"], state["top_k"], state["top_p"],
                            state["min_p"])


# --------------------------------------------------------------- plain forms --
def _plain_lora(state):
    case = state["case"]
    b, t, r = case["b"], case["t"], case["r"]
    x, y = state["x"].float().view(b, t, -1), state["y"].float().view(b, t, -1)
    ids = state["adapters"]
    some = ids.clamp(min=0)
    scale = torch.where(ids >= 0, state["scales"][some], 0.0)[:, None, None]
    low = scale * (x @ state["lora_A"].float()[some])
    up = state["lora_B"].float()
    at = 0
    parts = []
    for j, width in enumerate(_splits(case)):
        parts.append(low[..., j * r:(j + 1) * r] @ up[:, :, at:at + width][some])
        at += width
    return (y + torch.cat(parts, -1)).half().view(state["y"].shape)


def _plain_head(state):
    return (state["h"].float() @ state["weight"].float()).half()


def _plain_sample(state):
    logits = state["logits"]
    v = logits.size(1)
    l, order = torch.sort(logits.double(), dim=-1, descending=True, stable=True)
    temperature = state["temperature"].double()[:, None]
    greedy = temperature <= 0
    w = torch.exp((l - l[:, :1]) / torch.where(greedy, 1.0, temperature))
    place = torch.arange(v, device=l.device)
    k = torch.where(state["top_k"] > 0, state["top_k"], v)[:, None]
    w = torch.where((place < k) & (~greedy | (place == 0)), w, 0.0)
    upto = w.cumsum(-1)
    p = state["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (place == 0) | (upto - w < p * upto[:, -1:]), w, 0.0)
    w = torch.where(w >= state["min_p"].double()[:, None], w, 0.0)
    upto = w.cumsum(-1)
    at = (upto <= state["u"].double()[:, None] * upto[:, -1:]).sum(-1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(-1, keepdim=True) - 1)
    return order.gather(1, at)[:, 0], torch.log(w.gather(1, at) / upto[:, -1:])[:, 0].float()


# ------------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    state = prepare(case, seed)
    return {"lora": _exact_lora, "head": _exact_head, "sample": _exact_sample}[case["kind"]](case, state)


def _exact_lora(case, state):
    out = state["y"].double()
    r, edges = case["r"], np.cumsum([0] + _splits(case))
    for i, a in enumerate(state["adapters"].tolist()):
        if a < 0:
            continue
        x = state["x"][i].double().reshape(case["t"], -1)
        for j in range(len(edges) - 1):
            columns = slice(int(edges[j]), int(edges[j + 1]))
            low = torch.einsum("tk,kr->tr", x, state["lora_A"][a, :, j * r:(j + 1) * r].double())
            delta = torch.einsum("tr,rn->tn", low, state["lora_B"][a, :, columns].double())
            out[i][..., columns] += (state["scales"][a].double() * delta).view(out[i][..., columns].shape)
    return out


def _exact_head(case, state):
    h = state["h"].double()
    return torch.cat([h @ part.double() for part in state["weight"].split(16384, 1)], 1)


def _exact_sample(case, state):
    logits = state["logits"].cpu().numpy().astype(np.longdouble)
    u, temperature, top_k, top_p, min_p = (state[n].cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = [], []
    for i, row in enumerate(logits):
        order = np.lexsort((np.arange(row.size), -row))
        if not temperature[i] > 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        l = row[order][: int(top_k[i]) if top_k[i] > 0 else row.size]
        w = np.exp((l - l[0]) / np.longdouble(temperature[i]))
        if top_p[i] < 1:
            stay = 1 + int(np.searchsorted(np.cumsum(w), np.longdouble(top_p[i]) * w.sum()))
            w = w[:stay]
        w = w[w >= np.longdouble(min_p[i])]
        running = np.cumsum(w)
        at = int(np.searchsorted(running, np.longdouble(u[i]) * running[-1], side="right"))
        at = min(at, w.size - 1)
        tokens.append(int(order[at]))
        logprobs.append(float(np.log(w[at]) - np.log(running[-1])))
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.float64)


# ---------------------------------------------------------------- what it costs --
def work(case):
    b = case["b"]
    if case["kind"] == "lora":
        t, k, r, splits = case["t"], case["k"], case["r"], _splits(case)
        n, p = sum(splits), len(splits)
        ids = _adapters(case)
        used = len(set(ids) - {-1})
        rows = t * sum(a >= 0 for a in ids)
        return {"bytes": 2 * rows * k + 4 * b * t * n + 2 * used * r * (p * k + n) + 8 * b,
                "flops": 2 * rows * r * (p * k + n)}
    if case["kind"] == "head":
        k, v = case["k"], case["v"]
        return {"bytes": 2 * (b * k + k * v + b * v), "flops": 2 * b * k * v}
    return {"bytes": b * (2 * case["v"] + 36), "flops": 6 * b * case["v"]}
