"""Measured cases of the operators of a decode step: products with 4-bit
weights, rotary positions on several axes, attention over a sliding window
with sinks, and sampling from given random numbers.

``run`` computes them in their plain form, from elementary torch operations,
or (``own``) through the framework's graphs and runtime.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}
DEVICE = "cuda"


# ------------------------------------------------------------------- cases
def _q4(m, n, k, group, dtype, zeros):
    return {"op": "matvec_q4", "m": m, "n": n, "k": k, "group": group, "dtype": dtype,
            "zeros": zeros}


def _rope(batch, seq, heads, dim, axes, table, dtype, style):
    return {"op": "rope", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "axes": axes,
            "table": table, "dtype": dtype, "style": style}


def _attention(batch, new, cache, heads, kv_heads, dim, window, sinks, ragged, dtype):
    return {"op": "window_attention", "batch": batch, "new": new, "cache": cache, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks,
            "ragged": ragged, "dtype": dtype}


def _sample(rows, vocab, dtype, top_k, top_p, min_p):
    return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # the attention output projection of one request's token
        dict(_q4(1, 4096, 4096, 128, "bfloat16", False), name="q4_1x4096x4096"),
        # the up projection of 8 requests, weights with zero points
        dict(_q4(8, 14336, 4096, 64, "float16", True), name="q4_8x14336x4096_zeros"),
        # the vocabulary projection of 3 rows, an odd vocabulary
        dict(_q4(3, 100003, 5120, 128, "bfloat16", False), name="q4_3x100003x5120"),
        # queries and keys of one new token of 48 requests, plain positions
        dict(_rope(48, 1, 40, 128, 1, 8192, "bfloat16", "half"), name="rope_48x1x40x128"),
        # prefill of images: time, height and width positions
        dict(_rope(4, 4096, 32, 128, 3, 4096, "bfloat16", "half"), name="rope_4x4096x32x128_3axes"),
        # one request, one new token, short window: latency
        dict(_attention(1, 1, 4096, 32, 8, 128, 1024, 4, False, "bfloat16"),
             name="attention_decode_1x4096"),
        # 64 requests of different lengths, one new token each
        dict(_attention(64, 1, 8192, 32, 8, 128, 4096, 4, True, "bfloat16"),
             name="attention_decode_64x8192"),
        # prefill of one long prompt
        dict(_attention(1, 8192, 8192, 32, 8, 128, 2048, 4, False, "bfloat16"),
             name="attention_prefill_8192"),
        # chunks of 500 new tokens after caches of different lengths
        dict(_attention(4, 500, 2900, 16, 4, 64, 1000, 16, True, "float16"),
             name="attention_chunk_4x500"),
        # one request's token
        dict(_sample(1, 32768, "float32", True, True, False), name="sample_1x32768"),
        # a batch of requests, 16-bit logits with many equal values
        dict(_sample(64, 131072, "bfloat16", False, True, True), name="sample_64x131072"),
        # a large batch: some rows filtered, some drawn from all tokens
        dict(_sample(256, 100003, "float32", True, True, True), name="sample_256x100003"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matvec_q4", "rope", "window_attention", "sample"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "matvec_q4":
        group = rng.choice([32, 64, 128])
        return _q4(rng.choice([1, 1, 2, 3, 5, 8, 13, 16, 32]), _log_int(rng, 500, 60000),
                   group * max(1, _log_int(rng, 512, 8192) // group), group,
                   rng.choice(["bfloat16", "float16", "float32"]), rng.random() < 0.5)
    if op == "rope":
        tokens = _log_int(rng, 1, 16384)
        batch = min(tokens, _log_int(rng, 1, 64))
        return _rope(batch, max(1, tokens // batch), rng.choice([1, 4, 8, 17, 32]),
                     rng.choice([32, 64, 80, 96, 128]), rng.choice([1, 2, 3]),
                     _log_int(rng, 64, 20000), rng.choice(["bfloat16", "float16", "float32"]),
                     rng.choice(["half", "interleaved"]))
    if op == "window_attention":
        kv_heads, per = rng.choice([(8, 4), (8, 1), (4, 8), (2, 5), (1, 7), (4, 4)])
        dim = rng.choice([64, 64, 80, 128, 128])
        if rng.random() < 0.5:
            batch, new, cache = _log_int(rng, 1, 32), rng.choice([1, 1, 1, 2, 4]), _log_int(rng, 64, 8192)
        else:
            new = _log_int(rng, 40, 2500)
            batch, cache = rng.choice([1, 2, 3]), new + _log_int(rng, 1, 2500)
        return _attention(batch, new, cache, kv_heads * per, kv_heads, dim, _log_int(rng, 16, 4096),
                          rng.choice([0, 1, 4, 16, 33]), rng.random() < 0.7, dtype)
    return _sample(_log_int(rng, 1, 128), _log_int(rng, 500, 130000),
                   rng.choice(["bfloat16", "float16", "float32"]), rng.random() < 0.5,
                   rng.random() < 0.6, rng.random() < 0.4)


def _lengths(case):
    """Valid keys of each request's cache (the new tokens included)."""
    lo, hi = case["new"], case["cache"]
    span = hi - lo if case["ragged"] else 0
    return [hi - (b * 7919 + 131 * (b % 3)) % (span // 2 + 1) for b in range(case["batch"])]


def _sections(case):
    """Pairs of a head that each axis turns: the first axis the rest."""
    half, axes = case["dim"] // 2, case["axes"]
    each = half * 3 // 8 if axes == 3 else half // 2
    return [half - each * (axes - 1)] + [each] * (axes - 1)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEVICE)

    state = {"case": case}
    if case["op"] == "matvec_q4":
        m, n, k, g = case["m"], case["n"], case["k"], case["k"] // case["group"]
        sdt = torch.float32 if case["dtype"] == "float32" else dt
        state["x"] = normal(m, k).to(dt)
        state["qweight"] = torch.randint(0, 256, (n, k // 2), generator=gen, device=DEVICE,
                                         dtype=torch.uint8)
        state["scales"] = ((0.5 + uniform(n, g)) / (4.6 * k ** 0.5)).to(sdt)
        if case["zeros"]:
            state["zeros"] = (8 + 2 * uniform(n, g) - 1).to(sdt)
    elif case["op"] == "rope":
        b, s, d, p = case["batch"], case["seq"], case["dim"], case["table"]
        state["x"] = normal(b, s, case["heads"], d).to(dt)
        state["positions"] = torch.randint(0, p, (case["axes"], b, s), generator=gen, device=DEVICE,
                                           dtype=torch.int32)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
        angle = torch.arange(p, device=DEVICE, dtype=torch.float64)[:, None] * inv
        state["cos"], state["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    elif case["op"] == "window_attention":
        b, d = case["batch"], case["dim"]
        state["q"] = normal(b, case["new"], case["heads"], d).to(dt)
        state["k"] = normal(b, case["cache"], case["kv_heads"], d).to(dt)
        state["v"] = normal(b, case["cache"], case["kv_heads"], d).to(dt)
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    else:
        r = case["rows"]
        state["logits"] = (3 * normal(r, case["vocab"])).to(dt)
        state["u"] = uniform(r)
        state["temperature"] = 0.5 + uniform(r)
        if case["top_k"]:
            state["top_k"] = torch.randint(0, 100, (r,), generator=gen, device=DEVICE,
                                           dtype=torch.int32)
        if case["top_p"]:
            state["top_p"] = 0.5 + 0.55 * uniform(r)          # some rows above 1: no limit
        if case["min_p"]:
            state["min_p"] = 0.1 * uniform(r) - 0.02          # some rows below 0: no limit
    if own:
        state["fn"] = _compiled(case)
    return state


def _compiled(case):
    """The compiled graph that a program keeps."""
    from molten_b200 import graphs
    from molten_b200.codegen import compile_graph
    from molten_b200.runtime import MoltenRuntime

    dt = case["dtype"]
    if case["op"] == "matvec_q4":
        g = graphs.matvec_q4(case["m"], case["n"], case["k"], case["group"], dtype=dt,
                             zeros=case["zeros"])
    elif case["op"] == "rope":
        g = graphs.rope_positions(case["batch"], case["seq"], case["heads"], case["dim"],
                                  table=case["table"], sections=_sections(case), dtype=dt,
                                  style=case["style"])
    elif case["op"] == "window_attention":
        g = graphs.window_attention(case["batch"], case["new"], case["cache"], case["heads"],
                                    case["kv_heads"], case["dim"], window=case["window"],
                                    sinks=case["sinks"], dtype=dt)
    else:
        g = graphs.sample(case["rows"], case["vocab"], dtype=dt, top_k=case["top_k"],
                          top_p=case["top_p"], min_p=case["min_p"])
    return MoltenRuntime().compile(compile_graph(g, dtype=dt)[0])


INPUTS = {
    "matvec_q4": ("x", "qweight", "scales", "zeros"),
    "rope": ("x", "cos", "sin", "positions"),
    "window_attention": ("q", "k", "v", "lengths"),
    "sample": ("logits", "u", "temperature", "top_k", "top_p", "min_p"),
}


# --------------------------------------------------------------------- run
def run(state):
    op = state["case"]["op"]
    if own:
        return state["fn"](*(state[name] for name in INPUTS[op] if name in state))
    return PLAIN[op](state)


def _plain_q4(state):
    case, qw = state["case"], state["qweight"]
    q = torch.stack((qw & 15, qw >> 4), -1).view(case["n"], -1, case["group"]).float()
    zero = state["zeros"].float()[:, :, None] if case["zeros"] else 8.0
    w = ((q - zero) * state["scales"].float()[:, :, None]).view(case["n"], case["k"])
    return (state["x"].float() @ w.t()).to(state["x"].dtype)


def _plain_rope(state):
    case, x = state["case"], state["x"].float()
    sizes = torch.tensor(_sections(case), device=x.device)
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=x.device), sizes,
                                   output_size=case["dim"] // 2)
    rows = state["positions"].long()[axis].permute(1, 2, 0)              # [batch, seq, pair]
    pair = torch.arange(case["dim"] // 2, device=x.device)
    c, s = state["cos"][rows, pair][:, :, None], state["sin"][rows, pair][:, :, None]
    if case["style"] == "half":
        a, b = x.chunk(2, -1)
        out = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        out = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return out.to(state["x"].dtype)


def _plain_attention(state):
    case, q = state["case"], state["q"]
    b, new, heads, d = q.shape
    cache, kv = case["cache"], case["kv_heads"]
    per = heads // kv
    qs = q.float().view(b, new, kv, per, d).permute(0, 2, 3, 1, 4).reshape(b, kv, per * new, d)
    ks = state["k"].float().permute(0, 2, 3, 1)
    vs = state["v"].float().permute(0, 2, 1, 3)
    n = state["lengths"].long()[:, None, None]
    at = n - new + torch.arange(new, device=q.device)[:, None]
    key = torch.arange(cache, device=q.device)
    seen = (key <= at) & (key < n) & ((key > at - case["window"]) | (key < case["sinks"]))
    s = torch.matmul(qs, ks).view(b, kv, per, new, cache).mul_(d ** -0.5)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, kv, per * new, cache), vs).view(b, kv, per, new, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(b, new, heads, d).to(q.dtype)


def _plain_sample(state):
    # 64 bits: whether a token lies on this or that side of a border is the result
    case, x = state["case"], state["logits"].double()
    vocab = case["vocab"]
    t = state["temperature"].double()[:, None]
    y, order = torch.sort(x / t, dim=-1, descending=True, stable=True)
    w = torch.exp(y - y[:, :1])
    keep = torch.ones_like(w, dtype=torch.bool)
    if case["top_k"]:
        k = state["top_k"].long()[:, None]
        keep &= (torch.arange(vocab, device=x.device) < k) | (k <= 0)
        w = w * keep
    if case["top_p"]:
        p = state["top_p"].double()[:, None]
        before = w.cumsum(-1) - w
        keep &= (before < p * w.sum(-1, keepdim=True)) | (p >= 1)
    if case["min_p"]:
        keep &= w >= state["min_p"].double()[:, None]
    kept = torch.zeros_like(w).scatter_(-1, order, w * keep)
    cum = kept.cumsum(-1)
    goal = state["u"].double()[:, None] * cum[:, -1:]
    return (cum <= goal).sum(-1).to(torch.int32)


PLAIN = {"matvec_q4": _plain_q4, "rope": _plain_rope, "window_attention": _plain_attention,
         "sample": _plain_sample}


# -------------------------------------------------------------------- work
def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "matvec_q4":
        m, n, k = case["m"], case["n"], case["k"]
        groups = n * (k // case["group"]) * (2 if case["zeros"] else 1)
        return {"bytes": n * k // 2 + groups * size + (m * k + m * n) * size, "flops": 2 * m * n * k}
    if case["op"] == "rope":
        tokens = case["batch"] * case["seq"]
        x = tokens * case["heads"] * case["dim"]
        rows = min(tokens, case["table"])
        return {"bytes": 2 * x * size + 4 * case["axes"] * tokens + 4 * rows * case["dim"],
                "flops": 3 * x}
    if case["op"] == "window_attention":
        read = pairs = 0
        for n in _lengths(case):
            at = np.arange(n - case["new"], n)
            first = np.maximum(at - case["window"] + 1, 0)
            pairs += int((at - first + 1 + np.minimum(first, case["sinks"])).sum())
            read += int(n - first[0] + min(first[0], case["sinks"]))
        q = case["batch"] * case["new"] * case["heads"] * case["dim"]
        return {"bytes": (2 * q + 2 * read * case["kv_heads"] * case["dim"]) * size,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + 24 * case["rows"], "flops": 2 * n}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    return EXACT[case["op"]](case, prepare(case, seed))


def _exact_q4(case, state):
    q = torch.empty(case["n"], case["k"], dtype=torch.float64, device=DEVICE)
    q[:, 0::2] = state["qweight"] % 16
    q[:, 1::2] = state["qweight"] // 16
    spread = [state["scales"].double().repeat_interleave(case["group"], 1)]
    q -= state["zeros"].double().repeat_interleave(case["group"], 1) if case["zeros"] else 8
    q *= spread.pop()
    return torch.einsum("mk,nk->mn", state["x"].double(), q)


def _exact_rope(case, state):
    x = state["x"].double()
    half = case["dim"] // 2
    z = torch.empty(*x.shape[:3], half, dtype=torch.complex128, device=DEVICE)
    pairs = x.view(*x.shape[:3], 2, half) if case["style"] == "half" \
        else x.view(*x.shape[:3], half, 2).transpose(-1, -2)
    z.real, z.imag = pairs[..., 0, :], pairs[..., 1, :]
    start = 0
    for axis, width in enumerate(_sections(case)):
        part = slice(start, start + width)
        at = state["positions"][axis].long().flatten()
        turn = torch.complex(state["cos"][at, part].double(), state["sin"][at, part].double())
        z[..., part] *= turn.view(*x.shape[:2], 1, width)
        start += width
    parts = torch.stack((z.real, z.imag), -2)
    return (parts if case["style"] == "half" else parts.transpose(-1, -2)).reshape(x.shape)


def _exact_attention(case, state):
    per, new, d = case["heads"] // case["kv_heads"], case["new"], case["dim"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(_lengths(case)):
        i = torch.arange(n - new, n, device=DEVICE).view(1, -1, 1)
        j = torch.arange(n, device=DEVICE).view(1, 1, -1)
        hidden = (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
        for h in range(case["kv_heads"]):
            q = state["q"][b, :, h * per:(h + 1) * per].double().transpose(0, 1)
            s = q @ state["k"][b, :n, h].double().t() / math.sqrt(d)
            p = torch.softmax(s.masked_fill_(hidden, -math.inf), -1)
            out[b, :, h * per:(h + 1) * per] = (p @ state["v"][b, :n, h].double()).transpose(0, 1)
    return out


def _exact_sample(case, state):
    host = {k: v.double().cpu().numpy() for k, v in state.items() if torch.is_tensor(v)}
    tokens = np.zeros(case["rows"], dtype=np.int32)
    for r in range(case["rows"]):
        x = host["logits"][r]
        order = np.argsort(-x, kind="stable")
        w = np.exp((x[order] - x[order[0]]) / host["temperature"][r])
        count = w.size
        if case["top_k"] and host["top_k"][r] > 0:
            count = min(count, int(host["top_k"][r]))
        if case["top_p"] and host["top_p"][r] < 1:
            reach = np.cumsum(w[:count])
            count = int(np.searchsorted(reach, host["top_p"][r] * reach[-1], side="left")) + 1
        if case["min_p"]:
            count = min(count, int(np.sum(w >= host["min_p"][r])))
        chosen = np.sort(order[:count])
        v = np.exp((x[chosen] - x[order[0]]) / host["temperature"][r])
        reach = np.cumsum(v)
        tokens[r] = chosen[np.searchsorted(reach, host["u"][r] * reach[-1], side="right")]
    return torch.from_numpy(tokens)


EXACT = {"matvec_q4": _exact_q4, "rope": _exact_rope, "window_attention": _exact_attention,
         "sample": _exact_sample}
