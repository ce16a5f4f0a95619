"""Cases that measure the operators of a decoder layer's serving step over a paged key/value cache:
the residual's addition with the RMS norm (16-bit or 8-bit output), the rotary embedding with the
append to the cache, and the attention that reads the cache.

`run` computes a case in plain torch operations where `own` is false, and through the library's
operators (torch.ops.b200.*) where it is true.
"""
import math
import os
import random
import sys

import torch

own = False

E4M3_MAX = 448.0
MIN_AMAX = 1e-12  # the smallest absolute maximum that a scale is made of
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------- cases
def _norm(name, rows, cols, dtype="bf16", quant="none"):
    return {"name": name, "op": "add_rms_norm", "rows": rows, "cols": cols, "dtype": dtype, "quant": quant}


def _append(name, tokens, heads, kv_heads, dim, rot, page, dtype="bf16", fused=True):
    return {"name": name, "op": "rope_append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "page": page, "dtype": dtype, "fused": fused}


def _attn(name, seqs, q, kv, heads, kv_heads, dim, page, dtype="bf16", ragged=True, softcap=0.0, window=0, pad=0):
    return {"name": name, "op": "paged_attention", "seqs": seqs, "q": q, "kv": kv, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "softcap": softcap,
            "window": window, "pad": pad}


def listed():
    return [
        # one sequence's single token between two sublayers of the Llama-style model (width 2048)
        _norm("norm_token", 1, 2048),
        # its prefill at the benchmark's row chain size, 16-bit output
        _norm("norm_prefill", 16384, 8192),
        # an odd batch of tokens before an 8-bit product with one scale a row
        _norm("norm_rowquant", 777, 4096, "bf16", "row"),
        # a prompt before an 8-bit product with one scale for 128 columns, fp16
        _norm("norm_groupquant", 8192, 4096, "f16", "group"),
        # a step of 64 sequences, one token each, q / k / v as columns of one projection's output
        _append("append_step", 64, 32, 8, 128, 128, 16),
        # the prefill of the Llama-style model (8 prompts of 2048 tokens, 32 / 8 heads of 64)
        _append("append_prefill", 16384, 32, 8, 64, 64, 64, "bf16", False),
        # one chat: a single token over a short context (32 / 8 heads of 64)
        _attn("decode_one", 1, 1, 700, 32, 8, 64, 16, ragged=False),
        # a serving batch: 64 sequences of ragged lengths to 8192, heads of 128
        _attn("decode_batch", 64, 1, 8192, 32, 8, 128, 16),
        # few long contexts, capped scores, fp16
        _attn("decode_long", 3, 1, 65536, 16, 8, 128, 64, "f16", softcap=50.0),
        # tokens proposed ahead: 4 queries a sequence, every head its own keys, a sliding window
        _attn("verify_window", 16, 4, 3000, 16, 16, 128, 32, window=1024),
        # the prefill of the Llama-style model: 8 prompts of 2048
        _attn("prefill", 8, 2048, 2048, 32, 8, 64, 64, ragged=False),
        # chunks of prompts behind earlier context, ragged, with padded rows behind the last sequence
        _attn("prefill_chunks", 5, 1024, 6000, 32, 8, 128, 16, pad=37),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["add_rms_norm", "rope_append", "paged_attention", "paged_attention"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "add_rms_norm":
        quant = rng.choice(["none", "row", "group"])
        cols = _log(rng, 256, 16384)
        if quant == "group":
            cols = max(128, cols // 128 * 128)
        elif rng.random() < 0.7:
            cols = cols // 8 * 8
        rows = _log(rng, 1, min(16384, 16384 * 8192 // cols))
        c = _norm("", rows, cols, dtype, quant)
    elif op == "rope_append":
        heads, kv = rng.choice([(32, 8), (32, 32), (16, 2), (8, 1), (28, 4), (64, 8)])
        dim = rng.choice([64, 128])
        tokens = _log(rng, 1, 16384 * 2048 // (heads * dim))
        c = _append("", tokens, heads, kv, dim, rng.choice([dim, dim, dim // 2]), rng.choice([1, 16, 24, 32, 64, 128]),
                    dtype, rng.random() < 0.5)
    else:
        heads, kv = rng.choice([(32, 8), (16, 16), (16, 2), (8, 1), (28, 4), (64, 8)])
        dim = rng.choice([64, 128])
        page = rng.choice([1, 16, 24, 32, 64, 128])
        softcap = rng.choice([0.0, 0.0, 30.0, 50.0])
        window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
        kind = rng.choice(["one", "one", "few", "many"])
        if kind == "many":
            seqs = _log(rng, 1, 8)
            q = _log(rng, 9, 2048)
            kv_len = min(8192, q + (0 if rng.random() < 0.4 else _log(rng, 1, 6000)))
            q = min(q, max(9, 8 * 2048 * 2048 * 32 // (seqs * heads * kv_len)))  # the plain form's scores
        else:
            q = 1 if kind == "one" else rng.randint(2, 8)
            seqs = _log(rng, 1, 128)
            kv_len = max(q, _log(rng, 16, min(65536, 64 * 8192 * 1024 // (seqs * kv * dim))))
        c = _attn("", seqs, q, kv_len, heads, kv, dim, page, dtype, rng.random() < 0.7, softcap, window,
                  rng.choice([0, 0, rng.randint(1, 64)]))
    del c["name"]
    return c


def _lengths(c):
    """(queries, keys) of each sequence: the same for every seed, ragged ones between a quarter and the whole."""
    qs, ns = [], []
    for i in range(c["seqs"]):
        f = 1.0 if not c["ragged"] or i == 0 else 0.25 + 0.75 * ((i * 0.6180339887) % 1.0)
        q = max(1, round(c["q"] * f))
        qs.append(q)
        ns.append(max(q, round(c["kv"] * f)))
    return qs, ns


# ----------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, dtype=dt, generator=g)

    s = {"case": case}
    if case["op"] == "add_rms_norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = randn(rows, cols)
        s["residual"] = randn(rows, cols) * 2
        s["residual"][:, 5::97] *= 12  # the few large channels that trained models have
        s["weight"] = (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(dt)
        s["eps"] = 1e-5
    elif case["op"] == "rope_append":
        t, h, kv, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        if case["fused"]:
            qkv = randn(t, (h + 2 * kv) * d)
            s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], 1))
        else:
            s["q"], s["k"], s["v"] = randn(t, h, d), randn(t, kv, d), randn(t, kv, d)
        reach = 4096
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
        angles = torch.arange(reach, device=DEV, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
        pages = -(-t // page) + 3
        s["positions"] = torch.randint(0, reach, (t,), device=DEV, generator=g)
        order = torch.randperm(pages, device=DEV, generator=g)
        at = torch.arange(t, device=DEV)
        s["slots"] = order[at // page] * page + at % page
        s["k_cache"], s["v_cache"] = randn(pages, page, kv, d), randn(pages, page, kv, d)
    else:
        h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        qs, ns = _lengths(case)
        both = list(zip(qs, ns))
        random.Random(seed).shuffle(both)
        qs, ns = [x for x, _ in both], [x for _, x in both]
        used = [-(-n // page) for n in ns]
        pages = sum(used) + 2
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        table = torch.zeros(len(ns), max(used), dtype=torch.int32)
        first = 0
        for b, n in enumerate(used):
            table[b, :n] = order[first:first + n]
            first += n
        s["q"] = randn(sum(qs) + case["pad"], h, d) * 1.5
        s["k_cache"], s["v_cache"] = randn(pages, page, kv, d), randn(pages, page, kv, d)
        s["page_table"] = table.to(DEV)
        starts = [0]
        for q in qs:
            starts.append(starts[-1] + q)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor(ns, dtype=torch.int32, device=DEV)
        s["max_q"], s["max_kv"] = max(qs), max(ns)
        s["scale"] = d ** -0.5
    return s


# --------------------------------------------------------------------- run
_ops = None


def _library():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "torch-compile-backend_b200"))
        from compiler import runtime

        runtime.load()
        _ops = torch.ops.b200
    return _ops


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](_library(), state)
    return _PLAIN[op](state)


def _own_norm(ops, s):
    quant = s["case"]["quant"]
    if quant == "none":
        out, total = ops.add_rms_norm(s["x"], s["residual"], s["weight"], s["eps"])
        return {"out": out, "sum": total}
    out, scale, total = ops.add_rms_norm_quant(s["x"], s["residual"], s["weight"], s["eps"],
                                               128 if quant == "group" else 0)
    return {"out": out, "scale": scale, "sum": total}


def _own_append(ops, s):
    q = ops.rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"],
                        s["v_cache"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(ops, s):
    c = s["case"]
    return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["q_start"], s["kv_len"],
                               s["scale"], c["softcap"], c["window"], s["max_q"])


def _plain_norm(s):
    quant = s["case"]["quant"]
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    h = total.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    if quant == "none":
        return {"out": y.to(total.dtype), "sum": total}
    if quant == "group":
        y = y.unflatten(-1, (-1, 128))
    scale = y.abs().amax(-1, keepdim=True).clamp_min(MIN_AMAX) / E4M3_MAX
    out = (y / scale).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return {"out": out.flatten(1), "scale": scale.flatten(1), "sum": total}


def _rotate(x, cos, sin, rot):
    """Rotary embedding of x [t, heads, d] in 32 bits: the first `rot` columns, by halves."""
    x = x.float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_append(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    dt = s["q"].dtype
    q = _rotate(s["q"], cos, sin, c["rot"]).to(dt)
    s["k_cache"].flatten(0, 1)[s["slots"]] = _rotate(s["k"], cos, sin, c["rot"]).to(dt)
    s["v_cache"].flatten(0, 1)[s["slots"]] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(s):
    c = s["case"]
    t, h, d = s["q"].shape
    kv, page, group = c["kv_heads"], c["page"], h // c["kv_heads"]
    start, n = s["q_start"].long(), s["kv_len"].long()
    m = start[1:] - start[:-1]
    # keys and values of each sequence, by its pages: [seqs, kv heads, keys, d]
    key = torch.arange(s["max_kv"], device=DEV)
    slot = s["page_table"].long()[:, key // page] * page + key % page
    k = s["k_cache"].flatten(0, 1)[slot].float().transpose(1, 2)
    v = s["v_cache"].flatten(0, 1)[slot].float().transpose(1, 2)
    # queries, padded to the longest: [seqs, kv heads, queries, group, d]
    i = torch.arange(s["max_q"], device=DEV)
    token = (start[:-1, None] + i).clamp_max(t - 1)
    q = s["q"][token].float().unflatten(2, (kv, group)).transpose(1, 2)
    x = (q.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (-1, group)) * s["scale"]
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    at = (n - m)[:, None] + i  # each query's position
    seen = key <= at[:, :, None]
    if c["window"]:
        seen &= key > at[:, :, None] - c["window"]
    x = x.masked_fill(~seen[:, None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, group)).transpose(1, 2).flatten(2, 3)
    # back to one row a token; rows behind the last sequence are zero
    row = torch.arange(t, device=DEV)
    b = torch.searchsorted(start[1:], row, right=True).clamp_max(c["seqs"] - 1)
    o = o[b, (row - start[b]).clamp_max(s["max_q"] - 1)]
    return (o * (row < start[-1])[:, None, None]).to(s["q"].dtype)


_OWN = {"add_rms_norm": _own_norm, "rope_append": _own_append, "paged_attention": _own_attention}
_PLAIN = {"add_rms_norm": _plain_norm, "rope_append": _plain_append, "paged_attention": _plain_attention}


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "add_rms_norm":
        n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
        scales = {"none": 0, "row": rows, "group": n // 128}[case["quant"]]
        return {"bytes": 2 * n * 3 + 2 * cols + (2 if case["quant"] == "none" else 1) * n + 4 * scales, "flops": 6 * n}
    if case["op"] == "rope_append":
        t, d, h, kv = case["tokens"], case["dim"], case["heads"], case["kv_heads"]
        tables = min(t, 4096) * case["rot"] * 4
        return {"bytes": 2 * t * d * 2 * (h + 2 * kv) + tables + 16 * t, "flops": 3 * t * case["rot"] * (h + kv)}
    qs, ns = _lengths(case)
    h, kv, d, w = case["heads"], case["kv_heads"], case["dim"], case["window"]
    keys = pairs = 0
    for m, n in zip(qs, ns):
        first = n - m  # the first query's position
        keys += n if not w else n - max(0, first - w + 1)
        if not w:
            pairs += m * first + m * (m + 1) // 2
        else:
            short = min(m, max(0, w - 1 - first))  # queries that see less than a whole window
            pairs += (m - short) * w + short * first + short * (short + 1) // 2
    t = sum(qs)
    pages = sum(-(-n // case["page"]) for n in ns)
    return {"bytes": 2 * (2 * t * h * d + 2 * keys * kv * d) + 4 * pages + 8 * len(qs), "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The definition in 64 bits, one sequence (or block of rows) at a time."""
    s = prepare(case, seed)
    if case["op"] == "add_rms_norm":
        return _exact_norm(case, s)
    if case["op"] == "rope_append":
        return _exact_append(case, s)
    return _exact_attention(case, s)


def _exact_norm(case, s):
    outs, scales, sums = [], [], []
    for x, r in zip(s["x"].split(1024), s["residual"].split(1024)):
        total = (x.double() + r.double()).to(x.dtype)  # the sum is stored in 16 bits, and what is stored is normed
        h = total.double()
        y = h / torch.sqrt(torch.mean(h.square(), 1, keepdim=True) + s["eps"]) * s["weight"].double()
        sums.append(total)
        if case["quant"] == "none":
            outs.append(y)
            continue
        parts = y.reshape(y.shape[0], -1, 128 if case["quant"] == "group" else y.shape[1])
        top = parts.abs().max(2, keepdim=True).values.clamp(min=MIN_AMAX)
        scales.append((top / E4M3_MAX).squeeze(2))
        outs.append((parts * (E4M3_MAX / top)).reshape(y.shape))
    out = {"out": torch.cat(outs), "sum": torch.cat(sums)}
    if scales:
        out["scale"] = torch.cat(scales)
    return out


def _exact_append(case, s):
    half = case["rot"] // 2
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]

    def turned(x):
        x = x.double()
        z = torch.complex(x[:, :, :half].contiguous(), x[:, :, half:2 * half].contiguous())
        z = z * torch.complex(cos, sin)[:, None, :]
        return torch.cat([z.real, z.imag, x[:, :, 2 * half:]], 2)

    caches = {}
    for name, rows in (("k_cache", turned(s["k"])), ("v_cache", s["v"].double())):
        c = s[name].double()
        page, offset = s["slots"] // case["page"], s["slots"] % case["page"]
        c[page, offset] = rows
        caches[name] = c
    return {"q": turned(s["q"]), **caches}


def _exact_attention(case, s):
    starts, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["page_table"].tolist()
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        pages = table[b][:-(-n // case["page"])]
        k = s["k_cache"][pages].reshape(-1, *s["k_cache"].shape[2:])[:n].double()
        v = s["v_cache"][pages].reshape(-1, *s["v_cache"].shape[2:])[:n].double()
        m = starts[b + 1] - starts[b]
        for lo in range(0, m, 256):
            hi = min(m, lo + 256)
            at = torch.arange(n - m + lo, n - m + hi, device=DEV)
            keys = torch.arange(n, device=DEV)
            hide = keys[None, :] > at[:, None]
            if case["window"]:
                hide |= keys[None, :] <= at[:, None] - case["window"]
            q = s["q"][starts[b] + lo:starts[b] + hi].double()
            for j in range(case["kv_heads"]):
                x = torch.einsum("thd,nd->htn", q[:, j * group:(j + 1) * group], k[:, j]) * s["scale"]
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                p = torch.softmax(x.masked_fill(hide, -math.inf), 2)
                out[starts[b] + lo:starts[b] + hi, j * group:(j + 1) * group] = torch.einsum("htn,nd->thd", p, v[:, j])
    return out
