"""Cases that measure the 8-bit operators of a decoder layer's serving step: the product of e4m3
operands with a scale for each block of 128, the quantisation of the activations that enter it, the
append of rotated keys and values to an e4m3 cache, and the attention that reads such a cache.

`run` computes a case in plain torch operations where `own` is false, and through the library's
operators (torch.ops.b200.*) where it is true.
"""
import math
import os
import random
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_AMAX = 1e-12  # the smallest absolute maximum that a scale is made of
BLOCK = 128       # columns that share a scale
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"


# ------------------------------------------------------------------- cases
def _mm(name, m, k, n, out="bf16"):
    return {"name": name, "op": "scaled_mm", "m": m, "k": k, "n": n, "dtype": out}


def _quant(name, rows, cols, dtype="bf16", swiglu=False):
    return {"name": name, "op": "quant_groups", "rows": rows, "cols": cols, "dtype": dtype, "swiglu": swiglu}


def _append(name, tokens, heads, kv_heads, dim, rot, page, dtype="bf16", fused=True):
    return {"name": name, "op": "rope_append_quant", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "page": page, "dtype": dtype, "fused": fused}


def _attn(name, seqs, q, kv, heads, kv_heads, dim, page, dtype="bf16", ragged=True, softcap=0.0, window=0, pad=0):
    return {"name": name, "op": "paged_attention_quant", "seqs": seqs, "q": q, "kv": kv, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "softcap": softcap,
            "window": window, "pad": pad}


def listed():
    return [
        # one sequence's single token through the down projection of the Llama-style model (ffn 8192, width 2048)
        _mm("mm_token", 1, 8192, 2048),
        # a step of 64 sequences through the gate projection of a model of width 4096
        _mm("mm_batch", 64, 4096, 14336),
        # an odd batch of tokens, rows and columns that end inside a block, fp16
        _mm("mm_ragged", 777, 2064, 4100, "f16"),
        # a prompt batch at the benchmark's dominant product
        _mm("mm_prefill", 16384, 4096, 14336),
        # the attention's output of a step of 64 sequences, before its projection
        _quant("quant_step", 64, 4096),
        # gate and up of a prompt batch, before the down projection (the benchmark's rows)
        _quant("quant_swiglu", 16384, 8192, "bf16", True),
        # a step of 64 sequences, one token each, q / k / v as columns of one projection's output
        _append("append_step", 64, 32, 8, 128, 128, 16),
        # the prefill of the Llama-style model (8 prompts of 2048 tokens, 32 / 8 heads of 64)
        _append("append_prefill", 16384, 32, 8, 64, 64, 64, "bf16", False),
        # one chat: a single token over a short context (32 / 8 heads of 64)
        _attn("decode_one", 1, 1, 700, 32, 8, 64, 16, ragged=False),
        # a serving batch: 64 sequences of ragged lengths to 8192, heads of 128
        _attn("decode_batch", 64, 1, 8192, 32, 8, 128, 16),
        # tokens proposed ahead: 4 queries a sequence, capped scores in a sliding window, fp16
        _attn("verify_window", 16, 4, 3000, 16, 2, 128, 32, "f16", softcap=50.0, window=1024),
        # chunks of prompts behind earlier context, ragged, with padded rows behind the last sequence
        _attn("prefill_chunks", 5, 1024, 6000, 32, 8, 128, 16, pad=37),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["scaled_mm", "scaled_mm", "quant_groups", "rope_append_quant", "paged_attention_quant",
                     "paged_attention_quant"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "scaled_mm":
        k = _log(rng, 256, 16384)
        k = k // 16 * 16 if rng.random() < 0.4 else max(128, k // 128 * 128)
        n = _log(rng, 64, 32768)
        if rng.random() < 0.7:
            n = max(64, n // 64 * 64)
        m = _log(rng, 1, min(16384, 16384 * 4096 * 14336 // (k * n)))
        c = _mm("", m, k, n, rng.choice([dtype, dtype, dtype, "f32"]))
    elif op == "quant_groups":
        cols = _log(rng, 256, 16384)
        if rng.random() < 0.7:
            cols = cols // 128 * 128
        c = _quant("", _log(rng, 1, min(16384, 16384 * 8192 // cols)), cols, dtype, rng.random() < 0.5)
    elif op == "rope_append_quant":
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
def _quantised(x):
    """(codes, scales) of x's last dim in groups of 128, the last group what is left of it: what an earlier
    step, or the loading of a checkpoint, leaves."""
    cols = x.shape[-1]
    y = torch.nn.functional.pad(x.float(), (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    scale = y.abs().amax(-1, keepdim=True).clamp_min(MIN_AMAX) / E4M3_MAX
    return (y / scale).clamp(-E4M3_MAX, E4M3_MAX).flatten(-2)[..., :cols].to(E4M3), scale.squeeze(-1)


def _cache(pages, page, kv, d, g):
    """An e4m3 cache [pages, page, kv heads, d] and its scales, [pages, page, kv heads] with the places of a
    page side by side, filled by earlier steps."""
    codes = torch.empty(pages, page, kv, d, device=DEV, dtype=E4M3)
    scale = torch.empty(pages, kv, page, device=DEV).transpose(1, 2)
    step = max(1, (1 << 27) // (page * kv * d))
    for lo in range(0, pages, step):
        x = torch.randn(min(step, pages - lo), page, kv, d, device=DEV, generator=g)
        top = x.abs().amax(-1, keepdim=True) / E4M3_MAX
        codes[lo:lo + step] = (x / top).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
        scale[lo:lo + step] = top.squeeze(-1)
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, dtype=dt, generator=g)

    s = {"case": case}
    if case["op"] == "scaled_mm":
        m, k, n = case["m"], case["k"], case["n"]
        x = torch.randn(m, k, device=DEV, generator=g)
        x[:, 5::97] *= 12  # the few large channels that trained models have
        s["a"], s["a_scale"] = _quantised(x)
        del x
        # a linear layer's weight [n, k], with one scale for each 128 x 128 block of it
        w = torch.randn(n, k, device=DEV, generator=g) * k ** -0.5
        w = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))
        top = w.abs().amax((1, 3), keepdim=True) / E4M3_MAX
        w = (w / top).clamp(-E4M3_MAX, E4M3_MAX).flatten(2).flatten(0, 1)[:n, :k].to(E4M3).contiguous()
        s["b"], s["b_scale"] = w.t(), top.squeeze(3).squeeze(1).t()
    elif case["op"] == "quant_groups":
        s["x"] = randn(case["rows"], case["cols"] * (2 if case["swiglu"] else 1))
        s["x"][:, 5::97] *= 12
    elif case["op"] == "rope_append_quant":
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
        s["k_cache"], s["k_scale"] = _cache(pages, page, kv, d, g)
        s["v_cache"], s["v_scale"] = _cache(pages, page, kv, d, g)
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
        s["k_cache"], s["k_scale"] = _cache(pages, page, kv, d, g)
        s["v_cache"], s["v_scale"] = _cache(pages, page, kv, d, g)
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


def _own_mm(ops, s):
    return ops.scaled_mm(s["a"], s["b"], s["a_scale"], s["b_scale"], DTYPES[s["case"]["dtype"]])


def _own_quant(ops, s):
    out, scale = ops.quant_groups(s["x"], s["case"]["swiglu"])
    return {"out": out, "scale": scale}


def _own_append(ops, s):
    q = ops.rope_append_quant(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"], s["k_cache"],
                              s["v_cache"], s["k_scale"], s["v_scale"])
    return {"q": q, **{name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _own_attention(ops, s):
    c = s["case"]
    return ops.paged_attention_quant(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["page_table"],
                                     s["q_start"], s["kv_len"], s["scale"], c["softcap"], c["window"], s["max_q"])


def _plain_mm(s):
    (m, k), n = s["a"].shape, s["b"].shape[1]
    a = s["a"].float() * s["a_scale"].repeat_interleave(BLOCK, 1)[:, :k]
    b = s["b"].float() * s["b_scale"].repeat_interleave(BLOCK, 0)[:k].repeat_interleave(BLOCK, 1)[:, :n]
    return (a @ b).to(DTYPES[s["case"]["dtype"]])


def _plain_quant(s):
    y = s["x"].float()
    if s["case"]["swiglu"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    cols = y.shape[-1]
    y = torch.nn.functional.pad(y, (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    scale = y.abs().amax(-1, keepdim=True).clamp_min(MIN_AMAX) / E4M3_MAX
    out = (y / scale).clamp(-E4M3_MAX, E4M3_MAX).flatten(1)[:, :cols].to(E4M3)
    return {"out": out, "scale": scale.squeeze(-1)}


def _rotate(x, cos, sin, rot):
    """Rotary embedding of x [t, heads, d] in 32 bits: the first `rot` columns, by halves."""
    x = x.float()
    a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _store(cache, scales, slots, x):
    """The rows x [t, kv heads, d] to their slots, each in 8 bits with its own scale."""
    scale = x.abs().amax(-1, keepdim=True).clamp_min(MIN_AMAX) / E4M3_MAX
    codes = (x / scale).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    page = cache.shape[1]
    cache.view(torch.uint8)[slots // page, slots % page] = codes.view(torch.uint8)
    scales[slots // page, slots % page] = scale.squeeze(-1)


def _plain_append(s):
    rot = s["case"]["rot"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _rotate(s["q"], cos, sin, rot).to(s["q"].dtype)
    _store(s["k_cache"], s["k_scale"], s["slots"], _rotate(s["k"], cos, sin, rot))
    _store(s["v_cache"], s["v_scale"], s["slots"], s["v"].float())
    return {"q": q, **{name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _plain_attention(s):
    c = s["case"]
    t, h, d = s["q"].shape
    kv, page, group = c["kv_heads"], c["page"], h // c["kv_heads"]
    start, n = s["q_start"].long(), s["kv_len"].long()
    m = start[1:] - start[:-1]
    # keys and values of each sequence, by its pages: [seqs, kv heads, keys, d]
    key = torch.arange(s["max_kv"], device=DEV)
    pages, place = s["page_table"].long()[:, key // page], key % page

    def rows(name):
        codes = s[name + "_cache"].view(torch.uint8)[pages, place].view(E4M3)
        return (codes.float() * s[name + "_scale"][pages, place][..., None]).transpose(1, 2)

    k, v = rows("k"), rows("v")
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


_OWN = {"scaled_mm": _own_mm, "quant_groups": _own_quant, "rope_append_quant": _own_append,
        "paged_attention_quant": _own_attention}
_PLAIN = {"scaled_mm": _plain_mm, "quant_groups": _plain_quant, "rope_append_quant": _plain_append,
          "paged_attention_quant": _plain_attention}


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "scaled_mm":
        m, k, n, groups = case["m"], case["k"], case["n"], -(-case["k"] // BLOCK)
        out = 4 if case["dtype"] == "f32" else 2
        return {"bytes": m * k + k * n + 4 * groups * (m + -(-n // BLOCK)) + out * m * n, "flops": 2 * m * n * k}
    if case["op"] == "quant_groups":
        n = case["rows"] * case["cols"]
        wide = 2 if case["swiglu"] else 1
        return {"bytes": 2 * wide * n + n + 4 * case["rows"] * -(-case["cols"] // BLOCK), "flops": (7 if wide == 2 else 3) * n}
    if case["op"] == "rope_append_quant":
        t, d, h, kv = case["tokens"], case["dim"], case["heads"], case["kv_heads"]
        tables = min(t, 4096) * case["rot"] * 4
        return {"bytes": t * d * (4 * h + 6 * kv) + 8 * t * kv + tables + 16 * t,
                "flops": 3 * t * case["rot"] * (h + kv) + 3 * t * d * 2 * kv}
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
    return {"bytes": 2 * 2 * t * h * d + 2 * keys * kv * (d + 4) + 4 * pages + 8 * len(qs), "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The definition in 64 bits, a block of rows or one sequence at a time."""
    s = prepare(case, seed)
    return {"scaled_mm": _exact_mm, "quant_groups": _exact_quant, "rope_append_quant": _exact_append,
            "paged_attention_quant": _exact_attention}[case["op"]](case, s)


def _exact_mm(case, s):
    out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=DEV)
    for i, lo in enumerate(range(0, case["k"], BLOCK)):
        part = s["a"][:, lo:lo + BLOCK].double() @ s["b"][lo:lo + BLOCK].double()
        columns = s["b_scale"][i].double()[torch.arange(case["n"], device=DEV) // BLOCK]
        out += part * columns * s["a_scale"][:, i, None].double()
    return out


def _exact_rows(y):
    """(y over its scale, the scale) for the last dim."""
    top = y.abs().max(-1, keepdim=True).values.clamp(min=MIN_AMAX)
    return y * (E4M3_MAX / top), (top / E4M3_MAX).squeeze(-1)


def _exact_quant(case, s):
    outs, scales = [], []
    for x in s["x"].split(1024):
        y = x.double()
        if case["swiglu"]:
            y = y[:, :case["cols"]] * torch.sigmoid(y[:, :case["cols"]]) * y[:, case["cols"]:]
        parts = [_exact_rows(p) for p in y.split(BLOCK, 1)]
        outs.append(torch.cat([p for p, _ in parts], 1))
        scales.append(torch.stack([t for _, t in parts], 1))
    return {"out": torch.cat(outs), "scale": torch.cat(scales)}


def _exact_append(case, s):
    half = case["rot"] // 2
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]

    def turned(x):
        x = x.double()
        z = torch.complex(x[:, :, :half].contiguous(), x[:, :, half:2 * half].contiguous())
        z = z * torch.complex(cos, sin)[:, None, :]
        return torch.cat([z.real, z.imag, x[:, :, 2 * half:]], 2)

    out = {"q": turned(s["q"])}
    page, offset = s["slots"] // case["page"], s["slots"] % case["page"]
    for name, rows in (("k", turned(s["k"])), ("v", s["v"].double())):
        codes, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        codes[page, offset], scale[page, offset] = _exact_rows(rows)
        out[name + "_cache"], out[name + "_scale"] = codes, scale
    return {name: out[name] for name in ("q", "k_cache", "v_cache", "k_scale", "v_scale")}


def _exact_attention(case, s):
    starts, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["page_table"].tolist()
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        pages = torch.tensor(table[b][:-(-n // case["page"])], device=DEV)
        k, v = (s[c + "_cache"].view(torch.uint8)[pages].view(E4M3).double() * s[c + "_scale"][pages].double()[..., None]
                for c in "kv")
        k, v = k.flatten(0, 1)[:n], v.flatten(0, 1)[:n]
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
