"""e4m3 caches for the tests of the quantised append and attention."""
from __future__ import annotations

import torch

import quant_reference as quant
import serving_reference as ref


def quantised(x, order="phs"):
    """(codes, scales) of the rows of a cache [pages, page, heads, D]; NaN rows become NaN codes and
    scales.  `order` names the scales' memory order: p(age), s(lot), h(ead)."""
    y = x.double()
    scale = (y.abs().amax(-1).clamp_min(quant.MIN_AMAX) / quant.MAX).float()
    codes = (y / scale.double()[..., None]).clamp(-quant.MAX, quant.MAX).float().to(quant.E4M3)
    dims = ["psh".index(c) for c in order]
    scale = scale.permute(dims).contiguous().permute([dims.index(d) for d in range(3)])
    return codes, scale


def values(codes, scale):
    """What the codes stand for, in 64 bits."""
    return codes.double() * scale.double()[..., None]


def paged_inputs(*args, order="phs", spread=0, **kw):
    """serving_reference.paged_inputs with e4m3 caches: q, k_cache, v_cache, k_scale, v_scale, table,
    q_start, kv_len.  `spread`: the values' rows are scaled by 2^-spread .. 2^spread."""
    q, kc, vc, *rest = ref.paged_inputs(*args, **kw)
    if spread:
        g = torch.Generator(device=kc.device).manual_seed(9)
        e = torch.randint(-spread, spread + 1, vc.shape[:3], device=kc.device, generator=g)
        vc = vc.double() * 2.0 ** e[..., None].double()
    (k8, ks), (v8, vs) = quantised(kc, order), quantised(vc, order)
    return (q, k8, v8, ks, vs, *rest)


def attend(x, scale, softcap=0.0, window=0):
    """(out, sum_j p_j |v_j|) in 64 bits."""
    q, k8, v8, ks, vs, *rest = x
    return ref.paged_attention(q, values(k8, ks), values(v8, vs), *rest, scale, softcap, window)


def attention_close(got, x, scale, softcap=0.0, window=0):
    """serving_reference.attention_close for each sequence, on what the codes and scales stand for.
    Sequences of many query rows take values rounded to f16 (after a division by a power of two):
    beside bf16's half step that is nothing; f16 sequences may be close to the formula on such values."""
    q, k8, v8, ks, vs, table, q_start, kv_len = x
    want, size = attend(x, scale, softcap, window)
    if q.dtype != torch.float16:
        return ref.attention_close(got, want, size, q.dtype)
    near, near_size = ref.paged_attention(q, values(k8, ks), values(v8, vs).half(), table, q_start, kv_len, scale, softcap, window)
    starts = q_start.tolist()
    for a, b in zip([0, *starts], [*starts, len(q)]):
        if a == b:
            continue
        try:
            ref.attention_close(got[a:b], want[a:b], size[a:b], q.dtype)
        except AssertionError:
            ref.attention_close(got[a:b], near[a:b], near_size[a:b], q.dtype)
