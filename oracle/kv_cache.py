"""The quantized key/value cache and attention to it, in 64 bits, sequence by sequence (CPU restatement of the definitions in
rapid_h3_b200/kv_cache.py)."""
import math

import torch

from . import linear


def quantize(x, kind):
    """Codes and fp32 scales of rows x [..., D]: the arithmetic of the row quantizers; a row with a NaN or an infinity has codes 0 and a
    scale that is not finite."""
    flat = x.float().reshape(-1, x.shape[-1])
    finite = torch.isfinite(flat).all(1)
    q, s = linear.quantize_rows(torch.where(finite[:, None], flat, 0.0), "int8_rowwise" if kind == "int8" else "fp8_rowwise")
    s = torch.where(finite, s.reshape(-1), flat.abs().sum(1))
    return q.reshape(x.shape), s.reshape(x.shape[:-1])


def tokens(codes, scales, pages, n):
    """fp64 [n, heads, D] of the first n tokens of `pages`, and which of them exist."""
    page = codes.shape[2]
    out = torch.zeros(n, codes.shape[1], codes.shape[3], dtype=torch.float64)
    there = torch.zeros(n, dtype=torch.bool)
    for i in range(n):
        if i // page < len(pages) and 0 <= pages[i // page] < codes.shape[0]:
            at = pages[i // page], slice(None), i % page
            out[i] = codes.view(torch.uint8)[at].view(codes.dtype).double() * scales[at].double()[..., None]
            there[i] = True
    return out, there


def attention(q, cache, table, lens, starts, scale=None, causal=True, prefix=(), prefix_len=0):
    """out fp64 [T, heads, D] of q [T, heads, D]; cache: (k, v, k_scale, v_scale); rows of no sequence are NaN. Row r of sequence b is at
    position lens[b] - (starts[b + 1] - r), whatever its table and the call have room for."""
    k, v, ks, vs = cache
    t, heads, d = q.shape
    group = heads // k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.full((t, heads, d), float("nan"), dtype=torch.float64)
    kp, there_p = tokens(k, ks, prefix, prefix_len)
    vp, _ = tokens(v, vs, prefix, prefix_len)
    for b, n_all in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        m = max(0, min(n_all, len(table[b]) * k.shape[2]))
        kk, there = tokens(k, ks, table[b], m)
        vv, _ = tokens(v, vs, table[b], m)
        for r in range(max(lo, 0), min(hi, t)):
            seen = there.clone()
            if causal:
                seen[max(0, n_all - (hi - r) + 1):] = False
            keys, values = torch.cat([kp[there_p], kk[seen]]), torch.cat([vp[there_p], vv[seen]])
            for h in range(heads):
                if len(keys) == 0:
                    out[r, h] = 0
                else:
                    p = torch.softmax(scale * (keys[:, h // group] @ q[r, h].double()), 0)
                    out[r, h] = p @ values[:, h // group]
    return out
