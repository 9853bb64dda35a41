"""Operators of the quantized key/value cache whose speed is tracked (rapid_h3_b200.kv_cache), with their plain forms.

The cache holds the keys and values of a language model's attention (the text encoder's: grouped heads) as 8-bit codes
with one fp32 scale per token and head, in pages of `page` tokens: codes [pages, heads, page, D], scales [pages, heads,
page]. A batch is described by a page table [B, P], the number of cached tokens of each sequence `lens` [B] and the row
starts [B + 1]: rows starts[b] .. starts[b+1]-1 of a call are the last tokens of sequence b.

Kinds:
  write   quantize and store new keys and values, and read the stored rows back
  read    read spans of the cache back as bf16 rows
  attn    attention of new tokens to their sequences (causal among the new tokens, or not)
  shared  the same where all sequences continue one cached prefix

Where `own` is false, `run` computes the plain form in elementary torch operations and fp32; where it is true, it calls the
package. `exact` computes the same from the definitions in fp64, sequence by sequence.
"""
import math
import random

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # one decoding step of a batch of prompts being continued: a row per sequence, latency counts
        dict(name="write_tokens", kind="write", fmt="int8", dtype="bf16", batch=64, hkv=8, d=128, page=64, new=1, length=2000, ragged=1),
        # a batch of prompts of odd lengths, stored from the fp32 rows that the text encoder's linears give
        dict(name="write_prompts", kind="write", fmt="fp8", dtype="fp32", batch=37, hkv=8, d=128, page=16, new=900, length=900, ragged=1),
        # cached text tokens back as rows, head size 64, small pages
        dict(name="read_text", kind="read", fmt="fp8", dtype="bf16", batch=24, hkv=12, d=64, page=16, new=512, length=512, ragged=1),
        # a whole long sequence back (the token count of the full-resolution pass)
        dict(name="read_long", kind="read", fmt="int8", dtype="bf16", batch=1, hkv=8, d=128, page=64, new=36436, length=36436, ragged=0),
        # the smallest call: one sequence, one token, a short prompt
        dict(name="decode_one", kind="attn", fmt="int8", dtype="bf16", batch=1, hq=32, hkv=8, d=128, page=64, new=1, length=517, ragged=0, causal=True),
        # a decoding step of a batch of ragged sequences
        dict(name="decode_batch", kind="attn", fmt="int8", dtype="bf16", batch=48, hq=64, hkv=8, d=128, page=64, new=1, length=4096, ragged=1, causal=True),
        # few sequences of very long context, five query heads to a KV head
        dict(name="decode_long", kind="attn", fmt="fp8", dtype="bf16", batch=3, hq=20, hkv=4, d=128, page=64, new=1, length=120000, ragged=1, causal=True),
        # prompts of odd lengths appended to what their sequences hold
        dict(name="extend_prompts", kind="attn", fmt="int8", dtype="bf16", batch=10, hq=32, hkv=8, d=128, page=16, new=512, length=1536, ragged=1, causal=True),
        # a long text appended to a long context
        dict(name="extend_long", kind="attn", fmt="fp8", dtype="fp16", batch=1, hq=32, hkv=8, d=128, page=128, new=2011, length=18011, ragged=0, causal=True),
        # a few continuations of one template, latency counts
        dict(name="shared_few", kind="shared", fmt="int8", dtype="bf16", batch=6, hq=32, hkv=8, d=128, page=64, new=1, length=64, ragged=1, causal=True, prefix=700),
        # many samples drawn from one long prompt
        dict(name="shared_samples", kind="shared", fmt="int8", dtype="bf16", batch=64, hq=64, hkv=8, d=128, page=64, new=1, length=700, ragged=1, causal=True, prefix=12000),
        # prompts behind one template: all their tokens at once
        dict(name="shared_prompts", kind="shared", fmt="fp8", dtype="bf16", batch=24, hq=32, hkv=8, d=128, page=32, new=160, length=160, ragged=1, causal=True, prefix=1100),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    most = max((c for c in listed()), key=_cost)
    while True:
        kind = rng.choice(["write", "read", "attn", "attn", "attn", "shared", "shared"])
        hkv = rng.choice([1, 2, 4, 5, 8, 12, 16])
        d = rng.choice([64, 128, 128])
        c = dict(kind=kind, fmt=rng.choice(["int8", "fp8"]), dtype=rng.choice(["bf16", "bf16", "fp16"]), batch=_log(rng, 1, 96), hkv=hkv, d=d,
                 page=rng.choice([16, 32, 64, 128]), new=1, length=_log(rng, 1, 120000), ragged=rng.choice([0, 1]))
        if kind in ("write", "read"):
            c["dtype"] = rng.choice(["bf16", "fp16", "fp32"]) if kind == "write" else "bf16"
            c["new"] = rng.choice([1, _log(rng, 1, c["length"])])
        else:
            c["hq"] = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
            c["causal"] = rng.random() < 0.75
            c["new"] = rng.choice([1, 1, _log(rng, 1, c["length"])])
            if kind == "shared":
                c["prefix"] = _log(rng, 1, 20000)
        if c.get("hq", 1) > 64 or c["batch"] * c["length"] * hkv * d > 40_000_000 * 8:
            continue
        if c["batch"] * c["new"] * c.get("hq", 1) * (c["length"] + c.get("prefix", 0)) > 1_000_000_000:
            continue  # the scores of the plain form, padded
        if _cost(c) <= _cost(most):
            return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def _sizes(case):
    """(lens, news) of the case: how many tokens each sequence holds, how many of them are the call's rows."""
    r = random.Random("%d %d %d" % (case["batch"], case["length"], case["new"]))
    lens, news = [], []
    for _ in range(case["batch"]):
        n = case["new"] if not case["ragged"] else max(1, math.ceil(case["new"] * (1 - 0.9 * r.random())))
        old = max(0, case["length"] - case["new"])
        old = old if not case["ragged"] else math.ceil(old * (1 - 0.9 * r.random()))
        lens.append(old + n)
        news.append(n)
    return lens, news


def _visible(case):
    """Sum over the call's rows of the keys of its own sequence that a row sees."""
    lens, news = _sizes(case)
    if not case["causal"]:
        return sum(n * m for n, m in zip(news, lens))
    return sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(news, lens))


def work(case):
    lens, news = _sizes(case)
    rows, width = sum(news), case["hkv"] * case["d"]
    cached = 2 * case["hkv"] * (case["d"] + 4)          # bytes of a token's codes and scales, K and V
    if case["kind"] == "write":
        esize = 4 if case["dtype"] == "fp32" else 2
        # the new rows in, codes and scales out; the same back as bf16
        return {"bytes": rows * (2 * width * esize + cached) + rows * (cached + 4 * width), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": rows * (cached + 4 * width), "flops": 0}
    prefix = case.get("prefix", 0)
    keys = sum(lens) + prefix
    return {"bytes": keys * cached + 4 * rows * case["hq"] * case["d"], "flops": 4 * case["hq"] * case["d"] * (_visible(case) + prefix * rows)}


def _type(name):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


def _quantize(x, fmt):
    """(codes, scales) of fp32 rows x [..., D]: abs-max scale, round to nearest even."""
    top = 127.0 if fmt == "int8" else 448.0
    amax = x.abs().amax(-1)
    s = (amax / torch.full_like(amax, top)).clamp_min(1e-12)   # by a tensor: a true division
    y = (x / s.unsqueeze(-1)).clamp(-top, top)
    return (y.round().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)), s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)
    lens, news = _sizes(case)
    page, hkv, d, prefix = case["page"], case["hkv"], case["d"], case.get("prefix", 0)
    most = max(lens)
    per = [-(-n // page) for n in lens]
    pre = -(-prefix // page)
    total = sum(per) + pre + 3                                  # a few pages that nobody uses
    order = torch.randperm(total, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(case=dict(case), table=table, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
             starts=torch.tensor([0] + news, device=DEV).cumsum(0).to(torch.int32), prefix=order[at:at + pre].clone(),
             rows=sum(news), most_new=max(news), most_len=most)
    # what a cache holds: keys with an offset per channel, some tokens larger than others
    mean = torch.randn(hkv, 1, d, generator=g, device=DEV)

    def fill(offset):
        codes = torch.empty(total, hkv, page, d, dtype=torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn, device=DEV)
        scales = torch.empty(total, hkv, page, device=DEV)
        step = max(1, (1 << 26) // (hkv * page * d))
        for i in range(0, total, step):
            x = torch.randn(min(step, total - i), hkv, page, d, generator=g, device=DEV) + offset
            x *= 0.5 + torch.rand(x.shape[:-1], generator=g, device=DEV).unsqueeze(-1)
            codes[i:i + step], scales[i:i + step] = _quantize(x, case["fmt"])
        return codes, scales

    s["k"], s["ks"] = fill(mean)
    s["v"], s["vs"] = fill(0.3)
    if case["kind"] == "write":
        x = torch.randn(2, s["rows"], hkv, d, generator=g, device=DEV)
        x[0] += mean[:, 0]
        s["new_k"], s["new_v"] = (t.to(_type(case["dtype"])) for t in x)
    elif case["kind"] in ("attn", "shared"):
        s["q"] = (torch.randn(s["rows"], case["hq"], d, generator=g, device=DEV) * 1.5).to(_type(case["dtype"]))
    if own:  # the handles a program makes once
        from rapid_h3_b200 import kv_cache
        s["cache"] = kv_cache.KVCache(s["k"], s["v"], s["ks"], s["vs"])
        s["batch"] = kv_cache.Rows(s["table"], s["lens"], s["starts"])
    return s


def run(s):
    case = s["case"]
    if own:
        from rapid_h3_b200 import kv_cache
        if case["kind"] == "write":
            kv_cache.write(s["cache"], s["new_k"], s["new_v"], s["batch"])
            return kv_cache.read(s["cache"], s["batch"], s["rows"])
        if case["kind"] == "read":
            return kv_cache.read(s["cache"], s["batch"], s["rows"])
        if case["kind"] == "attn":
            return kv_cache.attention(s["q"], s["cache"], s["batch"], causal=case["causal"])
        return kv_cache.attention_shared(s["q"], s["cache"], s["batch"], s["prefix"], case["prefix"], causal=case["causal"])
    if case["kind"] == "write":
        return _plain_write(s)
    if case["kind"] == "read":
        return _plain_read(s)
    return _plain_attention(s)


# ---- plain forms ------------------------------------------------------------------------------------------------
def _row_places(s):
    """For each row of the call: its sequence, its number among the sequence's new rows, its position."""
    rows = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    i = rows - s["starts"].long()[b]
    return b, i, s["lens"].long()[b] - (s["starts"].long()[b + 1] - rows)


def _bytes(t):
    return t.view(torch.uint8)


def _plain_write(s):
    b, _, pos = _row_places(s)
    page = s["case"]["page"]
    pages, offs = s["table"].long()[b, pos // page], pos % page
    for codes, scales, x in ((s["k"], s["ks"], s["new_k"]), (s["v"], s["vs"], s["new_v"])):
        q, sc = _quantize(x.float(), s["case"]["fmt"])
        _bytes(codes)[pages, :, offs] = _bytes(q)
        scales[pages, :, offs] = sc
    return _plain_read(s)


def _rows_of(codes, scales, pages, offs):
    """fp32 [..., heads, D] of the tokens at (pages, offs)."""
    return _bytes(codes)[pages, :, offs].view(codes.dtype).float() * scales[pages, :, offs].unsqueeze(-1)


def _plain_read(s):
    b, _, pos = _row_places(s)
    page = s["case"]["page"]
    pages, offs = s["table"].long()[b, pos // page], pos % page
    return _rows_of(s["k"], s["ks"], pages, offs).to(torch.bfloat16), _rows_of(s["v"], s["vs"], pages, offs).to(torch.bfloat16)


def _plain_attention(s):
    case, page = s["case"], s["case"]["page"]
    b, i, _ = _row_places(s)
    hkv, group, d = case["hkv"], case["hq"] // case["hkv"], case["d"]
    lens, news = s["lens"].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    batch, most_new, most_len = len(lens), s["most_new"], s["most_len"]
    # padded queries [B, heads, new * group, D] and keys [B, heads, length, D]
    q = torch.zeros(batch, most_new, hkv, group, d, device=DEV)
    q[b, i] = s["q"].float().view(-1, hkv, group, d) * (d ** -0.5)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, hkv, most_new * group, d)
    pos = torch.arange(most_len, device=DEV)
    pages = s["table"].long()[:, pos // page]
    k = _rows_of(s["k"], s["ks"], pages, (pos % page).expand_as(pages)).permute(0, 2, 1, 3)
    t = torch.matmul(q, k.transpose(-1, -2)).view(batch, hkv, most_new, group, most_len)
    del k
    if case["causal"]:
        last = (lens - news)[:, None] + torch.arange(most_new, device=DEV)
    else:
        last = (lens - 1)[:, None].expand(batch, most_new)
    t.masked_fill_((pos > torch.minimum(last, lens[:, None] - 1).unsqueeze(-1))[:, None, :, None], -math.inf)
    prefix = case.get("prefix", 0)
    if prefix:
        pos = torch.arange(prefix, device=DEV)
        places = s["prefix"].long()[pos // page], pos % page
        kp = _rows_of(s["k"], s["ks"], *places).permute(1, 2, 0)                     # [heads, D, prefix]
        tp = torch.matmul(q.transpose(0, 1).reshape(hkv, -1, d), kp).view(hkv, batch, most_new, group, prefix).transpose(0, 1)
        t = torch.cat([tp, t], -1)
        del tp
    top = t.amax(-1, keepdim=True)
    t = (t - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = t.sum(-1, keepdim=True)
    t = (t / total.masked_fill(total == 0, 1.0)).view(batch, hkv, most_new * group, -1)
    v = _rows_of(s["v"], s["vs"], pages, (torch.arange(most_len, device=DEV) % page).expand_as(pages)).permute(0, 2, 1, 3)
    o = torch.matmul(t[..., prefix:], v)
    if prefix:
        vp = _rows_of(s["v"], s["vs"], *places).permute(1, 0, 2)
        o += torch.matmul(t[..., :prefix].transpose(0, 1).reshape(hkv, -1, prefix), vp).view(hkv, batch, most_new * group, d).transpose(0, 1)
    o = o.view(batch, hkv, most_new, group, d).transpose(1, 2)[b, i]
    return o.reshape(-1, case["hq"], d).to(s["q"].dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    lens, news = _sizes(case)
    page, d = case["page"], case["d"]
    table = s["table"].cpu().tolist()

    def tokens(codes, scales, ids, n):
        """fp64 [heads, n, D]: the first n tokens of the pages `ids`."""
        ids = torch.tensor(ids[:-(-n // page)], dtype=torch.int64, device=DEV)
        x = codes.view(torch.uint8).index_select(0, ids).view(codes.dtype).double() * scales.index_select(0, ids).double()[..., None]
        return x.transpose(0, 1).reshape(case["hkv"], -1, d)[:, :n]

    if case["kind"] == "write":
        found = []
        for x in (s["new_k"].double(), s["new_v"].double()):
            if case["fmt"] == "int8":
                step = (x.abs().amax(-1, keepdim=True) / 127).clamp_min(1e-12)
                found.append(torch.round(x / step) * step)
            else:
                step = (x.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-12)
                y = x / step
                # e4m3: 3 bits behind the leading one, the smallest exponent is -6
                unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                found.append(torch.round(y / unit) * unit * step)
        return tuple(found)
    if case["kind"] == "read":
        parts = [[tokens(c, sc, table[b], lens[b])[:, lens[b] - news[b]:].transpose(0, 1) for b in range(len(lens))]
                 for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
        return tuple(torch.cat(p) for p in parts)
    group, prefix = case["hq"] // case["hkv"], case.get("prefix", 0)
    if prefix:
        pre = [tokens(c, sc, s["prefix"].cpu().tolist(), prefix) for c, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
    out, at = [], 0
    for b, (m, n) in enumerate(zip(lens, news)):
        q = s["q"][at:at + n].double().view(n, case["hkv"], group, d)
        at += n
        k, v = tokens(s["k"], s["ks"], table[b], m), tokens(s["v"], s["vs"], table[b], m)
        hidden = None
        if case["causal"]:
            hidden = torch.arange(m, device=DEV)[None] > (m - n + torch.arange(n, device=DEV))[:, None]
        o = torch.empty(n, case["hkv"], group, d, dtype=torch.float64, device=DEV)
        for h in range(case["hkv"]):
            for first in range(0, n, 512):
                some = slice(first, min(n, first + 512))
                t = q[some, h] @ k[h].T / math.sqrt(d)                       # [rows, group, m]
                if hidden is not None:
                    t.masked_fill_(hidden[some, None], -math.inf)
                values = v[h]
                if prefix:
                    t = torch.cat([q[some, h] @ pre[0][h].T / math.sqrt(d), t], -1)
                    values = torch.cat([pre[1][h], values])
                o[some, h] = torch.softmax(t, -1) @ values
        out.append(o.reshape(n, case["hq"], d))
    return torch.cat(out)
