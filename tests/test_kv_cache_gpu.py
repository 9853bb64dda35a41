"""The quantized key/value cache on the GPU against the definitions in 64 bits (oracle/kv_cache.py).

Tolerance of attention, derived: the output is rounded once (eps / 2 of its value); every weight is rounded to fp16 (2^-11 of it),
computed with approximate exp2, log2 and reciprocal (2^-17 together, |log2 vs| <= 40) from a score that D / 16 tensor-core steps
sum in fp32 (2^-22 of the magnitudes' sum for each, the two products behind it included) and enters numerator and
denominator. Weights move the output by at most their relative error times sum_j p_j |v_j|."""
import random

import pytest
import torch

from oracle import kv_cache as okv

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from rapid_h3_b200 import _lib, kv_cache
    assert torch.cuda.is_available()
    _lib.lib()
    _lib.check_status()
    return kv_cache


def fill(cache, seed):
    """Random codes and scales in every slot of the cache, valid or not."""
    g = torch.Generator().manual_seed(seed)
    shape = tuple(cache.k.shape)
    for codes, scales, offset in ((cache.k, cache.k_scale, 0.5), (cache.v, cache.v_scale, 0.2)):
        x = (torch.randn(shape, generator=g) + offset) * (0.2 + torch.rand(shape[:3], generator=g)[..., None])
        q, s = okv.quantize(x, "int8" if cache.kind == 0 else "fp8")
        codes.view(torch.uint8).copy_(q.view(torch.uint8))
        scales.copy_(s)


def host(cache):
    return cache.k.cpu(), cache.v.cpu(), cache.k_scale.cpu(), cache.v_scale.cpu()


def batch(kv, lens, news, page, pages, seed, width=None):
    """(Rows, table, starts): pages drawn without repetition."""
    r = random.Random(seed)
    order = r.sample(range(pages), pages)
    width = width or max(1, max(-(-n // page) for n in lens))
    table, at = [], 0
    for n in lens:
        need = -(-n // page)
        table.append(order[at:at + need] + [0] * (width - need))
        at += need
    assert at <= pages
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (table, lens, starts)]
    return kv.Rows(*dev), table, starts


def check_attention(out, q, cache, table, lens, starts, **kw):
    k, v, ks, vs = host(cache)
    q = q.cpu()
    ref = okv.attention(q, (k, v, ks, vs), table, lens, starts, **kw)
    vabs = v.float().abs().to(v.dtype) if cache.kind else v.abs()
    mag = okv.attention(q, (k, vabs, ks, vs), table, lens, starts, **kw)
    scale = kw.get("scale") or q.shape[2] ** -0.5
    kmax = (k.float() * ks[..., None]).nan_to_num(0, 0, 0).abs().amax()
    s_abs = scale * float(q.double().abs().sum(-1).max() * kmax)
    d = q.shape[2]
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + mag * (2 ** -11 + 2 ** -17 + 2 * (d // 16 + 2) * 2 ** -22 * s_abs) + 1e-7
    rows = starts[-1]
    err = (out.cpu().double() - ref)[:rows].abs()
    assert torch.isfinite(out[:rows]).all()
    assert bool((err <= tol[:rows]).all()), float((err / tol[:rows]).max())


SHAPES = [  # kind, dtype, D, page, kv heads, group
    ("int8", torch.bfloat16, 128, 64, 2, 4),
    ("fp8", torch.bfloat16, 128, 16, 1, 8),
    ("int8", torch.float16, 64, 32, 3, 1),
    ("fp8", torch.float16, 64, 128, 2, 5),
    ("int8", torch.float16, 128, 128, 1, 16),
    ("fp8", torch.bfloat16, 64, 16, 1, 40),
]


@pytest.mark.parametrize("kind,dtype,d,page,heads,group", SHAPES)
@pytest.mark.parametrize("lens,news", [
    ([1], [1]), ([517], [1]), ([0, 5], [0, 2]), ([64, 1, 130, 257, 16], [1, 1, 1, 1, 1]), ([300, 37, 129], [7, 37, 20]), ([40, 128], [40, 3]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(kv, kind, dtype, d, page, heads, group, lens, news, causal):
    pages = sum(-(-n // page) for n in lens) + 2
    cache = kv.alloc(pages, heads, d, page, kind)
    fill(cache, 1)
    rows, table, starts = batch(kv, lens, news, page, pages, 2)
    g = torch.Generator().manual_seed(3)
    q = (torch.randn(starts[-1], heads * group, d, generator=g) * 1.5).to(dtype).cuda()
    out = kv.attention(q, cache, rows, causal=causal)
    check_attention(out, q, cache, table, lens, starts, causal=causal)


def strided(x, heads, extra):
    """x [T, heads, D] as a view into a wider buffer, as a slice of a qkv product is."""
    wide = torch.full((x.shape[0], heads + extra, x.shape[2]), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, 1:1 + heads] = x.cuda()
    return wide[:, 1:1 + heads]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,page,heads", [(128, 64, 8), (64, 16, 5), (128, 16, 1), (64, 128, 12)])
def test_write_stores_codes_and_scales_and_read_gives_them_back(kv, kind, dtype, d, page, heads):
    lens, news = [5, 300, 17, 0, 64], [5, 211, 1, 0, 2]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = kv.alloc(pages, heads, d, page, kind)
    fill(cache, 4)
    before = host(cache)
    rows, table, starts = batch(kv, lens, news, page, pages, 5)
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(starts[-1], heads, d, generator=g).to(dtype) for _ in range(2))
    k[0] = 0
    v[3, 0] *= 1e-20 if dtype != torch.float16 else 1e-7   # scales at their lower limit
    if dtype == torch.bfloat16:
        k[1] = torch.randint(-254, 255, (heads, d), generator=g).to(dtype)   # many ties: x / s is a half integer
        k[1, :, 0] = 254
    kv.write(cache, strided(k, heads, 3), strided(v, heads, 2), rows)
    want = [t.clone() for t in before]
    place = [(table[b][p // page], p % page) for b in range(len(lens)) for p in range(lens[b] - news[b], lens[b])]
    for codes, scales, x in ((want[0], want[2], k), (want[1], want[3], v)):
        q, s = okv.quantize(x, kind)
        for t, (pg, off) in enumerate(place):
            codes.view(torch.uint8)[pg, :, off] = q.view(torch.uint8)[t]
            scales[pg, :, off] = s[t]
    for got, ref in zip(host(cache), want):   # every other slot as it was
        assert torch.equal(got.view(torch.uint8), ref.view(torch.uint8))
    for back in (torch.bfloat16, torch.float16, torch.float32):
        out = [torch.full((starts[-1] + 2, heads, d), 7.0, dtype=back, device="cuda") for _ in range(2)]
        kv.read(cache, rows, starts[-1] + 2, back, out)
        for got, codes, scales in zip(out, want[:2], want[2:]):
            ref = torch.stack([codes[pg, :, off].float() * scales[pg, :, off, None] for pg, off in place]).to(back)
            assert torch.equal(got[:-2].cpu(), ref) and bool((got[-2:] == 7).all())


def test_rows_that_are_not_finite_read_back_as_nan_and_reach_nobody_else(kv):
    """A NaN or an infinity stays in its row's scale, and a masked row of that kind changes nothing."""
    for kind in ("int8", "fp8"):
        cache = kv.alloc(4, 2, 128, 16, kind)
        rows, table, starts = batch(kv, [40], [40], 16, 4, 7)
        g = torch.Generator().manual_seed(8)
        k, v = (torch.randn(40, 2, 128, generator=g).to(torch.bfloat16) for _ in range(2))
        q = torch.randn(40, 4, 128, generator=g).to(torch.bfloat16).cuda()
        kv.write(cache, k.cuda(), v.cuda(), rows)
        clean = kv.attention(q, cache, rows)
        k[30, 0, 5], k[31, 1, 0], v[32, 0, 127], v[33, 1, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
        kv.write(cache, k.cuda(), v.cuda(), rows)
        bk, bv = kv.read(cache, rows, 40)
        for back, x in ((bk, k), (bv, v)):
            bad = ~torch.isfinite(x).all(-1)
            assert bool(torch.isnan(back.cpu()[bad]).all()) and bool(torch.isfinite(back.cpu()[~bad]).all())
        out = kv.attention(q, cache, rows)
        assert torch.equal(out[:30], clean[:30])          # causal: the rows before see none of it
        assert bool(torch.isnan(out[33]).all())


def test_what_lies_in_slots_behind_a_sequence_does_not_matter(kv):
    """Unwritten slots with NaN codes (0x7f of e4m3), NaN and infinite scales."""
    for kind in ("int8", "fp8"):
        cache = kv.alloc(6, 1, 128, 64, kind)
        rows, table, starts = batch(kv, [70, 1, 0], [1, 1, 1], 64, 6, 9)
        for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            codes.view(torch.uint8).fill_(0x7F)
            scales.fill_(float("nan"))
            scales[..., ::2] = float("inf")
        whole = kv.Rows(rows.table, rows.lens, torch.tensor([0, 70, 71, 71], dtype=torch.int32, device="cuda"))
        g = torch.Generator().manual_seed(10)
        kv.write(cache, *(torch.randn(71, 1, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2)), whole)
        q = torch.randn(3, 8, 128, generator=g).to(torch.bfloat16).cuda()
        for causal in (True, False):
            out = kv.attention(q, cache, rows, causal=causal)
            check_attention(out, q, cache, table, [70, 1, 0], starts, causal=causal)
            assert bool((out[2] == 0).all())              # a row without a key


def test_values_without_sense_are_cut_to_what_exists(kv):
    """Pages outside the cache, lengths beyond the table, rows beyond the call's, negative lengths."""
    from rapid_h3_b200 import _lib
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = kv.alloc(4, 2, 128, 16, "int8")
    fill(cache, 11)
    before = host(cache)
    g = torch.Generator().manual_seed(12)
    table = [[0, 99, 2], [-1, 1, 3], [1, 2, 3], [0, 1, 2]]
    lens, starts = [40, 48, 1000, -5], [0, 2, 3, 4, 6]
    rows = kv.Rows(torch.tensor(table, **i32), torch.tensor(lens, **i32), torch.tensor(starts, **i32))
    q = torch.randn(6, 4, 128, generator=g).to(torch.bfloat16).cuda()
    out = kv.attention(q, cache, rows)
    check_attention(out, q, cache, table, lens, starts)
    with pytest.raises(RuntimeError, match="outside its cache"):
        _lib.check_status()
    # rows that lie nowhere: not written, read as zeros
    x = torch.randn(6, 2, 128, generator=g).to(torch.bfloat16).cuda()
    lost = kv.Rows(torch.tensor([[99, -7]], **i32), torch.tensor([20], **i32), torch.tensor([0, 6], **i32))
    kv.write(cache, x, x, lost)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(host(cache), before))
    assert all(bool((t == 0).all()) for t in kv.read(cache, lost, 6))
    with pytest.raises(RuntimeError, match="outside its cache"):
        _lib.check_status()
    # more rows named than the call has; fewer tokens than rows
    rows = kv.Rows(torch.tensor([[0, 1]], **i32), torch.tensor([3], **i32), torch.tensor([0, 500], **i32))
    out = kv.attention(q, cache, rows, causal=False)
    check_attention(out, q, cache, [[0, 1]], [3], [0, 6], causal=False)
    _lib.check_status()


@pytest.mark.parametrize("kind,dtype,d,page,heads,group", SHAPES)
@pytest.mark.parametrize("lens,news,prefix", [
    ([0], [1], 1), ([64, 1, 0, 130], [1, 1, 1, 1], 700), ([33, 160, 7], [33, 60, 0], 129), ([5, 300], [2, 9], 0),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_behind_a_shared_prefix(kv, kind, dtype, d, page, heads, group, lens, news, prefix, causal):
    pre = -(-prefix // page)
    pages = sum(-(-n // page) for n in lens) + pre + 2
    cache = kv.alloc(pages, heads, d, page, kind)
    fill(cache, 13)
    rows, table, starts = batch(kv, lens + [prefix], news + [0], page, pages, 14)
    ids = table[-1][:pre]
    rows = kv.Rows(rows.table[:-1], rows.lens[:-1], rows.starts[:-1])
    g = torch.Generator().manual_seed(15)
    q = (torch.randn(starts[-1], heads * group, d, generator=g) * 1.5).to(dtype).cuda()
    out = kv.attention_shared(q, cache, rows, torch.tensor(ids, dtype=torch.int32, device="cuda"), prefix, causal=causal)
    check_attention(out, q, cache, table[:-1], lens, starts[:-1], causal=causal, prefix=ids, prefix_len=prefix)


@pytest.mark.parametrize("kind,dtype,d,page,heads,group", SHAPES[:4])
@pytest.mark.parametrize("lens,news", [([700, 1, 333], [520, 1, 333]), ([2000], [65])])
def test_attention_of_many_rows(kv, kind, dtype, d, page, heads, group, lens, news):
    """Units of 256 rows over several key tiles, cut between CTAs."""
    pages = sum(-(-n // page) for n in lens) + 2
    cache = kv.alloc(pages, heads, d, page, kind)
    fill(cache, 21)
    rows, table, starts = batch(kv, lens, news, page, pages, 22)
    g = torch.Generator().manual_seed(23)
    q = (torch.randn(starts[-1], heads * group, d, generator=g) * 1.5).to(dtype).cuda()
    out = kv.attention(q, cache, rows)
    check_attention(out, q, cache, table, lens, starts)
