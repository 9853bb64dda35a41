"""The quantized key/value cache on the GPU against the definitions in 64 bits (oracle/kv_cache.py).

Tolerance of attention, derived: the output is rounded once (eps / 2 of its value); every weight is rounded to fp16 (2^-11 of it),
computed with approximate exp2, log2 and reciprocal (2^-17 together, |log2 vs| <= 40) from a score that D / 16 tensor-core steps
sum in fp32 (2^-22 of the magnitudes' sum for each, the two products behind it included) and enters numerator and
denominator. Weights move the output by at most their relative error times sum_j p_j |v_j|. The kernel for few rows adds K codes as code + 128 <= 255,
about twice the magnitudes, and the kernel for many rows rounds V to fp16 (2^-11 of a value, and 2^-25 of twice the largest row's magnitude where that
is more)."""
import random
import threading

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


@pytest.fixture(params=[False, True], ids=["few rows", "many rows"])
def path(kv, request):
    """Both kernels, whatever a call's sizes would choose."""
    before = kv.use_wide(request.param)
    yield
    kv.use_wide(before)


@pytest.fixture(params=[False, "apart", True], ids=["few rows", "few rows, prefix apart", "many rows"])
def prefix_path(kv, request):
    before = kv.use_wide(request.param)
    yield
    kv.use_wide(before)


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
    v_max = float((v.float().abs() * vs[..., None]).nan_to_num(0, 0, 0).amax())
    tol = torch.finfo(q.dtype).eps / 2 * ref.abs() + mag * (2 * 2 ** -11 + 2 ** -17 + 2 * (d // 16 + 2) * 2 ** -22 * 2 * s_abs) + 2 ** -24 * v_max + 1e-7
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
def test_attention(kv, path, kind, dtype, d, page, heads, group, lens, news, causal):
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


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes_are_those_of_the_rounded_quotients(kv, kind, dtype):
    """Rows of every magnitude, many of whose quotients lie at or next to a value between two codes."""
    n, heads, d, page = 1024, 8, 128, 128
    g = torch.Generator().manual_seed(7)
    exponent = torch.randint(-44, 120, (n, heads, 1), generator=g).float()   # scales down to their lower limit
    x = torch.rand(n, heads, d, generator=g) * 2 - 1
    top = 1 + torch.rand(n, heads, 1, generator=g)
    half = torch.randint(-254, 255, (n, heads, d), generator=g).float() / 254 * top.to(dtype).float()   # (k + 1/2) / 127 of the largest
    wiggle = 1 + torch.randint(-3, 4, (n, heads, d), generator=g).float() * 2.0**-23
    x = torch.where(torch.rand(n, heads, d, generator=g) < 0.7, half * wiggle, x)
    x[..., :1] = top
    x = (x * torch.exp2(exponent)).to(dtype)
    cache = kv.alloc(n // page, heads, d, page, kind)
    rows, table, starts = batch(kv, [n], [n], page, n // page, 8)
    kv.write(cache, x.cuda(), x.flip(0).cuda(), rows)
    q, s = okv.quantize(x, kind)
    order = torch.tensor(table[0])
    for of, want_q, want_s in ((0, q, s), (1, q.flip(0), s.flip(0))):
        codes, scales = (t.view(torch.uint8)[order] if t.dtype != torch.float32 else t[order] for t in host(cache)[of::2])
        assert torch.equal(scales.transpose(1, 2).reshape(n, heads), want_s)
        assert torch.equal(codes.transpose(1, 2).reshape(n, heads, d), want_q.contiguous().view(torch.uint8))


def test_rows_that_are_not_finite_read_back_as_nan_and_reach_nobody_else(kv, path):
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


def test_what_lies_in_slots_behind_a_sequence_does_not_matter(kv, path):
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


def test_values_without_sense_are_cut_to_what_exists(kv, path):
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
def test_attention_behind_a_shared_prefix(kv, prefix_path, kind, dtype, d, page, heads, group, lens, news, prefix, causal):
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
def test_attention_of_many_rows(kv, path, kind, dtype, d, page, heads, group, lens, news):
    """Units of 256 rows over several key tiles, cut between CTAs."""
    pages = sum(-(-n // page) for n in lens) + 2
    cache = kv.alloc(pages, heads, d, page, kind)
    fill(cache, 21)
    rows, table, starts = batch(kv, lens, news, page, pages, 22)
    g = torch.Generator().manual_seed(23)
    q = (torch.randn(starts[-1], heads * group, d, generator=g) * 1.5).to(dtype).cuda()
    out = kv.attention(q, cache, rows)
    check_attention(out, q, cache, table, lens, starts)


def test_a_long_context_joined_from_many_parts(kv, path):
    """One sequence over all of the chip: more parts than a joining CTA takes in at a time, and a tail of tiny weights."""
    for kind, dtype, d, heads, group in (("int8", torch.bfloat16, 128, 1, 2), ("fp8", torch.float16, 64, 1, 16)):
        n, page = 20011, 128
        pages = -(-n // page) + 1
        cache = kv.alloc(pages, heads, d, page, kind)
        fill(cache, 31)
        rows, table, starts = batch(kv, [n], [1], page, pages, 32)
        g = torch.Generator().manual_seed(33)
        q = (torch.randn(1, heads * group, d, generator=g) * 1.5).to(dtype).cuda()
        check_attention(kv.attention(q, cache, rows), q, cache, table, [n], starts)


def test_a_prefix_shared_by_many_rows(kv):
    """Enough rows and tokens that the prefix goes to the tensor-core tiles and the own parts do not; rows of one sequence lie in two units
    of the prefix pass."""
    heads, group, d, page, prefix = 4, 5, 128, 32, 1900
    lens, news = [3, 40, 0, 300, 129, 7] * 9, [1, 2, 1, 1, 3, 1] * 9
    pre = -(-prefix // page)
    pages = sum(-(-n // page) for n in lens) + pre + 2
    cache = kv.alloc(pages, heads, d, page, "int8")
    fill(cache, 34)
    rows, table, starts = batch(kv, lens + [prefix], news + [0], page, pages, 35)
    ids = table[-1][:pre]
    rows = kv.Rows(rows.table[:-1], rows.lens[:-1], rows.starts[:-1])
    g = torch.Generator().manual_seed(36)
    q = torch.randn(starts[-1], heads * group, d, generator=g).to(torch.bfloat16).cuda()
    before = None
    for use in (None, True, False):
        before = kv.use_wide(use) if before is None else (kv.use_wide(use), before)[1]
        out = kv.attention_shared(q, cache, rows, torch.tensor(ids, dtype=torch.int32, device="cuda"), prefix)
        check_attention(out, q, cache, table[:-1], lens, starts[:-1], prefix=ids, prefix_len=prefix)
    kv.use_wide(None)


def test_scales_of_very_different_size(kv, path):
    """V scales over 2^24 and K rows over 2^12: the largest tokens decide what matters, and later tiles bring larger ones."""
    cache = kv.alloc(8, 1, 128, 64, "int8")
    fill(cache, 37)
    rows, table, starts = batch(kv, [500], [40], 64, 8, 38)
    order = torch.tensor(table[0]).cuda()
    for i in range(8):
        cache.v_scale[order[i]] *= 2.0 ** (3 * i - 12)
        cache.k_scale[order[i]] *= 2.0 ** (i % 3 * 2 - 6)
    q = torch.randn(40, 4, 128, generator=torch.Generator().manual_seed(39)).to(torch.bfloat16)
    q[::3] *= 2.0 ** 20
    q[1::3] *= 2.0 ** -20
    q = q.cuda()
    check_attention(kv.attention(q, cache, rows, scale=1e-3), q, cache, table, [500], starts, scale=1e-3)
    check_attention(kv.attention(q[1::3].contiguous(), cache, kv.Rows(rows.table, rows.lens, torch.tensor([0, 13], dtype=torch.int32, device="cuda"))),
                    q[1::3], cache, table, [500], [0, 13])


def test_rows_behind_the_last_sequence_stay(kv, path):
    """A padded batch: more rows than starts[B] in q and out, which hold NaN."""
    cache = kv.alloc(6, 2, 64, 16, "fp8")
    fill(cache, 40)
    rows, table, starts = batch(kv, [17, 30], [1, 20], 16, 6, 41)
    q = torch.full((40, 4, 64), float("nan"), dtype=torch.bfloat16)
    q[:21] = torch.randn(21, 4, 64, generator=torch.Generator().manual_seed(42)).to(torch.bfloat16)
    out = torch.full((40, 6, 64), 5.0, dtype=torch.bfloat16, device="cuda")[:, 1:5]
    q = q.cuda()
    assert kv.attention(q, cache, rows, out=out) is out
    check_attention(out[:21], q[:21], cache, table, [17, 30], starts)
    assert bool((out[21:] == 5).all())
    pre = torch.tensor([5], dtype=torch.int32, device="cuda")
    kv.attention_shared(q, cache, rows, pre, 9, out=out)
    check_attention(out[:21], q[:21], cache, table, [17, 30], starts, prefix=[5], prefix_len=9)
    assert bool((out[21:] == 5).all())


def test_a_captured_step_follows_lengths_and_pages(kv, path):
    """Write, attention and read of one decoding step in a graph, replayed while sequences grow; an eager call of the same kind in between."""
    heads, group, d, page = 2, 4, 128, 16
    cache = kv.alloc(64, heads, d, page, "int8")
    dev = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(60, **dev).view(3, 20).contiguous()
    lens = torch.tensor([300, 1, 95], **dev)
    rows = kv.Rows(table, lens, torch.arange(4, **dev))
    fill(cache, 43)
    k, v = (torch.zeros(3, heads, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros(3, heads * group, d, dtype=torch.bfloat16, device="cuda")

    def step():
        kv.write(cache, k, v, rows)
        return kv.attention(q, cache, rows), kv.read(cache, rows, 3)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, back = step()
    g = torch.Generator().manual_seed(44)
    for i in range(3):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        if i:
            lens += 3
            table[1].copy_(table[1].flip(0))
        graph.replay()
        first = out.clone()
        other = kv.attention(q, cache, rows)
        graph.replay()
        assert torch.equal(first, out) and torch.equal(first, other)
        check_attention(out, q, cache, table.tolist(), lens.tolist(), [0, 1, 2, 3])
        place = [(table[b, (int(lens[b]) - 1) // page], (int(lens[b]) - 1) % page) for b in range(3)]
        for x, codes, scales in ((back[0], cache.k, cache.k_scale), (back[1], cache.v, cache.v_scale)):
            ref = torch.stack([codes[p, :, o].float() * scales[p, :, o, None] for p, o in place])
            assert torch.equal(x, ref.to(torch.bfloat16))


def test_a_captured_call_behind_a_prefix_with_rows_that_no_sequence_has(kv, prefix_path):
    """Rows before the first sequence and behind the last hold NaN and stay; lengths and the prefix's pages change between
    replays; a second graph of the same call is replayed on another stream meanwhile."""
    heads, group, d, page, prefix = 2, 3, 64, 16, 150
    cache = kv.alloc(80, heads, d, page, "int8")
    fill(cache, 46)
    dev = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(40, **dev).view(2, 20).contiguous()
    pre = torch.arange(40, 50, **dev)
    lens = torch.tensor([260, 33], **dev)
    rows = kv.Rows(table, lens, torch.tensor([2, 9, 42], **dev))
    q = torch.full((50, heads * group, d), float("nan"), dtype=torch.float16, device="cuda")
    outs = [torch.full_like(q, 3.0) for _ in range(2)]
    kv.attention_shared(q, cache, rows, pre, prefix, out=outs[0])   # kernels loaded
    outs[0].fill_(3.0)
    graphs = []
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(3):
                kv.attention_shared(q, cache, rows, pre, prefix, out=out)
    side = torch.cuda.Stream()
    g = torch.Generator().manual_seed(47)
    for i in range(3):
        q[2:42] = torch.randn(40, heads * group, d, generator=g).to(torch.float16).cuda()
        if i:
            lens += 13
            pre.copy_(pre.flip(0) if i == 1 else pre + 20)
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(4):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.current_stream().wait_stream(side)
        for out in outs:
            assert bool((out[:2] == 3).all()) and bool((out[42:] == 3).all())
            check_attention(out[2:42], q[2:42], cache, table.tolist(), lens.tolist(), [0, 7, 40], prefix=pre.tolist(), prefix_len=prefix)
        assert torch.equal(*outs)


def test_calls_on_two_streams_at_once(kv, path):
    """Each stream has counters and a workspace of its own: results as one after the other."""
    cache = kv.alloc(80, 2, 128, 64, "fp8")
    fill(cache, 45)
    cases = []
    for i, lens in enumerate(([4000], [300, 800, 64, 1])):
        rows, _, starts = batch(kv, lens, [1] * len(lens), 64, 80, 46 + i)
        q = torch.randn(starts[-1], 16, 128, generator=torch.Generator().manual_seed(i)).to(torch.float16).cuda()
        cases.append((q, rows, kv.attention(q, cache, rows), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (q, rows, _, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                outs[i].append(kv.attention(q, cache, rows))
    torch.cuda.synchronize()
    for got, (_, _, want, _) in zip(outs, cases):
        assert all(torch.equal(x, want) for x in got)


def test_calls_of_several_threads_on_one_stream(kv, prefix_path):
    """They share the stream's counters and workspace."""
    heads, group, d, page, prefix = 2, 4, 128, 64, 1000
    cache = kv.alloc(60, heads, d, page, "int8")
    fill(cache, 48)
    pre = torch.arange(16, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(49)
    calls = []
    for i in range(4):
        rows, _, _ = batch(kv, [70, 130, 9 + i], [1, 2, 1], page, 40, 50 + i)
        rows = kv.Rows(rows.table + 16, rows.lens, rows.starts)
        q = torch.randn(4, heads * group, d, generator=g).to(torch.bfloat16).cuda()
        calls.append((q, rows, kv.attention_shared(q, cache, rows, pre, prefix)))
    wrong, stream = [], torch.cuda.current_stream()

    def work(q, rows, want):
        with torch.cuda.stream(stream):
            for _ in range(100):
                if not torch.equal(kv.attention_shared(q, cache, rows, pre, prefix), want):
                    wrong.append(q)

    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_sequences_without_pages(kv, prefix_path):
    """A table of no columns: rows see the prefix alone, or nothing; nothing is written, zeros are read."""
    cache = kv.alloc(4, 2, 64, 32, "fp8")
    fill(cache, 51)
    before = host(cache)
    dev = dict(dtype=torch.int32, device="cuda")
    rows = kv.Rows(torch.empty(3, 0, **dev), torch.tensor([0, 5, 0], **dev), torch.tensor([0, 1, 1, 4], **dev))
    q = torch.randn(4, 6, 64, generator=torch.Generator().manual_seed(52)).to(torch.bfloat16).cuda()
    assert bool((kv.attention(q, cache, rows) == 0).all())
    out = kv.attention_shared(q, cache, rows, torch.tensor([3, 1], **dev), 33)
    check_attention(out, q, cache, [[], [], []], [0, 0, 0], [0, 1, 1, 4], prefix=[3, 1], prefix_len=33)
    kv.write(cache, q[:, :2], q[:, 2:4], rows)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(host(cache), before))
    assert all(bool((t == 0).all()) for t in kv.read(cache, rows, 4))
    none = torch.empty(0, **dev)
    assert bool((kv.attention_shared(q, cache, rows, none, 0) == 0).all())


def test_pages_behind_32_bit_offsets(kv, path):
    """A cache whose codes take more than 2^32 bytes: pages at its end are written, read and attended to."""
    page, heads, d = 128, 16, 128
    pages = (1 << 32) // (page * heads * d) + 40
    codes = [torch.empty(pages, heads, page, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    cache = kv.KVCache(*codes, *(torch.empty(pages, heads, page, device="cuda") for _ in range(2)))
    dev = dict(dtype=torch.int32, device="cuda")
    table = [[pages - 1, pages - 3], [pages - 2, 0]]
    rows = kv.Rows(torch.tensor(table, **dev), torch.tensor([200, 130], **dev), torch.tensor([0, 200, 330], **dev))
    g = torch.Generator().manual_seed(48)
    k, v = (torch.randn(330, heads, d, generator=g).to(torch.bfloat16) for _ in range(2))
    kv.write(cache, k.cuda(), v.cuda(), rows)
    q8, s8 = okv.quantize(k, "int8")
    assert torch.equal(kv.read(cache, rows, 330, torch.float32)[0].cpu(), q8.float() * s8[..., None])
    q = torch.randn(2, heads, d, generator=g).to(torch.bfloat16).cuda()
    last = kv.Rows(rows.table, rows.lens, torch.tensor([0, 1, 2], **dev))
    out = kv.attention(q, cache, last)
    small = [c[[0, pages - 3, pages - 2, pages - 1]] for c in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    check_attention(out, q, kv.KVCache(*(t.contiguous() for t in small)), [[3, 1], [2, 0]], [200, 130], [0, 1, 2])


def test_starts_that_do_not_ascend_are_reported_or_cut(kv, path):
    from rapid_h3_b200 import _lib
    cache = kv.alloc(40, 1, 64, 16, "int8")
    fill(cache, 49)
    dev = dict(dtype=torch.int32, device="cuda")
    rows = kv.Rows(torch.arange(40, **dev).view(4, 10), torch.tensor([160, 3, 160, 9], **dev), torch.tensor([0, 9, 2, 9, 1], **dev))
    q = torch.randn(9, 8, 64).to(torch.bfloat16).cuda()
    kv.attention(q, cache, rows)
    kv.read(cache, rows, 9)
    torch.cuda.synchronize()
    try:
        _lib.check_status()
    except RuntimeError as e:
        assert "ascending" in str(e)


def test_refusals(kv):
    dev = dict(dtype=torch.int32, device="cuda")
    cache = kv.alloc(4, 2, 64, 16, "int8")
    rows = kv.Rows(torch.zeros(1, 4, **dev), torch.ones(1, **dev), torch.tensor([0, 1], **dev))
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (x.cpu(), x.double(), x[..., :32], x[:, :1], torch.zeros(1, 2, 68, dtype=torch.bfloat16, device="cuda")[..., 2:66], x.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(RuntimeError):
            kv.write(cache, bad, x, rows)
        with pytest.raises(RuntimeError):
            kv.write(cache, x, bad, rows)
    with pytest.raises(RuntimeError):
        kv.write(cache, x, torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda"), rows)
    for bad in (q[:, :3], q.float(), q.cpu(), torch.zeros(1, 0, 64, dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(RuntimeError):
            kv.attention(bad, cache, rows)
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0), dict(out=q.float()), dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(RuntimeError):
            kv.attention(q, cache, rows, **kw)
    for pre, n in ((torch.zeros(2, **dev), 33), (torch.zeros(2, **dev), -1), (torch.zeros(2, device="cuda"), 3), (torch.zeros(2, 1, **dev), 3)):
        with pytest.raises(RuntimeError):
            kv.attention_shared(q, cache, rows, pre, n)
    for args in ((torch.zeros(1, 4, device="cuda"), rows.lens, rows.starts), (rows.table, torch.ones(2, **dev), rows.starts), (rows.table, rows.lens, rows.lens),
                 (rows.table[0], rows.lens, rows.starts), (torch.zeros(4, 4, **dev).t()[:1], rows.lens, rows.starts), (rows.table[:0], rows.lens[:0], rows.starts[:1])):
        with pytest.raises(RuntimeError):
            kv.Rows(*args)
    k, ks = cache.k, cache.k_scale
    for args in ((k, k[:2], ks, ks), (k.float(), k.float(), ks, ks), (k, k, ks.half(), ks), (k, k, ks[:, :1], ks), (k[:, :, ::2], k[:, :, ::2], ks[..., ::2], ks[..., ::2]),
                 (k.transpose(1, 2), k.transpose(1, 2), ks.transpose(1, 2), ks.transpose(1, 2))):
        with pytest.raises(RuntimeError):
            kv.KVCache(*args)
    with pytest.raises(RuntimeError):
        kv.read(cache, rows, 1, torch.float64)
    with pytest.raises(RuntimeError):
        kv.read(cache, rows, 1, torch.bfloat16, (x[:, :1], x))
    # calls without rows do nothing
    kv.write(cache, x[:0], x[:0], rows)
    assert kv.attention(q[:0], cache, rows).shape == (0, 4, 64) and kv.read(cache, rows, 0)[0].shape == (0, 2, 64)
