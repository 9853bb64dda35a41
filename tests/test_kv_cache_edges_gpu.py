"""Edges of the cache operators' definitions, both attention kernels on each: rows that are not finite, lengths and row starts that do not fit
the table or the call, V rows of very different size, outputs that overlap.

Tolerance, derived for each row and head: the output is rounded once (eps / 2 of its value). A weight moves it by its relative error times
sum_j p_j |v_j|, in numerator and denominator: 2^-11 for its rounding to fp16, 2^-14 for exponents of up to 2^9 (the score's and the V
scale's, in steps of 2^-15) and approximate exp2, log2 and reciprocal, and 2^-22 of the score's magnitude for each of D / 16 tensor-core steps and two
products (twice that, as K codes may enter as code + 128). The kernel for many rows rounds V (2^-11 of a value). There weights are fp16 whose
largest, with its V scale, is at least 2^3: one below 2^-14 is off by up to 2^-25 whatever its size, and its V at most 2^7 times the largest's."""
import pytest
import torch

from oracle import kv_cache as okv
from test_kv_cache_gpu import batch, fill, host, kv, path, prefix_path  # noqa: F401  (the fixtures of both kernels)

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def reference(q, cache, table, lens, starts, scale=None, causal=True, prefix=(), prefix_len=0):
    """(out, tolerance) fp64 [T, heads, D] from the definition; rows of no sequence are NaN."""
    k, v, ks, vs = host(cache)
    q = q.cpu().double()
    t, heads, d = q.shape
    group = heads // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    ref, tol = (torch.full((t, heads, d), float("nan"), dtype=torch.float64) for _ in range(2))
    pre = [okv.tokens(c, s, prefix, prefix_len) for c, s in ((k, ks), (v, vs))]
    for b, n in enumerate(lens):
        room = max(0, min(n, len(table[b]) * k.shape[2]))
        own = [okv.tokens(c, s, table[b], room) for c, s in ((k, ks), (v, vs))]
        for r in range(max(0, starts[b]), min(t, starts[b + 1])):
            seen = own[0][1] & (torch.arange(room) <= n - (starts[b + 1] - r) if causal else True)
            kk, vv = (torch.cat([p[0][p[1]], o[0][seen]]).repeat_interleave(group, 1) for p, o in zip(pre, own))
            if len(kk) == 0:
                ref[r], tol[r] = 0, 0
                continue
            p = torch.softmax(scale * torch.einsum("khd,hd->kh", kk, q[r]), 0)
            ref[r] = torch.einsum("kh,khd->hd", p, vv)
            mag = torch.einsum("kh,khd->hd", p, vv.abs())
            size = scale * torch.einsum("khd,hd->kh", kk.abs().amax(2, keepdim=True).expand_as(kk), q[r].abs()).amax(0)
            peak = (p * vv.abs().amax(2)).amax(0)
            tol[r] = (mag * (2 * 2**-11 + 2**-14 + 2 * (d // 16 + 2) * 2**-22 * 2 * size[:, None]) + len(kk) * 2**-21 * peak[:, None])
    return ref, tol


def check(out, q, cache, table, lens, starts, **kw):
    ref, tol = reference(q, cache, table, lens, starts, **kw)
    has = ~torch.isnan(tol).all(2).all(1)
    tol = tol + torch.finfo(q.dtype).eps / 2 * ref.abs() + torch.finfo(q.dtype).tiny
    err = (out.cpu().double() - ref).abs()[has]
    assert torch.isfinite(out.cpu()[has]).all()
    assert bool((err <= tol[has]).all()), float((err / tol[has]).max())


def randn(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_v_row_that_is_not_finite_reaches_the_rows_that_see_it(kv, prefix_path, kind, dtype, d, value):
    """V alone, K clean: every row that sees the key becomes NaN in that KV head, every other row and head stays as it was, bit for bit."""
    cache = kv.alloc(12, 2, d, 16, kind)
    rows, table, starts = batch(kv, [60, 9], [40, 9], 16, 8, 1)
    whole = kv.Rows(rows.table, rows.lens, torch.tensor([0, 60, 69], **I32))
    pre, pre_rows = torch.tensor([8, 11, 9], **I32), kv.Rows(torch.tensor([[8, 11, 9]], **I32), torch.tensor([37], **I32), torch.tensor([0, 37], **I32))
    k, v = (randn(s, 69, 2, d, dtype=dtype) for s in (2, 3))
    pk, pv = (randn(s, 37, 2, d, dtype=dtype) for s in (4, 5))
    q = randn(6, 49, 16, d, dtype=dtype).cuda()

    def outs():
        kv.write(cache, k.cuda(), v.cuda(), whole)
        kv.write(cache, pk.cuda(), pv.cuda(), pre_rows)
        return [kv.attention(q, cache, rows), kv.attention(q, cache, rows, causal=False), kv.attention_shared(q, cache, rows, pre, 37)]

    clean = outs()
    v[41, 1, d // 2] = value                    # position 41 of the first sequence, whose rows are positions 20 to 59
    sees = torch.zeros(49, dtype=torch.bool)
    sees[21:40] = True
    every = torch.arange(49) < 40
    for out, was, who in zip(outs(), clean, (sees, every, sees)):
        assert bool(torch.isnan(out[who.cuda()][:, 8:]).all())
        assert torch.equal(out[:, :8], was[:, :8]) and torch.equal(out[~who.cuda()], was[~who.cuda()])
    v[41, 1, d // 2] = 1
    pv[5, 0, 0] = value
    out = outs()[2]
    assert bool(torch.isnan(out[:, :8]).all()) and torch.isfinite(out[:, 8:]).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_k_row_that_is_not_finite_reaches_the_rows_that_see_it(kv, prefix_path, kind, dtype, value):
    """K alone, V clean, over 2,048 rows and heads: what codes of 0 leave of a score must not decide between a NaN and a key left out."""
    cache = kv.alloc(8, 1, 128, 16, kind)
    rows, table, starts = batch(kv, [70], [64], 16, 8, 1)
    whole = kv.Rows(rows.table, rows.lens, torch.tensor([0, 70], **I32))
    k, v = (randn(s, 70, 1, 128, dtype=dtype) for s in (2, 3))
    q = randn(4, 64, 32, 128, dtype=dtype).cuda()
    kv.write(cache, k.cuda(), v.cuda(), whole)
    clean = kv.attention(q, cache, rows)
    k[33, 0, 7] = value
    kv.write(cache, k.cuda(), v.cuda(), whole)
    assert bool(torch.isnan(kv.attention(q, cache, rows, causal=False)).all())
    out = kv.attention(q, cache, rows)
    assert torch.equal(out[:27], clean[:27]) and bool(torch.isnan(out[27:]).all())
    one = kv.Rows(rows.table, torch.zeros(1, **I32), torch.tensor([0, 64], **I32))
    assert bool(torch.isnan(kv.attention_shared(q, cache, one, rows.table[0].contiguous(), 70)).all())


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_query_that_is_not_finite_gives_nan_where_it_sees_a_key(kv, path, kind, dtype, value):
    """Its scores are infinite or NaN, and so is their softmax NaN: also where all of them are -inf. Without a key the row is 0."""
    cache = kv.alloc(6, 1, 64, 16, kind)
    fill(cache, 1)
    for page in (0, 1):
        cache.k[page] = torch.full((1, 16, 64), 1.0 - 2 * page, device="cuda").to(cache.k.dtype)      # scores of one sign
    rows = kv.Rows(torch.tensor([[0, 2], [1, 2], [2, 3], [4, 5]], **I32), torch.tensor([1, 16, 32, 0], **I32), torch.tensor([0, 1, 3, 23, 24], **I32))
    q = randn(2, 24, 4, 64, dtype=dtype)
    clean = kv.attention(q.cuda(), cache, rows)
    q[::2, 1::2, 9] = value
    out = kv.attention(q.cuda(), cache, rows)
    bad = torch.zeros(24, 4, dtype=torch.bool)
    bad[::2, 1::2] = True
    assert bool((out[23] == 0).all())
    bad[23] = False
    assert bool(torch.isnan(out[bad.cuda()]).all()) and torch.equal(out[~bad.cuda()], clean[~bad.cuda()])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("group", [3, 16])
def test_a_row_is_at_the_position_that_write_gave_it(kv, prefix_path, kind, group):
    """Lengths beyond the table, more rows named than the call has, rows named before the call's first: positions are lens - (starts[b + 1] - t) for
    every operator, and causal attention sees what lies up to there."""
    cache = kv.alloc(26, 2, 64, 16, kind)
    fill(cache, 1)
    q = randn(2, 30, 2 * group, 64).cuda()
    pre = torch.tensor([25, 24], **I32)
    for table, lens, starts in (
        ([[3, 7, 1, 9]], [70], [0, 10]),                                   # 64 tokens of room, positions 60 to 69
        ([[3, 7, 1, 9]], [1 << 30], [0, 30]),                              # all behind the room: a row sees all of it
        ([[3, 7, 1, 9]], [64], [0, 45]),                                   # the call has 30 rows: positions 19 to 48
        ([[3, 7, 1, 9], [2, 4, 6, 8]], [64, 50], [-20, 7, 100]),           # 20 rows before the call's first; 70 behind its last
        ([[3, 7, 1, 9], [2, 4, 6, 8], [10, 11, 12, 13]], [66, 20, 61], [0, 5, 28, 45]),   # the second has more rows than tokens
        ([[3, 7], [2, 4]], [-2147483648, 2147483647], [0, 15, 2147483647]),               # 32-bit ends
    ):
        rows = kv.Rows(torch.tensor(table, **I32), torch.tensor(lens, **I32), torch.tensor(starts, **I32))
        for causal in (True, False):
            check(kv.attention(q, cache, rows, causal=causal), q, cache, table, lens, starts, causal=causal)
        check(kv.attention_shared(q, cache, rows, pre, 19), q, cache, table, lens, starts, prefix=[25, 24], prefix_len=19)


def test_a_token_finds_itself(kv, path):
    """Rows written, and then attended to by queries that single out their own token, where the length is beyond the table."""
    cache = kv.alloc(4, 1, 64, 16, "int8")
    rows = kv.Rows(torch.tensor([[2, 0, 3, 1]], **I32), torch.tensor([70], **I32), torch.tensor([0, 26], **I32))
    at = torch.arange(26) + 44                                             # positions; the last six are beyond the table
    k = torch.zeros(26, 1, 64, dtype=torch.bfloat16)
    k[torch.arange(26), 0, torch.arange(26)] = 1
    v = randn(3, 26, 1, 64)
    kv.write(cache, k.cuda(), v.cuda(), rows)
    out = kv.attention((k * 1000).cuda(), cache, rows)
    back = kv.read(cache, rows, 26)[1]
    # other tokens' weights are e^-125; out and back are each rounded to bf16 (2^-8 of the value), out from V in fp16 (2^-11), whose sum is below 2^-6
    assert bool(((out - back).float().abs() <= 2**-6 * back.float().abs())[at < 64].all())
    assert bool((back[at >= 64] == 0).all())


@pytest.mark.parametrize("lens,starts", [
    ([160, 3, 160, 9], [0, 9, 2, 9, 1]), ([160, 3, 160, 9], [0, 5, 5, 4, 9]), ([160, 3, 160, 9], [3, 2, 5, 8, 9]), ([7] * 70, [0] * 60 + [9, 8] + [9] * 9),
])
@pytest.mark.parametrize("d", [64, 128])
def test_starts_that_do_not_ascend_are_reported_and_nothing_is_computed(kv, prefix_path, lens, starts, d):
    from rapid_h3_b200 import _lib
    cache = kv.alloc(40, 2, d, 16, "int8")
    fill(cache, 1)
    rows = kv.Rows(torch.arange(40, **I32).repeat(18)[:10 * len(lens)].view(len(lens), 10), torch.tensor(lens, **I32), torch.tensor(starts, **I32))
    q = randn(2, 9, 8, d).cuda()
    pre = torch.arange(30, **I32)
    good = kv.Rows(rows.table, rows.lens, torch.tensor([0] * len(lens) + [9], **I32))
    for call, kw in ((lambda r, out: kv.attention(q, cache, r, out=out), {}),
                     (lambda r, out: kv.attention_shared(q, cache, r, pre, 470, out=out), dict(prefix=pre.tolist(), prefix_len=470))):
        out = torch.full_like(q, 5.0)
        call(rows, out)
        with pytest.raises(RuntimeError, match="ascending"):
            _lib.check_status()
        assert bool((out == 5).all())
        call(good, out)                                                    # the next call is as any
        _lib.check_status()
        check(out, q, cache, rows.table.tolist(), lens, good.starts.tolist(), **kw)


@pytest.mark.parametrize("kind,dtype,d", [("int8", torch.bfloat16, 128), ("fp8", torch.bfloat16, 64), ("fp8", torch.float16, 128), ("int8", torch.float16, 64)])
@pytest.mark.parametrize("size", [12, 40, 90])
def test_a_large_v_row_costs_other_rows_nothing(kv, prefix_path, kind, dtype, d, size):
    """V rows 2^size times the others, at the beginning, inside and at the end of key tiles: rows that come before them, and rows that give
    them next to no weight, are as exact as without."""
    n, page = 420, 64
    cache = kv.alloc(10, 1, d, page, kind)
    rows, table, starts = batch(kv, [n], [n], page, 8, 1)
    k, v = (randn(s, n, 1, d).float() for s in (2, 3))
    k[:, :, :2] = 0
    big = [70, 127, 128, 200, 201, 419]
    v[big] *= 2.0 ** size
    k[big, :, 0] = 4.0                                    # found through two channels of q
    kv.write(cache, k.cuda(), v.cuda(), rows)
    q = randn(4, n, 4, d).float() * 0.3
    # the large rows' weights: 2^-(size + 20) and more (all that they add stays below fp16's largest)
    q[..., 0] = -0.7 * d ** 0.5 * (size + 20) / 4 * torch.tensor([1.0, 1.0, 0.9, 0.5 if dtype == torch.bfloat16 else 0.9])
    q = q.to(dtype).cuda()
    check(kv.attention(q, cache, rows), q, cache, table, [n], starts)
    pick = torch.tensor([0, 69, 70, 130, 300, 419])
    for r in pick.tolist():                               # single rows, and behind a prefix that holds large rows
        one = kv.Rows(rows.table, torch.tensor([r + 1], **I32), torch.tensor([0, 1], **I32))
        x = q[r:r + 1].contiguous()
        check(kv.attention(x, cache, one), x, cache, table, [r + 1], [0, 1])
    own = kv.Rows(torch.tensor([[8, 9]], **I32), torch.tensor([90], **I32), torch.tensor([0, 60], **I32))
    kv.write(cache, k[100:190].cuda(), (v[100:190] * 2.0**-5).cuda(), kv.Rows(own.table, own.lens, torch.tensor([0, 90], **I32)))
    x = q[-60:].contiguous()
    check(kv.attention_shared(x, cache, own, rows.table[0].contiguous(), n), x, cache, [[8, 9]], [90], [0, 60], prefix=table[0], prefix_len=n)


def test_v_scales_that_grow_and_fall_from_tile_to_tile(kv, path):
    """Every V row has a size of its own, over 2^60; and tiles whose rows are alike within 2^8, each tile of another size."""
    for seed, per_row in ((1, True), (2, False)):
        cache = kv.alloc(12, 2, 128, 64, "int8")
        fill(cache, seed)
        rows, table, starts = batch(kv, [700, 50], [90, 50], 64, 12, seed)
        g = torch.Generator().manual_seed(seed)
        e = torch.randint(-30, 31, (12, 2, 64), generator=g) if per_row else torch.randint(-30, 31, (12, 1, 1), generator=g) + torch.randint(-4, 5, (12, 2, 64), generator=g)
        cache.v_scale *= torch.exp2(e.float()).cuda()
        q = randn(seed + 2, 140, 6, 128).cuda()
        check(kv.attention(q, cache, rows), q, cache, table, [700, 50], starts)


@pytest.mark.parametrize("step", [20, 0, -20])
def test_k_scales_and_queries_of_very_different_size(kv, path, step):
    """Queries of 2^step with K rows over 2^12, the softmax scale such that the scores are some tens: held to a tolerance by each row's own scores."""
    cache = kv.alloc(8, 1, 128, 64, "int8")
    fill(cache, 1)
    rows, table, starts = batch(kv, [500], [40], 64, 8, 2)
    for i, p in enumerate(table[0]):
        cache.k_scale[p] *= 2.0 ** (i % 4 * 4 - 12)
    q = (randn(3, 40, 4, 128) * 2.0 ** step).cuda()
    check(kv.attention(q, cache, rows, scale=2.0 ** -step), q, cache, table, [500], starts, scale=2.0 ** -step)


def test_an_output_whose_rows_overlap_is_refused(kv):
    cache = kv.alloc(4, 2, 64, 16, "int8")
    fill(cache, 1)
    rows = kv.Rows(torch.arange(4, **I32).view(1, 4), torch.tensor([40], **I32), torch.tensor([0, 3], **I32))
    q = randn(2, 3, 4, 64).cuda()
    want = kv.attention(q, cache, rows)
    flat = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    for strides in ((0, 64), (64, 0), (256, 32), (64, 64), (128, 64), (200, 64), (64, 128), (0, 0), (192, 384)):
        with pytest.raises(RuntimeError, match="overlap"):
            kv.attention(q, cache, rows, out=flat.as_strided((3, 4, 64), (*strides, 1)))
    for strides in ((256, 64), (64, 192), (1024, 136), (72, 216), (96, 384), (192, 256), (192, 640)):     # token or head first, gaps, woven into one another
        out = flat.as_strided((3, 4, 64), (*strides, 1))
        kv.attention(q, cache, rows, out=out)
        assert torch.equal(out, want)
    one = kv.Rows(rows.table, rows.lens, torch.tensor([0, 1], **I32))
    kv.attention(q[:1], cache, one, out=flat.as_strided((1, 4, 64), (0, 64, 1)))       # one row only: its stride is nobody's


def test_the_output_may_be_the_query(kv, prefix_path):
    """Units in one CTA and cut between several, with and without a prefix."""
    for d, lens, news in ((128, [900, 70, 3000], [40, 1, 90]), (64, [20000], [2])):
        pages = sum(-(-n // 64) for n in lens) + 8
        cache = kv.alloc(pages, 2, d, 64, "int8")
        fill(cache, 1)
        rows, table, starts = batch(kv, lens, news, 64, pages - 8, 2)
        pre = torch.arange(pages - 8, pages, **I32)
        q = randn(3, starts[-1], 12, d).cuda()
        for call in (kv.attention, lambda *a, **kw: kv.attention_shared(*a, pre, 500, **kw)):
            x = q.clone()
            want = call(q, cache, rows)
            assert call(x, cache, rows, out=x) is x and torch.equal(x, want)


def test_no_gradient_passes(kv):
    """As documented: inputs may require one, outputs have none."""
    cache = kv.alloc(2, 2, 64, 16, "int8")
    rows = kv.Rows(torch.tensor([[0, 1]], **I32), torch.tensor([3], **I32), torch.tensor([0, 3], **I32))
    x = randn(1, 3, 2, 64).cuda().requires_grad_()
    kv.write(cache, x, x, rows)
    outs = [*kv.read(cache, rows, 3), kv.attention(x, cache, rows), kv.attention_shared(x, cache, rows, rows.table[0], 2)]
    assert not any(o.requires_grad or o.grad_fn is not None for o in outs)


def test_launches_are_counted(kv):
    from rapid_h3_b200 import _lib
    cache = kv.alloc(20, 2, 64, 16, "int8")
    fill(cache, 1)
    rows = kv.Rows(torch.tensor([[0, 1]], **I32), torch.tensor([3], **I32), torch.tensor([0, 3], **I32))
    x, pre = randn(1, 3, 2, 64).cuda(), torch.arange(2, 20, **I32)
    before = kv.use_wide(None)
    for use, call, want in ((None, lambda: kv.write(cache, x, x, rows), 1), (None, lambda: kv.write(cache, x[:0], x[:0], rows), 0), (None, lambda: kv.read(cache, rows, 3), 1),
                            (None, lambda: kv.read(cache, rows, 0), 0), (None, lambda: kv.attention(x, cache, rows), 1), (None, lambda: kv.attention(x[:0], cache, rows), 0),
                            ("apart", lambda: kv.attention_shared(x, cache, rows, pre, 280), 2), (True, lambda: kv.attention_shared(x, cache, rows, pre, 280), 1)):
        kv.use_wide(use)
        count = _lib.launch_count
        call()
        assert _lib.launch_count - count == want
    kv.use_wide(before)
