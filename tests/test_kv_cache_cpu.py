"""Refusals of the cache operators that need no GPU, the descriptors' checks, and the arithmetic that deals tiles to CTAs."""
import bisect
import ctypes
import random

import pytest
import torch

from rapid_h3_b200 import _lib, kv_cache

P = 4096  # an address that is never touched: the argument checks come first


CACHE_ARGS = dict(kc=P, vc=P, ks=P, vs=P, pages=8, heads=8, page=64, D=128)
BATCH_ARGS = dict(table=P, table_stride=4, per_seq=4, lens=P, starts=P, B=2)


def pack(a):
    v = list(a.values())
    tail = kv_cache._ROWS if len(v) == 23 else kv_cache._ATTN
    return kv_cache._TENSORS.pack(*v[:6]) + kv_cache._CACHE.pack(*v[6:14]) + kv_cache._BATCH.pack(*v[14:20]) + tail.pack(*v[20:])


def rows_args(**kw):
    return pack(dict(k=P, k_st=1024, k_sh=128, v=P, v_st=1024, v_sh=128, **CACHE_ARGS, **BATCH_ARGS, T=3, kind=0, dtype=0) | kw)


def attn_args(**kw):
    return pack(dict(q=P, q_st=1024, q_sh=128, out=P, o_st=1024, o_sh=128, **(CACHE_ARGS | dict(heads=2)), **BATCH_ARGS, T=3, group=4, prefix_table=0,
                     prefix_pages=0, prefix=0, scale=0.1, kind=0, dtype=0, causal=1) | kw)


CACHE = [(dict(kind=2), b"kind"), (dict(kind=-1), b"kind"), (dict(D=96), b"head size"), (dict(page=8), b"16, 32, 64 or 128"), (dict(page=48), b"16, 32, 64 or 128"),
         (dict(pages=0), b"bad cache shape"), (dict(heads=0), b"bad cache shape"), (dict(heads=2000), b"bad cache shape"), (dict(pages=1 << 40), b"too large"),
         (dict(ks=P + 4), b"aligned"), (dict(vs=0), b"must be set")]
BATCH = [(dict(B=0), b"bad batch"), (dict(B=1 << 20), b"bad batch"), (dict(per_seq=-1), b"bad batch"), (dict(table_stride=3), b"bad batch"),
         (dict(T=-1), b"rows"), (dict(T=1 << 30), b"rows"), (dict(lens=0), b"null"), (dict(starts=0), b"null"), (dict(table=0), b"null")]


@pytest.mark.parametrize("change,said", CACHE + BATCH + [(dict(dtype=3), b"dtype"), (dict(k=P + 2), b"16-byte"), (dict(v_sh=100), b"16-byte"), (dict(k_st=1), b"16-byte")])
def test_write_refuses(change, said):
    assert _lib.lib().rh3_kv_write(rows_args(**change), None) < 0 and said in _lib.lib().rh3_last_error_string()


@pytest.mark.parametrize("change,said", CACHE + BATCH + [(dict(dtype=-1), b"dtype"), (dict(k=P + 8), b"aligned"), (dict(v=0), b"must be set")])
def test_read_refuses(change, said):
    assert _lib.lib().rh3_kv_read(rows_args(**change), None) < 0 and said in _lib.lib().rh3_last_error_string()


@pytest.mark.parametrize("change,said", CACHE + BATCH + [
    (dict(dtype=2), b"dtype"), (dict(group=0), b"per KV head"), (dict(group=1 << 20), b"per KV head"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(prefix=1), b"prefix"), (dict(prefix=65, prefix_pages=1, prefix_table=P), b"prefix"), (dict(prefix=-1), b"prefix"),
    (dict(q=0), b"16-byte"), (dict(q_st=4), b"16-byte"), (dict(o_sh=129), b"16-byte"), (dict(out=P + 2), b"16-byte"), (dict(), b"workspace")])
def test_attention_refuses(change, said):
    lib = _lib.lib()
    assert lib.rh3_kv_attn(attn_args(**change), None, 0, P, None) < 0 and said in lib.rh3_last_error_string()
    if not change:
        need = lib.rh3_kv_attn_workspace_bytes(2, 4, 64, 128, 4, 2, 3, 0)
        assert need > 0
        assert lib.rh3_kv_attn(attn_args(), P, need - 1, P, None) < 0 and said in lib.rh3_last_error_string()
        assert lib.rh3_kv_attn(attn_args(), P + 16, need, P, None) < 0 and said in lib.rh3_last_error_string()
        assert lib.rh3_kv_attn(attn_args(), P, need, None, None) < 0 and b"counters" in lib.rh3_last_error_string()
        assert lib.rh3_kv_attn(None, P, need, P, None) < 0


def test_calls_without_rows_do_nothing():
    lib = _lib.lib()
    assert lib.rh3_kv_write(rows_args(T=0, k=0, v=0), None) == 0 and lib.rh3_kv_read(rows_args(T=0, k=0, v=0), None) == 0
    assert lib.rh3_kv_write(None, None) < 0 and lib.rh3_kv_read(None, None) < 0
    assert lib.rh3_kv_attn(attn_args(T=0, q=0, out=0), None, 0, None, None) == 0


def test_there_is_no_cpu_path():
    codes, scales = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.KVCache(codes, codes, scales, scales)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.Rows(i[None], i, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="kind"):
        kv_cache.alloc(1, 1, kind="int4", device="cpu")


def test_every_tile_has_one_owner_and_every_cut_unit_is_joined_once():
    """The device's arithmetic (runs, slots, parts), restated: units of any sizes dealt to any grid."""
    rng = random.Random(1)
    for _ in range(400):
        units = [rng.choice([1, 1, 2, 5, rng.randint(1, 300)]) for _ in range(rng.randint(1, 60))]
        grid = rng.choice([1, 2, 7, 148, rng.randint(1, 400)])
        w = sum(units)
        run = -(-w // grid)
        first = [sum(units[:i]) for i in range(len(units))]
        slots, whole, counters = {}, set(), {}
        for c in range(grid):
            x, x1 = min(w, c * run), min(w, (c + 1) * run)
            while x < x1:
                u = bisect.bisect_right(first, x) - 1
                k0 = x - first[u]
                k1 = min(units[u], k0 + x1 - x)
                if k0 == 0 and k1 == units[u]:
                    whole.add(u)
                else:
                    assert (c, k0 == 0) not in slots
                    slots[c, k0 == 0] = u, k0, k1
                    counters.setdefault(first[u] // run, set()).add(u)   # the word a cut unit's parts are counted in
                x += k1 - k0
        assert all(len(v) == 1 and c < grid for c, v in counters.items())
        cut = set()
        for u in range(len(units)):
            c, n = first[u] // run, (first[u] + units[u] - 1) // run - first[u] // run + 1
            if n > 1:
                parts = [slots[c, True]] + [slots[c + i, False] for i in range(1, n)]
                assert all(p[0] == u for p in parts) and parts[0][1] == 0 and parts[-1][2] == units[u]
                assert all(a[2] == b[1] for a, b in zip(parts, parts[1:]))
                cut.add(u)
        assert cut | whole == set(range(len(units))) and not cut & whole and len(slots) == sum(1 for s in slots)


@pytest.mark.parametrize("wide", [False, True])
def test_units_that_cost_something_to_begin_are_dealt_without_gaps(wide):
    """The same with what a unit weighs besides its tiles: positions up to the cost stand for tile 0, and (wide: weights are in keys, linear in
    the row tile, 128 to a key tile) positions behind the last tile for its end. The CTAs with parts are told from two positions."""
    rng = random.Random(3)
    cut = 0
    for _ in range(400):
        cost = rng.choice([640, 256, 0]) if wide else rng.choice([0, 2, 3])
        tiles = [rng.choice([1, 1, 2, 5, rng.randint(1, 300)]) for _ in range(rng.randint(1, 60))]
        grid = rng.choice([1, 2, 7, 148, rng.randint(1, 400)])
        # wide: keys of a unit as the weight has them, more or fewer than its tiles hold
        weight = [cost + max(1, kt * 128 - rng.randint(-100, 300)) if wide else kt + cost for kt in tiles]
        begin = [sum(weight[:i]) for i in range(len(tiles))]
        w = sum(weight)
        run = max(128 if wide else 1, -(-w // grid))

        def tile(u, y):
            if y >= weight[u]:
                return tiles[u]
            return 0 if y <= cost else min(tiles[u], -(-(y - cost) // 128) if wide else y - cost)

        slots, whole = {}, set()
        for c in range(grid):
            x, x1 = min(w, c * run), min(w, (c + 1) * run)
            while x < x1:
                u = bisect.bisect_right(begin, x) - 1
                y, end = x - begin[u], min(weight[u], x1 - begin[u])
                k0, k1 = tile(u, y), tile(u, end)
                x = begin[u] + end
                if k0 == k1:
                    continue
                if k0 == 0 and k1 == tiles[u]:
                    whole.add(u)
                else:
                    assert (c, k0 == 0) not in slots
                    slots[c, k0 == 0] = u, k0, k1
        firsts = set()
        for u, kt in enumerate(tiles):
            last = min(weight[u], cost + (kt - 1) * 128 + 1) - 1 if wide else cost + kt - 1
            c = (begin[u] + cost) // run
            n = (begin[u] + last) // run - c + 1
            assert (n == 1) == (u in whole)
            if n > 1:
                parts = [slots.pop((c, True))] + [slots.pop((c + i, False)) for i in range(1, n)]
                assert all(q[0] == u for q in parts) and parts[0][1] == 0 and parts[-1][2] == kt
                assert all(a[2] == b[1] for a, b in zip(parts, parts[1:]))
                assert c not in firsts   # the word its parts are counted in
                firsts.add(c)
                cut += 1
        assert not slots
    assert cut > 1000


def test_an_abandoned_call_leaves_no_counters_behind(monkeypatch):
    def failed(name, *args):
        ctypes.c_int.from_address(args[1]).value = 1

    monkeypatch.setattr(_lib, "call", failed)
    monkeypatch.setattr(_lib, "stream", lambda: 0)
    monkeypatch.setitem(kv_cache._SCRATCH, (0, 0), ("counters", "workspace"))
    with pytest.raises(RuntimeError, match="device status 1"):
        _lib.check_status()
    assert not kv_cache._SCRATCH


def test_a_prefix_falls_into_as_many_parts_as_the_workspace_holds():
    rng = random.Random(2)
    for _ in range(2000):
        units, kt = rng.randint(1, 400), rng.randint(1, 300)
        grid = min(rng.choice([148, 132]), units * kt)
        run = -(-units * kt // grid)
        room = min((kt - 1) // run + 2, kt)
        assert all((u * kt + kt - 1) // run - u * kt // run + 1 <= room for u in range(units))
