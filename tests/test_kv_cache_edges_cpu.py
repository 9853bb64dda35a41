"""What the cache operators decide on the host, against brute force."""
import copy
import itertools
import pickle
import random

import pytest
import torch

from rapid_h3_b200 import _lib, kv_cache


@pytest.mark.parametrize("t,heads", [(1, 1), (1, 4), (5, 1), (2, 2), (3, 4), (4, 3), (7, 5)])
def test_overlapping_rows_are_found(t, heads):
    d, found = 8, set()
    for st, sh in itertools.product(range(0, 80, 2), repeat=2):
        at = sorted(i * st + h * sh for i in range(t) for h in range(heads))
        overlap = any(b - a < d for a, b in zip(at, at[1:]))
        assert kv_cache._rows_overlap(t, heads, d, st, sh) == overlap, (st, sh)
        found.add(overlap)
    assert found == ({False} if t == heads == 1 else {False, True})


def test_scratch_of_many_streams_is_not_kept_for_ever(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False, raising=False)
    monkeypatch.setattr(kv_cache, "_SCRATCH", {})
    made = [kv_cache._scratch("cpu", 0, stream, 100) for stream in range(200)]
    assert len(kv_cache._SCRATCH) == kv_cache._KEPT_STREAMS
    assert kv_cache._scratch("cpu", 0, 199, 100)[0] is made[199][0] and kv_cache._scratch("cpu", 0, 0, 100)[0] is not made[0][0]
    big = kv_cache._scratch("cpu", 0, 199, kv_cache._KEPT_BYTES + 1)
    assert big[0] is made[199][0] and big[1].numel() == kv_cache._KEPT_BYTES + 1


def test_launches_of_a_call_are_counted():
    """A prefix with a pass of its own takes two."""
    lib, before = _lib.lib(), kv_cache.use_wide(None)
    sizes = lambda rows, prefix: (8, 4, 64, 128, 11, 64, rows, prefix)
    try:
        for use, want in ((False, 1), ("apart", 2), (True, 1)):
            kv_cache.use_wide(use)
            assert lib.rh3_kv_attn_launches(*sizes(64, 700)) == want and lib.rh3_kv_attn_launches(*sizes(64, 0)) == 1
        kv_cache.use_wide(None)
        assert lib.rh3_kv_attn_launches(*sizes(64, 12000)) == 2 and lib.rh3_kv_attn_launches(*sizes(64, 64)) == 1
        assert lib.rh3_kv_attn_launches(*sizes(0, 64)) == 0
    finally:
        kv_cache.use_wide(before)


@pytest.mark.parametrize("wide", [False, True])
def test_parts_of_a_prefix_fit_the_room_made_for_them(wide):
    """kv_plan's arithmetic, restated: what a unit weighs in the prefix pass, in tiles, or in keys with what it costs to begin; the CTAs with parts of a
    unit are those of its first and last tile's positions and all between, as the pass behind counts them; room is made for pre_splits."""
    rng = random.Random(1)
    full = 0
    for _ in range(4000):
        heads, tiles = rng.choice([1, 2, 8, 30]), rng.choice([1, 2, 7, rng.randint(1, 200)])
        prefix = rng.choice([1, 127, 128, 129, rng.randint(1, 40000)])
        kt, units = -(-prefix // 128), heads * tiles
        most = rng.choice([1, 2, 3]) * rng.choice([132, 148]) if not wide else rng.choice([132, 148])
        grid = min(units * kt, most)
        cost = 640 if wide else rng.choice([0, 2])
        unit = cost + (prefix if wide else kt)
        first, last = cost, cost + (kt - 1) * (128 if wide else 1)
        run = -(-units * unit // grid)
        if wide:
            run = max(run, 128)
        splits = min((last - first) // run + 2, kt)

        def tile(y):   # the first tile behind position y
            return kt if y >= unit else 0 if y <= cost else min(kt, -(-(y - cost) // 128) if wide else y - cost)

        parts = {}     # unit -> the CTAs that write a part of it
        for c in range(grid):
            x, x1 = min(units * unit, c * run), min(units * unit, (c + 1) * run)
            while x < x1:
                u, y = divmod(x, unit)
                end = min(unit, x1 - u * unit)
                if tile(y) < tile(end):
                    parts.setdefault(u, []).append(c)
                x = u * unit + end
        assert len(parts) == units
        for u, ctas in parts.items():
            x = u * unit
            assert ctas == list(range((x + first) // run, (x + last) // run + 1)) and len(ctas) <= splits
            full += len(ctas) == splits > 1
    assert full > 1000


def test_a_descriptor_that_is_copied_or_stored_describes_its_own_tensors(monkeypatch):
    """The addresses that calls take are those of the tensors that the object shows."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    codes, scales = [torch.zeros(2, 1, 16, 64, dtype=torch.int8) for _ in range(2)], [torch.zeros(2, 1, 16) for _ in range(2)]
    cache = kv_cache.KVCache(*codes, *scales)
    rows = kv_cache.Rows(torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32))
    for again in (copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        c, r = again(cache), again(rows)
        assert c._args == kv_cache.KVCache(c.k, c.v, c.k_scale, c.v_scale)._args
        assert r._args == kv_cache.Rows(r.table, r.lens, r.starts)._args
        assert (c.k.data_ptr() == cache.k.data_ptr()) == (r.lens.data_ptr() == rows.lens.data_ptr()) == (again is copy.copy)
    cache.v_scale += 1
    assert float(cache.v_scale.min()) == 1
    with pytest.raises(AttributeError):
        cache.v_scale = torch.zeros(2, 1, 16)
    class Named(kv_cache.KVCache):
        pass

    named = Named(*codes, *scales)
    named.name = "text"
    assert named.name == "text" and type(copy.copy(named)) is Named
    with pytest.raises(AttributeError):
        named.k = codes[0] + 1
    with pytest.raises(AttributeError):
        rows.lens = torch.zeros(1, dtype=torch.int32)
