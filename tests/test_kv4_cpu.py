"""The 4-bit cache without a GPU: the documented layout, the refusals of every entry point (all decided on the host before
any CUDA call), and the rotation table."""
import ctypes as C

import numpy as np
import pytest
import torch

from velox_inferer_b200 import Kv4Cache, ShapeError, Unsupported, _lib, rope_table

from . import kv4_ref as R

ERR_UNSUPPORTED, ERR_SHAPE = -1, -2


@pytest.mark.parametrize("D", [64, 128])
def test_block_layout_uses_every_byte_once(D):
    at = []
    for tau in range(16):
        at += [R.k_code_at(D, tau, b) for b in range(D // 2)] + [R.v_code_at(D, tau, b) for b in range(D // 2)]
        at += [R.k_scale_at(D, tau, g) for g in range(D // 16)] + [R.v_scale_at(D, tau, g) for g in range(D // 16)]
    assert sorted(at) == list(range(18 * D))


@pytest.mark.parametrize("D", [64, 128])
def test_lane_operands_are_contiguous(D):
    """What lane (g, t) of a warp needs lies at lane * (access size) in every plane."""
    for lane in range(32):
        g, t = lane // 4, lane % 4
        n = D // 8                                                       # bytes of one K row part / one V pair of pieces
        for h in range(2):
            got = [R.k_code_at(D, g + 8 * h, t * (D // 8) + i) for i in range(n)]
            assert got == [h * 4 * D + lane * n + i for i in range(n)]
            got = [R.v_code_at(D, 8 * h + 2 * t + j, g * (D // 16) + i) for j in range(2) for i in range(D // 16)]
            assert got == [8 * D + h * 4 * D + lane * n + i for i in range(n)]
        per = D // 64
        got = [R.k_scale_at(D, g + 8 * h, t * per + i) for h in range(2) for i in range(per)]
        assert got == [16 * D + lane * 2 * per + i for i in range(2 * per)]
        group = g * D // 8 // 16
        got = [R.v_scale_at(D, 8 * p + 2 * t + j, group) for p in range(2) for j in range(2)]
        assert got == [17 * D + (group * 4 + t) * 4 + i for i in range(4)]


def test_reference_quantiser_against_torch():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 128)) * np.exp(rng.standard_normal((50, 1)) * 3)).astype(np.float32)
    x[3] = 0
    x[4] = 1e-9
    x[5] = 1e6
    codes, scales = R.quantise(x, 16.0)
    amax = np.abs(x.reshape(50, 8, 16)).max(-1)
    want = (torch.from_numpy(amax * np.float32(16)) / torch.full((1,), 6.0)).clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(scales, want)
    back = R.values(codes, scales, 16.0)
    step = np.repeat(R.E4M3[scales], 16, -1) / 16
    live = (np.repeat(scales, 16, -1) > 0) & (np.repeat(scales, 16, -1) < 126)
    # half a step at the top of the grid is one scale; the scale itself may round down by 1/16 (of 6 of them)
    assert np.all(np.abs(back - x)[live] <= 1.5 * step[live])
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 2, dtype=np.float32)
    c, s = R.quantise(ties[None], 1.0)
    assert s[0, 0] == 0x38 and list(c[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 7]


def test_rope_table_far_positions():
    t = rope_table(200_001, 64, 1e6).numpy()
    for p in (0, 1, 199_999, 200_000):
        a = p * 1e6 ** (-np.arange(32) / 32)
        assert np.abs(t[p, :32] - np.cos(a)).max() <= 2.0 ** -24 and np.abs(t[p, 32:] - np.sin(a)).max() <= 2.0 ** -24


def test_cache_refusals():
    ok = torch.zeros(3, 2, 4, 18 * 64, dtype=torch.uint8)
    assert Kv4Cache(ok, 64, 64).bytes_per_token() == 2 * 72
    for bad, page, D, err in ((ok, 48, 64, Unsupported), (ok, 64, 96, Unsupported), (ok, 32, 64, ShapeError), (ok, 64, 128, ShapeError),
                              (ok.view(torch.int8), 64, 64, ShapeError), (ok[:, :1], 64, 64, ShapeError), (ok[0], 64, 64, ShapeError)):
        with pytest.raises(err):
            Kv4Cache(bad, page, D)
    with pytest.raises(ShapeError):
        Kv4Cache(ok, 64, 64, k_divisor=0.0)
    with pytest.raises(ShapeError):
        Kv4Cache(ok, 64, 64, v_divisor=float("nan"))


def _cache(**kw):
    f = dict(blocks=4096, pages=4, page_size=64, kv_heads=2, head_dim=128, k_divisor=16.0, v_divisor=16.0, reserved=0)
    f.update(kw)
    return _lib.Kv4CacheStruct(**f)


BAD_CACHES = [(dict(blocks=0), ERR_SHAPE), (dict(blocks=4104), ERR_UNSUPPORTED), (dict(pages=0), ERR_SHAPE),
              (dict(pages=1 << 25), ERR_UNSUPPORTED), (dict(page_size=8), ERR_UNSUPPORTED), (dict(page_size=48), ERR_UNSUPPORTED),
              (dict(head_dim=96), ERR_UNSUPPORTED), (dict(head_dim=256), ERR_UNSUPPORTED), (dict(kv_heads=0), ERR_SHAPE),
              (dict(k_divisor=0.0), ERR_SHAPE), (dict(v_divisor=-1.0), ERR_SHAPE), (dict(v_divisor=float("nan")), ERR_SHAPE)]

A = 1 << 20      # addresses no call below may reach: each is refused before any launch


def _attention(lib, cache=None, **kw):
    f = dict(q=A, qs=2048, out=2 * A, os=2048, table=A, cols=4, cu=A, kv=A, requests=2, tokens=4, heads=16, scale=0.1, causal=1, window=0,
             max_new=4, ws=A, ws_bytes=1 << 40)
    f.update(kw)
    c = _cache() if cache is None else cache
    return lib.velox_sm100_kv4_attention(f["q"], f["qs"], f["out"], f["os"], C.byref(c), f["table"], f["cols"], f["cu"], f["kv"], f["requests"],
                                         f["tokens"], f["heads"], f["scale"], f["causal"], f["window"], f["max_new"], f["ws"], f["ws_bytes"])


@pytest.mark.parametrize("kw,code", [
    (dict(heads=15), ERR_SHAPE), (dict(heads=0), ERR_SHAPE), (dict(requests=-1), ERR_SHAPE), (dict(tokens=-1), ERR_SHAPE),
    (dict(window=-1), ERR_SHAPE), (dict(scale=0.0), ERR_SHAPE), (dict(scale=float("nan")), ERR_SHAPE), (dict(scale=float("inf")), ERR_SHAPE),
    (dict(q=0), ERR_SHAPE), (dict(out=0), ERR_SHAPE), (dict(q=A + 2), ERR_UNSUPPORTED), (dict(qs=2047), ERR_SHAPE), (dict(qs=2049), ERR_UNSUPPORTED),
    (dict(os=2052), ERR_UNSUPPORTED), (dict(cu=0), ERR_SHAPE), (dict(kv=0), ERR_SHAPE), (dict(table=0), ERR_SHAPE), (dict(ws=0), ERR_SHAPE),
    (dict(ws_bytes=64), ERR_SHAPE), (dict(ws=A + 16), ERR_UNSUPPORTED), (dict(cols=(1 << 24) + 1), ERR_UNSUPPORTED),
    (dict(tokens=(1 << 27) + 1), ERR_UNSUPPORTED)])
def test_attention_refusals(kw, code):
    assert _attention(_lib.lib(), **kw) == code


def test_attention_of_nothing():
    for kw in (dict(requests=0), dict(tokens=0), dict(max_new=0)):
        assert _attention(_lib.lib(), q=0, out=0, ws=0, **kw) == 0


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_cache_struct_refusals(kw, code):
    lib, c = _lib.lib(), _cache(**kw)
    assert _attention(lib, cache=c) == code
    assert lib.velox_sm100_kv4_rows(C.byref(c), A, 3, A, A, 1) == code
    assert lib.velox_sm100_qk_norm_rope_kv4(None, 0, A, 4096, A, 4096, 0, None, None, None, 0, 0, 0, None, A, C.byref(c), None, 0, 0, 3, 0,
                                            1e-6, 0) == code


def test_cache_struct_size():
    assert C.sizeof(_lib.Kv4CacheStruct) == 40


def _rope(lib, **kw):
    f = dict(q=A, qs=512, k=A, ks=256, f32=0, qw=A, kw=A, rope=A, length=100, rot=128, inter=0, pos=A, qo=A, qos=512, ko=A, kos=256, of32=0, tokens=3,
             heads=4, kv=2, D=128, eps=1e-6)
    f.update(kw)
    return lib.velox_sm100_qk_norm_rope(f["q"], f["qs"], f["k"], f["ks"], f["f32"], f["qw"], f["kw"], f["rope"], f["length"], f["rot"], f["inter"],
                                        f["pos"], f["qo"], f["qos"], f["ko"], f["kos"], f["of32"], f["tokens"], f["heads"], f["kv"], f["D"],
                                        f["eps"], 0)


@pytest.mark.parametrize("kw,code", [
    (dict(D=80), ERR_UNSUPPORTED), (dict(rot=24), ERR_UNSUPPORTED), (dict(rot=144), ERR_SHAPE), (dict(rot=0), ERR_SHAPE), (dict(length=0), ERR_SHAPE),
    (dict(pos=0), ERR_SHAPE), (dict(q=0), ERR_SHAPE), (dict(ko=0), ERR_SHAPE), (dict(qs=511), ERR_SHAPE), (dict(qs=516), ERR_UNSUPPORTED),
    (dict(k=A + 8), ERR_UNSUPPORTED), (dict(qw=A + 4), ERR_UNSUPPORTED), (dict(rope=A + 8), ERR_UNSUPPORTED), (dict(tokens=-1), ERR_SHAPE),
    (dict(heads=0, kv=0), ERR_SHAPE), (dict(heads=-1), ERR_SHAPE), (dict(eps=-1.0), ERR_SHAPE), (dict(eps=float("nan")), ERR_SHAPE)])
def test_norm_rope_refusals(kw, code):
    assert _rope(_lib.lib(), **kw) == code


def test_norm_rope_of_nothing():
    assert _rope(_lib.lib(), tokens=0) == 0


def _plan(lib, **kw):
    f = dict(cached=A, new=A, requests=2, table=A, cols=3, free=A, n_free=5, taken=A, taken_out=A, page=64, tokens=9, cu=A, kv=A, pos=A, slots=A,
             status=A, ticket=A)
    f.update(kw)
    return lib.velox_sm100_kv4_plan(*f.values())


@pytest.mark.parametrize("kw,code", [
    (dict(page=8), ERR_UNSUPPORTED), (dict(requests=-1), ERR_SHAPE), (dict(tokens=-1), ERR_SHAPE), (dict(cols=-1), ERR_SHAPE), (dict(n_free=-1), ERR_SHAPE),
    (dict(cached=0), ERR_SHAPE), (dict(table=0), ERR_SHAPE), (dict(free=0), ERR_SHAPE), (dict(taken=0), ERR_SHAPE), (dict(taken_out=0), ERR_SHAPE),
    (dict(cu=0), ERR_SHAPE), (dict(kv=0), ERR_SHAPE), (dict(pos=0), ERR_SHAPE), (dict(slots=0), ERR_SHAPE), (dict(status=0), ERR_SHAPE), (dict(ticket=0), ERR_SHAPE)])
def test_plan_refusals(kw, code):
    assert _plan(_lib.lib(), **kw) == code


def test_workspace_refusals():
    lib = _lib.lib()
    for heads, kv, D in ((0, 1, 128), (15, 2, 128), (16, 0, 128), (16, 2, 96)):
        assert lib.velox_sm100_kv4_attention_workspace(heads, kv, D) == -1


# ---- how the attention kernels cut a step (restated from csrc/kv4_items.cuh) ---------------------------

def _share(total, i, n):
    return total * i // n


def _block_of(u, total, n):
    return ((u + 1) * n + total - 1) // total - 1


def _cut(items, grid, min_run, extra):
    """For items of `items[i]` tiles: {item: {block: (k0, k1, first, begin, end)}}."""
    units = [nt + extra for nt in items]
    total = sum(units)
    cap = min(grid, max(len(items), total // min_run))
    even = cap // len(items) * len(items)
    n = max(even, min(len(items), cap)) if even * 16 >= cap * 15 or total < 8 * cap else cap
    held = {i: {} for i in range(len(items))}
    for c in range(n):
        begin, end = _share(total, c, n), _share(total, c + 1, n)
        assert end > begin
        first = 0
        for i, nt in enumerate(items):
            stop = first + nt + extra
            if stop > begin and first < end:
                tile_at = lambda x: 0 if x <= 0 else nt if x >= nt + extra else x * nt // (nt + extra)  # noqa: E731,B023
                k0, k1 = tile_at(max(begin, first) - first), tile_at(end - first)
                f, l = _block_of(first, total, n), _block_of(stop - 1, total, n)
                assert _share(total, f, n) <= first < _share(total, f + 1, n)
                assert _share(total, l, n) <= stop - 1 < _share(total, l + 1, n)
                b = f + (tile_at(_share(total, f + 1, n) - first) == 0)
                e = l - (tile_at(_share(total, l, n) - first) == nt)
                held[i][c] = (k0, k1, f, b, e)
            first = stop
    return held


@pytest.mark.parametrize("extra", [1, 3])
def test_every_tile_is_in_one_block_and_the_counts_agree(extra):
    rng = np.random.default_rng(extra)
    for _ in range(400):
        items = [int(x) for x in rng.choice([1, 1, 2, 3, 5, 17, 64, 300], rng.choice([1, 2, 3, 8, 20, 64]))]
        held = _cut(items, int(rng.choice([1, 2, 7, 148, 296])), 4, extra)
        slots = set()
        for i, nt in enumerate(items):
            parts = {c: x for c, x in held[i].items() if x[0] < x[1]}
            assert [t for c in sorted(parts) for t in range(*parts[c][:2])] == list(range(nt))
            assert len({x[2:] for x in parts.values()}) == 1
            _, _, first, begin, end = next(iter(parts.values()))
            assert sorted(parts) == list(range(begin, end + 1))         # what the join waits for
            for c in parts:
                if begin != end:                                          # a parked part has a place of its own
                    assert (c, c == first) not in slots
                    slots.add((c, c == first))


def _cut_by_items(items, grid, parts):
    """Items by themselves: {item: {block: (k0, k1, begin, end)}}, whole or in `parts` runs, several whole ones per block where
    there are more items than blocks."""
    held = {i: {} for i in range(len(items))}
    total = len(items) * parts
    blocks = min(grid, total)
    for c in range(blocks):
        begin, end = _share(total, c, blocks), _share(total, c + 1, blocks)
        for i in range(begin // parts, (end - 1) // parts + 1):
            nt, first = items[i], i * parts
            some = min(parts, nt)
            tile_at = lambda x: 0 if x <= 0 else nt if x >= some else x * nt // some  # noqa: E731,B023
            k0, k1 = tile_at(max(begin, first) - first), tile_at(end - first)
            if k0 < k1:
                f = _block_of(first, total, blocks)
                held[i][c] = (k0, k1, f, f + some - 1)
    return held


def test_items_cut_by_themselves_hold_every_tile_once():
    rng = np.random.default_rng(10)
    for _ in range(800):
        items = [int(x) for x in rng.choice([1, 1, 2, 3, 5, 17, 64, 300], rng.choice([1, 2, 3, 8, 20, 64, 300]))]
        grid = int(rng.choice([1, 2, 7, 148, 296]))
        parts = int(rng.integers(1, max(1, grid // len(items)) + 1))
        held = _cut_by_items(items, grid, parts)
        for i, nt in enumerate(items):
            assert [t for c in sorted(held[i]) for t in range(*held[i][c][:2])] == list(range(nt))
            _, _, begin, end = next(iter(held[i].values()))
            assert sorted(held[i]) == list(range(begin, end + 1))         # what the join waits for
            if begin != end:                                              # a block of a shared item has no other
                assert all(sum(c in held[k] for k in range(len(items))) == 1 for c in held[i])
