"""The operators between the q|k|v and o linears over the 4-bit cache, against plain 64-bit forms (kv4_ref.py)."""
import numpy as np
import pytest
import torch

from velox_inferer_b200 import Kv4Cache, Kv4Step, ShapeError, rope_table

from . import kv4_ref as R
from .gpu_util import backend

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# ---- plan --------------------------------------------------------------------------------------------

PLANS = [  # cached, new, page, cols, free, taken, tokens
    ([0], [1], 16, 1, 1, 0, 1),
    ([16, 15, 17], [1, 1, 1], 16, 3, 9, 2, 3),
    ([5, 0, 64, 63, 128], [0, 70, 0, 2, 1], 64, 4, 20, 3, 80),          # nothing new, padded rows
    ([100, 10], [300, 50], 32, 40, 4, 1, 350),                          # pages run out inside the first request
    ([100, 10], [30, 500], 32, 5, 40, 0, 530),                          # the table row is full
    ([7, 7, 7], [9, 9, 9], 16, 4, 6, 0, 20),                            # more new tokens than rows
    ([-3, 4], [5, -2], 16, 2, 4, 0, 8),                                 # negative lengths count as none
    ([], [], 64, 0, 0, 0, 5),
    ([3], [4], 128, 2, 0, 0, 4),                                        # no pages at all, one is there
    ([1000000], [3000], 128, 8000, 30, 0, 3000),
]


def run_plan(b, cached, new, page, table, free, taken, tokens, inplace):
    step = Kv4Step(b, len(cached), tokens)
    for x in (step.cu, step.kv_lens, step.positions, step.slots, step.status):
        x.fill_(-77)
    t, out = i32([taken]), i32([-5])
    tab = i32(table).reshape(table.shape)
    b.kv4_plan(i32(cached), i32(new), tab, i32(free), t, page, step, None if inplace else out)
    assert step.ticket.item() == 0
    used = (t if inplace else out).item()
    if not inplace:
        assert t.item() == taken
    return tab.cpu().numpy(), step, used


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(case, inplace):
    cached, new, page, cols, n_free, taken, tokens = PLANS[case]
    rng = np.random.default_rng(case)
    ids = rng.permutation(10000)
    free = ids[:n_free]
    table = np.full((len(cached), cols), -9, dtype=np.int64)
    for b_, c in enumerate(cached):
        h = min(max(0, -(-c // page)), cols)
        table[b_, :h] = rng.integers(0, 9000, h)
    want = R.plan(cached, new, table, free, taken, page, tokens)
    tab, step, used = run_plan(backend(), cached, new, page, table, free, taken, tokens, inplace)
    assert np.array_equal(tab, want[0])
    for got, w in zip((step.cu, step.kv_lens, step.positions, step.slots), want[1:5]):
        assert np.array_equal(got.cpu().numpy(), w)
    assert used == want[5] and step.status.item() == want[6]


@pytest.mark.parametrize("requests", [511, 512, 513, 1500])
def test_plan_many_requests(requests):
    rng = np.random.default_rng(requests)
    cached, new = rng.integers(0, 300, requests), rng.integers(0, 40, requests) * (rng.random(requests) < 0.7)
    page, cols, tokens = 16, 22, int(new.sum()) + 100
    table = rng.integers(0, 9000, (requests, cols))
    free = rng.permutation(20000)[:5000]
    want = R.plan(cached, new, table, free, 7, page, tokens)
    tab, step, used = run_plan(backend(), cached, new, page, table, free, 7, tokens, False)
    assert np.array_equal(tab, want[0])
    for got, w in zip((step.cu, step.kv_lens, step.positions, step.slots), want[1:5]):
        assert np.array_equal(got.cpu().numpy(), w)
    assert used == want[5] and step.status.item() == want[6]


def test_plan_page_ids_past_the_slots():
    """Ids whose slots would pass 32 bits, or negative ones, in the table and in the free list: no slot."""
    tab, step, _ = run_plan(backend(), [5, 5, 16], [1, 20, 20], 16, np.array([[-7, 0, 0], [1 << 27, 0, 0], [3, 0, 0]]), [1 << 28, (1 << 27) - 1], 0, 41, False)
    assert np.array_equal(tab, [[-7, 0, 0], [1 << 27, 1 << 28, 0], [3, (1 << 27) - 1, -1]])
    slots = step.slots.cpu().numpy()
    last = ((1 << 27) - 1) * 16
    assert np.all(slots[:21] == -1) and np.array_equal(slots[21:37], last + np.arange(16)) and np.all(slots[37:] == -1)
    assert step.kv_lens.tolist() == [6, 25, 32] and step.status.item() == 1


# ---- norms, rotation, store --------------------------------------------------------------------------

def inputs(T, hq, hkv, D, dtype, seed, wide=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    mk = lambda h: torch.randn(T, h, D, generator=g, device=DEV).to(dtype)  # noqa: E731
    if not wide:
        return mk(hq) * 2, mk(hkv) * 3, mk(hkv)
    # views into one q|k|v buffer
    big = torch.randn(T, (hq + 2 * hkv) * D + 24, generator=g, device=DEV).to(dtype)
    cut = lambda a, h: big[:, a: a + h * D].view(T, h, D) if T else mk(h)  # noqa: E731
    return cut(8, hq), cut(8 + hq * D, hkv), cut(16 + (hq + hkv) * D, hkv)


def f64(t):
    return t.detach().double().cpu().numpy()


def close_rows(got, x, weight, eps, offset, rope, pos, inter):
    """got against the 64-bit form: 14 single-precision roundings of each product that enters a value (13 sums of positive
    squares, halved by the root, root, quotient, two products; three more in the rotation), plus the output's own."""
    want = R.norm_rope(x, weight, eps, offset, rope, pos, inter)
    mag = R.norm_rope(x, weight, eps, offset, None, pos, inter)
    if rope is not None:   # |a cos| + |b sin|, by the triangle inequality at most |a| + |b|
        rot = rope.shape[1]
        m = np.abs(mag)
        if inter:
            s = m[..., 0:rot:2] + m[..., 1:rot:2]
            m[..., 0:rot:2], m[..., 1:rot:2] = s, s
        else:
            s = m[..., : rot // 2] + m[..., rot // 2: rot]
            m[..., : rot // 2], m[..., rot // 2: rot] = s, s
        mag = m
    live = np.ones(len(pos), bool) if rope is None else (pos >= 0) & (pos < rope.shape[0])
    out = 2.0 ** -24 if got.dtype == torch.float32 else 2.0 ** -8
    err = np.abs(f64(got) - want)[live]
    assert np.all(err <= (14 * 2.0 ** -24 * np.abs(mag) + out * np.abs(want) * (1 + 1e-5) + 1e-30)[live]), err.max()
    return live


@pytest.mark.parametrize("T,hq,hkv,D,rot,inter,offset,dt,odt", [
    (1, 64, 8, 128, 128, False, False, "bf16", "bf16"), (5, 3, 1, 128, 64, True, False, "f32", "f32"),
    (300, 7, 3, 64, 64, False, True, "bf16", "f32"), (33, 16, 16, 64, 32, False, False, "f32", "bf16"),
    (2100, 10, 2, 128, 128, True, False, "bf16", "bf16"), (17, 1, 5, 128, 16, False, True, "bf16", "bf16"), (9, 64, 8, 64, 16, True, False, "f32", "f32")])
def test_norm_rope(T, hq, hkv, D, rot, inter, offset, dt, odt):
    b = backend()
    dts = {"bf16": torch.bfloat16, "f32": torch.float32}
    q, k, _ = inputs(T, hq, hkv, D, dts[dt], T, wide=T % 2 == 1)
    g = torch.Generator(device=DEV).manual_seed(T + 1)
    qw, kw = torch.rand(D, generator=g, device=DEV) + 0.5, torch.randn(D, generator=g, device=DEV)
    rope = rope_table(5000, rot, 1e4).to(DEV)
    pos = torch.randint(-3, 5003, (T,), generator=g, device=DEV, dtype=torch.int32)
    qo, ko = torch.full((T, hq, D), 9.0, dtype=dts[odt], device=DEV), torch.full((T, hkv, D), 9.0, dtype=dts[odt], device=DEV)
    b.qk_norm_rope(q, k, qw, kw, rope, pos, qo, ko, 1e-5, offset, inter)
    p = pos.cpu().numpy()
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        live = close_rows(got, f64(x), w.cpu().numpy(), 1e-5, offset, rope.cpu().numpy(), p, inter)
        assert np.all(f64(got)[~live] == 9.0)


@pytest.mark.parametrize("weight,rope", [(True, False), (False, True), (False, False)])
def test_norm_rope_parts(weight, rope):
    b = backend()
    q, k, _ = inputs(21, 4, 2, 128, torch.bfloat16, 3)
    w = torch.rand(128, device=DEV) if weight else None
    tab = rope_table(100, 128).to(DEV) if rope else None
    pos = torch.arange(21, dtype=torch.int32, device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    b.qk_norm_rope(q, k, w, None, tab, pos if rope else None, qo, ko)
    for got, x, ww in ((qo, q, w), (ko, k, None)):
        close_rows(got, f64(x), None if ww is None else ww.cpu().numpy(), 1e-6, False, None if tab is None else tab.cpu().numpy(), pos.cpu().numpy(), False)


def test_norm_rope_in_place_and_alone():
    b = backend()
    q, k, _ = inputs(40, 8, 2, 128, torch.bfloat16, 4)
    w, tab = torch.rand(128, device=DEV), rope_table(100, 128).to(DEV)
    pos = torch.arange(40, dtype=torch.int32, device=DEV)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    b.qk_norm_rope(q, k, w, w, tab, pos, qo, ko)
    k2 = torch.empty_like(k)
    b.qk_norm_rope(None, k, None, w, tab, pos, None, k2)
    b.qk_norm_rope(q, None, w, None, tab, pos, q, None)     # in place
    assert torch.equal(qo, q) and torch.equal(ko, k2)


def make_cache(pages, hkv, page, D, seed=0, kdiv=16.0, vdiv=8.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = torch.randint(0, 256, (pages, hkv, page // 16, 18 * D), generator=g, device=DEV, dtype=torch.uint8)
    return Kv4Cache(s, page, D, kdiv, vdiv)


@pytest.mark.parametrize("T,hq,hkv,D,page,dt,weight,rope", [
    (1, 64, 8, 128, 64, "bf16", True, True), (50, 6, 3, 64, 16, "bf16", True, True), (2048, 8, 2, 128, 128, "bf16", True, True),
    (33, 0, 1, 128, 32, "f32", True, True), (70, 4, 4, 64, 64, "f32", False, False), (19, 2, 2, 128, 16, "bf16", False, True)])
def test_store_and_rows(T, hq, hkv, D, page, dt, weight, rope):
    b = backend()
    dtype = torch.bfloat16 if dt == "bf16" else torch.float32
    q, k, v = inputs(T, max(hq, 1), hkv, D, dtype, T, wide=T % 2 == 0)
    if hq == 0:
        q = None
    pages = -(-T // page) + 3
    cache = make_cache(pages, hkv, page, D)
    before = cache.storage.cpu().numpy().copy()
    rng = np.random.default_rng(T)
    slots = rng.permutation(pages * page)[:T]
    if T > 10:
        slots[3], slots[5] = -1, pages * page      # outside the cache
    w = torch.randn(D, device=DEV) if weight else None
    tab = rope_table(3000, D // 2).to(DEV) if rope else None
    pos = rng.integers(0, 3000, T)
    qo = None if q is None else torch.empty_like(q).contiguous()
    b.qk_norm_rope_kv4(q, k, v, w, w, tab, i32(pos) if rope else None, i32(slots), cache, qo, 1e-6)
    nw, nt = None if w is None else w.cpu().numpy(), None if tab is None else tab.cpu().numpy()
    if q is not None:
        close_rows(qo, f64(q), nw, 1e-6, False, nt, pos, False)
    kk = R.norm_rope(f64(k), nw, 1e-6, False, nt, pos, False).astype(np.float32)
    want = R.Cache(before, page, D, cache.k_divisor, cache.v_divisor)
    for t in range(T):
        if 0 <= slots[t] < pages * page:
            want.write(int(slots[t]), kk[t], f64(v)[t].astype(np.float32))
    assert np.array_equal(cache.storage.cpu().numpy(), want.s)      # the written rows and everything between them
    for odt in (torch.float32, torch.bfloat16):
        ko, vo = torch.full((T, hkv, D), 5.0, dtype=odt, device=DEV), torch.full((T, hkv, D), 5.0, dtype=odt, device=DEV)
        b.kv4_rows(cache, i32(slots), ko, vo)
        for t in range(T):
            if 0 <= slots[t] < pages * page:
                rk, rv = want.read(int(slots[t]))
                for got, x in ((ko, rk), (vo, rv)):
                    assert torch.equal(got[t].cpu(), torch.from_numpy(x.astype(np.float32)).to(odt))
            else:
                assert torch.all(ko[t] == 5) and torch.all(vo[t] == 5)
        only = torch.empty(T, hkv, D, dtype=odt, device=DEV).fill_(5)
        b.kv4_rows(cache, i32(slots), None, only)
        assert torch.equal(only, vo)


def test_store_ties_extremes_and_nonfinite():
    """Ties, zeros, values past the grid's ends: the documented bytes. A NaN element is stored as some code and leaves
    its group finite; infinities saturate."""
    b = backend()
    x = torch.zeros(8, 1, 64, device=DEV)
    x[0, 0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 2) / 16
    x[1] = 1e-8
    x[2] = -1e8
    x[3, 0, ::2] = -0.1
    x[4, 0, 5] = 448 * 6 / 16
    x[5, 0, 5] = float("nan")
    x[5, 0, 6] = 1.0
    x[6, 0, 17] = float("-inf")
    cache = make_cache(1, 1, 16, 64, kdiv=16.0, vdiv=16.0)
    slots = i32(np.arange(8))
    b.kv4_store(x, x, slots, cache)
    want = R.Cache(np.zeros_like(cache.storage.cpu().numpy()), 16, 64, 16.0, 16.0)
    for t in (0, 1, 2, 3, 4, 7):
        want.write(t, f64(x)[t].astype(np.float32), f64(x)[t].astype(np.float32))
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    b.kv4_rows(cache, slots, ko, vo)
    for t in (0, 1, 2, 3, 4, 7):
        assert np.array_equal(f64(ko)[t], want.read(t)[0]) and np.array_equal(f64(vo)[t], want.read(t)[1])
    assert torch.isfinite(ko).all() and torch.isfinite(vo).all()
    # 1 beside the NaN: scale e4m3(16 / 6 = 2.667) = 2.75, code e2m1(16 / 2.75 = 5.8) = 6
    assert ko[6, 0, 17].item() == -168.0 and ko[5, 0, 6].item() == 6 * 2.75 / 16


# ---- attention ---------------------------------------------------------------------------------------

def scene(lens, new, hq, hkv, D, page, seed=0, spare=0, qscale=1.0, kdiv=16.0, vdiv=8.0):
    """Random cache (all bytes random, then real rows in the requests' pages), table, queries."""
    rng = np.random.default_rng(seed)
    need = [-(-l // page) for l in lens]
    pages = sum(need) + 3
    ids = rng.permutation(pages)
    cols = max(need + [0]) + 1
    table, at = np.full((len(lens), cols), -1, dtype=np.int64), 0
    cache = make_cache(pages, hkv, page, D, seed, kdiv, vdiv)
    slots = []
    for b_, n in enumerate(need):
        table[b_, :n] = ids[at: at + n]
        at += n
        slots += [int(table[b_, j // page]) * page + j % page for j in range(lens[b_])]
    g = torch.Generator(device=DEV).manual_seed(seed)
    if slots:
        k = torch.randn(len(slots), hkv, D, generator=g, device=DEV)
        k *= torch.exp(0.5 * torch.randn(hkv, D, generator=g, device=DEV))
        v = torch.randn(len(slots), hkv, D, generator=g, device=DEV)
        backend().kv4_store(k, v, i32(slots), cache)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    T = int(cu[-1]) + spare
    q = (torch.randn(T, hq, D, generator=g, device=DEV) * qscale).to(torch.bfloat16)
    return cache, table, cu, q, T


def check(cache, table, cu, lens, q, out, fill, scale, causal, window, rows=None):
    ref = R.Cache(cache.storage.cpu().numpy(), cache.page_size, cache.head_dim, cache.k_divisor, cache.v_divisor)
    want, spread, reach = R.attention(f64(q), ref, table, cu, lens, scale, causal, window)
    got = f64(out)
    none = np.isnan(want)
    assert np.all(got[none] == fill)
    bound = R.attention_bound(want, spread, reach, max(list(lens) + [1]), 2688 / cache.v_divisor, cache.head_dim)
    bad = ~none & ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.abs(got - want)[bad].max(), np.argwhere(bad)[:5], int(bad.sum()))


ATTN = [  # lens, new, hq, hkv, D, page, causal, window, spare
    ([1], [1], 8, 1, 128, 16, True, 0, 0),
    ([1, 2, 3], [1, 1, 1], 4, 2, 64, 16, True, 0, 2),
    ([17, 15, 16, 0, 33], [1, 1, 1, 0, 1], 16, 2, 128, 16, True, 0, 3),
    ([700], [1], 64, 8, 128, 64, True, 0, 0),
    ([1500, 1, 260, 31], [1, 1, 1, 1], 8, 1, 128, 32, True, 0, 0),
    ([900, 300], [1, 1], 28, 4, 64, 128, True, 0, 1),
    ([500, 80], [1, 1], 16, 1, 128, 64, True, 0, 0),                  # sixteen query heads on one kv head
    ([333, 64, 65], [3, 2, 1], 8, 2, 64, 64, True, 0, 0),             # a drafter's tokens
    ([600, 40], [4, 1], 8, 8, 128, 16, True, 100, 2),                 # window, ungrouped
    ([300], [1], 8, 2, 128, 64, False, 0, 0),
    ([90], [5], 10, 2, 64, 32, False, 7, 0),                          # window without causality
    ([0, 5], [1, 1], 8, 2, 128, 16, True, 0, 0),                      # a row that sees nothing
    ([3], [7], 4, 1, 64, 16, True, 0, 0),                             # more new rows than tokens: the first see nothing
    ([40], [40], 8, 2, 128, 64, True, 0, 3),                          # a whole prompt
    ([200, 129, 61], [200, 65, 61], 16, 2, 128, 64, True, 0, 5),
    ([150, 90], [20, 90], 14, 2, 64, 16, True, 33, 0),
    ([260, 7, 130], [19, 1, 64], 8, 1, 128, 32, False, 0, 1),
    ([300], [257], 5, 1, 128, 128, True, 0, 0),
    ([1000, 3, 500], [100, 1, 33], 2, 2, 64, 32, True, 0, 0),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(case):
    lens, new, hq, hkv, D, page, causal, window, spare = ATTN[case]
    b = backend()
    cache, table, cu, q, T = scene(lens, new, hq, hkv, D, page, case, spare)
    out = torch.full((T, hq, D), 0.75, dtype=torch.bfloat16, device=DEV)
    ws = b.kv4_workspace(hq, hkv, D)
    args = (cache, i32(table), i32(cu), i32(lens), ws)
    b.kv4_attention(q, out, *args, causal=causal, window=window, max_new=max(new))
    check(cache, table, cu, lens, q, out, 0.75, D ** -0.5, causal, window)
    again = torch.full_like(out, 0.75)                                 # same workspace: the same bits
    b.kv4_attention(q, again, *args, causal=causal, window=window, max_new=max(new))
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    again.fill_(0.75)                                                  # without the hint
    b.kv4_attention(q, again, *args, causal=causal, window=window)
    check(cache, table, cu, lens, q, again, 0.75, D ** -0.5, causal, window)


@pytest.mark.parametrize("requests", [33, 64, 257, 300, 513, 700])
@pytest.mark.parametrize("new", [1, 30])
def test_attention_many_requests(requests, new):
    """More requests than a warp, a block of the decode kernel (256) and one of the prefill kernel (512) count at once."""
    b = backend()
    rng = np.random.default_rng(requests)
    fresh = rng.integers(0, 2, requests) if new == 1 else np.where(rng.random(requests) < 0.1, rng.integers(17, new + 1, requests), 1)
    lens = fresh + rng.integers(0, 40, requests)
    cache, table, cu, q, T = scene(list(lens), list(fresh), 2, 1, 64, 16, requests, 2)
    out = torch.full((T, 2, 64), 0.75, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32(lens), b.kv4_workspace(2, 1, 64), max_new=int(fresh.max()))
    check(cache, table, cu, lens, q, out, 0.75, 0.125, True, 0)


@pytest.mark.parametrize("qscale,scale", [(1e-3, 1.0), (300.0, 0.02), (1e20, 1e-21), (0.0, 1.0)])
def test_attention_query_ranges(qscale, scale):
    b = backend()
    cache, table, cu, q, T = scene([200, 50], [1, 20], 8, 2, 128, 32, 5, 0, qscale)
    q[:, 0] *= 1e-6                                                    # heads of very different size
    out = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32([200, 50]), b.kv4_workspace(8, 2, 128), scale=scale)
    check(cache, table, cu, [200, 50], q, out, 0, scale, True, 0)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_one_nan_row(new):
    """A query with a NaN gives NaN in its own row and head, nowhere else."""
    b = backend()
    cache, table, cu, q, T = scene([300], [new], 16, 2, 128, 64, 6)
    out, ref = torch.zeros(T, 16, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(T, 16, 128, dtype=torch.bfloat16, device=DEV)
    ws = b.kv4_workspace(16, 2, 128)
    args = (cache, i32(table), i32(cu), i32([300]), ws)
    b.kv4_attention(q, ref, *args, max_new=new)
    q[new // 2, 5, 17] = float("nan")
    b.kv4_attention(q, out, *args, max_new=new)
    assert torch.isnan(out[new // 2, 5]).all()
    out[new // 2, 5] = ref[new // 2, 5]
    assert torch.equal(out, ref)


@pytest.mark.parametrize("new", [1, 40])
def test_attention_pages_outside_the_cache(new):
    b = backend()
    lens = [260, 100]
    cache, table, cu, q, T = scene(lens, [new, 1], 8, 2, 128, 32, 7)
    table[0, 1], table[0, 5], table[1, 0] = -1, cache.pages, 1 << 30
    out = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32(lens), b.kv4_workspace(8, 2, 128), max_new=new)
    check(cache, table, cu, lens, q, out, 0, 128 ** -0.5, True, 0)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_pages_shared_by_requests(new, page):
    """A common prefix: the same page ids in several rows of the table, and twice in one."""
    b = backend()
    lens = [150 + new, 70 + new, 3 * page + new]
    cache, table, cu, q, T = scene(lens, [new] * 3, 8, 2, 64, page, 12)
    table[1, :2], table[2, 1] = table[0, :2], table[2, 0]
    out = torch.zeros(T, 8, 64, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32(lens), b.kv4_workspace(8, 2, 64), max_new=new)
    check(cache, table, cu, lens, q, out, 0, 0.125, True, 0)


@pytest.mark.parametrize("heads,kv_heads,D", [(64, 1, 64), (33, 1, 128), (100, 2, 64), (3, 3, 128), (48, 2, 128)])
def test_attention_group_sizes(heads, kv_heads, D):
    """Groups of 1 to 64 query heads, with one and two new tokens."""
    b = backend()
    lens, new = [290, 40, 7], [1, 2, 1]
    cache, table, cu, q, T = scene(lens, new, heads, kv_heads, D, 32, heads)
    out = torch.zeros(T, heads, D, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32(lens), b.kv4_workspace(heads, kv_heads, D), max_new=2)
    check(cache, table, cu, lens, q, out, 0, D ** -0.5, True, 0)


@pytest.mark.parametrize("new", [1, 30])
def test_attention_unwritten_bytes_do_not_leak(new):
    """Every byte behind a request's last token may hold anything (0xff: scales that E4M3 calls NaN)."""
    b = backend()
    lens = [new + 70, new + 3]
    cache, table, cu, q, T = scene(lens, [new, new], 8, 2, 64, 64, 8)
    out, ref = torch.zeros(T, 8, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(T, 8, 64, dtype=torch.bfloat16, device=DEV)
    args = (i32(table), i32(cu), i32(lens), b.kv4_workspace(8, 2, 64))
    b.kv4_attention(q, ref, cache, *args, max_new=new)
    dirty = R.Cache(cache.storage.cpu().numpy().copy(), 64, 64, 16.0, 8.0)
    live = {int(table[i, j // 64]) * 64 + j % 64 for i in range(2) for j in range(lens[i])}
    for slot in range(cache.pages * 64):
        if slot not in live:
            blk, at = dirty.block(slot)
            for x in at:
                blk[:, x] = 0xff
    c2 = Kv4Cache(torch.from_numpy(dirty.s).to(DEV), 64, 64, 16.0, 8.0)
    b.kv4_attention(q, out, c2, *args, max_new=new)
    assert torch.equal(out, ref)


def test_attention_strides_and_lengths_past_the_table():
    b = backend()
    cache, table, cu, q, T = scene([200], [3], 8, 2, 128, 64, 9)
    wide = torch.full((T, 2048), 0.5, dtype=torch.bfloat16, device=DEV)
    wide[:, 512: 1536] = q.view(T, 1024)
    big = torch.full((T, 3000), 0.5, dtype=torch.bfloat16, device=DEV)
    out = big[:, 1000: 2024].view(T, 8, 128)
    ref = torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    ws = b.kv4_workspace(8, 2, 128)
    b.kv4_attention(q, ref, cache, i32(table), i32(cu), i32([200]), ws)
    b.kv4_attention(wide[:, 512: 1536].view(T, 8, 128), out, cache, i32(table), i32(cu), i32([200]), ws)
    assert torch.equal(out, ref) and torch.all(big[:, :1000] == 0.5) and torch.all(big[:, 2024:] == 0.5)
    # a length the table cannot hold stops at the table's end
    short = table[:, :3]
    b.kv4_attention(q, out, cache, i32(short), i32(cu), i32([100000]), ws)
    check(cache, short, cu, [192], q, out.contiguous(), 0, 128 ** -0.5, True, 0)


def test_attention_leaves_out_requests_past_the_hint():
    b = backend()
    cache, table, cu, q, T = scene([100, 60], [1, 40], 8, 1, 128, 64, 10)
    out = torch.full((T, 8, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    b.kv4_attention(q, out, cache, i32(table), i32(cu), i32([100, 60]), b.kv4_workspace(8, 1, 128), max_new=1)
    assert torch.all(out[1:] == 3.0) and not torch.any(out[0] == 3.0)


def test_attention_python_refusals():
    b = backend()
    cache, table, cu, q, T = scene([20], [2], 8, 2, 128, 64, 11)
    ws, out = b.kv4_workspace(8, 2, 128), torch.zeros(T, 8, 128, dtype=torch.bfloat16, device=DEV)
    ok = dict(q=q, out=out, cache=cache, table=i32(table), cu=i32(cu), kv_lens=i32([20]), workspace=ws)
    for name, bad in (("q", q.float()), ("out", q), ("out", out[:, :4]), ("q", q.transpose(0, 1)), ("table", i32(table)[:0]), ("table", torch.tensor(table)),
                      ("cu", i32(cu)[:1]), ("kv_lens", i32([20, 3])), ("workspace", ws[:100]), ("workspace", ws.cpu()), ("cu", i32(cu).long())):
        with pytest.raises(ShapeError):
            b.kv4_attention(**{**ok, name: bad})


# ---- together ----------------------------------------------------------------------------------------

def test_steps_together_captured_and_on_a_stream():
    """Two prefill steps and decode steps of three requests as they are used: plan, norm + rotation + store, attention.
    The decode step is captured once and replayed; two graphs with their own step and workspace run side by side."""
    b = backend()
    hq, hkv, D, page = 8, 2, 128, 32
    rope, w = rope_table(500, D).to(DEV), torch.rand(D, device=DEV) + 0.5

    class Lane:
        def __init__(self, seed):
            self.cache = make_cache(40, hkv, page, D, seed)
            self.ref = R.Cache(self.cache.storage.cpu().numpy().copy(), page, D, 16.0, 8.0)
            self.free, self.taken = i32(np.random.default_rng(seed).permutation(40)), i32([0])
            self.table = torch.full((3, 9), -1, dtype=torch.int32, device=DEV)
            self.cached = i32([0, 0, 0])
            self.ws = b.kv4_workspace(hq, hkv, D)
            self.lens = np.zeros(3, np.int64)

        def arrays(self, rows):
            g = torch.Generator(device=DEV).manual_seed(rows)
            mk = lambda h: torch.randn(rows, h, D, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
            self.q, self.k, self.v = mk(hq), mk(hkv), mk(hkv)
            self.qo, self.out = torch.zeros_like(self.q), torch.full_like(self.q, 0.5)
            self.step = Kv4Step(b, 3, rows)

        def call(self, new, most):
            b.kv4_plan(self.cached, new, self.table, self.free, self.taken, page, self.step)
            b.qk_norm_rope_kv4(self.q, self.k, self.v, w, w, rope, self.step.positions, self.step.slots, self.cache, self.qo)
            b.kv4_attention(self.qo, self.out, self.cache, self.table, self.step.cu, self.step.kv_lens, self.ws, max_new=most)
            self.cached.add_(new)

        def verify(self, new):
            cu = np.concatenate([[0], np.cumsum(new)])
            pos = np.concatenate([self.lens[i] + np.arange(new[i]) for i in range(3)]).astype(np.int64)
            n = int(cu[-1])
            assert np.array_equal(self.step.positions.cpu().numpy()[:n], pos) and self.step.status.item() == 0
            assert np.all(self.step.positions.cpu().numpy()[n:] == -1)
            kk = R.norm_rope(f64(self.k)[:n], w.cpu().numpy(), 1e-6, False, rope.cpu().numpy(), pos, False).astype(np.float32)
            slots = self.step.slots.cpu().numpy()
            for t in range(n):
                self.ref.write(int(slots[t]), kk[t], f64(self.v)[t].astype(np.float32))
            assert np.array_equal(self.ref.s, self.cache.storage.cpu().numpy())
            self.lens += new
            close_rows(self.qo[:n], f64(self.q)[:n], w.cpu().numpy(), 1e-6, False, rope.cpu().numpy(), pos, False)
            check(self.cache, self.table.cpu().numpy(), cu, self.lens, self.qo, self.out, 0.5, D ** -0.5, True, 0)

    lanes = [Lane(1), Lane(2)]
    for new in ([70, 3, 31], [1, 40, 30]):
        for lane in lanes:
            lane.arrays(int(sum(new)) + 2)
            lane.call(i32(new), max(new))
            lane.verify(np.array(new))
    one = i32([1, 1, 1])
    streams, graphs = [torch.cuda.Stream() for _ in lanes], []
    for lane, st in zip(lanes, streams):
        lane.arrays(4)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):                       # a side stream, outside any graph
            lane.call(one, 1)
        st.synchronize()
        lane.verify(np.array([1, 1, 1]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            lane.call(one, 1)
        graphs.append(graph)
    for round_ in range(35):                              # pages are taken on the way
        for lane in lanes:
            g = torch.Generator(device=DEV).manual_seed(round_)
            for x in (lane.q, lane.k, lane.v):
                x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for lane in lanes:
            if round_ % 7 == 0 or round_ > 32:
                lane.verify(np.array([1, 1, 1]))
            else:
                _advance(lane, w, rope)
    assert b.debug_status() == 0


def _advance(lane, w, rope):
    """Keeps the reference's cache in step without the (slow) comparison."""
    pos = lane.lens.copy()
    kk = R.norm_rope(f64(lane.k)[:3], w.cpu().numpy(), 1e-6, False, rope.cpu().numpy(), pos, False).astype(np.float32)
    slots = lane.step.slots.cpu().numpy()
    for t in range(3):
        lane.ref.write(int(slots[t]), kk[t], f64(lane.v)[t].astype(np.float32))
    lane.lens += 1


def test_attention_long_cache_past_32_bits():
    """A cache of more than 2^32 bytes whose used pages lie at its end."""
    b = backend()
    hkv, D, page = 8, 128, 64
    pages = (1 << 32) // (hkv * page * 144) + 200
    storage = torch.empty(pages, hkv, page // 16, 18 * D, dtype=torch.uint8, device=DEV)
    cache = Kv4Cache(storage, page, D, 16.0, 16.0)
    ids = np.arange(pages - 5, pages)
    slots = np.concatenate([i * page + np.arange(page) for i in ids])
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(len(slots), hkv, D, generator=g, device=DEV) for _ in range(2))
    b.kv4_store(k, v, i32(slots), cache)
    small = Kv4Cache(storage[-5:].clone(), page, D, 16.0, 16.0)
    q = torch.randn(21, 16, D, generator=g, device=DEV).to(torch.bfloat16)
    outs = []
    for c, tab in ((cache, ids), (small, np.arange(5))):
        ws = b.kv4_workspace(16, hkv, D)
        out = torch.zeros(21, 16, D, dtype=torch.bfloat16, device=DEV)
        b.kv4_attention(q, out, c, i32([tab, tab]), i32([0, 1, 21]), i32([320, 300]), ws)
        ko, vo = torch.empty(3, hkv, D, device=DEV), torch.empty(3, hkv, D, device=DEV)
        b.kv4_rows(c, i32([tab[0] * page, tab[4] * page + 63, tab[2] * page + 1]), ko, vo)
        outs.append((out, ko, vo))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    check(small, np.array([np.arange(5)] * 2), np.array([0, 1, 21]), [320, 300], q, outs[1][0], 0, D ** -0.5, True, 0)


def _chosen(lens, new, G, hkv, rows, tile, extra, join, grid):
    """Which cut csrc/kv4_items.cuh takes for causal requests without a window: 0 equal runs, else parts per item."""
    items = []
    for length, n in zip(lens, new):
        for t in range(-(-n * G // rows)):
            hi = min(length, length - n + (min((t + 1) * rows, n * G) - 1) // G + 1)
            items += [max(1, -(-hi // tile))] * hkv
    n, total, longest = len(items), sum(items) + extra * len(items), max(items)
    cap = min(grid, max(n, total // 4))
    each = grid // n
    blocks = cap if total >= 8 * cap or not each else max(n, cap // n * n)
    equal, whole = total // blocks + 2 * extra + join, (1 if each else -(-n // grid)) * (longest + extra)
    s = min(each, longest // 4)
    alike = -(-longest // s) + extra + join if s > 1 else whole
    return 0 if min(whole, alike) > equal else 1 if whole <= alike else s


@pytest.mark.parametrize("lens,new,hq,hkv,D,want", [
    ([3000], [256], 16, 2, 128, "parts"),                                # prefill: both halves of an item joined
    ([2500, 70], [40, 33], 9, 3, 64, "parts"),                           # a short item beside it has fewer parts
    ([9000] + [120] * 30, [64] + [100] * 30, 8, 2, 128, "equal"),
    ([130] * 90, [100] * 90, 8, 2, 64, "whole"),                         # more items than blocks
    ([20000, 300], [1, 1], 8, 2, 128, "parts"),
    ([5000, 40, 900], [2, 3, 1], 8, 1, 64, "parts"),
    ([40000] + [90] * 60, [1] * 61, 8, 2, 128, "equal"),
    ([300] * 330, [1] * 330, 8, 1, 128, "whole"),
])
def test_attention_every_cut(lens, new, hq, hkv, D, want):
    """Equal runs, items in parts, whole items: the results, bit for bit the same from call to call."""
    b = backend()
    sms, G = torch.cuda.get_device_properties(0).multi_processor_count, hq // hkv
    if max(new) * G > 32:
        mode = _chosen(lens, new, G, hkv, 256, 128, 3, 6, sms)
    else:
        mode = _chosen(lens, new, G, hkv, 8 if max(new) * G <= 8 else 16, 256, 1, 3, 2 * sms)
    assert {0: "equal", 1: "whole"}.get(mode, "parts") == want
    cache, table, cu, q, T = scene(lens, new, hq, hkv, D, 64, len(lens), 1)
    out = torch.full((T, hq, D), 0.75, dtype=torch.bfloat16, device=DEV)
    args = (cache, i32(table), i32(cu), i32(lens), b.kv4_workspace(hq, hkv, D))
    b.kv4_attention(q, out, *args, max_new=max(new))
    check(cache, table, cu, lens, q, out, 0.75, D ** -0.5, True, 0)
    again = torch.full_like(out, 0.75)
    b.kv4_attention(q, again, *args, max_new=max(new))
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
