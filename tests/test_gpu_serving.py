"""The operators for serving many sequences, through the C ABI, against plain forms in 64 bits (serving_oracle.py): rotary
positions, attention over a paged cache, the pages' own operations, beam selection, and a run of them together."""
import ctypes as C

import numpy as np
import pytest

import serving_oracle as so
from serving_cases import BEAM_SHAPES, beam_case

pytestmark = pytest.mark.gpu


def normal(r, *shape, std=1.0):
    return (r.standard_normal(shape) * std).astype(np.float16)


def close(got, want, tol, what=""):
    got = got.astype(np.float64)
    assert got.shape == want.shape
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3])


# ---- rotary positions ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,heads,hd,rot,half", [(1, 1, 2, 2, False), (1, 32, 128, 128, False), (5, 3, 80, 80, True), (17, 8, 128, 64, True),
                                                 (9, 4, 64, 16, False), (3, 5, 7, 6, False), (4, 2, 9, 4, True), (300, 6, 72, 36, True),
                                                 (2, 1, 256, 256, True), (33, 2, 48, 0, False), (2, 3, 1024, 1024, False), (70, 12, 96, 24, False)])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_matches_the_formula(tl, T, heads, hd, rot, half, inverse):
    r = np.random.default_rng([T, heads, hd, rot])
    x = normal(r, T, heads, hd, std=2.0)
    pos = r.integers(0, 1 << 20, T).astype(np.int32)
    pos[0] = [0, 1, 2 ** 31 - 1][T % 3]
    f, mag = tl.rotary_frequencies(max(rot, 2), scaling="ramp", factor=4.0, trained_len=2048, low=1, high=32)
    f = f[:rot // 2]
    want, tol = so.rotary(x, pos, f, mag, half, inverse)
    close(tl.rotary(x, pos, f, mag, half, inverse), want, tol)
    close(tl.rotary(x, pos, f, mag, half, inverse, in_place=True), want, tol, "in place")


def test_rotary_leaves_padding_and_turns_back(tl):
    r = np.random.default_rng(5)
    x, f = normal(r, 12, 4, 64), tl.rotary_frequencies(64)[0]
    pos = np.array([3, -1, 70000, -5, 0, 1, 2, -2 ** 31, 9, 8, 7, 6], np.int32)
    old = normal(r, 12, 4, 64)
    y = tl.rotary(x, pos, f, out=old)
    assert np.array_equal(y[pos < 0], old[pos < 0])
    # forward, then inverse: two roundings of at most |x| + |y| of a pair each
    back = tl.rotary(y, pos, f, inverse=True, out=old)
    size = np.abs(x.astype(np.float64)).reshape(12, 4, 32, 2).sum(-1).repeat(2, -1)
    assert (np.abs(back.astype(np.float64) - x)[pos >= 0] <= (3 * so.EPS16 * size + 2 * so.TINY16)[pos >= 0]).all()
    assert tl.device_status() == 0


def test_rotary_gradient_is_the_inverse_turn(tl):
    """d/dx sum(g * R x) = R^T g, checked against differences of the formula."""
    r = np.random.default_rng(6)
    x, g = r.standard_normal((2, 1, 16)), normal(r, 2, 1, 16)
    pos, (f, mag) = np.array([5, 4000], np.int32), tl.rotary_frequencies(12, scaling="ramp", factor=2.0, trained_len=512, low=1, high=32)
    for half in (False, True):
        got = tl.rotary(g, pos, f, mag, half, inverse=True)
        h = 1e-6
        num = np.zeros_like(x)
        for i in np.ndindex(*x.shape):
            d = np.zeros_like(x)
            d[i] = h
            num[i] = ((so.rotary(x + d, pos, f, mag, half)[0] - so.rotary(x - d, pos, f, mag, half)[0]) * g).sum() / (2 * h)
        tol = so.rotary(g, pos, f, mag, half, True)[1] + 1e-7
        close(got, num, tol)


def test_rotary_of_a_strided_slice(tl):
    """Heads 2..4 of a wider buffer, by-head output: what lies between the rows stays."""
    r = np.random.default_rng(7)
    T, W, hd = 6, 9, 24
    x, f = normal(r, T, W, hd), tl.rotary_frequencies(24)[0]
    pos = np.arange(T, dtype=np.int32) * 1000
    for off in (0, 1):                       # 16-byte aligned, and not
        dx, dp, df = tl.DeviceBuffer.from_numpy(np.concatenate([x.reshape(-1), np.zeros(8, np.float16)])), tl.DeviceBuffer.from_numpy(pos), tl.DeviceBuffer.from_numpy(f)
        do = tl.DeviceBuffer.from_numpy(np.full(3 * T * 32 + 8, 7.0, np.float16))
        start = 2 * hd + off
        tl.check(tl.load().tl_rotary_f16(dx.ptr + 2 * start, do.ptr + 2 * off, dp.ptr, df.ptr, 1.0, T, 3, hd, hd, 1, 0, W * hd, hd, 32, T * 32, None), "rotary")
        flat = np.concatenate([x.reshape(-1), np.zeros(8, np.float16)])
        xs = np.stack([[flat[start + t * W * hd + h * hd:][:hd] for h in range(3)] for t in range(T)])
        want, tol = so.rotary(xs, pos, f, 1.0, True)
        got = do.to_numpy(np.float16, (3 * T * 32 + 8,))[off:off + 3 * T * 32].reshape(3, T, 32).swapaxes(0, 1)
        close(got[..., :hd], want, tol, off)
        assert (got[..., hd:] == 7).all()


@pytest.mark.parametrize("T,heads,hd,rot,half", [(1500, 40, 128, 128, False), (4099, 3, 64, 64, False), (9000, 1, 128, 64, True), (1481, 32, 128, 128, True),
                                                 (3000, 5, 80, 40, False), (2222, 12, 96, 48, True), (1200, 2, 36, 20, True), (20011, 2, 10, 6, False),
                                                 (1300, 300, 8, 8, False), (800, 2, 1024, 1024, False), (1000, 4, 512, 512, True), (70000, 1, 16, 2, False)])
def test_rotary_of_many_tokens(tl, T, heads, hd, rot, half):
    """More tokens than CTAs are resident: a CTA turns several, padding among them."""
    r = np.random.default_rng([T, heads, hd])
    x, old = normal(r, T, heads, hd, std=2.0), normal(r, T, heads, hd)
    pos = r.integers(0, 1 << 20, T).astype(np.int32)
    pos[r.random(T) < 0.1] = -1
    f, mag = tl.rotary_frequencies(rot, scaling="parts" if rot > 2 else "unscaled", factor=4.0, trained_len=2048, low=1, high=4)
    live = pos >= 0
    for inverse in (False, True):
        want, tol = so.rotary(x[live], pos[live], f, mag, half, inverse)
        got = tl.rotary(x, pos, f, mag, half, inverse, out=old)
        close(got[live], want, tol)
        assert np.array_equal(got[~live], old[~live])
        got = tl.rotary(x, pos, f, mag, half, inverse, in_place=True)
        close(got[live], want, tol, "in place")
        assert np.array_equal(got[~live], x[~live])
    assert tl.device_status() == 0


@pytest.mark.parametrize("hd,rot", [(8, 8), (7, 6)])
def test_rotary_of_the_most_tokens(tl, hd, rot):
    """2^31 - 1 tokens, all padding but the last; they share one row of in and out."""
    lib, T = tl.load(), 2 ** 31 - 1
    x, f, last = normal(np.random.default_rng(8), 1, 1, hd), tl.rotary_frequencies(rot)[0], np.array([5], np.int32)
    dx, do, df, dp = tl.DeviceBuffer.from_numpy(x), tl.DeviceBuffer.from_numpy(np.zeros(hd, np.float16)), tl.DeviceBuffer.from_numpy(f), tl.DeviceBuffer(4 * T)
    tl.check(lib.tl_memset(dp.ptr, 0xff, dp.nbytes, None), "memset")
    tl.check(lib.tl_memcpy_h2d(dp.ptr + 4 * (T - 1), last.ctypes.data, 4, None), "h2d")
    tl.synchronize()
    tl.check(lib.tl_rotary_f16(dx.ptr, do.ptr, dp.ptr, df.ptr, 1.0, T, 1, hd, rot, 0, 0, 0, hd, 0, hd, None), "rotary")
    want, tol = so.rotary(x, last, f)
    close(do.to_numpy(np.float16, x.shape), want, tol)
    assert tl.device_status() == 0


def test_rotary_of_the_widest_token(tl):
    """49981 heads of 42966 elements, two below 2^31 in all; they share one row of in and out."""
    heads, hd = 49981, 42966
    assert heads * hd == 2 ** 31 - 2
    x = normal(np.random.default_rng(9), 1, 1, hd)
    dx, do, dp = tl.DeviceBuffer.from_numpy(x), tl.DeviceBuffer.from_numpy(np.zeros(hd + 64, np.float16)), tl.DeviceBuffer.from_numpy(np.zeros(1, np.int32))
    tl.check(tl.load().tl_rotary_f16(dx.ptr, do.ptr, dp.ptr, None, 1.0, 1, heads, hd, 0, 0, 0, heads * hd, 0, heads * hd, 0, None), "rotary")
    got = do.to_numpy(np.float16, (hd + 64,))
    assert np.array_equal(got[:hd], x[0, 0]) and (got[hd:] == 0).all() and tl.device_status() == 0


# ---- the way into the cache ------------------------------------------------------------------------------------------
def filled_cache(tl, r, layers, page, kv, hd, lens, by_head=False, spare=3, max_pages=None, garbage=True):
    """A cache whose row i holds lens[i] tokens in random pages, with anything at all in the slots never written."""
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    width = max_pages or max(1, max(counts) + 1)
    k, v = normal(r, layers, pages, page, kv, hd), normal(r, layers, pages, page, kv, hd)
    order = r.permutation(pages).astype(np.int32)
    table, refs, at = np.full((len(lens), width), -1, np.int32), np.zeros(pages, np.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        refs[order[at:at + n]] = 1
        at += n
        if garbage and lens[i] % page:
            for a in (k, v):
                a[:, table[i, n - 1], lens[i] % page:] = np.array([np.nan, np.inf, -np.inf, 65504], np.float16)[r.integers(0, 4, a[:, 0, lens[i] % page:].shape)]
    c = tl.PagedCache(layers, pages, page, kv, hd, len(lens), width, by_head, k, v)
    c.set_state(table, np.asarray(lens, np.int32), refs)
    return c, k, v, table, refs


def row_tokens(a, table, n, page):
    """[n, kv, hd] of one row from a pool [pages, page, kv, hd]"""
    t = np.arange(n)
    return a[table[t // page], t % page]


@pytest.mark.parametrize("page,kv,hd,heads,rot,half,by_head", [(16, 8, 128, 32, 128, False, False), (1, 1, 64, 1, 64, True, False),
                                                               (24, 3, 80, 15, 40, True, True), (5, 2, 7, 4, 6, False, False),
                                                               (16, 2, 64, 0, 64, False, True), (8, 4, 32, 8, 0, False, False)])
def test_append_stores_at_the_row_and_position(tl, page, kv, hd, heads, rot, half, by_head):
    r = np.random.default_rng([page, kv, hd])
    lens = [3 * page, 1, 2 * page + 1, 0, page, 4]
    c, k, v, table, refs = filled_cache(tl, r, 2, page, kv, hd, lens, by_head)
    rows = np.array([2, 0, 0, 1, 4, 2, 5, 5], np.int32)
    pos = np.array([2 * page, 0, 3 * page - 1, 0, page - 1, 0, -1, 3], np.int32)
    q = normal(r, 8, heads, hd) if heads else None
    nk, nv = normal(r, 8, kv, hd), normal(r, 8, kv, hd)
    f = tl.rotary_frequencies(rot)[0] if rot else None
    got_q = c.append(1, q, nk, nv, pos, f, 1.25, half, rows)
    fr = np.zeros(0) if f is None else f
    wk, tk = so.rotary(nk, pos, fr, 1.25, half)
    if heads:
        wq, tq = so.rotary(q, pos, fr, 1.25, half)
        live = pos >= 0
        close(got_q[live], wq[live], tq[live], "q")
        assert (got_q[~live] == 0).all()
    gk, gv = c.pools()
    seen = np.zeros(k.shape[1:3], bool)
    for i in range(8):
        if pos[i] >= 0:
            at = (1, table[rows[i], pos[i] // page], pos[i] % page)
            seen[at[1:]] = True
            close(gk[at], wk[i], tk[i], "k")
            assert np.array_equal(gv[at], nv[i])
    for got, old in ((gk, k), (gv, v)):          # nothing else has changed
        assert np.array_equal(got[0].view(np.uint16), old[0].view(np.uint16))
        assert np.array_equal(got[1][~seen].view(np.uint16), old[1][~seen].view(np.uint16))
    assert tl.device_status() == 0


@pytest.mark.parametrize("T,page,kv,hd,heads,rot,half,by_head", [(3001, 16, 8, 128, 32, 128, False, False), (2500, 24, 3, 80, 15, 40, True, True),
                                                                 (5000, 16, 1, 64, 1, 64, True, False), (2000, 64, 32, 128, 32, 128, True, False),
                                                                 (4000, 5, 2, 7, 4, 6, False, False), (2222, 16, 2, 64, 0, 64, False, True),
                                                                 (1700, 8, 4, 32, 64, 0, False, False), (1333, 16, 2, 36, 9, 20, True, False)])
def test_append_of_a_prompt(tl, T, page, kv, hd, heads, rot, half, by_head):
    """Thousands of tokens of three rows in any order: a CTA moves several, all three tensors of them."""
    r = np.random.default_rng([T, page, kv, hd])
    lens = [T // 2, T // 3, T - T // 2 - T // 3]
    c, k, v, table, refs = filled_cache(tl, r, 2, page, kv, hd, lens, by_head, garbage=False)
    rows = np.repeat(np.arange(3), lens).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    order = r.permutation(T)
    rows, pos = rows[order], pos[order]
    pos[r.random(T) < 0.05] = -1
    live = pos >= 0
    q = normal(r, T, heads, hd) if heads else None
    nk, nv = normal(r, T, kv, hd), normal(r, T, kv, hd)
    f = tl.rotary_frequencies(rot)[0] if rot else None
    got_q = c.append(1, q, nk, nv, pos, f, 0.75, half, rows)
    fr = np.zeros(0) if f is None else f
    if heads:
        wq, tq = so.rotary(q[live], pos[live], fr, 0.75, half)
        close(got_q[live], wq, tq, "q")
        assert (got_q[~live] == 0).all()
    wk, tk = so.rotary(nk[live], pos[live], fr, 0.75, half)
    gk, gv = c.pools()
    at = table[rows[live], pos[live] // page], pos[live] % page
    close(gk[1][at], wk, tk, "k")
    assert np.array_equal(gv[1][at], nv[live])
    seen = np.zeros(k.shape[1:3], bool)
    seen[at] = True
    for got, old in ((gk, k), (gv, v)):          # nothing else has changed
        assert np.array_equal(got[0], old[0]) and np.array_equal(got[1][~seen], old[1][~seen])
    assert tl.device_status() == 0


def test_append_never_follows_bad_ids(tl):
    r = np.random.default_rng(9)
    page, kv, hd = 8, 2, 32
    c, k, v, table, refs = filled_cache(tl, r, 1, page, kv, hd, [8, 8, 8, 8, 8], garbage=False)
    table[3, 0], table[4, 0] = k.shape[1], -7
    c.set_state(table, [8] * 5, refs)
    rows = np.array([0, 5, -1, 3, 4, 1, 2], np.int32)
    pos = np.array([1, 0, 0, 0, 0, 16, 2 ** 31 - 1], np.int32)     # row 1 has room for 16 tokens, entry 1 is -1
    nk, nv = normal(r, 7, kv, hd), normal(r, 7, kv, hd)
    c.append(0, None, nk, nv, pos, None, rows=rows)
    gk, gv = c.pools()
    assert tl.device_status() == 1
    k[0, table[0, 0], 1], v[0, table[0, 0], 1] = nk[0], nv[0]
    assert np.array_equal(gk, k) and np.array_equal(gv, v)


# ---- attention over pages --------------------------------------------------------------------------------------------
def check_attention(tl, c, k, v, table, lens, page, q, scale=None, rows=None, got=None):
    B, heads, hd = q.shape
    kv = k.shape[2]
    out, lse = c.attend(0, q, scale, rows) if got is None else got
    for b in range(B):
        row = b if rows is None else rows[b]
        n = 0 if row < 0 else lens[row]
        kk, vv = (row_tokens(a, table[row], n, page) for a in (k, v)) if n else (np.zeros((0, kv, hd)),) * 2
        for h in range(heads):
            j = h // (heads // kv)
            o, l, to, tl_ = so.attend(q[b, h], kk[:, j], vv[:, j], hd ** -0.5 if scale is None else scale)
            close(out[b, h], o, to, (b, h, n))
            if n == 0:
                assert (out[b, h] == 0).all() and lse[b, h] == -np.inf
            else:
                assert abs(lse[b, h] - l) <= tl_, (b, h, n, lse[b, h], l, tl_)
    return out, lse


LENS = [1, 0, 15, 16, 17, 33, 2, 64, 129, 300, 1000]


@pytest.mark.parametrize("hd,kv,group,page,by_head", [(128, 8, 4, 16, False), (64, 1, 1, 16, False), (80, 3, 5, 24, True), (128, 2, 8, 1, False),
                                                      (256, 2, 3, 64, False), (96, 2, 16, 16, True), (40, 1, 7, 100, False), (8, 2, 2, 3, False),
                                                      (192, 1, 12, 32, False), (128, 4, 1, 16, False), (64, 1, 40, 16, False), (256, 1, 20, 8, True),
                                                      (7, 2, 3, 5, False), (33, 1, 17, 16, True), (136, 2, 9, 16, False)])
def test_attention_over_pages(tl, hd, kv, group, page, by_head):
    r = np.random.default_rng([hd, kv, group, page])
    c, k, v, table, _ = filled_cache(tl, r, 1, page, kv, hd, LENS, by_head)
    q = normal(r, len(LENS), kv * group, hd, std=1.5)
    out, lse = check_attention(tl, c, k[0], v[0], table, LENS, page, q)
    again = c.attend(0, q)
    assert np.array_equal(out, again[0]) and np.array_equal(lse, again[1])       # the same call, the same bits
    assert tl.device_status() == 0


@pytest.mark.parametrize("B,low,high,kv,group,hd,page", [(1, 1, 1, 32, 1, 128, 16), (1, 333, 333, 32, 1, 128, 16), (1, 20011, 20011, 1, 8, 128, 16),
                                                         (1, 9000, 9000, 8, 4, 64, 64), (3, 1, 7000, 2, 4, 128, 24), (200, 1, 90, 2, 2, 64, 16),
                                                         (65, 30, 500, 4, 3, 80, 32), (300, 0, 3, 1, 1, 128, 16),
                                                         (1, 30000, 30000, 1, 16, 64, 16), (2, 6000, 9000, 1, 12, 256, 32), (1, 15000, 15000, 2, 3, 192, 8)])
def test_attention_split_over_the_length(tl, B, low, high, kv, group, hd, page):
    r = np.random.default_rng([B, high, kv])
    lens = r.integers(low, high + 1, B).tolist()
    c, k, v, table, _ = filled_cache(tl, r, 1, page, kv, hd, lens)
    q = normal(r, B, kv * group, hd, std=1.5)
    check_attention(tl, c, k[0], v[0], table, lens, page, q)
    assert tl.device_status() == 0


@pytest.mark.parametrize("B,low,high,kv,group,hd,page", [(11, 0, 1000, 2, 16, 128, 16), (1, 20011, 20011, 1, 9, 128, 16), (3, 1, 7000, 2, 12, 112, 24),
                                                         (100, 0, 90, 1, 10, 128, 8), (5, 100, 3000, 2, 25, 128, 64)])
def test_attention_of_wide_groups(tl, B, low, high, kv, group, hd, page):
    """Nine and more query heads a KV head at 97..128 elements."""
    r = np.random.default_rng([B, high, group])
    lens = r.integers(low, high + 1, B).tolist()
    c, k, v, table, _ = filled_cache(tl, r, 1, page, kv, hd, lens)
    check_attention(tl, c, k[0], v[0], table, lens, page, normal(r, B, kv * group, hd, std=1.5))
    assert tl.device_status() == 0


def test_attention_of_large_scores_and_values(tl):
    """Scores over hundreds apart, growing and falling, and values at the type's limits."""
    r = np.random.default_rng(12)
    hd, page = 128, 16
    for order in (1, -1):
        c, k, v, table, _ = filled_cache(tl, r, 1, page, 1, hd, [777, 64], garbage=False)
        ramp = np.linspace(-20, 20, 777)[::order]
        t = np.arange(777)
        k[0, table[0, t // page], t % page, 0] = (ramp[:, None] * np.sign(r.standard_normal(hd))[None]).astype(np.float16)
        v[0, table[0, t // page], t % page, 0] = (r.choice([-65504.0, 65504.0, 1.0], (777, hd))).astype(np.float16)
        state = c.state()
        c = tl.PagedCache(1, k.shape[1], page, 1, hd, 2, table.shape[1], k=k, v=v)
        c.set_state(*state)
        q = normal(r, 2, 6, hd, std=4.0)
        check_attention(tl, c, k[0], v[0], table, [777, 64], page, q)


@pytest.mark.parametrize("n,at,gap,hd,group,page", [(4096, 0, 17.5, 128, 4, 16), (4096, 2000, 16.25, 64, 1, 16), (131072, 0, 17.5, 128, 8, 16),
                                                    (131072, 65536, 16.25, 128, 1, 64), (20011, 0, 18.0, 256, 3, 32), (20011, 77, 17.0, 96, 12, 16),
                                                    (3000, 0, 17.5, 65, 2, 16)])
def test_attention_keeps_weights_far_below_the_largest(tl, n, at, gap, hd, group, page):
    """One key `gap` nats above all others, whose value is 0 where theirs are 1: what comes out is the sum of the small weights.
    The scores are exact sums; scaling by log2 e costs 2^-23 of up to 26 twice; a weight is held to 2^-40 of the largest; the sums of
    products and of weights add at most n / 16 times with 2^-24 each; then one rounding."""
    r = np.random.default_rng([n, hd])
    c, k, v, table, refs = filled_cache(tl, r, 1, page, 1, hd, [n], garbage=False)
    k[:], v[:] = 0, 1
    k[0, table[0, at // page], at % page, 0, :64] = gap / 64
    v[0, table[0, at // page], at % page] = 0
    c = tl.PagedCache(1, k.shape[1], page, 1, hd, 1, table.shape[1], k=k, v=v)
    c.set_state(table, [n], refs)
    out, lse = c.attend(0, np.ones((1, group, hd), np.float16), 1.0)
    rest = (n - 1) * np.exp(-gap)
    want = np.full((1, group, hd), rest / (1 + rest))
    close(out, want, want * (so.EPS16 + 2.0 ** -17 + 2.0 ** -40 * np.exp(gap) + n / 8 * 2.0 ** -24) + so.TINY16)
    assert (np.abs(lse - (gap + np.log1p(rest))) <= 2.0 ** -17 + n / 16 * 2.0 ** -24).all()
    assert tl.device_status() == 0


def test_attention_takes_a_row_list_with_padding(tl):
    r = np.random.default_rng(13)
    lens = [40, 7, 0, 300]
    c, k, v, table, _ = filled_cache(tl, r, 1, 16, 2, 64, lens)
    rows = [3, -1, 0, 3, 2, 1, -1]
    q = normal(r, len(rows), 6, 64)
    check_attention(tl, c, k[0], v[0], table, lens, 16, q, rows=rows)
    assert tl.device_status() == 0


@pytest.mark.parametrize("hd", [64, 7])
def test_attention_never_follows_bad_ids(tl, hd):
    """Pages outside the pool count as tokens that are not there; rows and lengths outside their tables as empty or cut."""
    r = np.random.default_rng(14)
    lens = [50, 50, 16, 50, 30, 20]
    c, k, v, table, refs = filled_cache(tl, r, 1, 16, 1, hd, lens, max_pages=4, garbage=False)
    bad = table.copy()
    bad[0, 1] = k.shape[1]
    bad[1, :4] = [-1, -9, 2 ** 31 - 1, -2 ** 31]
    c.set_state(bad, [50, 50, -4, 50, 1 << 20, 20], refs)
    q = normal(r, 8, 4, hd)
    rows = [0, 1, 2, 3, 4, 5, 6, -3]
    out, lse = c.attend(0, q, rows=rows)
    assert tl.device_status() == 1
    sound = {0: [t for t in range(50) if t // 16 != 1], 1: [], 2: [], 3: list(range(50)), 4: list(range(32)), 5: list(range(20)), 6: [], 7: []}
    for b, ts in sound.items():
        t = np.array(ts, int)
        kk, vv = (a[0][table[rows[b], t // 16], t % 16, 0] if len(ts) else np.zeros((0, hd)) for a in (k, v))
        for h in range(4):
            o, l, to, tl_ = so.attend(q[b, h], kk, vv, hd ** -0.5)
            close(out[b, h], o, to, (b, h))
            assert (lse[b, h] == l) if not ts else abs(lse[b, h] - l) <= tl_
    out, lse = c.attend(0, q[3:4], rows=[3])                                      # and nothing is left behind
    check_attention(tl, c, k[0], v[0], table, lens, 16, q[3:4], rows=[3], got=(out, lse))
    assert tl.device_status() == 0


@pytest.mark.parametrize("hd", [64, 7])
def test_attention_shows_a_nan_where_there_is_one(tl, hd):
    """A NaN in a stored key or value reaches the results of its row's heads, and no other's."""
    r = np.random.default_rng(17)
    lens = [100, 100, 100]
    c, k, v, table, refs = filled_cache(tl, r, 1, 16, 2, hd, lens, garbage=False)
    k[0, table[1, 2], 5, 1, 3] = np.nan
    v[0, table[2, 6], 3, 0, 2] = np.nan
    c = tl.PagedCache(1, k.shape[1], 16, 2, hd, 3, table.shape[1], k=k, v=v)
    c.set_state(table, lens, refs)
    q = normal(r, 3, 4, hd)
    out, lse = c.attend(0, q)
    assert np.isnan(out[1, 2:]).all() and np.isnan(lse[1, 2:]).all()
    assert np.isnan(out[2, :2, 2]).all() and not np.isnan(np.delete(out[2, :2], 2, 1)).any() and not np.isnan(lse[2]).any()
    assert not np.isnan(out[0]).any() and not np.isnan(out[1, :2]).any() and not np.isnan(out[2, 2:]).any()
    check_attention(tl, c, k[0], v[0], table, lens, 16, q[:1], rows=[0], got=(out[:1], lse[:1]))


def test_attention_with_padded_rows_of_q_and_out_and_no_lse(tl):
    r = np.random.default_rng(15)
    lens, heads, hd = [70, 3, 0], 8, 64
    c, k, v, table, _ = filled_cache(tl, r, 1, 16, 2, hd, lens)
    pitch = heads * hd + 24
    q = normal(r, 3, pitch)
    dq, do = tl.DeviceBuffer.from_numpy(q), tl.DeviceBuffer.from_numpy(np.full((3, pitch), 5, np.float16))
    w = tl.DeviceBuffer.from_numpy(np.zeros(32 << 20, np.uint8))
    tl.check(tl.load().tl_paged_attn_decode_f16(C.byref(c.c), 0, dq.ptr, do.ptr, None, None, 3, heads, hd ** -0.5, pitch, pitch, w.ptr, w.nbytes, None), "attn")
    got = do.to_numpy(np.float16, (3, pitch))
    assert (got[:, heads * hd:] == 5).all()
    ref = c.attend(0, np.ascontiguousarray(q[:, :heads * hd].reshape(3, heads, hd)))
    assert np.array_equal(got[:, :heads * hd].reshape(3, heads, hd), ref[0])
    check_attention(tl, c, k[0], v[0], table, lens, 16, q[:, :heads * hd].reshape(3, heads, hd), got=ref)


def test_attention_beyond_32_bit_offsets(tl):
    """Pages whose values lie more than 2^32 elements into the pool (a stride between small pages makes it so)."""
    r = np.random.default_rng(16)
    page, kv, hd, pages, stride = 16, 1, 128, 9, 1 << 29
    lib = tl.load()
    bytes_ = ((pages - 1) * stride + page * hd) * 2
    kbuf, vbuf = tl.DeviceBuffer(bytes_), tl.DeviceBuffer(bytes_)
    k, v = normal(r, pages, page, kv, hd), normal(r, pages, page, kv, hd)
    for buf, a in ((kbuf, k), (vbuf, v)):
        for p in range(pages):
            x = np.ascontiguousarray(a[p])
            tl.check(lib.tl_memcpy_h2d(buf.ptr + 2 * p * stride, x.ctypes.data, x.nbytes, None), "h2d")
            tl.synchronize()
    lens = [page * 8, 5]
    table = np.full((2, 8), -1, np.int32)
    table[0] = [8, 1, 2, 3, 7, 5, 6, 0]
    table[1, 0] = 4
    c = tl.PagedCache(1, pages, page, kv, hd, 2, 8)
    refs = np.ones(pages, np.int32)
    c.set_state(table, lens, refs)
    c.c.k_pages, c.c.v_pages, c.c.page_stride, c.c.layer_stride = kbuf.ptr, vbuf.ptr, stride, pages * stride
    q = normal(r, 2, 4, hd)
    check_attention(tl, c, k, v, table, lens, page, q)
    nk, nv = normal(r, 1, kv, hd), normal(r, 1, kv, hd)
    c.append(0, None, nk, nv, [page * 8 - 1 - 7 * page], None, rows=[0])         # slot 15 of page 8
    k[8, page - 1], v[8, page - 1] = nk[0], nv[0]
    c.copy([8], [4])
    k[4], v[4] = k[8], v[8]
    check_attention(tl, c, k, v, table, lens, page, q)
    assert tl.device_status() == 0


# ---- the pages' own operations ------------------------------------------------------------------------------------------
def same_books(c, pg):
    for got, want, name in zip(c.state(), (pg.table, pg.lengths, pg.refs), ("table", "lengths", "refs")):
        assert np.array_equal(got, want), name


@pytest.mark.parametrize("seed,pages,page,rows,width,layers,kv,hd,by_head", [(1, 40, 4, 6, 9, 2, 2, 16, False), (2, 300, 16, 40, 12, 1, 1, 8, True),
                                                                            (3, 2500, 3, 1500, 5, 1, 1, 7, False), (4, 9, 1, 3, 4, 3, 3, 24, False),
                                                                            (5, 1024, 8, 64, 40, 1, 2, 8, False)])
def test_pages_over_many_steps(tl, seed, pages, page, rows, width, layers, kv, hd, by_head):
    r = np.random.default_rng(seed)
    k, v = normal(r, layers, pages, page, kv, hd), normal(r, layers, pages, page, kv, hd)
    c, pg = tl.PagedCache(layers, pages, page, kv, hd, rows, width, by_head, k, v), so.Pages(pages, page, rows, width)
    refused = 0
    for step in range(40):
        what = step % 4
        if what == 1:
            parents = np.arange(rows)
            some = r.random(rows) < 0.4
            parents[some] = r.integers(-1, rows, some.sum())
            pg.fork(parents)
            c.fork(parents)
        elif what == 3 and step % 8 == 3:
            drop = np.where(r.random(rows) < 0.4, -1, np.arange(rows))
            pg.fork(drop)
            c.fork(drop)
            moved, live, moves = pg.compact()
            got = c.compact()
            assert np.array_equal(got[0], moved) and got[1] == live
            for s, d in moves:
                k[:, d], v[:, d] = k[:, s], v[:, s]
        else:
            new = r.integers(0, 2 if what else page + 2, rows)
            want, copies = pg.reserve(new)
            assert c.reserve(new) == want
            refused += want != 0
            for s, d, n in copies:
                k[:, d, :n], v[:, d, :n] = k[:, s, :n], v[:, s, :n]
        same_books(c, pg)
        if want_contents(step):
            gk, gv = c.pools()
            assert np.array_equal(gk, k) and np.array_equal(gv, v), step
    assert tl.device_status() == 0


def want_contents(step):
    return step % 5 == 4 or step > 36


def test_fork_of_many_rows(tl):
    """More rows than 32 bytes each fill shared memory with."""
    r = np.random.default_rng(23)
    rows, width, pages = 7001, 11, 300
    c, pg = tl.PagedCache(1, pages, 2, 1, 8, rows, width), so.Pages(pages, 2, rows, width)
    n = r.integers(0, width + 1, rows)
    pg.table = np.where(np.arange(width) < n[:, None], r.integers(0, pages, (rows, width)), -1).astype(np.int32)
    pg.lengths = (2 * n).astype(np.int32)
    pg.refs = np.bincount(pg.table[pg.table >= 0], minlength=pages).astype(np.int32)
    c.set_state(pg.table, pg.lengths, pg.refs)
    for share in (0.9, 0.3, 1.0):
        parents = np.where(r.random(rows) < share, r.integers(-1, rows, rows), np.arange(rows))
        c.fork(parents)
        pg.fork(parents)
        same_books(c, pg)
    assert tl.device_status() == 0


def test_pages_refuse_without_changing_anything(tl):
    c, pg = tl.PagedCache(1, 6, 4, 1, 8, 4, 3), so.Pages(6, 4, 4, 3)
    for new in ([5, 3, 0, 0], [1, 1, 1, 1]):
        assert c.reserve(new) == pg.reserve(new)[0] == 0
    c.fork([0, 1, 0, 0])
    pg.fork([0, 1, 0, 0])
    for new in ([1, 1, 1, 1], [9, 0, 0, 0], [0, 9, 0, 0], [2, 2, 2, 2]):           # no page left for every copy; more than max_pages
        want, _ = pg.reserve(new)
        assert c.reserve(new) == want
        same_books(c, pg)
    assert tl.device_status() == 0
    assert c.reserve([0, -1, 0, 0]) == 1                                         # no such number of tokens
    assert tl.device_status() == 1
    same_books(c, pg)
    table, lengths, refs = c.state()
    bad = table.copy()
    assert lengths[0] % 4                                                        # its next token goes into its last page
    bad[0, lengths[0] // 4] = 77
    c.set_state(bad, lengths, refs)
    assert c.reserve([1, 0, 0, 0]) == 1 and tl.device_status() == 1               # an entry that names no page
    c.set_state(table, lengths, refs)
    c.fork([0, 4, -2, 3])                                                        # parents that are no rows: those rows stay
    assert tl.device_status() == 1
    same_books(c, pg)
    c.copy([0, 9, 2], [3, 1, -1])
    assert tl.device_status() == 1


def test_pages_refused_for_their_counts_keep_them(tl):
    """A count below the number of rows that let go of the page: refused, and every count as it was."""
    for rows, page, lens, counts, new in ((3, 4, [2, 0, 0], [0], [1, 0, 0]), (3, 4, [2, 2, 0], [1], [1, 1, 0]), (4, 4, [2, 2, 2, 0], [-3], [1, 1, 1, 2]),
                                          (1500, 8, [3] * 1500, [1498], [1] * 1500), (1500, 8, [3] * 1500, [0], [1] * 1499 + [0])):
        c = tl.PagedCache(1, 6, page, 1, 8, rows, 3)
        table, refs = np.full((rows, 3), -1, np.int32), np.zeros(6, np.int32)
        table[np.array(lens) > 0, 0] = 2
        refs[2] = counts[0]
        table[rows - 1, 0], refs[4] = 4, 1                # a sound page beside it
        lens = lens[:-1] + [1]
        c.set_state(table, lens, refs)
        assert c.reserve(new) == 1 and tl.device_status() == 1
        for got, want in zip(c.state(), (table, lens, refs)):
            assert np.array_equal(got, want), (rows, got, want)


def test_pages_wanted_beyond_32_bits_are_refused(tl):
    """4096 rows that ask for 2^20 pages each, of a table of 16 GB: 2^32 in all, which 32 bits hold as 0."""
    rows, width = 4096, 1 << 20
    c = tl.PagedCache(1, 64, 1, 1, 8, rows, 4)
    lib, big = tl.load(), tl.DeviceBuffer(4 * rows * width)
    tl.check(lib.tl_memset(big.ptr, 0xff, big.nbytes, None), "memset")
    c.c.page_table, c.c.max_pages = big.ptr, width
    for new in (np.full(rows, width), np.r_[np.full(rows - 1, width), 5]):
        assert c.reserve(new) == 5
        assert (c._lengths.to_numpy(np.int32, (rows,)) == 0).all() and (c._refs.to_numpy(np.int32, (64,)) == 0).all()
    new = np.zeros(rows)
    new[[0, rows - 1]] = [3, 60]
    assert c.reserve(new) == 0
    head, tail = np.empty(4, np.int32), np.empty(61, np.int32)
    tl.check(lib.tl_memcpy_d2h(tl._np_ptr(head), big.ptr, head.nbytes, None), "d2h")
    tl.check(lib.tl_memcpy_d2h(tl._np_ptr(tail), big.ptr + 4 * (rows - 1) * width, tail.nbytes, None), "d2h")
    tl.synchronize()
    assert head.tolist() == [0, 1, 2, -1] and tail.tolist() == list(range(3, 63)) + [-1]
    assert tl.device_status() == 0


@pytest.mark.parametrize("shape,by_head", [((2, 30, 16, 4, 64), False), ((3, 12, 5, 3, 7), False), ((1, 40, 8, 2, 24), True)])
def test_page_copies(tl, shape, by_head):
    r = np.random.default_rng(21)
    k, v = normal(r, *shape), normal(r, *shape)
    c = tl.PagedCache(*shape, 2, 4, by_head, k, v)
    src, dst = [1, 3, -1, 5, 9, 0], [2, 4, 6, 5, 8, 11]
    c.copy(src, dst)
    for s, d in zip(src, dst):
        if s >= 0:
            k[:, d], v[:, d] = k[:, s], v[:, s]
    gk, gv = c.pools()
    assert np.array_equal(gk, k) and np.array_equal(gv, v) and tl.device_status() == 0


def test_pages_with_gaps_between_tokens_and_heads(tl):
    """Strides wider than the rows: contents move, gaps stay."""
    r = np.random.default_rng(22)
    L, P, s, H, d = 2, 6, 4, 3, 8
    for hs, ts in ((8, 40), (16, 48), (80, 16)):          # heads packed; neither; by head with gaps
        ps = max(ts * s, hs * H) + 8
        flat = normal(r, 2, L * P * ps)
        bufs = [tl.DeviceBuffer.from_numpy(a) for a in flat]
        c = tl.PagedCache(L, P, s, H, d, 3, 4)
        c.c.k_pages, c.c.v_pages, c.c.layer_stride, c.c.page_stride, c.c.token_stride, c.c.head_stride = bufs[0].ptr, bufs[1].ptr, P * ps, ps, ts, hs
        pg = so.Pages(P, s, 3, 4)
        for new in ([3, 0, 0],):
            assert c.reserve(new) == pg.reserve(new)[0] == 0
        c.fork([0, 0, 0])
        pg.fork([0, 0, 0])
        want, copies = pg.reserve([1, 1, 0])
        assert c.reserve([1, 1, 0]) == want == 0 and len(copies) == 2
        c.copy([copies[0][1]], [5])
        for a in flat:
            def at(l, p, t, h):
                return slice(l * P * ps + p * ps + t * ts + h * hs, l * P * ps + p * ps + t * ts + h * hs + d)
            for src, dst, n in copies + [(copies[0][1], 5, s)]:
                for l in range(L):
                    for t in range(n):
                        for h in range(H):
                            a[at(l, dst, t, h)] = a[at(l, src, t, h)]
        for a, b in zip(flat, bufs):
            assert np.array_equal(b.to_numpy(np.float16, a.shape), a), (hs, ts)
        same_books(c, pg)


# ---- beams ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("batch,beams,vocab,k", BEAM_SHAPES)
@pytest.mark.parametrize("with_finished", [False, True])
def test_beam_selection(tl, batch, beams, vocab, k, with_finished):
    x, s, fin = beam_case(batch, beams, vocab, 1)
    pad = min(2, vocab - 1)
    with np.errstate(all="ignore"):
        want = so.beam_select(x, s, beams, k, fin if with_finished else None, pad)
    got = tl.beam_select(x, s, beams, k, fin if with_finished else None, pad)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    # the log of the sum is good to 2^-21 (32-bit exponentials), and the result rounded once
    close(got[0], want[0], np.abs(want[0]) * 2.0 ** -24 + 2.0 ** -21)
    again = tl.beam_select(x, s, beams, k, fin if with_finished else None, pad)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))


def test_beam_selection_first_step_and_nothing_left(tl):
    r = np.random.default_rng(31)
    x = normal(r, 8, 1000, std=3)
    x[:4] = x[0]                                                     # all beams of an entry start out alike, one is live
    s = np.array([0, -np.inf, -np.inf, -np.inf, -1, -np.inf, -np.inf, np.nan], np.float32)
    want = so.beam_select(x, s, 4, 8)
    got = tl.beam_select(x, s, 4, 8)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    got = tl.beam_select(x, np.full(8, -np.inf, np.float32), 4, 5)      # no live beam: the first candidates, at -inf
    assert (got[0] == -np.inf).all() and np.array_equal(got[2], [np.arange(5)] * 2) and np.array_equal(got[1], [[0] * 5, [4] * 5])
    got = tl.beam_select(np.full((2, 1000), -np.inf, np.float16), np.zeros(2, np.float32), 2, 3)
    assert (got[0] == -np.inf).all() and np.array_equal(got[2], [[0, 1, 2]]) and np.array_equal(got[1], [[0, 0, 0]])
    got = tl.beam_select(np.zeros((3, 700), np.float16), np.zeros(3, np.float32), 3, 70)   # every candidate equal: the lowest indices
    assert np.array_equal(got[2][0], np.arange(70)) and (got[1] == 0).all()
    z = np.full((1, 700), -0.0, np.float16)
    z[0, 500:] = 0.0
    assert np.array_equal(tl.beam_select(z, [0.0], 1, 9)[2][0], np.arange(9))              # -0 equals +0


@pytest.mark.parametrize("batch,beams,vocab,k", [(2, 4, 5000, 8), (3, 2, 20000, 100), (1, 8, 70001, 16), (300, 3, 900, 5), (2, 128, 300, 128)])
def test_beam_selection_where_scores_leave_no_room_for_logits(tl, batch, beams, vocab, k):
    """Scores so large that many candidates are equal in 64 bits: the lowest beams, then the lowest tokens, whatever their logits."""
    r = np.random.default_rng([34, beams, vocab])
    rows = batch * beams
    x = r.choice([0.0, -0.5, 3.0, 5.0], (rows, vocab)).astype(np.float16)
    x[r.random((rows, vocab)) < 0.2] = -np.inf
    for n, big in enumerate((-1e30, 3e38, 2.0 ** 90)):
        s = np.full(rows, big, np.float32)
        if n == 0:
            s[::beams * 2] = -4.0                            # some entries have a beam with room
        want = so.beam_select(x, s, beams, k)
        got = tl.beam_select(x, s, beams, k)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), big
        close(got[0], want[0], np.abs(want[0]) * 2.0 ** -24 + 2.0 ** -21)
    # below 2^60 the steps are 128: the few logits within half a step of 0 are equal, and so are the many at -400
    x = np.full((rows, vocab), -400, np.float16)
    for row in x:
        row[r.permutation(vocab)[:min(vocab, k // 2 + 1)]] = r.choice([0.0, 2.0, 9.0], min(vocab, k // 2 + 1))
    s = np.full(rows, 2.0 ** 60, np.float32)
    want, got = so.beam_select(x, s, beams, k), tl.beam_select(x, s, beams, k)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]) and np.array_equal(got[0], want[0].astype(np.float32))


@pytest.mark.parametrize("batch,beams,vocab,k", [(3, 8, 32000, 16), (1, 4, 700, 100), (2, 16, 20001, 64), (1, 3, 50, 120)])
def test_beam_selection_with_beams_marked_by_a_large_score(tl, batch, beams, vocab, k):
    """One live beam an entry and the others at -1e9 or lower, as for a search's first step: the live one's candidates come first, and
    where there are too few of them (masked ones count as -inf) the marked beams' follow, in order."""
    r = np.random.default_rng([36, beams, vocab, k])
    rows = batch * beams
    for mark in (-1e9, -1e20, -3e38):
        x = (r.standard_normal((rows, vocab)) * 3).astype(np.float16)
        live = np.arange(batch) * beams + r.integers(0, beams, batch)
        s = np.full(rows, mark, np.float32)
        s[live] = -r.random(batch)
        for some in (vocab, k // 2):                     # the live beam's tokens that are not masked
            for row in live:
                x[row, r.permutation(vocab)[some:]] = -np.inf
            want = so.beam_select(x, s, beams, k)
            got = tl.beam_select(x, s, beams, k)
            sure = want[0] > mark / 2 if mark == -1e9 else np.ones(want[0].shape, bool)      # at -1e9 the log-sums' rounding decides
            assert np.array_equal(got[1][sure], want[1][sure]) and np.array_equal(got[2][sure], want[2][sure]), (mark, some)
            close(got[0], want[0], np.abs(want[0]) * 2.0 ** -24 + 2.0 ** -21)


@pytest.mark.parametrize("batch,beams,vocab", [(5, 4, 3001), (3, 128, 200)])
def test_beam_selection_writes_the_scores_in_place(tl, batch, beams, vocab):
    """Both kernels: the second shape has more candidates than one CTA joins."""
    x, s, fin = beam_case(batch, beams, vocab, 2)
    with np.errstate(all="ignore"):
        want = so.beam_select(x, s, beams, beams, fin, 0)
    assert want[3] > 1e-6
    lib, need = tl.load(), C.c_size_t(0)
    tl.check(lib.tl_beam_select_workspace(batch, beams, vocab, beams, C.byref(need)), "ws")
    w = tl.DeviceBuffer.from_numpy(np.zeros(max(16, need.value), np.uint8))
    dx, ds, df, dp, dt = (tl.DeviceBuffer.from_numpy(a) for a in (x, s, fin, np.zeros(batch * beams, np.int32), np.zeros(batch * beams, np.int32)))
    tl.check(lib.tl_beam_select_f16(dx.ptr, vocab, ds.ptr, df.ptr, 0, batch, beams, vocab, beams, ds.ptr, dp.ptr, dt.ptr, w.ptr, w.nbytes, None), "select")
    assert np.array_equal(dp.to_numpy(np.int32, (batch, beams)), want[1]) and np.array_equal(dt.to_numpy(np.int32, (batch, beams)), want[2])
    close(ds.to_numpy(np.float32, (batch, beams)), want[0], np.abs(want[0]) * 2.0 ** -24 + 2.0 ** -21)


@pytest.mark.parametrize("stride,off", [(1004, 0), (1001, 0), (1008, 3)])
def test_beam_selection_with_row_strides(tl, stride, off):
    """Rows that start at any 2-byte boundary; what lies behind a row is not read as a candidate."""
    r = np.random.default_rng(32)
    rows, vocab, k = 6, 1000, 6
    flat = np.full(rows * stride + 8, 60000, np.float16)
    x = normal(r, rows, vocab, std=3)
    for i in range(rows):
        flat[off + i * stride: off + i * stride + vocab] = x[i]
    s = (-r.random(rows)).astype(np.float32)
    need = C.c_size_t(0)
    lib = tl.load()
    tl.check(lib.tl_beam_select_workspace(2, 3, vocab, k, C.byref(need)), "ws")
    w = tl.DeviceBuffer.from_numpy(np.zeros(max(16, need.value), np.uint8))
    dx, ds, outs = tl.DeviceBuffer.from_numpy(flat), tl.DeviceBuffer.from_numpy(s), [tl.DeviceBuffer(2 * k * 4) for _ in range(3)]
    tl.check(lib.tl_beam_select_f16(dx.ptr + 2 * off, stride, ds.ptr, None, 0, 2, 3, vocab, k, outs[0].ptr, outs[1].ptr, outs[2].ptr, w.ptr, w.nbytes, None), "select")
    want = so.beam_select(x, s, 3, k)
    assert np.array_equal(outs[1].to_numpy(np.int32, (2, k)), want[1]) and np.array_equal(outs[2].to_numpy(np.int32, (2, k)), want[2])


def select_rows(tl, x, s, beams, k, stride, off):
    """Selection from rows `stride` apart that start `off` values into a buffer of 60000s; checked against the values in 64 bits: each
    beam's tokens are its first ones by (logit, lowest token), and what is left out is no better but for the rounding of the log-sums."""
    rows, vocab = x.shape
    batch = rows // beams
    lib, need = tl.load(), C.c_size_t(0)
    flat = np.full(off + rows * stride + 8, 60000, np.float16)
    flat[off:off + rows * stride].reshape(rows, stride)[:, :vocab] = x
    tl.check(lib.tl_beam_select_workspace(batch, beams, vocab, k, C.byref(need)), "ws")
    w, dx, ds = (tl.DeviceBuffer.from_numpy(a) for a in (np.zeros(max(16, need.value), np.uint8), flat, np.asarray(s, np.float32)))
    out = [tl.DeviceBuffer.from_numpy(np.full(batch * k, -7, np.int32)) for _ in range(3)]
    tl.check(lib.tl_beam_select_f16(dx.ptr + 2 * off, stride, ds.ptr, None, 0, batch, beams, vocab, k, *(o.ptr for o in out), w.ptr, w.nbytes, None), "select")
    values = so.beam_values(x, s).reshape(batch, beams * vocab)
    parents, tokens = (o.to_numpy(np.int32, (batch, k)) for o in out[1:])
    at = (parents - np.arange(batch)[:, None] * beams).astype(np.int64) * vocab + tokens
    assert at.min() >= 0 and at.max() < beams * vocab and all(len(set(a)) == k for a in at)
    logits = np.minimum(np.where(np.isnan(x), -np.inf, x.astype(np.float64)), 65504.0)
    for b in range(batch):
        for beam in range(beams):
            chosen = tokens[b][parents[b] == b * beams + beam]
            row = logits[b * beams + beam]
            assert np.array_equal(chosen, np.argsort(-row, kind="stable")[:len(chosen)]), (b, beam)
    got, want = np.take_along_axis(values, at, 1), -np.sort(-values, axis=1)[:, :k]
    with np.errstate(invalid="ignore"):
        assert ((got == want) | (np.abs(got - want) <= 2.0 ** -20)).all()
    close(out[0].to_numpy(np.float32, (batch, k)), got, np.abs(got) * 2.0 ** -24 + 2.0 ** -21)


@pytest.mark.parametrize("batch,beams,vocab,k,stride,off", [(1, 16, 20001, 64, 20001, 0), (1, 16, 20001, 64, 20004, 3), (1, 16, 40000, 64, 40000, 0),
                                                            (2, 128, 25003, 8, 25003, 1), (300, 2, 20480, 16, 20480, 0), (600, 1, 9001, 1, 9001, 5),
                                                            (1, 8, 16385, 128, 16392, 0), (40, 16, 8193, 33, 8200, 7)])
def test_beam_selection_over_several_windows(tl, batch, beams, vocab, k, stride, off):
    """Rows (chunks of them) of more than 8192 logits: random, rising, falling, all equal, masked but for a few, with NaN and infinities,
    and large where the first window has seen nothing of it."""
    r = np.random.default_rng([35, batch, beams, vocab, k])
    rows = batch * beams
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float16)
    for i in range(rows):
        kind = i % 9
        if kind == 1:
            x[i] = np.linspace(-9, 9, vocab)
        elif kind == 2:
            x[i] = np.linspace(9, -9, vocab)
        elif kind == 3:
            x[i] = 2.5
        elif kind == 4:
            keep = r.permutation(vocab)[:20]
            kept = x[i, keep]
            x[i] = -np.inf
            x[i, keep] = kept
        elif kind == 5:
            x[i, r.random(vocab) < 0.3] = np.nan
            x[i, r.integers(vocab)] = -np.inf
        elif kind == 6:
            x[i, r.random(vocab) < 0.01] = np.inf
        elif kind == 7:
            x[i, vocab // 2:] += np.float16(20)
        elif kind == 8:
            x[i] = r.choice([1.0, 1.5, -0.0, 0.0], vocab)
    select_rows(tl, x, -r.random(rows).astype(np.float32), beams, k, stride, off)
    assert tl.device_status() == 0


def test_beam_selection_of_other_sizes_in_the_same_workspace(tl):
    """Zeroed once, then calls of any sizes: what one leaves behind is no counter of the next. More entries than one launch takes as well."""
    shapes = [(2, 4, 5000, 4), (300, 3, 40, 3), (2, 4, 5000, 4), (4100, 2, 17, 5), (1, 8, 30000, 128), (9001, 1, 9, 9), (64, 8, 600, 16)]
    lib, need = tl.load(), C.c_size_t(0)
    size = 16
    for batch, beams, vocab, k in shapes:
        tl.check(lib.tl_beam_select_workspace(batch, beams, vocab, k, C.byref(need)), "ws")
        size = max(size, need.value)
    w = tl.DeviceBuffer.from_numpy(np.zeros(size, np.uint8))
    for n, (batch, beams, vocab, k) in enumerate(shapes):
        r = np.random.default_rng([33, n])
        x, s = normal(r, batch * beams, vocab, std=3), -r.random(batch * beams).astype(np.float32)
        fin = (r.random(batch * beams) < 0.2).astype(np.uint8)
        dx, ds, df = (tl.DeviceBuffer.from_numpy(a) for a in (x, s, fin))
        out = [tl.DeviceBuffer.from_numpy(np.full(batch * k, -7, np.int32)) for _ in range(3)]
        tl.check(lib.tl_beam_select_f16(dx.ptr, vocab, ds.ptr, df.ptr, 1, batch, beams, vocab, k, *(o.ptr for o in out), w.ptr, w.nbytes, None), "select")
        values = so.beam_values(x, s, fin, 1).reshape(batch, beams * vocab)
        parents, tokens = (o.to_numpy(np.int32, (batch, k)) for o in out[1:])
        at = (parents - np.arange(batch)[:, None] * beams).astype(np.int64) * vocab + tokens
        assert at.min() >= 0 and at.max() < beams * vocab and all(len(set(a)) == k for a in at), n
        # values nearer to one another than the logs of the sums are good to may change places
        got, want = np.take_along_axis(values, at, 1), -np.sort(-values, axis=1)[:, :k]
        with np.errstate(invalid="ignore"):
            assert ((got == want) | (np.abs(got - want) <= 2.0 ** -20)).all(), n
        close(out[0].to_numpy(np.float32, (batch, k)), got, np.abs(got) * 2.0 ** -24 + 2.0 ** -21, n)


def test_beam_selection_of_the_largest_vocabulary(tl):
    """2^31 - 1 equal logits but for two: the last, and one in the middle."""
    lib, vocab, need = tl.load(), 2 ** 31 - 1, C.c_size_t(0)
    tl.check(lib.tl_beam_select_workspace(1, 1, vocab, 1, C.byref(need)), "ws")
    dx, ds = tl.DeviceBuffer(2 * vocab), tl.DeviceBuffer.from_numpy(np.array([-1.5], np.float32))
    w, out = tl.DeviceBuffer.from_numpy(np.zeros(max(16, need.value), np.uint8)), [tl.DeviceBuffer(4) for _ in range(3)]
    tl.check(lib.tl_memset(dx.ptr, 0, dx.nbytes, None), "memset")
    for at, value in ((vocab - 1, 4.0), (1 << 30, 3.0)):
        one = np.array([value], np.float16)
        tl.check(lib.tl_memcpy_h2d(dx.ptr + 2 * at, one.ctypes.data, 2, None), "h2d")
        tl.synchronize()
    tl.check(lib.tl_beam_select_f16(dx.ptr, vocab, ds.ptr, None, 0, 1, 1, vocab, 1, *(o.ptr for o in out), w.ptr, w.nbytes, None), "select")
    want = -1.5 + np.array([4.0]) - np.log(vocab - 2 + np.exp(4.0) + np.exp(3.0))
    close(out[0].to_numpy(np.float32, (1,)), want, np.abs(want) * 2.0 ** -24 + 2.0 ** -21)
    assert out[2].to_numpy(np.int32, (1,)).tolist() == [vocab - 1] and out[1].to_numpy(np.int32, (1,)) == 0
    assert tl.device_status() == 0


@pytest.mark.parametrize("outer,rows,pitch,used", [(1, 1, 8, 8), (2, 5, 24, 17), (3, 4, 70000, 69993), (2, 7, 33, 33), (4, 64, 4096, 1000)])
def test_beam_reorder(tl, outer, rows, pitch, used):
    r = np.random.default_rng([outer, rows, pitch])
    src, dst = normal(r, outer, rows, pitch), normal(r, outer, rows, pitch)
    parents = r.integers(0, rows, rows).astype(np.int32)
    if rows > 3:
        parents[2] = -1
    got = tl.beam_reorder(src, dst, parents, used)
    want = dst.copy()
    for i, p in enumerate(parents):
        if p >= 0:
            want[:, i, :used] = src[:, p, :used]
    assert np.array_equal(got, want) and tl.device_status() == 0
    if rows > 3:
        parents[0], parents[1] = rows, -2
        got = tl.beam_reorder(src, dst, parents, used)
        want[:, :2] = dst[:, :2]
        assert np.array_equal(got, want) and tl.device_status() == 1


# ---- nothing to do, threads ----------------------------------------------------------------------------------------
def test_calls_with_nothing_to_do(tl):
    h = lambda *n: np.zeros(n, np.float16)  # noqa: E731
    f = tl.rotary_frequencies(16)[0]
    c = tl.PagedCache(1, 4, 8, 2, 16, 3, 2)
    assert tl.rotary(h(0, 2, 16), [], f).shape == (0, 2, 16)
    assert c.append(0, h(0, 4, 16), h(0, 2, 16), h(0, 2, 16), [], f).shape == (0, 4, 16)
    out, lse = c.attend(0, h(0, 4, 16))
    assert out.shape == (0, 4, 16) and lse.shape == (0, 4)
    c.copy([], [])
    assert c.reserve([0, 0, 0]) == 0
    moved, live = c.compact()
    assert (moved == -1).all() and live == 0
    assert all(a.shape == (0, 3) for a in tl.beam_select(h(0, 9), [], 2, 3))
    dst = normal(np.random.default_rng(1), 2, 3, 8)
    assert np.array_equal(tl.beam_reorder(h(2, 3, 8), dst, [0, 0, 0], 0), dst) and tl.beam_reorder(h(0, 3, 8), h(0, 3, 8), [0, 0, 0], 8).shape == (0, 3, 8)
    table, lengths, refs = c.state()
    assert (table == -1).all() and (lengths == 0).all() and (refs == 0).all() and tl.device_status() == 0


def test_host_threads_with_workspaces_of_their_own(tl):
    """Four threads at once, each with its own cache and arrays: every result as from one alone."""
    from concurrent.futures import ThreadPoolExecutor

    def work(i):
        r = np.random.default_rng([61, i])
        hd, lens = (64, 96, 192, 256)[i], [300, 0, 17, 1200]
        c, k, v, table, _ = filled_cache(tl, r, 1, 16, 2, hd, lens)
        x, s = normal(r, 8, 5000 + i, std=3), -r.random(8).astype(np.float32)
        q = normal(r, 4, 6, hd, std=1.5)
        want = so.beam_select(x, s, 4, 8)
        for _ in range(10):
            check_attention(tl, c, k[0], v[0], table, lens, 16, q)
            got = tl.beam_select(x, s, 4, 8)
            assert want[3] < 1e-6 or (np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]))
            assert c.reserve([1, 0, 0, 0]) in (0, 5)
            lens[0] = int(c.state()[1][0])
            lens[0] -= 1
            c.set_state(*(a if j != 1 else lens for j, a in enumerate(c.state())))
        return True

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))
    assert tl.device_status() == 0


# ---- bad ids and the rest of the library ---------------------------------------------------------------------------
def test_bad_ids_are_no_concern_of_a_model(tl):
    """An id outside its table is reported by tl_device_status, not by the next call of a model, and hides no timeout."""
    from tensorlib_b200 import synth
    lib = tl.load()
    m = tl.Llama2(synth.TINY, numerics=tl.FAST)
    m.init_random(7)
    want = m.generate([3, 5, 7], 8)[0]
    c = tl.PagedCache(1, 6, 4, 1, 8, 2, 3)
    c.fork([0, 9])
    assert np.array_equal(m.generate([3, 5, 7], 8)[0], want)
    assert tl.device_status() == 1 and tl.device_status() == 0
    tl.check(lib.tl_selftest_unposted_exchange(256, None), "tl_selftest_unposted_exchange")
    c.fork([0, 9])
    tl.synchronize()
    assert tl.device_status() == 6 and tl.device_status() == 1 and tl.device_status() == 0
    m.close()


# ---- together ------------------------------------------------------------------------------------------------------
def test_a_beam_search_over_pages_matches_one_over_copied_sequences(tl):
    """Select, fork, reserve, append and attend for 3 entries of 4 beams over 2 layers and 30 steps, against beams that carry
    their whole history with them. Queries, keys, values and logits are functions of the token and step alone."""
    r = np.random.default_rng(41)
    batch, beams, vocab, layers, kv, heads, hd, page, steps = 3, 4, 50, 2, 2, 6, 64, 8, 30
    rows = batch * beams
    emb = normal(r, vocab, 2, heads + 2 * kv, hd)
    lm = normal(r, vocab, vocab, std=2)
    f, mag = tl.rotary_frequencies(hd, scaling="parts", factor=4.0, trained_len=16, low=1, high=4)
    c = tl.PagedCache(layers, 120, page, kv, hd, rows, 8)
    hist = [[] for _ in range(rows)]
    scores = np.where(np.arange(rows) % beams == 0, 0.0, -np.inf).astype(np.float32)
    fin = np.zeros(rows, np.uint8)
    tokens = np.arange(rows) // beams
    for step in range(steps):
        assert c.reserve(np.ones(rows, np.int32)) == 0
        hist = [h + [int(t)] for h, t in zip(hist, tokens)]
        pos = np.full(rows, step, np.int32)
        e = emb[tokens]
        for layer in range(layers):
            q = c.append(layer, np.ascontiguousarray(e[:, layer, :heads]), np.ascontiguousarray(e[:, layer, heads:heads + kv]),
                         np.ascontiguousarray(e[:, layer, heads + kv:]), pos, f, mag, True)
            out, lse = c.attend(layer, q)
            if step % 7 == 6 or step == steps - 1:
                for i in range(rows):
                    k = np.stack([so.rotary(emb[t, layer, heads:heads + kv][None], [s], f, mag, True)[0][0] for s, t in enumerate(hist[i])]).astype(np.float16)
                    v = np.stack([emb[t, layer, heads + kv:] for t in hist[i]])
                    for h in range(heads):
                        o, l, to, tl_ = so.attend(q[i, h], k[:, h // 3], v[:, h // 3], hd ** -0.5)
                        # keys here are rounded from 64 bits, there from 32: a step of fp16 apart where the two fall apart
                        slack = 2 * 2 * so.EPS16 * (np.abs(k[:, h // 3]).astype(np.float64) @ np.abs(q[i, h]).astype(np.float64)).max() * hd ** -0.5
                        close(out[i, h], o, to + slack * np.abs(v[:, h // 3]).astype(np.float64).max(0), (step, i, h))
                        assert abs(lse[i, h] - l) <= tl_ + slack
        logits = np.stack([lm[t] + np.float16(0.01 * (step % 3)) for t in tokens]).astype(np.float16)
        want = so.beam_select(logits, scores, beams, beams, fin, 1)
        got = tl.beam_select(logits, scores, beams, beams, fin, 1)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]), step
        parents, tokens, scores = got[1].reshape(-1), got[2].reshape(-1), got[0].reshape(-1)
        c.fork(parents)
        hist = [list(hist[p]) for p in parents]
        fin = fin[parents] | (tokens == 1)
        table, lengths, refs = c.state()
        want_refs = np.zeros_like(refs)
        np.add.at(want_refs, table[table >= 0], 1)
        assert np.array_equal(refs, want_refs)
        if step % 10 == 9:
            c.compact()
    assert tl.device_status() == 0


def test_a_whole_step_replayed_from_a_graph(tl):
    """Fork, reserve, append, attend, select and compact captured once and replayed: the books move on with every replay."""
    torch = pytest.importorskip("torch")
    r = np.random.default_rng(52)
    lib = tl.load()
    rows, page, kv, heads, hd, width, pages = 6, 4, 2, 4, 32, 8, 60
    c, pg = tl.PagedCache(1, pages, page, kv, hd, rows, width), so.Pages(pages, page, rows, width)
    k, v = c.pools()
    assert c.reserve([3, 0, 5, 0, 1, 0]) == pg.reserve([3, 0, 5, 0, 1, 0])[0] == 0
    parents, ones = np.array([0, 0, 2, 2, 4, 4], np.int32), np.ones(rows, np.int32)
    need, bneed, aneed = C.c_size_t(0), C.c_size_t(0), C.c_size_t(0)
    tl.check(lib.tl_paged_workspace(rows, pages, C.byref(need)), "ws")
    tl.check(lib.tl_beam_select_workspace(3, 2, 90, 2, C.byref(bneed)), "ws")
    tl.check(lib.tl_paged_attn_workspace(heads, kv, hd, C.byref(aneed)), "ws")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    t = dict(par=cuda(parents), one=cuda(ones), pos=cuda(np.zeros(rows, np.int32)), res=cuda(np.zeros(4, np.int32)), moved=cuda(np.zeros(pages, np.int32)),
             q=cuda(normal(r, rows, heads, hd)), k=cuda(normal(r, rows, kv, hd)), v=cuda(normal(r, rows, kv, hd)), x=cuda(normal(r, rows, 90, std=2)),
             s=torch.zeros(rows, device="cuda"), f=cuda(tl.rotary_frequencies(hd)[0]), o=torch.zeros(rows, heads, hd, dtype=torch.float16, device="cuda"),
             qo=torch.zeros(rows, heads, hd, dtype=torch.float16, device="cuda"), sc=torch.zeros(3, 2, device="cuda"),
             ip=torch.zeros(3, 2, dtype=torch.int32, device="cuda"), it=torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
             w=torch.zeros(need.value, dtype=torch.uint8, device="cuda"), bw=torch.zeros(max(16, bneed.value), dtype=torch.uint8, device="cuda"),
             aw=torch.zeros(max(16, aneed.value), dtype=torch.uint8, device="cuda"))
    p = {n: a.data_ptr() for n, a in t.items()}
    cc = C.byref(c.c)
    lengths = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def step(st):
        tl.check(lib.tl_paged_fork(cc, p["par"], st), "fork")
        tl.check(lib.tl_paged_reserve_f16(cc, p["one"], p["res"], p["w"], t["w"].numel(), st), "reserve")
        tl.check(lib.tl_memcpy_d2d(lengths.data_ptr(), c._lengths.ptr, 4 * rows, st), "lengths")
        torch.sub(lengths, t["one"], out=t["pos"])                    # the new token's position
        tl.check(lib.tl_rotary_append_f16(cc, 0, p["q"], p["qo"], p["k"], p["v"], None, p["pos"], p["f"], 1.0, rows, heads, hd, 1, heads * hd, heads * hd,
                                          kv * hd, st), "append")
        tl.check(lib.tl_paged_attn_decode_f16(cc, 0, p["qo"], p["o"], None, None, rows, heads, hd ** -0.5, heads * hd, heads * hd, p["aw"], t["aw"].numel(), st), "attn")
        tl.check(lib.tl_beam_select_f16(p["x"], 90, p["s"], None, 0, 3, 2, 90, 2, p["sc"], p["ip"], p["it"], p["bw"], t["bw"].numel(), st), "select")
        tl.check(lib.tl_paged_compact_f16(cc, p["moved"], p["res"] + 4, p["w"], t["w"].numel(), st), "compact")

    torch.cuda.synchronize()
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=stream):
        step(torch.cuda.current_stream().cuda_stream)
    nk, nv, q = (t[n].cpu().numpy() for n in ("k", "v", "q"))
    f = tl.rotary_frequencies(hd)[0]
    for rep in range(5):
        g.replay()
        torch.cuda.synchronize()
        pg.fork(parents)
        status, copies = pg.reserve(ones)
        assert status == 0 and t["res"].cpu().numpy()[0] == 0
        for s, d, n in copies:
            k[:, d, :n], v[:, d, :n] = k[:, s, :n], v[:, s, :n]
        pos = pg.lengths - 1
        wk, tk = so.rotary(nk, pos, f, 1.0, True)
        for i in range(rows):
            at = (0, pg.table[i, pos[i] // page], pos[i] % page)
            k[at], v[at] = wk[i].astype(np.float16), nv[i]
        wq, tq = so.rotary(q, pos, f, 1.0, True)
        close(t["qo"].cpu().numpy(), wq, tq)
        before = pg.table.copy()
        moved, live, moves = pg.compact()
        kk, vv = k.copy(), v.copy()
        for s, d in moves:
            k[:, d], v[:, d] = k[:, s], v[:, s]
        same_books(c, pg)
        assert np.array_equal(t["moved"].cpu().numpy(), moved) and t["res"].cpu().numpy()[1] == live
        gk, gv = c.pools()
        for i in range(rows):                     # what the rows hold: values bit for bit, keys to their rounding
            n = pg.lengths[i]
            assert np.array_equal(row_tokens(gv[0], pg.table[i], n, page), row_tokens(v[0], pg.table[i], n, page))
            d = row_tokens(gk[0], pg.table[i], n, page).astype(np.float64) - row_tokens(k[0], pg.table[i], n, page).astype(np.float64)
            assert (np.abs(d) <= 2 * so.EPS16 * np.abs(row_tokens(k[0], pg.table[i], n, page).astype(np.float64)) + 2.0 ** -18).all()
        k[0], v[0] = gk[0], gv[0]
        for i in range(rows):
            keys, vals = row_tokens(k[0], pg.table[i], pg.lengths[i], page), row_tokens(v[0], pg.table[i], pg.lengths[i], page)
            for h in range(heads):
                o, l, to, _ = so.attend(t["qo"].cpu().numpy()[i, h], keys[:, h // 2], vals[:, h // 2], hd ** -0.5)
                close(t["o"].cpu().numpy()[i, h], o, to, (rep, i, h))
        want = so.beam_select(t["x"].cpu().numpy(), np.zeros(rows), 2, 2)
        assert np.array_equal(t["it"].cpu().numpy(), want[2]) and np.array_equal(t["ip"].cpu().numpy(), want[1])
    del g
    assert tl.device_status() == 0


def test_on_two_streams_and_from_a_graph(tl):
    """The calls enqueue on the stream that they are given; captured once, replayed on changed inputs."""
    torch = pytest.importorskip("torch")
    r = np.random.default_rng(51)
    lib = tl.load()
    lens, heads, hd, page = [900, 31, 0, 2000], 8, 64, 16
    c, k, v, table, _ = filled_cache(tl, r, 1, page, 2, hd, lens)
    beams, vocab, kk = 4, 5000, 8
    need = C.c_size_t(0)
    tl.check(lib.tl_beam_select_workspace(1, beams, vocab, kk, C.byref(need)), "ws")
    streams = [torch.cuda.Stream() for _ in range(2)]
    state = []
    for i in range(2):
        q, x = normal(r, 4, heads, hd), normal(r, beams, vocab, std=3)
        s = dict(q=torch.from_numpy(q).cuda(), out=torch.zeros(4, heads, hd, dtype=torch.float16, device="cuda"),
                 w=torch.zeros(32 << 20, dtype=torch.uint8, device="cuda"), x=torch.from_numpy(x).cuda(), s=torch.zeros(beams, device="cuda"),
                 v=torch.zeros(kk, device="cuda"), p=torch.zeros(kk, dtype=torch.int32, device="cuda"), t=torch.zeros(kk, dtype=torch.int32, device="cuda"),
                 bw=torch.zeros(max(need.value, 16), dtype=torch.uint8, device="cuda"))
        state.append((q, x, s))
    torch.cuda.synchronize()

    def call(s, stream):
        tl.check(lib.tl_paged_attn_decode_f16(C.byref(c.c), 0, s["q"].data_ptr(), s["out"].data_ptr(), None, None, 4, heads, hd ** -0.5, heads * hd,
                                              heads * hd, s["w"].data_ptr(), s["w"].numel(), stream), "attn")
        tl.check(lib.tl_beam_select_f16(s["x"].data_ptr(), vocab, s["s"].data_ptr(), None, 0, 1, beams, vocab, kk, s["v"].data_ptr(), s["p"].data_ptr(),
                                        s["t"].data_ptr(), s["bw"].data_ptr(), s["bw"].numel(), stream), "select")

    def verify(i):
        q, x, s = state[i]
        ref = c.attend(0, q)[0]
        assert np.array_equal(s["out"].cpu().numpy(), ref)
        assert np.array_equal(s["t"].cpu().numpy(), so.beam_select(x, np.zeros(beams), beams, kk)[2][0])
    for rep in range(20):
        for i in range(2):
            call(state[i][2], streams[i].cuda_stream)
    torch.cuda.synchronize()
    verify(0)
    verify(1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        call(state[0][2], torch.cuda.current_stream().cuda_stream)
    for rep in range(3):
        q, x = normal(r, 4, heads, hd), normal(r, beams, vocab, std=3)
        state[0] = (q, x, state[0][2])
        state[0][2]["q"].copy_(torch.from_numpy(q))
        state[0][2]["x"].copy_(torch.from_numpy(x))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        verify(0)
    del g
    assert tl.device_status() == 0
