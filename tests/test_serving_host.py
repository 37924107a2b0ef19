"""CPU suite of the operators for serving many sequences: what needs no device (rotation frequencies, workspace sizes), the
refusals, which come before the device is asked for, and the sanity of the shared cases."""
import ctypes as C
import math

import numpy as np
import pytest

import serving_oracle as so
import tensorlib_b200 as tl
from serving_cases import BEAM_SHAPES, beam_case

P = 4096            # a pointer that nobody follows: every call here is refused before


def test_frequencies_follow_their_formulas():
    for rot in (2, 64, 96, 128):
        i = np.arange(rot // 2)
        f, mag = tl.rotary_frequencies(rot)
        assert mag == 1.0 and np.allclose(f, 10000.0 ** (-2 * i / rot), rtol=1e-13, atol=0)
        assert np.allclose(tl.rotary_frequencies(rot, scaling="linear", factor=8.0)[0], f / 8, rtol=1e-13, atol=0)
        if rot > 2:
            g = tl.rotary_frequencies(rot, scaling="base", factor=8.0)[0]
            assert np.allclose(g, (10000.0 * 8 ** (rot / (rot - 2))) ** (-2 * i / rot), rtol=1e-13, atol=0)
            assert math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12)             # the slowest pair is divided by the whole factor
        g = tl.rotary_frequencies(rot, scaling="parts", factor=8.0, trained_len=4096, low=1, high=4)[0]
        turns = 4096 * f / (2 * np.pi)
        w = np.clip((turns - 1) / 3, 0, 1)
        assert np.allclose(g, (1 - w) * f / 8 + w * f, rtol=1e-12, atol=0)
        g, mag = tl.rotary_frequencies(rot, scaling="ramp", factor=8.0, trained_len=4096, low=1, high=32)
        assert abs(mag - (0.1 * math.log(8) + 1)) < 1e-6
        lo = max(math.floor(rot * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000))), 0)
        hi = min(math.ceil(rot * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000))), rot - 1)
        w = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        assert np.allclose(g, (1 - w) * f + w * f / 8, rtol=1e-12, atol=0)


def test_ramp_where_no_pair_turns_as_often_as_low():
    """trained_len below 2 pi low: every pair, the first among them, is on the scaled side."""
    for rot, trained, low in ((64, 6.0, 1.0), (64, 3.0, 1.0), (2, 1.0, 1.0), (128, 2 * math.pi * 4, 4.0 * (1 + 1e-9)), (8, 0.01, 2.0)):
        f = tl.rotary_frequencies(rot)[0]
        g = tl.rotary_frequencies(rot, scaling="ramp", factor=8.0, trained_len=trained, low=low, high=32)[0]
        assert np.allclose(g, f / 8, rtol=1e-13, atol=0), (rot, trained, low, g / f)
    # and as soon as the first one does, it is kept
    assert tl.rotary_frequencies(64, scaling="ramp", factor=8.0, trained_len=7.0, low=1.0, high=32)[0][0] == 1.0


def test_frequencies_refuse():
    for kw in (dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=8, base=1.0), dict(rot_dim=8, base=math.nan),
               dict(rot_dim=8, scaling="linear", factor=0.5), dict(rot_dim=8, scaling="parts", factor=2.0),
               dict(rot_dim=8, scaling="ramp", factor=2.0, trained_len=100.0, low=4.0, high=4.0)):
        with pytest.raises(tl.TLError) as e:
            tl.rotary_frequencies(**kw)
        assert e.value.status == 1
    assert tl.load().tl_rotary_frequencies(8, 1e4, 5, 1.0, 1.0, 1.0, 2.0, P, C.byref(C.c_float(0))) == 1


def cache(**kw):
    d = dict(k_pages=P, v_pages=P, layer_stride=1 << 20, page_stride=16 * 1024, token_stride=1024, head_stride=128, n_layers=2, n_pages=9,
             page_size=16, n_kv_heads=8, head_dim=128, n_rows=4, max_pages=8, page_table=P, lengths=P, ref_counts=P)
    d.update(kw)
    return C.byref(tl.tl_paged_cache(**d))


BAD_CACHES = [dict(n_layers=0), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(head_dim=-1), dict(n_rows=0), dict(max_pages=0),
              dict(page_table=None), dict(max_pages=1 << 30, page_size=2)]
BAD_POOLS = [dict(k_pages=None), dict(v_pages=None), dict(page_stride=0), dict(token_stride=-1), dict(head_stride=0), dict(layer_stride=0),
             dict(page_size=1 << 20, head_dim=1 << 10, max_pages=1)]


def refused(rc, status=1):
    assert rc == status, (rc, tl.load().tl_last_error())


def test_cache_calls_refuse_what_cannot_be_a_cache():
    lib = tl.load()
    ws = 1 << 25
    for bad in BAD_CACHES + BAD_POOLS:
        c = cache(**bad)
        refused(lib.tl_paged_reserve_f16(c, P, P, P, ws, None))
        refused(lib.tl_paged_copy_f16(c, P, P, 1, None))
        refused(lib.tl_paged_compact_f16(c, P, P, P, ws, None))
        refused(lib.tl_rotary_append_f16(c, 0, P, P, P, P, None, P, P, 1.0, 1, 8, 128, 0, 1024, 1024, 1024, None))
        refused(lib.tl_paged_attn_decode_f16(c, 0, P, P, P, None, 1, 8, 1.0, 1024, 1024, P, ws, None))
    for bad in BAD_CACHES + [dict(lengths=None), dict(ref_counts=None)]:
        refused(lib.tl_paged_fork(cache(**bad), P, None))
    refused(lib.tl_paged_fork(cache(), None, None))
    refused(lib.tl_paged_fork(None, P, None))
    refused(lib.tl_paged_copy_f16(cache(), None, P, 1, None))
    refused(lib.tl_paged_copy_f16(cache(), P, P, -1, None))
    for bad in (dict(lengths=None), dict(ref_counts=None)):
        refused(lib.tl_paged_reserve_f16(cache(**bad), P, P, P, ws, None))
    refused(lib.tl_paged_compact_f16(cache(ref_counts=None), P, P, P, ws, None))
    need = C.c_size_t(0)
    assert lib.tl_paged_workspace(4, 9, C.byref(need)) == 0
    for w, n in ((None, ws), (P + 8, ws), (P, need.value - 1)):
        refused(lib.tl_paged_reserve_f16(cache(), P, P, w, n, None))
        refused(lib.tl_paged_compact_f16(cache(), P, P, w, n, None))
    refused(lib.tl_paged_workspace(0, 9, C.byref(need)))


def test_rotary_refuses():
    lib = tl.load()
    ok = dict(i=P, o=P, pos=P, f=P, t=3, h=8, d=128, rot=128, half=0, its=1024, ihs=128, ots=1024, ohs=128)

    def call(**kw):
        a = {**ok, **kw}
        return lib.tl_rotary_f16(a["i"], a["o"], a["pos"], a["f"], 1.0, a["t"], a["h"], a["d"], a["rot"], a["half"], 0, a["its"], a["ihs"],
                                 a["ots"], a["ohs"], None)
    for bad in (dict(t=-1), dict(h=0), dict(d=0), dict(rot=129), dict(rot=127), dict(rot=130), dict(d=2048, rot=1026), dict(half=2), dict(i=None),
                dict(o=None), dict(pos=None), dict(f=None), dict(ots=2048), dict(its=-1), dict(ihs=-8), dict(o=2 * P, ots=-1024), dict(o=2 * P, ohs=-1), dict(h=1 << 20, d=1 << 12)):
        refused(call(**bad))
    c = cache()
    for layer, rest in ((2, (None, P, P, 1.0, 1, 8, 128, 0)), (-1, (None, P, P, 1.0, 1, 8, 128, 0)), (0, (None, P, P, 1.0, 5, 8, 128, 0)),
                        (0, (None, None, P, 1.0, 1, 8, 128, 0)), (0, (None, P, None, 1.0, 1, 8, 128, 0)), (0, (None, P, P, 1.0, 1, 8, 130, 0)),
                        (0, (None, P, P, 1.0, 1, -1, 128, 0)), (0, (None, P, P, 1.0, 1, 8, 128, 3))):
        refused(lib.tl_rotary_append_f16(c, layer, P, P, P, P, *rest, 1024, 1024, 1024, None))
    refused(lib.tl_rotary_append_f16(c, 0, None, P, P, P, None, P, P, 1.0, 1, 8, 128, 0, 1024, 1024, 1024, None))
    refused(lib.tl_rotary_append_f16(c, 0, P, P, P, P, None, P, P, 1.0, 1, 8, 128, 0, 1024, 2048, 1024, None))
    for strides in ((-1024, -1024, 1024), (1024, 1024, -1024)):
        refused(lib.tl_rotary_append_f16(c, 0, P, P, P, P, None, P, P, 1.0, 1, 8, 128, 0, *strides, None))


def test_helpers_refuse_arrays_of_other_sizes():
    """Before anything is allocated: the kernels read as much as the sizes say."""
    h = lambda *s: np.zeros(s, np.float16)  # noqa: E731
    c = tl.PagedCache.__new__(tl.PagedCache)      # no device here: only what the checks look at
    c.shape, c.by_head, c._attn_work, c._table, c._lengths, c._refs = (1, 4, 8, 2, 16), False, None, None, None, None
    c.c = cache(n_layers=1, n_pages=4, page_size=8, n_kv_heads=2, head_dim=16, n_rows=3, max_pages=2)._obj
    f = tl.rotary_frequencies(16)[0]
    for call in (lambda: tl.rotary(h(3, 2, 16), [0, 1], f), lambda: tl.rotary(h(3, 2, 16).astype(np.float32), [0, 1, 2], f),
                 lambda: tl.rotary(h(3, 2, 16), [0, 1, 2], f, out=h(3, 2, 8)),
                 lambda: tl.PagedCache(1, 4, 8, 2, 16, 3, 2, k=h(1, 4, 8, 2, 8)),
                 lambda: c.set_state(np.zeros((3, 3)), np.zeros(3), np.zeros(4)),
                 lambda: c.fork([0, 1]), lambda: c.reserve([1, 1, 1, 1]), lambda: c.copy([0, 1], [2]),
                 lambda: c.append(0, None, h(3, 2, 16), h(2, 2, 16), [0, 0, 0]), lambda: c.append(0, None, h(3, 1, 16), h(3, 1, 16), [0, 0, 0]),
                 lambda: c.append(0, h(2, 4, 16), h(3, 2, 16), h(3, 2, 16), [0, 0, 0]),
                 lambda: c.append(0, None, h(3, 2, 16), h(3, 2, 16), [0, 0]),
                 lambda: c.append(0, None, h(3, 2, 16), h(3, 2, 16), [0, 0, 0], rows=[1, 2]),
                 lambda: c.attend(0, h(3, 4, 8)), lambda: c.attend(0, h(3, 4, 16), rows=[0, 1]), lambda: tl.beam_select(h(5, 9), np.zeros(5), 2, 2), lambda: tl.beam_select(h(4, 9), np.zeros(3), 2, 2),
                 lambda: tl.beam_select(h(4, 9), np.zeros(4), 0, 2), lambda: tl.beam_select(h(4, 9), np.zeros(4), 2, 2, finished=[0, 1]),
                 lambda: tl.beam_reorder(h(1, 3, 8), h(1, 2, 8), [0, 0, 0], 8), lambda: tl.beam_reorder(h(1, 3, 8), h(1, 3, 8), [0, 0], 8)):
        with pytest.raises(ValueError):
            call()


def test_helpers_refuse_numbers_that_do_not_fit():
    """Whole numbers of 32 bits, 8 for the marks of finished beams: nothing is cut off or wrapped round."""
    h = lambda *s: np.zeros(s, np.float16)  # noqa: E731
    c = tl.PagedCache.__new__(tl.PagedCache)
    c.shape, c.by_head, c._attn_work, c._table, c._lengths, c._refs = (1, 4, 8, 2, 16), False, None, None, None, None
    c.c = cache(n_layers=1, n_pages=4, page_size=8, n_kv_heads=2, head_dim=16, n_rows=3, max_pages=2)._obj
    f = tl.rotary_frequencies(16)[0]
    for bad in (2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1, 1.5, np.nan, np.inf):
        for call in (lambda: tl.rotary(h(3, 2, 16), [0, bad, 1], f), lambda: c.fork([0, 1, bad]), lambda: c.reserve([1, bad, 0]),
                     lambda: c.copy([0, bad], [1, 2]), lambda: c.copy([0, 1], [2, bad]), lambda: c.set_state(np.zeros((3, 2)), [0, 0, bad], np.zeros(4)),
                     lambda: c.append(0, None, h(2, 2, 16), h(2, 2, 16), [0, bad]), lambda: c.append(0, None, h(2, 2, 16), h(2, 2, 16), [0, 1], rows=[bad, 0]),
                     lambda: c.attend(0, h(1, 4, 16), rows=[bad]), lambda: tl.beam_reorder(h(1, 3, 8), h(1, 3, 8), [0, bad, 0], 8),
                     lambda: tl.beam_select(h(2, 9), np.zeros(2), 2, 2, finished=[0, bad])):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        tl.beam_select(h(2, 9), np.zeros(2), 2, 2, finished=[0, 256])


def test_attention_refuses():
    lib = tl.load()
    ws = 1 << 25

    def call(c=None, layer=0, q=P, out=P, batch=2, heads=8, scale=1.0, w=P, n=ws):
        return lib.tl_paged_attn_decode_f16(c or cache(), layer, q, out, None, None, batch, heads, scale, 1024, 1024, w, n, None)
    for bad in (dict(layer=2), dict(q=None), dict(out=None), dict(batch=-1), dict(batch=5), dict(heads=9), dict(heads=0), dict(scale=math.inf),
                dict(scale=math.nan), dict(w=None), dict(w=P + 4), dict(c=cache(lengths=None)), dict(batch=65536, c=cache(n_rows=1 << 20))):
        refused(call(**bad))
    refused(call(c=cache(head_dim=264)), status=4)
    for strides in ((-1024, 1024), (1024, -1024)):
        refused(lib.tl_paged_attn_decode_f16(cache(), 0, P, P, None, None, 2, 8, 1.0, *strides, P, ws, None))
    need = C.c_size_t(0)
    for heads, kv, d in ((32, 32, 128), (64, 1, 256), (7, 7, 8), (128, 128, 256)):
        assert lib.tl_paged_attn_workspace(heads, kv, d, C.byref(need)) == 0 and need.value <= 32 << 20
        if need.value:
            refused(call(c=cache(n_kv_heads=kv, head_dim=d), heads=heads, n=need.value - 1))
    for bad in ((8, 3, 128), (0, 1, 128), (8, 8, 257)):
        refused(lib.tl_paged_attn_workspace(*bad, C.byref(need)))


def test_attention_refuses_a_scale_that_overflows():
    """Finite, but not times log2 e: a score of 0 would have become a NaN."""
    for scale in (3e38, -2.4e38):
        refused(tl.load().tl_paged_attn_decode_f16(cache(), 0, P, P, None, None, 2, 8, scale, 1024, 1024, P, 1 << 25, None))


def test_beam_calls_refuse():
    lib = tl.load()
    ws = 1 << 25

    def call(x=P, stride=100, s=P, fin=None, pad=0, batch=2, beams=4, vocab=100, k=8, w=P, n=ws, o=P):
        return lib.tl_beam_select_f16(x, stride, s, fin, pad, batch, beams, vocab, k, o, P, P, w, n, None)
    for bad in (dict(x=None), dict(s=None), dict(o=None), dict(stride=99), dict(fin=P, pad=100), dict(fin=P, pad=-1), dict(batch=-1), dict(beams=0),
                dict(beams=129), dict(k=0), dict(k=129), dict(vocab=0), dict(beams=1, vocab=5, stride=5, k=6), dict(beams=128, vocab=1 << 25, stride=1 << 25),
                dict(w=None), dict(w=P + 2)):
        refused(call(**bad))
    need = C.c_size_t(0)
    assert lib.tl_beam_select_workspace(2, 4, 100, 8, C.byref(need)) == 0
    if need.value:
        refused(call(n=need.value - 1))
    for a in ((None, P, P, 1, 2, 8, 8, 8, 8, 8), (P, None, P, 1, 2, 8, 8, 8, 8, 8), (P, 2 * P, None, 1, 2, 8, 8, 8, 8, 8), (P, P, P, 1, 2, 8, 8, 8, 8, 8),
              (P, 2 * P, P, -1, 2, 8, 8, 8, 8, 8), (P, 2 * P, P, 1, 2, 8, -8, 8, 8, 8), (P, 2 * P, P, 1, 2, 8, 8, 8, -8, 8), (P, 2 * P, P, 1, 2, 9, 8, 8, 16, 16), (P, 2 * P, P, 1, 2, 9, 16, 16, 8, 8)):
        refused(lib.tl_beam_reorder_f16(*a, None))


def test_a_workspace_for_a_batch_serves_the_smaller_ones():
    lib, need = tl.load(), C.c_size_t(0)
    for beams, vocab, k in ((4, 32000, 8), (1, 32000, 1), (8, 128256, 16), (1, 131072, 64), (5, 1001, 10), (16, 50000, 16), (64, 65537, 128), (3, 1 << 22, 4),
                            (128, 32000, 64), (1, 2000000, 128)):
        most = 0
        for batch in [*range(1, 700), 4095, 4096, 4097, 5000]:
            assert lib.tl_beam_select_workspace(batch, beams, vocab, k, C.byref(need)) == 0
            assert need.value >= most, (beams, vocab, k, batch)
            most = need.value
            assert lib.tl_beam_select_f16(P, vocab, P, None, 0, batch, beams, vocab, k, P, P, P, P, need.value - 1, None) == 1


@pytest.mark.skipif(tl.device_count() != 0, reason="host-only behaviour: a GPU is present")
def test_sound_calls_without_a_device_report_that():
    lib = tl.load()
    ws = 1 << 25
    for rc in (lib.tl_paged_fork(cache(), P, None), lib.tl_paged_reserve_f16(cache(), P, P, P, ws, None), lib.tl_paged_copy_f16(cache(), P, P, 0, None),
               lib.tl_paged_compact_f16(cache(), P, P, P, ws, None), lib.tl_paged_attn_decode_f16(cache(), 0, P, P, None, None, 0, 8, 1.0, 0, 0, P, ws, None),
               lib.tl_rotary_f16(P, P, P, P, 1.0, 0, 8, 128, 128, 0, 0, 0, 0, 0, 0, None),
               lib.tl_beam_select_f16(P, 100, P, None, 0, 0, 4, 100, 8, P, P, P, P, ws, None),
               lib.tl_beam_reorder_f16(P, 2 * P, P, 0, 2, 8, 8, 8, 8, 8, None),
               lib.tl_rotary_append_f16(cache(), 0, P, P, P, P, None, P, P, 1.0, 1, 8, 128, 0, 1024, 1024, 1024, None)):
        refused(rc, status=2)


def test_beam_cases_have_no_near_ties():
    """Neighbours of the selection are equal or at least 1e-6 apart, so that their order does not hang on a rounding."""
    for batch, beams, vocab, k in BEAM_SHAPES:
        x, s, fin = beam_case(batch, beams, vocab, 1)
        with np.errstate(all="ignore"):
            for f in (None, fin):
                assert so.beam_select(x, s, beams, k, f, min(2, vocab - 1))[3] > 1e-6, (batch, beams, vocab)


def test_the_page_oracle_keeps_its_books():
    r = np.random.default_rng(3)
    pg = so.Pages(60, 4, 6, 12)
    for step in range(200):
        if step % 3 == 0:
            pg.fork([int(r.integers(-1, 6)) if r.random() < 0.5 else i for i in range(6)])
        elif step % 7 == 0:
            pg.compact()
        else:
            pg.reserve(r.integers(0, 4, 6))
        want = np.zeros(60, np.int32)
        np.add.at(want, pg.table[pg.table >= 0], 1)
        assert np.array_equal(want, pg.refs)
        assert all((pg.table[i] >= 0).sum() == -(-pg.lengths[i] // 4) for i in range(6))
