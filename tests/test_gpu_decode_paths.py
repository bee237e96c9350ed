"""Paths of the decode-step calls that only larger or rarer calls take: tiles of one sequence's rows that are done
again, large chunks of logits in every type, rope with several units a thread."""
import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import FLOATS, assert_within, dev, logits_adjust, narrow, rope, rounding, widen
from hipmem import synchronize
from kurumi_amd import DType
from test_gpu_logits_adjust import call as logits_call, everything
from test_gpu_rope import call as rope_call, untouched
from test_gpu_sdpa_prefix import Case

pytestmark = pytest.mark.gpu


def one_slot(c):
    """Whether the tiles write the output themselves: no partial results."""
    return K.sdpa_prefix_scratch(c.args()) == 0


# One sequence's rows fill tiles of 128 (128 or 256 of them a kv head): batch, q_len, q_heads, kv_heads, d, prefix, own
# keys. The first two are one block of keys, whose tile writes the output itself; the others leave partial results.
JOINT = [(2, 128, 1, 1, 32, 0, 30), (2, 128, 2, 2, 64, 7, 25), (2, 128, 2, 1, 64, 0, 200), (2, 128, 2, 1, 64, 70, 200), (1, 256, 1, 1, 96, 0, 200),
         (1, 256, 1, 1, 96, 300, 70), (2, 64, 4, 1, 128, 70, 200)]
# So many sequences that a tile's keys are one split of several blocks.
JOINT_MANY = [(33, 128, 8, 8, 32, 20, 130)]


def joint_cases():
    return [(dt, *size) for size in JOINT for dt in FLOATS] + [(DType.BF16, *size) for size in JOINT_MANY]


@pytest.mark.parametrize("dt,nb,nt,nh,kv,d,prefix,own", joint_cases())
def test_queries_of_a_full_tile_that_see_nothing_or_infinities(hip, dt, nb, nt, nh, kv, d, prefix, own):
    """Lengths below the number of queries (the first queries see no own key, without a prefix nothing at all), an
    infinity and a NaN in the last own key, garbage behind the lengths."""
    print(f"sdpa_prefix full tiles {dt.name} {nb}x{nt}x{nh}x{kv}x{d} prefix {prefix}", flush=True)
    lens = [own - 9 * (b % 3) if b % 4 else min(own, nt // 2) - b % 7 for b in range(nb)]
    c = Case(dt, nb, nt, nh, kv, d, prefix, own, lens=lens, garbage=np.nan)
    assert one_slot(c) == (nb == 33 or prefix + own <= 32)
    c.v[lens[0] - 1, 0, 5] = narrow(np.array([np.inf], np.float32), dt)[0]
    if nb > 1:
        c.v[c.seq_rows + lens[1] - 1, 0, 6] = narrow(np.array([np.nan], np.float32), dt)[0]
    o, l = c.check(hip)
    unseen = nt - lens[0]
    assert unseen > 0
    if prefix == 0:
        assert (o[0, :unseen] == 0).all() and np.isneginf(l[0, :unseen]).all()
    assert np.isfinite(widen(o[0, :-1], dt)).all() and np.isposinf(widen(o[0, -1, : nh // kv, 5], dt)).all()


@pytest.mark.parametrize("dt,nb,nt,nh,kv,d,prefix,own", joint_cases())
def test_full_tiles_with_pages_that_are_none(hip, dt, nb, nt, nh, kv, d, prefix, own):
    print(f"sdpa_prefix full tiles, absent pages {dt.name} {nb}x{nt}x{nh}x{kv}x{d}", flush=True)
    c = Case(dt, nb, nt, nh, kv, d, prefix, own, lens=[own - 5 * (b % 3) for b in range(nb)], page=4)
    c.pages[0, 1], c.pages[-1, 3] = -1, c.npages
    c.check(hip)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("prefix", [33, 160])
def test_full_tiles_that_go_from_the_prefix_to_the_own_keys(hip, dt, prefix):
    """Several blocks of both in one tile's split."""
    print(f"sdpa_prefix full tiles, both runs {dt.name} prefix {prefix}", flush=True)
    Case(dt, 33, 128, 4, 4, 64, prefix, 168, lens=[168 - b % 50 if b % 5 else 130 for b in range(33)]).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
def test_full_tiles_of_infinite_scores(hip, dt):
    """Every key of the prefix scores -inf with some queries and +inf with others."""
    c = Case(dt, 1, 128, 1, 1, 32, 40, 150, lens=[150])
    inf = narrow(np.array([np.inf], np.float32), dt)[0]
    c.pk[:, 0, 7] = inf
    zero = widen(c.q[..., 7], dt) == 0
    assert not zero.any()
    o, l = c.check(hip)
    up = widen(c.q[0, :, 0, 7], dt) > 0
    assert np.isnan(widen(o[0, up], dt)).all() and np.isposinf(l[0, up]).all() and np.isfinite(widen(o[0, ~up], dt)).all()


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("size", [(3, 1, 8, 2, 128, 500, 60), (70, 1, 4, 4, 64, 300, 40), (2, 128, 2, 1, 96, 100, 200), (5, 2, 4, 2, 32, 90, 20)], ids=str)
def test_the_output_does_not_depend_on_lse(hip, dt, size):
    """lse is of another sum than the output in 16 bits: asked for or not, the output has the same bits."""
    c = Case(dt, *size)
    with_lse, without = c.run(hip)[0], c.run(hip, lse=None)[0]
    np.testing.assert_array_equal(with_lse, without)


# ---- logits_adjust: chunks of 8192 logits, which take a row for every CU at least ----


@pytest.mark.parametrize("dt,out", [(d, o) for d in FLOATS for o in FLOATS])
def test_large_chunks_in_every_type(hip, dt, out):
    """Two chunks of an odd vocabulary a row, more tokens than a work-group counts in one round."""
    rows, vocab, history = 140, 8501, 9001
    print(f"logits_adjust {dt.name} -> {out.name} {rows}x{vocab} history {history}", flush=True)
    rng = np.random.default_rng(3)
    x = narrow(rng.standard_normal((rows, vocab)) * 4, dt)
    kw = everything(rng, rows, vocab, history, 40)
    got = logits_call(hip, x, dt, out, pad=3, lead=1, **kw)
    want, tol = logits_adjust(widen(x, dt), out=out, **kw)
    assert_within(widen(got, out), want, tol, "logits")


@pytest.mark.parametrize("dt", FLOATS)
def test_large_chunks_in_place(hip, dt):
    rng = np.random.default_rng(4)
    rows, vocab = 260, 4001
    x = narrow(rng.standard_normal((rows, vocab)) * 3, dt)
    kw = everything(rng, rows, vocab, 500, 30)
    np.testing.assert_array_equal(logits_call(hip, x, dt, dt, in_place=True, **kw), logits_call(hip, x, dt, dt, **kw))


@pytest.mark.parametrize("vocab,history", [(8192, 8192), (8193, 16385), (16384, 40000)])
def test_large_chunks_of_whole_and_nearly_whole_rounds(hip, vocab, history):
    rng = np.random.default_rng(vocab)
    rows = 256 if vocab == 8192 else 128
    x = narrow(rng.standard_normal((rows, vocab)), DType.BF16)
    kw = everything(rng, rows, vocab, history, 3)
    kw["lens"][:8] = [history, history - 1, 8192, 8191, 0, 1, 8193, history]
    np.minimum(kw["lens"], history, out=kw["lens"])
    got = logits_call(hip, x, DType.BF16, DType.F32, **kw)
    want, tol = logits_adjust(widen(x, DType.BF16), **kw)
    assert_within(got, want, tol, "logits")


# ---- rope: work-groups of two units a thread and more ----


@pytest.mark.parametrize("dt,t,h,d,rot,layout,pad", [
    (DType.BF16, 6000, 4, 128, 128, K.ROPE_HALF, 0),       # several tokens a work-group
    (DType.F16, 2001, 25, 128, 64, K.ROPE_INTERLEAVED, 0),  # more units a token than a work-group takes
    (DType.F32, 1000, 16, 128, 128, K.ROPE_HALF, 0),
    (DType.BF16, 6000, 1, 256, 200, K.ROPE_HALF, 8),       # many tokens of few units
    (DType.BF16, 600, 9, 80, 20, K.ROPE_INTERLEAVED, 1),   # single elements
])
def test_rope_with_several_units_a_thread(hip, dt, t, h, d, rot, layout, pad):
    print(f"rope {dt.name} {t}x{h}x{d} rot {rot} layout {layout} pad {pad}", flush=True)
    rng = np.random.default_rng(t)
    x, v = (narrow(rng.standard_normal((t, h, d), np.float32), dt) for _ in range(2))
    pos, freqs, out_rows = rng.integers(0, 100000, t), K.rope_freqs(rot), t + 5
    rows = rng.permutation(out_rows)[:t].astype(np.int32)
    rows[::97] = -1
    q, k, vc = rope_call(hip, dt, x, pos, freqs, rot, layout=layout, v=v, rows=rows, out_rows=out_rows, pad=pad)
    want, tol = rope(widen(x, dt), pos, list(freqs)[: rot // 2], rot, layout)
    assert_within(widen(q, dt), want, tol + rounding(want, dt), "q")
    kept = rows >= 0
    np.testing.assert_array_equal(k[rows[kept]], q[kept])
    np.testing.assert_array_equal(vc[rows[kept]], v[kept])
    np.testing.assert_array_equal(q[..., rot:], x[..., rot:])
    rest = np.setdiff1d(np.arange(out_rows), rows[kept])
    assert untouched(k[rest]) and untouched(vc[rest])


@pytest.mark.parametrize("dt", [DType.BF16, DType.F32])
def test_rope_in_place_with_several_units_a_thread(hip, dt):
    """q, k and v of a projection's rows; q and k turned where they lie."""
    t, hq, hk, d = 6000, 12, 4, 128
    rng = np.random.default_rng(8)
    row = (hq + 2 * hk) * d
    x = narrow(rng.standard_normal((t, row), np.float32), dt)
    pos, freqs, w = rng.integers(0, 9999, t).astype(np.int32), K.rope_freqs(d), dt.width
    dx, dp = dev(x), dev(pos)
    hip.rope(K.RopeArgs(dtype=dt, layout=K.ROPE_HALF, scale=1.0, tokens=t, q_heads=hq, kv_heads=hk, head_dim=d, rot_dim=d, freqs=freqs, positions=dp.ptr,
                        q=dx.ptr, q_token_stride=row, q_head_stride=d, q_out=dx.ptr, q_out_token_stride=row, q_out_head_stride=d,
                        k=dx.ptr + hq * d * w, k_token_stride=row, k_head_stride=d, k_out=dx.ptr + hq * d * w, k_out_row_stride=row,
                        k_out_head_stride=d, out_rows=t))
    synchronize()
    got, turned = dx.numpy(dt.storage, (t, row)), (hq + hk) * d
    want, tol = rope(widen(x[:, :turned], dt).reshape(t, hq + hk, d), pos, list(freqs), d, K.ROPE_HALF)
    assert_within(widen(got[:, :turned], dt).reshape(want.shape), want, tol + rounding(want, dt), "q, k")
    np.testing.assert_array_equal(got[:, turned:], x[:, turned:])


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("garbage", [0.0, np.nan])
@pytest.mark.parametrize("nb,nt,nh,kv,d,prefix,own,page", [
    (3, 1, 8, 2, 128, 300, 90, 8), (2, 1, 4, 2, 64, 0, 700, 1), (40, 2, 8, 2, 96, 500, 60, 16),  # a few rows of a sequence
    (2, 40, 4, 2, 64, 130, 200, 4),                                                            # tiles of 128 rows
    (2, 128, 2, 1, 32, 0, 200, 4), (1, 128, 2, 2, 128, 70, 333, 1), (33, 128, 8, 8, 32, 20, 130, 8)],  # prefix and own keys in one pass
    ids=lambda x: str(x))
def test_keys_of_absent_pages_are_masked_like_others(hip, dt, garbage, nb, nt, nh, kv, d, prefix, own, page):
    """The same bits as keys that score -inf in their place: the rows go through the same tiles (a row that is done by
    itself, as one whose sums are not finite, has other roundings, and takes a hundred times as long). What the
    cache's first page holds, or an unused one, does not matter."""
    print(f"sdpa_prefix absent pages masked {dt.name} {nb}x{nt}x{nh}x{kv}x{d} prefix {prefix} own {own} pages of {page}", flush=True)
    lens = [own - 7 * (b % 4) for b in range(nb)]
    c = Case(dt, nb, nt, nh, kv, d, prefix, own, lens=lens, page=page)
    c.q[..., 0] = narrow(np.abs(widen(c.q[..., 0], dt)) + 0.1, dt)
    absent = [(0, 0), (0, 3), (nb - 1, 2), (nb - 1, (lens[-1] - 1) // page), (nb // 2, 1)]
    keys, values, pages = c.k.copy(), c.v.copy(), c.pages.copy()
    for b, i in absent:
        at = int(pages[b, i]) * page
        c.k[at : at + page, :, 0] = narrow(np.array([-np.inf], np.float32), dt)[0]
    want = c.run(hip)
    c.k, c.v = keys, values
    for n, (b, i) in enumerate(absent):
        at = int(pages[b, i]) * page
        if garbage != 0:
            c.v[at : at + page] = narrow(np.array([garbage], np.float32), dt)[0]
        c.pages[b, i] = (-1, c.npages, 2 ** 31 - 1, -2 ** 31, c.npages + 5)[n]
    for x, y in zip(c.run(hip), want):
        np.testing.assert_array_equal(x, y)
