"""ku_hip_rope: rotary positions and the store into a cache, against the formula in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import FLOATS, assert_within, dev, narrow, rope, rounding, widen
from hipmem import DevBuf, check, hip as hiprt, synchronize
from kurumi_amd import DType, Graph, Tensor

pytestmark = pytest.mark.gpu
FILL = 0x5A  # bytes of a cache before the call


def call(hip, dt, x, positions, freqs, rot, *, layout=K.ROPE_HALF, scale=1.0, inverse=False, v=None, rows=None, out_rows=None,
         pad=0, lead=0, heads_first=False, stream=None):
    """q = k = x through one call: q_out whole, and the k and v caches. `pad` elements follow every input
    head and `lead` come before the first, so that strides and alignment vary; `heads_first` stores the
    cache as [heads, rows, d]."""
    t, h, d = x.shape
    out_rows = t if out_rows is None else out_rows

    def strided(a):
        buf = np.zeros((t, h, d + pad), a.dtype)
        buf[..., :d] = a
        return dev(np.concatenate([np.zeros(lead, a.dtype), buf.ravel()]))

    w = dt.width
    dx, dv, dp, dr = strided(x), strided(v) if v is not None else None, dev(positions.astype(np.int32)), dev(rows)
    dq = dev(np.full((t, h, d), FILL, np.uint8).repeat(w, -1))
    dk, dvo = (dev(np.full(out_rows * h * d * w, FILL, np.uint8)) for _ in range(2))
    rs, hs = (d, out_rows * d) if heads_first else (h * d, d)
    a = K.RopeArgs(dtype=dt, layout=layout, inverse=int(inverse), scale=scale, tokens=t, q_heads=h, kv_heads=h, head_dim=d, rot_dim=rot,
                   freqs=freqs, positions=dp.ptr, q=dx.ptr + lead * w, q_token_stride=h * (d + pad), q_head_stride=d + pad,
                   q_out=dq.ptr, q_out_token_stride=h * d, q_out_head_stride=d, k=dx.ptr + lead * w, k_token_stride=h * (d + pad),
                   k_head_stride=d + pad, k_out=dk.ptr, k_out_row_stride=rs, k_out_head_stride=hs, rows=dr.ptr if dr else None, out_rows=out_rows)
    if v is not None:
        a.v, a.v_token_stride, a.v_head_stride = dv.ptr + lead * w, h * (d + pad), d + pad
        a.v_out, a.v_out_row_stride, a.v_out_head_stride = dvo.ptr, rs, hs
    hip.rope(a, stream)
    synchronize()
    shape = (h, out_rows, d) if heads_first else (out_rows, h, d)
    kc, vc = (b.numpy(dt.storage, shape) for b in (dk, dvo))
    if heads_first:
        kc, vc = kc.transpose(1, 0, 2), vc.transpose(1, 0, 2)
    return dq.numpy(dt.storage, (t, h, d)), kc, vc


def untouched(bits):
    return (np.ascontiguousarray(bits).view(np.uint8) == FILL).all()


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("t,h,d,rot,layout,pad,lead", [
    (1, 1, 2, 2, K.ROPE_HALF, 0, 0),
    (1, 8, 128, 128, K.ROPE_HALF, 0, 0),
    (1, 8, 128, 128, K.ROPE_INTERLEAVED, 0, 0),
    (7, 3, 64, 32, K.ROPE_HALF, 8, 0),      # part of a head, whole 16-byte pieces
    (7, 3, 64, 32, K.ROPE_INTERLEAVED, 8, 8),
    (33, 5, 80, 20, K.ROPE_INTERLEAVED, 0, 0),  # pairs that are no whole piece
    (33, 5, 80, 20, K.ROPE_HALF, 0, 0),
    (5, 2, 72, 48, K.ROPE_HALF, 0, 0),      # an odd number of copied pieces
    (9, 4, 96, 96, K.ROPE_HALF, 1, 3),      # unaligned rows and pointer
    (9, 4, 33, 22, K.ROPE_INTERLEAVED, 0, 1),  # an odd head
    (300, 2, 256, 256, K.ROPE_HALF, 0, 0),
    (260, 6, 64, 64, K.ROPE_INTERLEAVED, 0, 0),
    (4, 7, 16, 0, K.ROPE_HALF, 0, 0),       # nothing turned: a copy into the cache
])
def test_rope_matches_the_formula(hip, dt, t, h, d, rot, layout, pad, lead):
    print(f"rope {dt.name} {t}x{h}x{d} rot {rot} layout {layout} pad {pad} lead {lead}", flush=True)
    rng = np.random.default_rng(t * 1000 + d)
    x, v = (narrow(rng.standard_normal((t, h, d)), dt) for _ in range(2))
    pos = rng.integers(-5, 100000, t)
    freqs = K.rope_freqs(rot)
    out_rows = t + 11
    rows = rng.permutation(out_rows)[:t].astype(np.int32)
    if t > 4:
        rows[1], rows[3] = -1, out_rows  # neither is stored
    q, k, vc = call(hip, dt, x, pos, freqs, rot, layout=layout, v=v, rows=rows, out_rows=out_rows, pad=pad, lead=lead, heads_first=t % 2 == 0)
    want, tol = rope(widen(x, dt), pos, list(freqs)[: rot // 2], rot, layout)
    tol = tol + rounding(want, dt)
    assert_within(widen(q, dt), want, tol, "q")
    kept = (rows >= 0) & (rows < out_rows)
    np.testing.assert_array_equal(k[rows[kept]], q[kept])  # one input: one result, wherever it goes
    np.testing.assert_array_equal(vc[rows[kept]], v[kept])
    np.testing.assert_array_equal(q[..., rot:], x[..., rot:])
    rest = np.setdiff1d(np.arange(out_rows), rows[kept])
    assert untouched(k[rest]) and untouched(vc[rest])


@pytest.mark.parametrize("layout", [K.ROPE_HALF, K.ROPE_INTERLEAVED])
@pytest.mark.parametrize("scaling", [K.ROPE_LINEAR, K.ROPE_BASE, K.ROPE_BY_PARTS])
def test_rope_scaled_for_long_contexts_at_far_positions(hip, layout, scaling):
    print(f"rope far positions, layout {layout} scaling {scaling}", flush=True)
    t, h, d = 40, 3, 64
    rng = np.random.default_rng(11)
    x = rng.standard_normal((t, h, d)).astype(np.float32)
    pos = np.concatenate([rng.integers(0, 1 << 20, t - 4), [0, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]])
    freqs = K.rope_freqs(d, 500000.0, scaling, factor=8.0, trained_len=4096.0, low=1.0, high=4.0)
    q, _, _ = call(hip, DType.F32, x, pos, freqs, d, layout=layout, scale=1.25)
    want, tol = rope(x, pos, list(freqs), d, layout, scale=1.25)
    assert_within(q, want, tol, "q")


@pytest.mark.parametrize("dt", FLOATS)
def test_inverse_is_the_gradient(hip, dt):
    """<R x, y> = <x, R' y> for the transpose R', and differences of the forward call agree with it."""
    t, h, d, rot = 6, 2, 64, 48
    print(f"rope inverse {dt.name}", flush=True)
    rng = np.random.default_rng(5)
    pos, freqs = rng.integers(0, 5000, t), K.rope_freqs(rot)
    g = narrow(rng.standard_normal((t, h, d)), dt)
    got, _, _ = call(hip, dt, g, pos, freqs, rot, scale=0.5, inverse=True)
    want, tol = rope(widen(g, dt), pos, list(freqs), rot, K.ROPE_HALF, scale=0.5, inverse=True)
    assert_within(widen(got, dt), want, tol + rounding(want, dt), "gradient")
    if dt == DType.F32:
        x, e = rng.standard_normal((t, h, d)).astype(np.float32), np.zeros((t, h, d), np.float32)
        e[3, 1, 7] = 1.0  # the map is linear: its column is a difference of any size
        up, _, _ = call(hip, dt, x + e, pos, freqs, rot, scale=0.5)
        down, _, _ = call(hip, dt, x - e, pos, freqs, rot, scale=0.5)
        column = (up.astype(np.float64) - down) / 2
        # features past rot keep their values: a column of the identity, untouched by scale
        assert abs((column * g).sum() - want[3, 1, 7]) < 64 * 2.0 ** -20


def test_matches_the_graph_builder(hip):
    """ku_rope's half layout, whole head, base 10000, positions 0.. as a graph."""
    s, h, d = 50, 4, 64
    x = np.random.default_rng(2).standard_normal((h, s, d)).astype(np.float32)
    g = Graph()
    n = g.input([h, s, d], DType.F32)
    graph = hip.eval_with(g, g.rope(n), {n: Tensor.from_numpy(x)}).numpy()
    q, _, _ = call(hip, DType.F32, np.ascontiguousarray(x.transpose(1, 0, 2)), np.arange(s), K.rope_freqs(d), d)
    # the graph's angles are f32 products of positions below 50: off by 50 * 2^-23 of the features' sizes
    np.testing.assert_allclose(q.transpose(1, 0, 2), graph, rtol=0, atol=8 * 50 * 2.0 ** -23 * np.abs(x).max())


@pytest.mark.parametrize("dt", [DType.F32, DType.BF16])
@pytest.mark.parametrize("layout,rot,d", [(K.ROPE_HALF, 64, 64), (K.ROPE_INTERLEAVED, 20, 33)])
def test_in_place_inside_a_projection(hip, dt, layout, rot, d):
    """q and k turned where they lie in the rows [q | k | v] of one projection; v and the gap stay."""
    print(f"rope in place {dt.name} {layout}", flush=True)
    t, hq, hk, gap = 70, 6, 2, 5
    row = (hq + 2 * hk) * d + gap
    rng = np.random.default_rng(8)
    x = narrow(rng.standard_normal((t, row)), dt)
    pos = rng.integers(0, 9999, t).astype(np.int32)
    dx, dp, freqs, w = dev(x), dev(pos), K.rope_freqs(rot), dt.width
    a = K.RopeArgs(dtype=dt, layout=layout, scale=1.0, tokens=t, q_heads=hq, kv_heads=hk, head_dim=d, rot_dim=rot, freqs=freqs, positions=dp.ptr,
                   q=dx.ptr, q_token_stride=row, q_head_stride=d, q_out=dx.ptr, q_out_token_stride=row, q_out_head_stride=d,
                   k=dx.ptr + hq * d * w, k_token_stride=row, k_head_stride=d, k_out=dx.ptr + hq * d * w, k_out_row_stride=row,
                   k_out_head_stride=d, out_rows=t)
    hip.rope(a)
    got = dx.numpy(dt.storage, (t, row))
    turned = (hq + hk) * d
    want, tol = rope(widen(x[:, :turned], dt).reshape(t, hq + hk, d), pos, list(freqs), rot, layout)
    assert_within(widen(got[:, :turned], dt).reshape(want.shape), want, tol + rounding(want, dt), "q, k")
    np.testing.assert_array_equal(got[:, turned:], x[:, turned:])


def test_infinities_and_nan_stay_in_their_pair(hip):
    t, h, d = 3, 2, 32
    x = np.random.default_rng(1).standard_normal((t, h, d)).astype(np.float32)
    x[1, 0, 3], x[2, 1, 20] = np.inf, np.nan
    q, _, _ = call(hip, DType.F32, x, np.array([0, 5, 9]), K.rope_freqs(16), 16)
    bad = ~np.isfinite(q)
    want = np.zeros_like(bad)
    want[1, 0, [3, 11]] = want[2, 1, 20] = True
    np.testing.assert_array_equal(bad, want)


def test_cache_past_2_to_32_elements(hip):
    """A row whose offset needs more than 32 bits."""
    d, h = 128, 8
    out_rows = (1 << 32) // (d * h) + 3  # f16: 8 GiB
    cache = DevBuf(out_rows * h * d * 2)
    x = narrow(np.random.default_rng(3).standard_normal((2, h, d)), DType.F16)
    rows = np.array([out_rows - 1, 0], np.int32)
    dx, dr, dp = dev(x), dev(rows), dev(np.zeros(2, np.int32))
    a = K.RopeArgs(dtype=DType.F16, scale=1.0, tokens=2, kv_heads=h, head_dim=d, rot_dim=d, freqs=K.rope_freqs(d), positions=dp.ptr, k=dx.ptr,
                   k_token_stride=h * d, k_head_stride=d, k_out=cache.ptr, k_out_row_stride=h * d, k_out_head_stride=d, rows=dr.ptr,
                   out_rows=out_rows)
    hip.rope(a)
    synchronize()
    for t, r in enumerate(rows):
        got = np.empty((h, d), np.uint16)
        check(hiprt().hipMemcpy(got.ctypes.data, cache.ptr + int(r) * h * d * 2, got.nbytes, 2), "hipMemcpy D2H")
        np.testing.assert_array_equal(got, x[t])  # position 0 turns by nothing


def test_on_a_stream_of_the_caller(hip):
    rng = np.random.default_rng(4)
    x, pos = rng.standard_normal((20, 4, 64)).astype(np.float32), rng.integers(0, 99, 20)
    s = C.c_void_p()
    check(hiprt().hipStreamCreate(C.byref(s)), "hipStreamCreate")
    a, _, _ = call(hip, DType.F32, x, pos, K.rope_freqs(64), 64, stream=s.value)
    b, _, _ = call(hip, DType.F32, x, pos, K.rope_freqs(64), 64)
    check(hiprt().hipStreamDestroy(s), "hipStreamDestroy")
    np.testing.assert_array_equal(a, b)
