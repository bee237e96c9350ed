"""ku_hip_sdpa_prefix: attention over a shared prefix and each sequence's own keys, against the definition
in 64 bits, with tolerances from the arithmetic (decode_ref.sdpa_prefix)."""
import ctypes as C

import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import FLOATS, assert_within, dev, narrow, sdpa_prefix, widen
from hipmem import DevBuf, check, hip as hiprt, synchronize
from kurumi_amd import DType, Graph, Tensor

pytestmark = pytest.mark.gpu


class Case:
    """Inputs of one call on the device, and its result in 64 bits."""

    def __init__(self, dt, nb, nt, nh, kv, d, prefix, own_max, lens=None, page=0, seed=0, spread=2.0, pad=0, heads_first=False, garbage=None):
        rng = np.random.default_rng(seed + nb + 10 * nt + 100 * nh + prefix + own_max)
        self.dt, self.dims, self.page, self.scale = dt, (nb, nt, nh, kv, d), page, float(np.float32(1 / np.sqrt(d)))
        self.prefix, self.own_max = prefix, own_max
        per = -(-own_max // page) if page else 0
        self.seq_rows = 0 if page else own_max + 3
        self.npages = nb * per + 2
        rows = self.npages * page if page else nb * self.seq_rows
        self.pages = rng.permutation(self.npages)[: nb * per].reshape(nb, per).astype(np.int32) if page and own_max else None
        self.lens = np.asarray(lens if lens is not None else rng.integers(0, own_max + 1, nb), np.int32) if own_max else None
        q = narrow(rng.standard_normal((nb, nt, nh, d)) * spread, dt)
        self.q, self.pk, self.pv = q, *(narrow(rng.standard_normal((prefix, kv, d)), dt) if prefix else None for _ in range(2))
        self.k, self.v = (narrow(rng.standard_normal((rows, kv, d)), dt) if own_max else None for _ in range(2))
        if garbage is not None and own_max:  # everything that no query may see
            used = np.zeros(rows, bool)
            for b in range(nb):
                j = np.arange(max(0, min(int(self.lens[b]), own_max)))
                used[(self.pages[b][j // page].astype(np.int64) * page + j % page) if page else b * self.seq_rows + j] = True
            bad = narrow(np.array([garbage], np.float32), dt)[0]
            self.k[~used], self.v[~used] = bad, bad
        self.pad, self.heads_first = pad, heads_first

    def strided(self, a):
        """[rows, kv, d] as it lies on the device: heads first or rows first, `pad` elements after each head."""
        rows, kv, d = a.shape
        if self.heads_first:
            a = a.transpose(1, 0, 2)
        buf = np.zeros((*a.shape[:2], d + self.pad), a.dtype)
        buf[..., :d] = a
        s = (d + self.pad, rows * (d + self.pad)) if self.heads_first else (kv * (d + self.pad), d + self.pad)
        return dev(buf), s

    def args(self, scratch=False, **more):
        nb, nt, nh, kv, d = self.dims
        self.held = held = [dev(self.q)]
        self.out, self.lse = DevBuf(self.q.nbytes + 64), DevBuf(4 * nb * nt * nh)
        a = K.SdpaPrefixArgs(dtype=self.dt, scale=self.scale, batch=nb, q_len=nt, q_heads=nh, kv_heads=kv, head_dim=d, q=held[0].ptr,
                             q_batch_stride=nt * nh * d, q_token_stride=nh * d, q_head_stride=d, out=self.out.ptr, out_batch_stride=nt * nh * d,
                             out_token_stride=nh * d, out_head_stride=d, lse=self.lse.ptr, prefix_len=self.prefix, own_max=self.own_max)
        if self.prefix:
            (bk, s), (bv, _) = self.strided(self.pk), self.strided(self.pv)
            a.prefix_k, a.prefix_v, a.prefix_row_stride, a.prefix_head_stride = bk.ptr, bv.ptr, *s
            held += [bk, bv]
        if self.own_max:
            (bk, s), (bv, _), bl = self.strided(self.k), self.strided(self.v), dev(self.lens)
            a.own_k, a.own_v, a.own_row_stride, a.own_head_stride, a.own_lens = bk.ptr, bv.ptr, *s, bl.ptr
            a.own_rows, a.own_seq_rows = len(self.k), self.seq_rows
            held += [bk, bv, bl]
            if self.page:
                held.append(dev(self.pages))
                a.pages, a.page_size, a.pages_per_seq = held[-1].ptr, self.page, self.pages.shape[1]
        for name, value in more.items():
            setattr(a, name, value)
        if scratch:
            n = K.sdpa_prefix_scratch(a)
            held.append(dev(np.full(n, 0xFF, np.uint8)))  # NaN in every float
            a.scratch, a.scratch_bytes = held[-1].ptr, n
        return a

    def results(self):
        nb, nt, nh, kv, d = self.dims
        synchronize()
        return self.out.numpy(self.dt.storage, self.q.shape), self.lse.numpy(np.float32, (nb, nt, nh))

    def run(self, hip, **more):
        hip.sdpa_prefix(self.args(**more))
        return self.results()

    def want(self):
        w = lambda x: None if x is None else widen(x, self.dt)  # noqa: E731
        lens = None if self.lens is None else np.clip(self.lens, 0, self.own_max)
        return sdpa_prefix(w(self.q), w(self.pk), w(self.pv), w(self.k), w(self.v), lens, self.scale, seq_rows=self.seq_rows, pages=self.pages,
                           page=self.page, npages=self.npages, dt=self.dt)

    def check(self, hip, what="", **more):
        o, l = self.run(hip, **more)
        wo, wl, to, tl = self.want()
        assert_within(widen(o, self.dt), wo, to, f"out {what}")
        assert_within(l, wl, tl, f"lse {what}")
        return o, l


SIZES = [  # batch, q_len, q_heads, kv_heads, d, prefix, own_max, page
    (1, 1, 1, 1, 8, 1, 0, 0),
    (1, 1, 1, 1, 64, 0, 1, 0),
    (2, 1, 4, 2, 32, 63, 5, 0),
    (3, 1, 8, 2, 128, 64, 64, 16),
    (3, 2, 8, 8, 64, 65, 33, 8),
    (5, 3, 6, 2, 80, 257, 77, 8),
    (4, 1, 32, 4, 128, 1000, 200, 64),
    (33, 1, 16, 2, 96, 300, 40, 1),
    (2, 40, 4, 1, 64, 130, 90, 0),
    (2, 150, 6, 2, 128, 70, 170, 32),
    (1, 300, 2, 2, 40, 100, 300, 0),
    (7, 17, 3, 3, 128, 0, 50, 16),
    (2, 1, 64, 1, 64, 500, 33, 0),        # many heads on one kv head: a whole tile of one sequence's rows
    (2, 1, 4, 2, 64, 0, 700, 8),          # more pages than a wave has lanes
    (1, 1, 2, 1, 32, 3, 300, 1),          # a page for each key
    (1, 140, 2, 1, 64, 50, 400, 1),
    (64, 1, 8, 8, 64, 100, 130, 16),      # more units than CUs: the longest sequences first
    (61, 1, 8, 8, 32, 64, 40, 0),
    (70, 1, 8, 4, 64, 31, 129, 32),       # more sequences than a wave has lanes
    (20, 1, 16, 4, 128, 5000, 600, 16),   # many splits of either part
    (40, 3, 8, 2, 128, 1500, 20, 0),      # shared tiles over the prefix
    (3, 257, 4, 2, 96, 700, 300, 0),      # joint tiles, split
]


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_matches_the_definition(hip, dt, size):
    nb, nt, nh, kv, d, prefix, own_max, page = size
    print(f"sdpa_prefix {dt.name} {size}", flush=True)
    Case(dt, nb, nt, nh, kv, d, prefix, own_max, page=page).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("size", [(6, 182, 8, 2, 96, 30, 453, 16), (6, 182, 8, 2, 96, 30, 453, 0), (8, 128, 4, 2, 64, 20, 500, 8), (3, 200, 8, 4, 128, 95, 77, 0)],
                         ids=lambda s: "x".join(map(str, s)))
def test_tiles_whose_prefix_is_a_block_or_three(hip, dt, size):
    """A tile goes from the prefix to the own keys after an odd number of blocks: its waves may be a block apart."""
    Case(dt, *size[:7], page=size[7], lens=[size[6]] * size[0]).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("page", [1, 8])
@pytest.mark.parametrize("size", [(32, 33, 16, 8, 32, 5, 1100), (64, 70, 4, 4, 128, 40, 600), (33, 104, 8, 8, 64, 5, 700)], ids=lambda s: "x".join(map(str, s)))
def test_runs_of_more_pages_than_a_wave_has_lanes(hip, dt, size, page):
    Case(dt, *size, page=page, lens=[size[6] - 7 * (b % 5) for b in range(size[0])]).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
def test_lengths_zero_one_and_past_the_range(hip, dt):
    """No own keys, one, fewer than queries; lengths outside [0, own_max] are taken into it."""
    print(f"sdpa_prefix lengths {dt.name}", flush=True)
    for prefix in (0, 70):
        c = Case(dt, 6, 3, 4, 2, 64, prefix, 20, lens=[0, 1, 2, 3, -5, 99])
        o, l = c.check(hip, f"prefix {prefix}")
        if prefix == 0:  # queries that see nothing
            assert (o[0] == 0).all() and np.isneginf(l[0]).all() and (o[4] == 0).all() and (o[1, :2] == 0).all() and np.isneginf(l[1, :2]).all()


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("garbage", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("page", [0, 16])
def test_what_no_query_sees_does_not_matter(hip, dt, garbage, page):
    """NaN, infinities and the largest values behind the lengths and in unused pages."""
    print(f"sdpa_prefix garbage {dt.name} {garbage} {page}", flush=True)
    args = (dt, 4, 2, 4, 2, 64, 100, 90)
    Case(*args, lens=[0, 33, 64, 90], page=page, garbage=garbage).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
def test_values_that_an_earlier_query_does_not_see(hip, dt):
    """The last own key holds an infinity and a NaN: the last query alone sees them."""
    print(f"sdpa_prefix causal infinities {dt.name}", flush=True)
    for nt in (4, 140):
        c = Case(dt, 2, nt, 2, 1, 64, 70, 200, lens=[150, 171])
        last = [149, c.seq_rows + 170]
        c.v[last[0], 0, 5] = narrow(np.array([np.inf], np.float32), dt)[0]
        c.v[last[1], 0, 6] = narrow(np.array([np.nan], np.float32), dt)[0]
        o, _ = c.check(hip, f"q_len {nt}")
        assert np.isfinite(widen(o[:, :-1], dt)).all()
        assert np.isposinf(widen(o[0, -1, :, 5], dt)).all() and np.isnan(widen(o[1, -1, :, 6], dt)).all()


@pytest.mark.parametrize("dt", FLOATS)
def test_infinite_scores(hip, dt):
    """Keys whose scores are -inf for some queries weigh nothing; a query with nothing else, or with a
    score of +inf, has NaN as the definition does."""
    print(f"sdpa_prefix infinite scores {dt.name}", flush=True)
    c = Case(dt, 2, 1, 2, 1, 32, 80, 10, lens=[10, 10])
    c.q[:] = narrow(np.abs(widen(c.q, dt)) + 0.1, dt)
    c.pk[3:40, 0, 7] = narrow(np.array([-np.inf], np.float32), dt)[0]
    c.check(hip, "-inf")
    c.pk[:, 0, 7] = c.pk[3, 0, 7]
    c.k[: c.seq_rows, 0, 7] = c.pk[3, 0, 7]  # sequence 0 has nothing left
    o, l = c.check(hip, "all -inf")
    assert np.isnan(widen(o[0], dt)).all() and np.isneginf(l[0]).all()
    c.pk[5, 0, 7] = narrow(np.array([np.inf], np.float32), dt)[0]
    o, l = c.check(hip, "+inf")
    assert np.isnan(widen(o, dt)).all() and np.isposinf(l).all()


@pytest.mark.parametrize("dt", FLOATS)
def test_large_scores(hip, dt):
    """Scores of hundreds, rising along the keys: the maximum moves all the way."""
    print(f"sdpa_prefix large scores {dt.name}", flush=True)
    c = Case(dt, 2, 1, 4, 2, 64, 500, 100, spread=40.0)
    order = np.argsort(widen(c.pk, dt)[:, 0] @ widen(c.q, dt)[0, 0, 0])
    c.pk, c.pv = c.pk[order], c.pv[order]
    c.check(hip)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("heads_first,pad", [(True, 0), (False, 8), (True, 16)])
def test_strides(hip, dt, heads_first, pad):
    print(f"sdpa_prefix strides {dt.name} {heads_first} {pad}", flush=True)
    Case(dt, 3, 2, 6, 3, 72, 150, 70, heads_first=heads_first, pad=pad).check(hip)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("nb,nt", [(2, 1), (40, 2), (2, 70)])
def test_rows_of_keys_that_repeat_or_overlap(hip, dt, nb, nt):
    """A row stride of nothing, and one of less than a row: the keys are views of each other."""
    print(f"sdpa_prefix overlapping rows {dt.name} {nb} {nt}", flush=True)
    d, prefix = 64, 90
    c = Case(dt, nb, nt, 2, 1, d, prefix, 0)
    for stride in (0, 16):
        flat = narrow(np.random.default_rng(5).standard_normal(prefix * stride + d), dt)
        c.pk = c.pv = np.stack([flat[j * stride : j * stride + d] for j in range(prefix)])[:, None]
        buf = dev(flat)
        hip.sdpa_prefix(c.args(prefix_k=buf.ptr, prefix_v=buf.ptr, prefix_row_stride=stride, prefix_head_stride=0))
        o, l = c.results()
        wo, wl, to, tl = c.want()
        assert_within(widen(o, dt), wo, to, f"out, stride {stride}")
        assert_within(l, wl, tl, f"lse, stride {stride}")


@pytest.mark.parametrize("dt", [DType.F32, DType.BF16])
def test_values_near_the_largest(hip, dt):
    """Sums of values that overflow where their mean does not."""
    for nb, nt in ((2, 1), (40, 2), (1, 130)):
        c = Case(dt, nb, nt, 2, 1, 32, 70, 10, lens=[10] * nb)
        big = narrow(np.array([2.5e38], np.float32), dt)[0]
        c.pv[:, 0, 3], c.v[:, 0, 3] = big, big
        o, _ = c.run(hip)
        want = float(widen(np.array([big]), dt)[0])
        # the probabilities add up to one within the sums' and the output's roundings
        assert (np.abs(widen(o[..., 3], dt) / want - 1) < (100 * 2.0 ** -24 if dt == DType.F32 else 2.0 ** -8)).all()


def test_strides_of_queries_and_outputs(hip):
    """Queries inside the rows of a projection, a head's outputs next to each other."""
    nb, nt, nh, d = 3, 5, 4, 64
    c = Case(DType.BF16, nb, nt, nh, 2, d, 100, 40)
    row = nh * d + 128
    wide = np.zeros((nb, nt, row), np.uint16)
    wide[..., : nh * d] = c.q.reshape(nb, nt, nh * d)
    dq = dev(wide)
    hip.sdpa_prefix(c.args(q=dq.ptr, q_batch_stride=nt * row, q_token_stride=row, out_batch_stride=nh * nt * d, out_token_stride=d,
                           out_head_stride=nt * d))
    o, l = c.results()
    wo, wl, to, tl = c.want()
    assert_within(widen(o.reshape(nb, nh, nt, d).transpose(0, 2, 1, 3), DType.BF16), wo, to, "out")
    assert_within(l, wl, tl, "lse")


@pytest.mark.parametrize("dt", FLOATS)
def test_pages_that_are_none_of_the_caches(hip, dt):
    """The keys of a page whose index is negative or past the cache count as not there; indices behind
    the length are never looked at."""
    print(f"sdpa_prefix bad pages {dt.name}", flush=True)
    c = Case(dt, 3, 1, 4, 2, 64, 50, 64, lens=[64, 40, 5], page=8)
    c.pages[0, 2], c.pages[1, 0] = -1, c.npages
    c.pages[1, 5:] = 2 ** 31 - 1
    c.pages[2, 1:] = -2 ** 31
    c.check(hip)
    c = Case(dt, 2, 1, 4, 2, 64, 0, 16, lens=[16, 16], page=8)
    c.pages[0, :] = -1  # no key at all
    o, l = c.check(hip, "no page")
    assert (o[0] == 0).all() and np.isneginf(l[0]).all()


@pytest.mark.parametrize("dt", FLOATS)
def test_one_page_in_several_sequences(hip, dt):
    c = Case(dt, 4, 1, 4, 1, 64, 30, 48, lens=[48, 48, 20, 33], page=16)
    c.pages[1:] = c.pages[0]
    c.check(hip)


def test_joins_by_lse(hip):
    """Two calls over halves of the keys join into one over all of them."""
    c = Case(DType.F32, 3, 1, 4, 2, 64, 200, 0)
    o, l = c.run(hip)
    halves = []
    for part in (slice(0, 90), slice(90, 200)):
        p = Case(DType.F32, 3, 1, 4, 2, 64, 200, 0)
        p.pk, p.pv, p.prefix = c.pk[part], c.pv[part], part.stop - part.start
        halves.append(p.run(hip))
    ls = np.stack([h[1] for h in halves]).astype(np.float64)
    w = np.exp(ls - ls.max(0))
    joined = (np.stack([h[0] for h in halves]) * w[..., None]).sum(0) / w.sum(0)[..., None]
    np.testing.assert_allclose(joined, o, atol=4e-6, rtol=0)
    np.testing.assert_allclose(ls.max(0) + np.log(w.sum(0)), l, atol=4e-6, rtol=0)


def test_matches_the_graph_attention(hip):
    """Without own keys and with one head a kv head it is ku_sdpa without a mask."""
    s, h, d = 96, 4, 64
    c = Case(DType.F32, 1, s, h, h, d, s, 0, spread=1.0)
    g = Graph()
    q, k, v = (g.input([1, h, s, d], DType.F32) for _ in range(3))
    feeds = {n: Tensor.from_numpy(np.ascontiguousarray(x.reshape(s, h, d).transpose(1, 0, 2)[None])) for n, x in ((q, c.q), (k, c.pk), (v, c.pv))}
    graph = hip.eval_with(g, g.sdpa(q, k, v, False), feeds).numpy()[0].transpose(1, 0, 2)
    o, _ = c.check(hip)
    _, _, to, _ = c.want()
    assert_within(graph, o[0], 2 * to[0], "graph")


@pytest.mark.parametrize("dt", FLOATS)
def test_a_scratch_of_the_callers_and_repeated_calls_agree(hip, dt):
    print(f"sdpa_prefix scratch {dt.name}", flush=True)
    for size in ((5, 1, 8, 2, 64, 900, 70), (2, 60, 4, 2, 64, 300, 100)):
        c = Case(dt, *size)
        first = c.run(hip)
        for scratch in (True, True, False):
            for x, y in zip(first, c.run(hip, scratch=scratch)):
                np.testing.assert_array_equal(x, y)


def test_a_batch_without_sequences_and_one_head_of_outputs(hip):
    c = Case(DType.F32, 1, 1, 2, 1, 32, 10, 0)
    hip.sdpa_prefix(c.args(batch=0, q=None, out=None))
    c.check(hip)
    o1, _ = c.run(hip)
    o2, _ = c.run(hip, lse=None)
    np.testing.assert_array_equal(o1, o2)


@pytest.mark.parametrize("dt", FLOATS)
def test_no_keys_at_all(hip, dt):
    c = Case(dt, 5, 2, 6, 3, 72, 0, 0)
    assert K.sdpa_prefix_scratch(c.args()) == 0
    o, lse = c.run(hip)
    assert (o == 0).all() and (lse == -np.inf).all()


def test_own_cache_past_2_to_32_elements(hip):
    """A cache of 8 GiB a tensor: the last page and the last sequence lie past 2^32 elements."""
    kv, d, page = 8, 128, 16
    npages = (1 << 32) // (kv * d * page) + 2
    rows = npages * page
    rng = np.random.default_rng(1)
    bufs = [DevBuf(rows * kv * d * 2) for _ in range(2)]
    c = Case(DType.F16, 1, 1, kv, kv, d, 0, 20, lens=[20], page=page)
    table = np.array([[npages - 1, npages - 2]], np.int32)
    for buf, x in zip(bufs, (c.k, c.v)):
        for p in table[0]:
            part = np.ascontiguousarray(x[p % c.npages * page : (p % c.npages + 1) * page])
            check(hiprt().hipMemcpy(buf.ptr + int(p) * page * kv * d * 2, part.ctypes.data, part.nbytes, 1), "hipMemcpy H2D")
    dp = dev(table)
    hip.sdpa_prefix(c.args(own_k=bufs[0].ptr, own_v=bufs[1].ptr, own_rows=rows, pages=dp.ptr))
    c.pages = table % c.npages
    o, l = c.results()
    wo, wl, to, tl = c.want()
    assert_within(widen(o, DType.F16), wo, to, "out")
    assert_within(l, wl, tl, "lse")
