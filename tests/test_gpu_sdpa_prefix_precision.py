"""How many bits ku_hip_sdpa_prefix keeps of its probabilities: keys whose probabilities round the same way,
very many keys far below the largest, and heads of up to 32 features."""
import numpy as np
import pytest

from decode_ref import narrow, widen
from kurumi_amd import DType
from test_gpu_sdpa_prefix import Case

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {DType.BF16: 2.0 ** -8, DType.F16: 2.0 ** -11}  # of a value of 16 bits, relative to it
STEP_BITS = {DType.BF16: 7, DType.F16: 10}             # a value in [1, 2) lies 2^-bits from its neighbours

# batch, q_len, q_heads, kv_heads: a few rows, whose waves deal the keys; rows of many sequences in tiles of 128;
# rows of one sequence that fill such tiles
ROWS = [(1, 1, 1, 1), (70, 1, 1, 1), (1, 128, 1, 1)]


def two_levels(dt, rows, d, n, own, p, big):
    """Keys of score 0 where `big`, of score ln p elsewhere (scale makes it so: q and k are 1 and -1 in one feature)."""
    nb, nt, nh, kv = rows
    c = Case(dt, nb, nt, nh, kv, d, 0, n if own else 0, lens=[n] * nb if own else None)
    c.prefix, c.scale = 0 if own else n, float(np.float32(-np.log(p)))
    c.q[:], one = 0, narrow(np.array([1.0, -1.0]), dt)
    c.q[..., 0] = one[0]
    keys = np.zeros((n, 1, d), c.q.dtype)
    keys[~big, 0, 0] = one[1]
    return c, keys, np.where(big, 0.0, 1.0)[:, None, None].repeat(d, 2)


def place(c, keys, values, own):
    if own:
        for b in range(c.dims[0]):
            at = b * c.seq_rows
            c.k[at : at + len(keys)], c.v[at : at + len(keys)] = keys, narrow(values, c.dt)
    else:
        c.pk, c.pv = keys, narrow(values, c.dt)


@pytest.mark.parametrize("dt", [DType.BF16, DType.F16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("own", [False, True], ids=["shared", "own"])
@pytest.mark.parametrize("rows", ROWS, ids=lambda r: "x".join(map(str, r)))
def test_probabilities_that_round_the_same_way_leave_no_bias(hip, dt, d, own, rows):
    """All values 1, all keys but one in 32 at one probability, whose rounding is off by nearly half a step: a mean of
    ones is one. Numerator and denominator add the same roundings in other orders, n of them at most, each
    off by n u of the sum: 2 n u = 2^-15.4 together, under half of the step of 2^-8 or 2^-11 below 1, so the output is 1
    (heads of 32 hold a probability to 2^-16 and more and add it unrounded: the same).
    (A quotient of rounded and unrounded sums would be off by the rounding, nearly 2^-8 or 2^-11.)
    The causal mask of several queries leaves the earlier ones fewer keys, of both kinds.
    lse is of the unrounded sum: a probability is off by 8 u (its exponent's rounding, exp2), the sum by n u, its
    logarithm's value by 4 u (|lse| + 1)."""
    print(f"sdpa_prefix bias {dt.name} d {d} own {own} {rows}", flush=True)
    n = 192
    p = 0.5 * (1 + HALF[dt] * 0.97)
    big = np.arange(n) % 32 == 0
    c, keys, values = two_levels(dt, rows, d, n, own, p, big)
    place(c, keys, np.ones_like(values), own)
    o, lse = c.run(hip)
    np.testing.assert_array_equal(widen(o, dt), 1.0)
    ps = np.where(big, 1.0, np.exp(-np.float64(c.scale)))
    nt = rows[1]
    want = np.array([np.log(ps[: n - (nt - 1 - t) if own else n].sum()) for t in range(nt)])[None, :, None]
    assert (np.abs(lse - want) <= (n + 12) * U + 4 * U * (np.abs(want) + 1)).all()


@pytest.mark.parametrize("dt", [DType.BF16, DType.F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nb,nt", [(1, 1), (70, 1), (2, 128)])
def test_a_mean_of_ones_over_thousands_of_far_keys(hip, dt, d, nb, nt):
    """4096 keys at 2^-21.05 of the largest, all values 1, on 256 kv heads of one set of keys (so that one unit meets them
    all): the far keys are 2^-9.05 of the sum, numerator and denominator alike. Their roundings differ by 2 n u = 2^-11
    of the sums at most, the output by its own half step: either sum without the far keys would be off by more."""
    n, p = 4097, 2.0 ** -21.05
    c, keys, values = two_levels(dt, (nb, nt, 256, 256), d, n, False, p, np.arange(n) == 0)
    c.pk, c.pv = keys, narrow(np.ones_like(values), dt)
    o, lse = c.run(hip, prefix_head_stride=0)
    assert (np.abs(widen(o, dt) - 1) <= 2 * n * U + HALF[dt]).all()
    want = np.log(1 + (n - 1) * np.exp(-np.float64(c.scale)))
    # a far key is off by 8 u and its exponent's rounding, 4 u a power of two; few of them weigh much
    assert (np.abs(lse - want) <= (n + 100) * U).all()


@pytest.mark.parametrize("dt", [DType.BF16, DType.F16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("own", [False, True], ids=["shared", "own"])
@pytest.mark.parametrize("rows", ROWS, ids=lambda r: "x".join(map(str, r)))
@pytest.mark.parametrize("power", [-18.3, -22.5, -25.5])
def test_keys_far_below_the_largest_still_count(hip, dt, d, own, rows, power):
    """One key in 32 holds zeros and stands 2^18 to 2^25 above the others, which hold 30000: what they add up to is the
    whole output. A probability is rounded to half a step, in f16 to 2^-32 of the largest at least (values
    are held 2^7 times as large, with 2^-25 as the least half step), and is off by 4 u of its exponent before that;
    the sums over n keys by n u each, the output by half a step."""
    print(f"sdpa_prefix far below {dt.name} d {d} own {own} {rows} 2^{power}", flush=True)
    n = 192
    big = np.arange(n) % 32 == 0
    c, keys, values = two_levels(dt, rows, d, n, own, 2.0 ** power, big)
    value = widen(narrow(np.array([30000.0]), dt), dt)[0]
    place(c, keys, values * value, own)
    o, _ = c.run(hip)
    p, nt = np.exp(-np.float64(c.scale)), rows[1]
    for t in range(nt):
        left = n - (nt - 1 - t) if own else n
        small, large = int((~big[:left]).sum()), int(big[:left].sum())
        want = small * p * value / (large + small * p)
        tol = want * (HALF[dt] + 8 * U + 4 * U * abs(power) + 2 * n * U + HALF[dt])
        if dt == DType.F16:
            tol += small * 2.0 ** -32 * value / large + 2.0 ** -25
        got = widen(o[:, t], dt)
        assert (np.abs(got - want) <= tol).all(), (t, got.ravel()[:3], want, tol)


@pytest.mark.parametrize("dt", [DType.BF16, DType.F16])
@pytest.mark.parametrize("d", [8, 32])
@pytest.mark.parametrize("own", [False, True], ids=["shared", "own"])
@pytest.mark.parametrize("rows", ROWS, ids=lambda r: "x".join(map(str, r)))
def test_heads_of_32_hold_a_probability_as_two_values(hip, dt, d, own, rows):
    """Two keys of which one holds zeros, a query's probabilities different from the next one's: the output is one
    probability times a value. Two values of 16 bits hold a probability to the square of half a step (f16: to
    2^-32 at least), which is a hundredth of the output's own half step or less."""
    print(f"sdpa_prefix two values {dt.name} d {d} own {own} {rows}", flush=True)
    rng = np.random.default_rng(d)
    nb, nt, nh, kv = rows
    for trial in range(4):
        c = Case(dt, nb, nt, nh, kv, d, 0 if own else 2, 2 + nt - 1 if own else 0, lens=[2 + nt - 1] * nb if own else None)
        c.scale = 1.0
        c.q[:] = 0
        c.q[..., 0] = narrow(rng.uniform(0.1, 2.0, c.q.shape[:3]), dt)
        minus = narrow(np.array([-1.0]), dt)[0]
        # own keys: the first two are seen by all queries; the later ones score -inf-like, -1000 times a query
        keys, values = np.zeros((2 + nt - 1 if own else 2, kv, d), c.q.dtype), np.zeros((2 + nt - 1 if own else 2, kv, d))
        keys[1, :, 0] = minus
        keys[2:, :, 0] = narrow(np.array([-30000.0]), dt)[0]
        values[1] = rng.uniform(1, 2, (kv, d))
        place(c, keys, values, own)
        o, _ = c.run(hip)
        p = np.exp(-widen(c.q[..., 0], dt))[..., None]
        v = widen(narrow(values[1, 0], dt), dt)
        want = p * v / (1 + p)
        step = 2.0 ** (np.floor(np.log2(want)) - STEP_BITS[dt])
        extra = want * (HALF[dt] ** 2 + 40 * U) + (2.0 ** -32 * 2 if dt == DType.F16 else 0)
        got = widen(o, dt)
        assert (np.abs(got - want) <= step / 2 + extra).all(), np.abs(got - want).max()
