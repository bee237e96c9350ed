"""ku_hip_logits_adjust: penalties, biases and grammar masks on logits, against the formula in 64 bits."""
import numpy as np
import pytest

import kurumi_amd as K
from decode_ref import FLOATS, assert_within, csr, dev, logits_adjust, narrow, packed, widen
from hipmem import synchronize
from kurumi_amd import DType

pytestmark = pytest.mark.gpu


def call(hip, x, dt, out, *, tokens=None, lens=None, prompts=None, rep=None, pres=None, freq=None, bias=None, mask=None, mask_index=None,
         pad=0, lead=0, in_place=False, stream=None):
    """The call on a [rows, vocab] array of dt's storage; `pad` elements follow every row, `lead` precede the first."""
    rows, vocab = x.shape

    def strided(a):
        buf = np.full((rows, vocab + pad), 0x33, a.dtype)
        buf[:, :vocab] = a
        return np.concatenate([np.zeros(lead, a.dtype), buf.ravel()])

    keep = [dev(strided(x))]
    dy = keep[0] if in_place else dev(strided(np.zeros((rows, vocab), out.storage)))

    def p(v, dtype=np.int32):
        if v is None:
            return None
        keep.append(dev(np.ascontiguousarray(v, dtype)))
        return keep[-1].ptr

    a = K.LogitsArgs(dtype=dt, out_dtype=out, rows=rows, vocab=vocab, logits=keep[0].ptr + lead * dt.width, logits_stride=vocab + pad,
                     out=dy.ptr + lead * out.width, out_stride=vocab + pad, repetition=p(rep, np.float32), presence=p(pres, np.float32),
                     frequency=p(freq, np.float32))
    if tokens is not None:
        a.tokens, a.tokens_stride, a.history, a.lens, a.prompt_lens = p(tokens), tokens.shape[1], tokens.shape[1], p(lens), p(prompts)
    if bias is not None:
        ids, vals, offsets = csr(bias)
        a.bias_ids, a.bias_values, a.bias_offsets, a.bias_count = p(ids if len(ids) else [0]), p(vals if len(vals) else [0.0], np.float32), p(offsets), len(ids)
    if mask is not None:
        words = packed(mask)
        a.mask, a.mask_rows, a.mask_stride, a.mask_index = p(words, np.uint32), words.shape[0], words.shape[1], p(mask_index)
    hip.logits_adjust(a, stream)
    synchronize()
    whole = dy.numpy(out.storage, (lead + rows * (vocab + pad),))[lead:].reshape(rows, vocab + pad)
    if pad:
        assert (whole[:, vocab:] == np.array(0x33, out.storage)).all(), "what follows a row was written"
    return whole[:, :vocab].copy()


def everything(rng, rows, vocab, history, n_bias):
    tokens = rng.integers(0, vocab, (rows, history)).astype(np.int32)
    tokens[:, ::3] %= max(1, vocab // 7)
    tokens[:, 5::11] = -1  # padding
    if history > 3:
        tokens[:, 3] = vocab  # one past the end
    lens = rng.integers(0, history + 1, rows)
    lens[0] = history
    masks = rng.random((max(1, rows // 2), vocab)) < 0.5
    masks[0] = False  # a grammar state that allows nothing
    return dict(tokens=tokens, lens=lens, prompts=(lens * rng.random(rows)).astype(np.int32), rep=1 + rng.random(rows, np.float32),
                pres=rng.random(rows, np.float32), freq=rng.random(rows, np.float32) * np.float32(0.1),
                bias=[[(int(i), float(np.float32(w))) for i, w in zip(rng.integers(0, vocab, n_bias), rng.standard_normal(n_bias) * 5)]
                      for _ in range(rows)], mask=masks, mask_index=rng.integers(-1, len(masks), rows))


@pytest.mark.parametrize("dt,out", [(d, o) for d in FLOATS for o in FLOATS])
@pytest.mark.parametrize("rows,vocab,history,pad,lead", [(1, 1, 1, 0, 0), (3, 1001, 64, 0, 0), (2, 4096, 200, 8, 0), (5, 8193, 33, 3, 1)])
def test_matches_the_formula(hip, dt, out, rows, vocab, history, pad, lead):
    print(f"logits_adjust {dt.name} -> {out.name} {rows}x{vocab} history {history} pad {pad}", flush=True)
    rng = np.random.default_rng(rows * 7 + vocab)
    x = narrow(rng.standard_normal((rows, vocab)) * 4, dt)
    kw = everything(rng, rows, vocab, history, 9)
    got = call(hip, x, dt, out, pad=pad, lead=lead, **kw)
    want, tol = logits_adjust(widen(x, dt), out=out, **kw)
    assert_within(widen(got, out), want, tol, "logits")


@pytest.mark.parametrize("rows,vocab,history", [(4, 50257, 2000), (1, 131072, 40000), (64, 32000, 100), (300, 2000, 7)])
def test_larger_sizes(hip, rows, vocab, history):
    print(f"logits_adjust {rows}x{vocab} history {history}", flush=True)
    rng = np.random.default_rng(vocab)
    x = narrow(rng.standard_normal((rows, vocab)) * 4, DType.BF16)
    kw = everything(rng, rows, vocab, history, 300)
    got = call(hip, x, DType.BF16, DType.F32, **kw)
    want, tol = logits_adjust(widen(x, DType.BF16), **kw)
    assert_within(got, want, tol, "logits")


@pytest.mark.parametrize("part", ["none", "repetition", "presence", "frequency", "bias", "mask", "all generated", "whole history"])
def test_each_part_by_itself(hip, part):
    rng = np.random.default_rng(6)
    rows, vocab, history = 3, 700, 50
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    every = everything(rng, rows, vocab, history, 20)
    hist = {k: every[k] for k in ("tokens", "lens", "prompts")}
    kw = {"none": {}, "repetition": {**hist, "rep": every["rep"]}, "presence": {**hist, "pres": every["pres"]},
          "frequency": {**hist, "freq": every["freq"]}, "bias": {"bias": every["bias"]}, "mask": {"mask": every["mask"], "mask_index": every["mask_index"]},
          "all generated": {**every, "prompts": None}, "whole history": {**every, "prompts": None, "lens": None}}[part]
    got = call(hip, x, DType.F32, DType.F32, **kw)
    want, tol = logits_adjust(x, **kw)
    assert_within(got, want, tol, part)
    if part == "none":
        np.testing.assert_array_equal(got, x)


def test_a_mask_row_a_row_without_an_index(hip):
    rng = np.random.default_rng(9)
    x, mask = rng.standard_normal((4, 333)).astype(np.float32), rng.random((6, 333)) < 0.5
    got = call(hip, x, DType.F32, DType.F32, mask=mask)
    np.testing.assert_array_equal(got, np.where(mask[:4], x, -np.inf))
    # an index that no mask row has leaves its row unmasked
    got = call(hip, x, DType.F32, DType.F32, mask=mask, mask_index=np.array([5, 6, -7, 0]))
    np.testing.assert_array_equal(got, np.where(np.stack([mask[5], np.ones(333, bool), np.ones(333, bool), mask[0]]), x, -np.inf))


def test_repeated_bias_ids_add_in_list_order(hip):
    """1 + 2^24 - 2^24: a sum whose order shows."""
    x = np.zeros((2, 5000), np.float32)
    lists = [[(4321, 1.0), (4321, 2.0 ** 24), (4321, -(2.0 ** 24))], [(4321, 2.0 ** 24), (4321, -(2.0 ** 24)), (17, 3.0), (4321, 1.0)]]
    for _ in range(3):
        got = call(hip, x, DType.F32, DType.F32, bias=lists)
        assert got[0, 4321] == 0.0 and got[1, 4321] == 1.0 and got[1, 17] == 3.0 and np.count_nonzero(got) == 2


def test_bias_ids_and_lengths_out_of_range_are_taken_into_it(hip):
    x = np.zeros((2, 100), np.float32)
    got = call(hip, x, DType.F32, DType.F32, bias=[[(-1, 9.0), (100, 9.0), (2 ** 31 - 1, 9.0)], [(99, 2.0)]])
    assert got[1, 99] == 2.0 and np.count_nonzero(got) == 1
    tokens = np.array([[1, 2, 3], [4, 5, 6]], np.int32)
    kw = dict(tokens=tokens, lens=np.array([-4, 99]), prompts=np.array([2, -1]), freq=np.ones(2, np.float32))
    got = call(hip, x, DType.F32, DType.F32, **kw)
    want = np.zeros((2, 100))
    want[1, 4:7] = -1
    np.testing.assert_array_equal(got, want)


def test_counts_of_one_token_repeated(hip):
    """A count past 16 bits."""
    n = 70000
    tokens = np.full((1, n), 77, np.int32)
    got = call(hip, np.zeros((1, 200), np.float32), DType.F32, DType.F32, tokens=tokens, freq=np.full(1, 0.5, np.float32), prompts=np.array([3]))
    assert got[0, 77] == -0.5 * (n - 3) and np.count_nonzero(got) == 1


def test_infinities_and_nan(hip):
    x = np.zeros((1, 64), np.float32)
    x[0, :4] = [np.inf, -np.inf, np.nan, np.nan]
    mask = np.ones((1, 64), bool)
    mask[0, 3] = False
    got = call(hip, x, DType.F32, DType.F32, tokens=np.arange(64, dtype=np.int32)[None], rep=np.full(1, 2.0, np.float32), mask=mask)
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2]) and got[0, 3] == -np.inf


@pytest.mark.parametrize("dt", FLOATS)
def test_in_place(hip, dt):
    rng = np.random.default_rng(12)
    x = narrow(rng.standard_normal((6, 4999)) * 3, dt)
    kw = everything(rng, 6, 4999, 77, 12)
    np.testing.assert_array_equal(call(hip, x, dt, dt, in_place=True, **kw), call(hip, x, dt, dt, **kw))


def test_no_rows_is_no_call(hip):
    hip.logits_adjust(K.LogitsArgs(dtype=DType.F32, out_dtype=DType.F32, vocab=10, out_stride=10))
