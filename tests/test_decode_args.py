"""Argument checks of the decode-step calls (rope, sdpa_prefix, logits_adjust). They come before the
backend, so every refusal is tested without a GPU: with the check passed, a null backend is what is named."""
import ctypes as C
import math
import re
from pathlib import Path

import numpy as np
import pytest

import kurumi_amd as K
from kurumi_amd import DType

ROOT = Path(__file__).resolve().parent.parent
P = 1 << 20  # a well-aligned address; nothing is read there, since no backend is given


def said(call: str, args) -> str:
    assert getattr(K.lib(), call)(None, args, None) == -1
    return K.last_error()


def accepted(call: str, args) -> bool:
    return said(call, args) == f"{call}: null backend handle"


@pytest.mark.parametrize("cls,c_name", [(K.RopeArgs, "KuHipRopeArgs"), (K.SdpaPrefixArgs, "KuHipSdpaPrefixArgs"),
                                        (K.LogitsArgs, "KuHipLogitsArgs")])
def test_python_blocks_mirror_the_header(cls, c_name):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "kurumi_hip.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % c_name, text, re.S).group(1)
    widths, names = {"uint32_t": 4, "float": 4, "size_t": 8, "int64_t": 8}, []
    for line in body.split(";"):
        m = re.match(r"\s*(?:const )?(\w+) (.*)", line.strip(), re.S)
        if m:
            names += [(n.strip().lstrip("* "), 8 if "*" in n else widths[m.group(1)]) for n in m.group(2).split(",")]
    assert [(n, getattr(cls, n).size) for n, _ in cls._fields_] == names


def test_a_block_takes_only_its_own_fields():
    with pytest.raises(TypeError, match="no field 'token'"):
        K.RopeArgs(token=3)


# ---- rope_freqs ----


def test_rope_freqs_follow_the_formulas():
    base = np.array([10000.0 ** (-2 * i / 64) for i in range(32)])
    np.testing.assert_allclose(list(K.rope_freqs(64)), base, rtol=1e-15)
    np.testing.assert_allclose(list(K.rope_freqs(64, scaling=K.ROPE_LINEAR, factor=4.0)), base / 4, rtol=1e-15)
    ntk = list(K.rope_freqs(64, scaling=K.ROPE_BASE, factor=4.0))
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], base[-1] / 4, rel_tol=1e-13)  # the ends: kept, and divided
    parts = np.array(list(K.rope_freqs(64, scaling=K.ROPE_BY_PARTS, factor=8.0, trained_len=4096, low=1, high=4)))
    turns = 4096 * base / (2 * math.pi)
    np.testing.assert_allclose(parts[turns >= 4], base[turns >= 4], rtol=1e-15)
    np.testing.assert_allclose(parts[turns <= 1], base[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    g = (turns[mid] - 1) / 3
    assert mid.any()
    np.testing.assert_allclose(parts[mid], base[mid] * g + base[mid] / 8 * (1 - g), rtol=1e-14)
    assert list(K.rope_freqs(2, scaling=K.ROPE_BASE, factor=4.0)) == [1.0]  # one pair: nothing to spread


@pytest.mark.parametrize("kw,what", [
    (dict(rot_dim=7), "even"), (dict(rot_dim=8, base=0.0), "base"), (dict(rot_dim=8, base=math.inf), "base"),
    (dict(rot_dim=8, scaling=9), "unknown scaling"), (dict(rot_dim=8, scaling=1, factor=0.0), "factor"),
    (dict(rot_dim=8, scaling=3, factor=2.0, trained_len=0.0), "trained_len"),
    (dict(rot_dim=8, scaling=3, factor=2.0, trained_len=64.0, low=4.0, high=4.0), "low must be less"),
])
def test_rope_freqs_refusals(kw, what):
    with pytest.raises(K.KuError, match=what):
        K.rope_freqs(**kw)


# ---- rope ----


def rope_args(**kw):
    a = K.RopeArgs(dtype=DType.BF16, layout=K.ROPE_HALF, scale=1.0, tokens=5, q_heads=4, kv_heads=2, head_dim=64, rot_dim=32,
                   freqs=K.rope_freqs(32), positions=P, q=2 * P, q_token_stride=512, q_head_stride=64, q_out=4 * P,
                   q_out_token_stride=256, q_out_head_stride=64, k=3 * P, k_token_stride=512, k_head_stride=64, k_out=5 * P,
                   k_out_row_stride=128, k_out_head_stride=64, v=6 * P, v_token_stride=512, v_head_stride=64, v_out=7 * P,
                   v_out_row_stride=128, v_out_head_stride=64, rows=8 * P, out_rows=100)
    for name, value in kw.items():
        assert hasattr(K.RopeArgs, name), name
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    {}, dict(tokens=0), dict(tokens=0, q=None, k=None, v=None, positions=None, rows=None), dict(tokens=0, q=None, q_out=None, k=None, v=None, rows=None),
    dict(rot_dim=0, freqs=None, positions=None), dict(q=None, q_out=None), dict(k=None, k_out=None, v=None, v_out=None),
    dict(v=None, v_out=None), dict(rows=None), dict(q_out=2 * P, q_out_token_stride=512),  # in place
    dict(k_out=3 * P, k_out_row_stride=512, rows=None), dict(q_token_stride=0),  # a broadcast input
    dict(q_out_token_stride=64, q_out_head_stride=320),  # heads outermost
    dict(q=2 * P + 2, q_token_stride=513),  # unaligned
])
def test_rope_accepts(kw):
    assert accepted("ku_hip_rope", rope_args(**kw)), K.last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(size=8), "sizeof"), (dict(dtype=int(DType.I32)), "dtype"), (dict(dtype=int(DType.F64)), "dtype"), (dict(layout=2), "layout"),
    (dict(head_dim=0), "head_dim"), (dict(rot_dim=31), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(head_dim=512, rot_dim=258), "rot_dim"),
    (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(tokens=1 << 31), "tokens"), (dict(q_heads=1 << 15), "heads"),
    (dict(q=None), "without its input"), (dict(k_out=None), "without its output"), (dict(q=None, q_out=None, k=None, k_out=None, v=None, v_out=None), "nothing"),
    (dict(q_heads=0), "q_heads"), (dict(kv_heads=0), "kv_heads"), (dict(freqs=None), "freqs"), (dict(positions=None), "positions"),
    (dict(positions=P + 2), "aligned"), (dict(rows=P + 1), "aligned"), (dict(q=2 * P + 1), "aligned"),
    (dict(rows=None, out_rows=4), "out_rows"), (dict(out_rows=1 << 31), "cache rows"), (dict(q_token_stride=-512), "negative"),
    (dict(q_out_head_stride=63), "overlap"), (dict(q_out_token_stride=255), "overlap"), (dict(k_out_row_stride=0), "overlap"),
    (dict(q_out=2 * P + 128), "overlaps its input"), (dict(q_out=2 * P), "overlaps its input"),
    (dict(k_out=3 * P, k_out_row_stride=512), "no rows"), (dict(q_token_stride=1 << 62), "address space"),
    (dict(tokens=(1 << 31) - 1, head_dim=2, rot_dim=0, q_heads=1, q_head_stride=0, q_token_stride=2, q_out_head_stride=0, q_out_token_stride=2,
          k=None, k_out=None, v=None, v_out=None, q_out=1 << 40), "one launch"),
])
def test_rope_refusals(kw, what):
    assert re.search(what, said("ku_hip_rope", rope_args(**kw)))


def test_rope_refuses_frequencies_that_are_not_finite():
    f = K.rope_freqs(32)
    f[3] = math.inf
    assert "freqs must be finite" in said("ku_hip_rope", rope_args(freqs=f))


# ---- sdpa_prefix ----


def sdpa_args(**kw):
    a = K.SdpaPrefixArgs(dtype=DType.BF16, scale=0.125, batch=3, q_len=2, q_heads=8, kv_heads=2, head_dim=64, q=P, q_batch_stride=1024,
                         q_token_stride=512, q_head_stride=64, out=2 * P, out_batch_stride=1024, out_token_stride=512, out_head_stride=64,
                         lse=3 * P, prefix_len=1000, prefix_k=4 * P, prefix_v=5 * P, prefix_row_stride=128, prefix_head_stride=64,
                         own_max=50, own_lens=6 * P, own_k=7 * P, own_v=8 * P, own_row_stride=128, own_head_stride=64, own_rows=160,
                         own_seq_rows=50)
    for name, value in kw.items():
        assert hasattr(K.SdpaPrefixArgs, name), name
        setattr(a, name, value)
    return a


PAGED = dict(pages=9 * P, page_size=16, pages_per_seq=4)


@pytest.mark.parametrize("kw", [
    {}, dict(batch=0), dict(batch=0, q=None, out=None, own_k=None, own_v=None, own_lens=None, pages=None, own_rows=0), dict(lse=None), dict(prefix_len=0, prefix_k=None, prefix_v=None), dict(own_max=0, own_lens=None, own_k=None, own_v=None),
    PAGED, dict(batch=1, own_seq_rows=0), dict(head_dim=8), dict(q_heads=2), dict(q_token_stride=0), dict(prefix_row_stride=0),
    dict(dtype=int(DType.F32), head_dim=4),
])
def test_sdpa_prefix_accepts(kw):
    assert accepted("ku_hip_sdpa_prefix", sdpa_args(**kw)), K.last_error()
    assert K.sdpa_prefix_scratch(sdpa_args(**kw)) < 1 << 40


@pytest.mark.parametrize("kw,what", [
    (dict(size=8), "sizeof"), (dict(dtype=int(DType.F8E4M3)), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(q_len=0), "positive"), (dict(kv_heads=0), "positive"), (dict(kv_heads=3), "multiple of kv_heads"), (dict(batch=1 << 31), "queries"),
    (dict(prefix_len=1 << 31), "keys"), (dict(own_max=1 << 31), "keys"), (dict(q_len=1 << 28, batch=1), "queries"),
    (dict(q=None), "null device pointer"), (dict(out=None), "null device pointer"), (dict(prefix_v=None), "null device pointer"),
    (dict(own_k=None), "null device pointer"), (dict(own_lens=None), "own_lens"), (dict(q=P + 8), "16-byte aligned"),
    (dict(lse=3 * P + 2), "4-byte aligned"), (dict(scratch=P + 4), "scratch must be 16-byte"), (dict(q_head_stride=60), "16 bytes"),
    (dict(prefix_row_stride=68), "16 bytes"), (dict(own_head_stride=4), "16 bytes"), (dict(out_head_stride=56), "overlap"),
    (dict(out_token_stride=0), "overlap"), (dict(out=P), "out overlaps q"), (dict(out=P + 512), "out overlaps q"),
    (dict(own_seq_rows=49), "own_seq_rows"), (dict(own_rows=149), "own_rows does not hold"), (dict(q_batch_stride=-1024), "negative"),
    ({**PAGED, "page_size": 12}, "power of two"), ({**PAGED, "page_size": 0}, "power of two"), ({**PAGED, "pages_per_seq": 3}, "pages_per_seq"),
    (dict(batch=1 << 20, q_len=1, q_heads=64, kv_heads=64, head_dim=8, q_batch_stride=512, q_head_stride=8, out_batch_stride=512,
          out_head_stride=8, out=1 << 42, own_max=1, own_rows=1 << 20, own_seq_rows=1), "one launch"),
    ({**PAGED, "own_rows": 15}, "no page"), ({**PAGED, "pages": 9 * P + 2}, "4-byte aligned"),
])
def test_sdpa_prefix_refusals(kw, what):
    assert re.search(what, said("ku_hip_sdpa_prefix", sdpa_args(**kw)))
    with pytest.raises(K.KuError, match=what):
        K.sdpa_prefix_scratch(sdpa_args(**kw))


def test_sdpa_prefix_refuses_a_scratch_that_is_too_small():
    need = K.sdpa_prefix_scratch(sdpa_args())
    assert accepted("ku_hip_sdpa_prefix", sdpa_args(scratch=16 * P, scratch_bytes=need))
    if need:
        assert "scratch_bytes" in said("ku_hip_sdpa_prefix", sdpa_args(scratch=16 * P, scratch_bytes=need - 1))


# ---- logits_adjust ----


def logits_args(**kw):
    a = K.LogitsArgs(dtype=DType.F16, out_dtype=DType.F32, rows=4, vocab=1001, logits=P, logits_stride=1001, out=2 * P, out_stride=1001,
                     history=64, tokens=3 * P, tokens_stride=64, lens=4 * P, prompt_lens=5 * P, repetition=6 * P, presence=7 * P,
                     frequency=8 * P, bias_ids=9 * P, bias_values=10 * P, bias_offsets=11 * P, bias_count=12, mask=12 * P, mask_rows=2,
                     mask_stride=32, mask_index=13 * P)
    for name, value in kw.items():
        assert hasattr(K.LogitsArgs, name), name
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    {}, dict(rows=0), dict(tokens=None, lens=None, prompt_lens=None), dict(mask=None, mask_index=None), dict(mask_index=None, mask_rows=4),
    dict(bias_ids=None, bias_values=None, bias_offsets=None), dict(tokens_stride=0), dict(logits_stride=0), dict(history=0),
    dict(out=P, out_dtype=int(DType.F16)), dict(repetition=None, presence=None, frequency=None), dict(lens=None, prompt_lens=None),
    # what holds no elements may have no address
    dict(bias_count=0, bias_ids=None, bias_values=None), dict(history=0, tokens=None), dict(mask_rows=0, mask=None),
    dict(rows=0, logits=None, out=None, tokens=None, lens=None, prompt_lens=None, repetition=None),
])
def test_logits_adjust_accepts(kw):
    assert accepted("ku_hip_logits_adjust", logits_args(**kw)), K.last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(size=8), "sizeof"), (dict(dtype=int(DType.I64)), "dtype"), (dict(out_dtype=int(DType.F64)), "out_dtype"), (dict(vocab=0), "vocab"),
    (dict(vocab=1 << 31), "vocab"), (dict(logits=None), "null logits"), (dict(out=None), "null logits or out"), (dict(logits=P + 1), "aligned"),
    (dict(out_stride=1000), "overlap"), (dict(logits_stride=-1), "negative"), (dict(out=P), "without being the same"),
    (dict(out=P + 16, out_dtype=int(DType.F16)), "without being the same"), (dict(tokens=None), "without tokens"), (dict(history=1 << 31), "history"),
    (dict(bias_ids=None), "go together"), (dict(bias_offsets=None), "go together"), (dict(bias_count=1 << 31), "bias_count"),
    (dict(mask=None), "mask_index without mask"), (dict(mask_index=None), "fewer mask rows"), (dict(mask_stride=-1), "negative"),
    (dict(tokens=3 * P + 2), "aligned"), (dict(mask=12 * P + 1), "aligned"), (dict(rows=1 << 40), "too many|address space"),
    (dict(rows=1 << 24), "too many rows"),
])
def test_logits_adjust_refusals(kw, what):
    assert re.search(what, said("ku_hip_logits_adjust", logits_args(**kw)))


@pytest.mark.parametrize("call", ["ku_hip_rope", "ku_hip_sdpa_prefix", "ku_hip_logits_adjust"])
def test_null_arguments(call):
    assert said(call, None) == f"{call}: null arguments"


def test_null_arguments_of_the_scratch_size():
    assert K.lib().ku_hip_sdpa_prefix_scratch(None) == C.c_size_t(-1).value
    assert "null arguments" in K.last_error()
