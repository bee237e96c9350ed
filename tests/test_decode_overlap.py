"""Buffers of the decode-step calls that share memory: refused where a byte is written that another buffer has, and
taken where their runs only lie between each other's. The checks come before the backend: no GPU is needed."""
import itertools
import random

import pytest

import kurumi_amd as K
from kurumi_amd import DType
from test_decode_args import P, PAGED, accepted, logits_args, rope_args, said, sdpa_args


def bytes_of(start, inner, axes, width):
    """The bytes of contiguous runs of `inner` elements along (n, stride) axes."""
    out = set()
    for steps in itertools.product(*(range(n) for n, _ in axes)):
        at = start + sum(i * s for i, (_, s) in zip(steps, axes)) * width
        out.update(range(at, at + inner * width))
    return out


def test_layouts_drawn_at_random_against_their_bytes():
    """rope with q, k, v and their outputs at random places and strides of one small buffer: refused for sharing exactly
    where a byte of an output is another buffer's (its own input's too, but for the same places)."""
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for trial in range(6000):
        d, tokens, hq, hk = rng.choice([1, 2, 4]), rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 3]), rng.choice([1, 2])
        width, dt = rng.choice([(2, DType.BF16), (4, DType.F32)])
        row = rng.choice([(hq + 2 * hk) * d, (hq + 2 * hk) * d + 3, 40])

        def layout(heads):
            kind = rng.random()
            token, head = (row, d) if kind < 0.5 else (d, tokens * d + rng.randint(0, 2)) if kind < 0.8 else (rng.randint(0, 30), rng.randint(0, 9))
            return P + rng.choice([0, hq * d, (hq + hk) * d, rng.randint(0, 80)]) * width, token, head

        parts = {}
        for name, heads in (("q", hq), ("k", hk), ("v", hk)):
            x = layout(heads)
            parts[name] = (heads, x, x if rng.random() < 0.4 else layout(heads))
        kw = {}
        for name, (heads, x, y) in parts.items():
            step = "token" if name == "q" else "row"
            kw |= {name: x[0], f"{name}_token_stride": x[1], f"{name}_head_stride": x[2], f"{name}_out": y[0], f"{name}_out_{step}_stride": y[1],
                   f"{name}_out_head_stride": y[2]}
        args = rope_args(dtype=int(dt), tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=d, rot_dim=0, freqs=None, positions=None, rows=None,
                         out_rows=tokens, **kw)
        message = said("ku_hip_rope", args)
        if "rows that overlap" in message:
            continue  # an output whose own rows share bytes: another check
        sets = {n: [bytes_of(z[0], d, ((tokens, z[1]), (heads, z[2])), width) for z in (x, y)] for n, (heads, x, y) in parts.items()}
        clash = False
        for n, (heads, x, y) in parts.items():
            same = x[0] == y[0] and (tokens == 1 or x[1] == y[1]) and (heads == 1 or x[2] == y[2])
            clash |= bool(sets[n][0] & sets[n][1]) and not same
            clash |= any(sets[n][1] & sets[m][i] for m in parts if m != n for i in (0, 1))
        assert ("overlap" in message) == clash, (trial, message, parts, tokens, d, width)
        assert clash or message == "ku_hip_rope: null backend handle"
        seen[clash] += 1
    assert min(seen.values()) > 300, seen


@pytest.mark.parametrize("kw,what", [
    (dict(q_out=3 * P), "input of another"), (dict(q_out=6 * P + 64), "input of another"), (dict(k_out=2 * P), "input of another"),
    (dict(v_out=3 * P + 1024), "input of another"), (dict(k_out=7 * P), "two outputs"), (dict(v_out=4 * P), "two outputs"),
    (dict(q_out=P - 512), "positions or rows"), (dict(v_out=8 * P), "positions or rows"),
    (dict(v_out=5 * P + 64, k_out_row_stride=256, v_out_row_stride=256), "two outputs"),
])
def test_rope_refuses_outputs_on_other_buffers(kw, what):
    assert what in said("ku_hip_rope", rope_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(k_out=5 * P, k_out_row_stride=256, v_out=5 * P + 256, v_out_row_stride=256),  # keys and values side by side in a row
    dict(k_out=5 * P, k_out_head_stride=128, k_out_row_stride=256, v_out=5 * P + 128, v_out_head_stride=128, v_out_row_stride=256),  # in a head
    dict(q=2 * P, q_out=2 * P, q_out_token_stride=512, k=2 * P + 512, v=2 * P + 768),  # in place inside a projection's rows
    dict(q=2 * P, q_out=2 * P + 512, q_out_token_stride=512),  # into the gaps of its own rows
    dict(k=3 * P, v=3 * P),  # inputs may share
])
def test_rope_takes_buffers_between_each_other(kw):
    assert accepted("ku_hip_rope", rope_args(**kw)), K.last_error()


@pytest.mark.parametrize("more", [{}, PAGED])
@pytest.mark.parametrize("kw,what", [
    (dict(out=4 * P), "overlaps an input"), (dict(out=5 * P + 128000), "overlaps an input"), (dict(out=7 * P), "overlaps an input"),
    (dict(out=8 * P + 160 * 256 - 16), "overlaps an input"), (dict(out=6 * P), "overlaps an input"), (dict(lse=P + 4), "overlaps an input"),
    (dict(lse=4 * P + 256), "overlaps an input"), (dict(lse=2 * P), "out, lse and scratch overlap"),
    (dict(lse=2 * P + 3 * 2 * 8 * 64 * 2 - 4), "out, lse and scratch overlap"), (dict(scratch=P), "overlaps an input"),
    (dict(scratch=5 * P), "overlaps an input"), (dict(scratch=2 * P), "out, lse and scratch overlap"), (dict(scratch=3 * P), "out, lse and scratch overlap"),
])
def test_sdpa_prefix_refuses_what_is_written_on_other_buffers(kw, what, more):
    if "scratch" in kw:
        kw = {**kw, "scratch_bytes": 1 << 40}
    assert what in said("ku_hip_sdpa_prefix", sdpa_args(**kw, **more))


def test_sdpa_prefix_refuses_an_output_on_the_page_table():
    assert "overlaps an input" in said("ku_hip_sdpa_prefix", sdpa_args(**PAGED, out=9 * P))
    assert accepted("ku_hip_sdpa_prefix", sdpa_args(out=9 * P)), "no pages: nothing lies there"


@pytest.mark.parametrize("kw", [
    dict(q_token_stride=1024, q_batch_stride=2048, out=P + 1024, out_token_stride=1024, out_batch_stride=2048),  # outputs between the queries
    dict(prefix_len=0, out=4 * P), dict(own_max=0, out=7 * P), dict(lse=2 * P + 3 * 2 * 8 * 64 * 2),
    dict(prefix_k=4 * P, prefix_v=4 * P, own_k=4 * P, own_v=4 * P),  # inputs may share
])
def test_sdpa_prefix_takes_buffers_beside_each_other(kw):
    assert accepted("ku_hip_sdpa_prefix", sdpa_args(**kw)), K.last_error()


@pytest.mark.parametrize("kw", [dict(out=3 * P), dict(out=4 * P), dict(out=5 * P), dict(out=6 * P), dict(out=7 * P), dict(out=8 * P), dict(out=9 * P),
                                dict(out=10 * P), dict(out=11 * P), dict(out=12 * P), dict(out=13 * P), dict(out=3 * P + 4 * (3 * 64 + 63))])
def test_logits_adjust_refuses_an_output_on_what_it_reads(kw):
    assert "overlaps an array that is read" in said("ku_hip_logits_adjust", logits_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(dtype=int(DType.F32), logits_stride=2002, out=P + 4 * 1001, out_stride=2002),  # beside each row
    dict(out=12 * P, mask=None, mask_index=None), dict(out=9 * P, bias_ids=None, bias_values=None, bias_offsets=None),
    dict(tokens=14 * P, history=64, tokens_stride=1065, dtype=int(DType.F32), out=14 * P + 256, out_stride=1065, logits=P),  # behind each row's tokens
])
def test_logits_adjust_takes_buffers_between_each_other(kw):
    assert accepted("ku_hip_logits_adjust", logits_args(**kw)), K.last_error()
