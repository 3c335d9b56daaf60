"""The operators of a step of several answers to one prompt, as far as they go without a device: what they refuse, the scratch they
ask for, and the frequencies of rotary positions against their formulas."""
import ctypes as C
import math

import numpy as np
import pytest

from nfai_b200 import _lib

# addresses that are never followed: a call without a context ends before any of them is
BASE = 1 << 20


def refusal(name, *args):
    """The text of a refused call. Arguments are checked before the context, so a good call without one says that it is missing."""
    lib = _lib.load()
    assert getattr(lib, name)(None, *args) == _lib.ERR_ARG
    return lib.nfai_last_error(None).decode()


ROPE = dict(x=BASE, x_dtype=_lib.F32, x_stride=0, rows=3, qH=4, kvH=2, d=64, dims=64, layout=0, freqs=BASE, magnitude=1.0,
            positions=BASE, slots=BASE, q=BASE, k=BASE, v=BASE, out_dtype=_lib.F16, cache_rows=10, stream=None)
ATTN = dict(q=BASE, kp=BASE, vp=BASE, prefix=100, ko=BASE, vo=BASE, capacity=50, lens=BASE, dtype=_lib.F16, B=3, qH=8, kvH=2, d=64,
            scale=0.0, out=BASE, scratch=BASE, scratch_bytes=1 << 30, stream=None)
RULES = dict(logits=BASE, rows=2, V=100, history=BASE, history_stride=5, history_len=BASE, repetition=BASE, frequency=BASE,
             presence=BASE, bias_start=BASE, bias_ids=BASE, bias=BASE, n_bias=3, masks=BASE, n_masks=2, mask_rows=BASE,
             out=BASE + (1 << 16), stream=None)


@pytest.mark.parametrize("change,says", [
    ({}, "ctx is null"), ({"rows": 0}, "ctx is null"), ({"slots": None}, "ctx is null"), ({"dims": 0, "freqs": None, "positions": None}, "ctx is null"),
    ({"qH": 0, "q": None}, "ctx is null"), ({"kvH": 0, "k": None, "v": None}, "ctx is null"), ({"x_stride": 8 * 64}, "ctx is null"),
    ({"x": None}, "null"), ({"q": None}, "null"), ({"k": None}, "null"), ({"v": None}, "null"), ({"freqs": None}, "null"), ({"positions": None}, "null"),
    ({"x_dtype": 3}, "type"), ({"out_dtype": -1}, "type"), ({"dims": 66}, "dims"), ({"dims": 63}, "dims"), ({"d": 0}, "1 .. 65536"),
    ({"qH": 0, "kvH": 0}, "1 .. 65536"), ({"layout": 2}, "layout"), ({"x_stride": 511}, "shorter"), ({"rows": 1 << 31}, "too many"),
    ({"qH": 65536, "d": 65536}, "too long"), ({"x": BASE + 2}, "aligned"), ({"q": BASE + 1}, "aligned"), ({"slots": BASE + 2}, "aligned"),
    ({"freqs": BASE + 4}, "aligned")])
def test_rope_refusals(change, says):
    assert says in refusal("nfai_op_rope_rows", *{**ROPE, **change}.values())


@pytest.mark.parametrize("change,says", [
    ({}, "ctx is null"), ({"prefix": 0, "kp": None, "vp": None}, "ctx is null"), ({"capacity": 0, "ko": None, "vo": None}, "ctx is null"),
    ({"B": 0, "q": None, "scratch": None, "scratch_bytes": 0}, "ctx is null"), ({"scale": 0.25}, "ctx is null"),
    ({"q": None}, "null"), ({"kp": None}, "null"), ({"vp": None}, "null"), ({"ko": None}, "null"), ({"vo": None}, "null"), ({"lens": None}, "null"),
    ({"out": None}, "null"), ({"scratch": None}, "null"), ({"dtype": 7}, "type"), ({"qH": 7}, "multiple"), ({"kvH": 0}, "multiple"),
    ({"d": 60}, "head size"), ({"d": 264}, "head size"), ({"d": 0}, "head size"), ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"),
    ({"scale": math.inf}, "scale"), ({"B": 1 << 22}, "too many"), ({"prefix": 1 << 30}, "too many"), ({"q": BASE + 8}, "aligned"),
    ({"scratch": BASE + 128}, "aligned"), ({"scratch_bytes": 16}, "too small")])
def test_attention_refusals(change, says):
    assert says in refusal("nfai_op_attn_shared", *{**ATTN, **change}.values())


@pytest.mark.parametrize("change,says", [
    ({}, "ctx is null"), ({"rows": 0}, "ctx is null"), ({"out": BASE}, "ctx is null"),
    ({k: None for k in ("history", "history_len", "repetition", "frequency", "presence")}, "ctx is null"),
    ({"n_bias": 0, "bias_start": None, "bias_ids": None, "bias": None}, "ctx is null"), ({"n_masks": 0, "masks": None}, "ctx is null"),
    ({"mask_rows": None}, "ctx is null"), ({"mask_rows": None, "n_masks": 1}, "mask of its own"),
    ({"logits": None}, "null"), ({"out": None}, "null"), ({"V": 0}, "vocabulary"), ({"V": (1 << 31) - 1}, "too many"),
    ({"bias_ids": None}, "biases"), ({"bias": None}, "biases"), ({"bias_start": None}, "biases"), ({"masks": None}, "masks"),
    ({"out": BASE + 400}, "overlaps"), ({"out": BASE - 4}, "overlaps"), ({"history": BASE + 1}, "aligned"), ({"logits": BASE + 2}, "aligned")])
def test_rules_refusals(change, says):
    assert says in refusal("nfai_op_logit_rules", *{**RULES, **change}.values())


def test_scratch_sizes():
    need = _lib.load().nfai_op_attn_shared_scratch_bytes
    assert need(_lib.F16, 0, 8, 2, 64, 10, 10) == 0 and need(_lib.F16, 2, 7, 2, 64, 10, 10) == 0 and need(9, 2, 8, 2, 64, 10, 10) == 0
    for dtype in (_lib.F32, _lib.F16, _lib.BF16):
        for B, qH, kvH, d, P, cap in ((1, 32, 8, 64, 1, 0), (64, 32, 8, 128, 32768, 1024), (256, 32, 8, 64, 1500, 2048), (3, 16, 1, 256, 100003, 7)):
            n = need(dtype, B, qH, kvH, d, P, cap)
            assert 0 < n < 1 << 30 and n % 256 == 0


def frequencies(dims, base, scaling, factor=0.0, a=0.0, b=0.0, trained=0):
    out, magnitude = (C.c_double * (dims // 2))(), C.c_float()
    _lib.check(_lib.load().nfai_rope_frequencies(dims, base, scaling, factor, a, b, trained, out, C.byref(magnitude)))
    return np.array(out), magnitude.value


def test_frequencies():
    plain, one = frequencies(64, 500000.0, 0)
    want = 500000.0 ** (-np.arange(32) / 32)
    assert np.allclose(plain, want, rtol=1e-14) and one == 1.0
    linear, one = frequencies(64, 500000.0, 1, 4.0)
    assert np.allclose(linear, want / 4, rtol=1e-14) and one == 1.0
    # bands: by turns within the trained context
    bands, one = frequencies(64, 500000.0, 2, 8.0, 1.0, 4.0, 8192)
    turns = 8192 * want / (2 * math.pi)
    assert np.allclose(bands[turns >= 4], want[turns >= 4], rtol=1e-14) and np.allclose(bands[turns <= 1], want[turns <= 1] / 8, rtol=1e-14)
    between = (turns > 1) & (turns < 4)
    keep = (turns[between] - 1) / 3
    assert between.any() and np.allclose(bands[between], want[between] * (keep + (1 - keep) / 8), rtol=1e-12) and one == 1.0
    # yarn: a ramp over pairs between the one that turns 32 times and the one that turns once
    yarn, mag = frequencies(64, 500000.0, 3, 16.0, 32.0, 1.0, 4096)
    first = [64 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(500000.0)) for t in (32.0, 1.0)]
    lo, hi = math.floor(first[0]), math.ceil(first[1])
    ramp = np.clip((np.arange(32) - lo) / (hi - lo), 0, 1)
    assert 0 < lo < hi < 32 and np.allclose(yarn, want * (1 - ramp) + want / 16 * ramp, rtol=1e-12)
    assert mag == np.float32(0.1 * math.log(16.0) + 1.0)


@pytest.mark.parametrize("args", [(0, 1e4, 0), (63, 1e4, 0), (64, 1.0, 0), (64, math.nan, 0), (64, 1e4, 4), (64, 1e4, 1, 0.5), (64, 1e4, 2, 8.0, 4.0, 1.0, 8192),
                                  (64, 1e4, 2, 8.0, 1.0, 4.0, 0), (64, 1e4, 3, 8.0, 1.0, 32.0, 4096), (64, 1e4, 3, 8.0, 32.0, 0.0, 4096)])
def test_frequencies_refused(args):
    with pytest.raises(_lib.NfaiError) as e:
        frequencies(*args)
    assert e.value.code == _lib.ERR_ARG


def test_scratch_of_the_largest_step_serves_every_smaller_one():
    """A host allocates once, for the largest batch, prompt and capacity that it will run; what a call needs (the text of a refusal says it) is
    never more."""
    need = _lib.load().nfai_op_attn_shared_scratch_bytes

    def used(**sizes):
        text = refusal("nfai_op_attn_shared", *{**ATTN, **sizes, "scratch_bytes": 0}.values())
        assert "too small: 0 < " in text, text
        return int(text.rsplit(" ", 1)[1])
    batches = [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 37, 63, 64, 65, 74, 128, 129, 200, 256, 300, 600]
    prefixes = [0, 1, 129, 300, 700, 1500, 2500, 3130, 4000, 9000, 20000, 32768, 100003]
    capacities = [0, 1, 40, 64, 300, 512, 1024, 5000]
    for dtype in (_lib.F32, _lib.F16):
        for qH, kvH, d in ((32, 8, 64), (32, 8, 128), (16, 16, 64), (16, 1, 128), (6, 2, 32), (20, 1, 256), (48, 2, 80)):
            sizes = dict(dtype=dtype, qH=qH, kvH=kvH, d=d)
            before = {}
            for B in batches:
                for P in prefixes:
                    for cap in capacities:
                        n = need(dtype, B, qH, kvH, d, P, cap)
                        assert n % 256 == 0 and n >= max(before.get((P, cap), 0), used(B=B, prefix=P, capacity=cap, **sizes)), (sizes, B, P, cap)
                        before[P, cap] = n
                for a, b in zip(prefixes, prefixes[1:]):
                    assert all(before[a, cap] <= before[b, cap] for cap in capacities), (sizes, B, a, b)
                for a, b in zip(capacities, capacities[1:]):
                    assert all(before[P, a] <= before[P, b] for P in prefixes), (sizes, B, a, b)


def test_scratch_is_not_far_above_what_a_step_uses():
    """The bound goes by the most parts that any smaller step is cut into: at most so much per CTA of the GPU, or per row of the output."""
    need = _lib.load().nfai_op_attn_shared_scratch_bytes
    for dtype, B, qH, kvH, d, P, cap in ((_lib.F16, 64, 32, 8, 128, 32768, 1024), (_lib.F16, 256, 32, 8, 64, 1500, 2048), (_lib.F16, 2, 32, 8, 64, 300, 128),
                                         (_lib.F32, 9, 8, 2, 32, 1000, 512), (_lib.BF16, 8, 32, 8, 128, 2011, 1024), (_lib.F16, 600, 32, 8, 128, 100003, 5000)):
        # 148 CTAs with 256 rows each of the shared rows' parts, up to 592 with 16 of the own rows', and a row of each for every query head
        assert need(dtype, B, qH, kvH, d, P, cap) <= (148 * 256 + 592 * 16 + 2 * B * qH) * (d + 2) * 4 + 1024


@pytest.mark.parametrize("scale", [3.4e38, 2.4e38])
def test_a_scale_that_leaves_float32_is_refused(scale):
    """The kernels use scale * log2(e)."""
    assert "scale" in refusal("nfai_op_attn_shared", *{**ATTN, "scale": scale}.values())
    assert "ctx is null" in refusal("nfai_op_attn_shared", *{**ATTN, "scale": 2.3e38}.values())
