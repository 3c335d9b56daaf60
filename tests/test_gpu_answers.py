"""The operators of a step of several answers to one prompt (rotary rows, attention over shared rows, rules on logits) against their
formulas in 64 bits, one by one and as a step.

Tolerances follow from the arithmetic. A rounding to type t is off by at most half a step, eps(t) / 2 of the value; u below is that of
float32, 2^-24."""
import ctypes as C
import math
import threading

import numpy as np
import pytest

from nfai_b200 import _lib

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": (torch.float32, _lib.F32), "f16": (torch.float16, _lib.F16), "bf16": (torch.bfloat16, _lib.BF16)}


def at(t):
    return t.data_ptr() if t is not None else None


def run(ctx, name, *args, stream=None):
    """On the context's stream where `stream` is None (the call waits), else there."""
    if stream is None:
        torch.cuda.synchronize()
    _lib.check(getattr(_lib.load(), name)(ctx.handle, *args, stream), ctx.handle)


def half_step(kind):
    return torch.finfo(kind).eps / 2


# ---- rotary rows ---------------------------------------------------------------------------------------------------------
def rope_args(rows, qH, kvH, d, dims, layout, x, out, cache, seed, stride=None, far=1000000, slots="mixed", offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xt, ot = TYPES[x][0], TYPES[out][0]
    width = (qH + 2 * kvH) * d
    stride = stride or width
    flat = torch.randn(rows * stride + offset, generator=g, device="cuda").to(xt)
    s = dict(x=flat[offset:], xt=xt, ot=ot, rows=rows, qH=qH, kvH=kvH, d=d, dims=dims, layout=layout, stride=stride, cache=cache)
    s["freqs"] = torch.tensor([500000.0 ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=torch.float64, device="cuda")
    s["magnitude"] = float(np.float32(1.1))
    s["positions"] = torch.randint(0, far, (rows,), generator=g, device="cuda", dtype=torch.int32)
    s["slots"] = None if slots is None else torch.randperm(cache, generator=g, device="cuda")[:rows].to(torch.int32)
    if slots == "mixed" and rows > 2:  # rows that go nowhere
        s["slots"][0], s["slots"][1] = -1, cache
    s["q"] = torch.full((rows, qH * d), 7.0, device="cuda", dtype=ot)
    s["k"] = torch.randn(cache, kvH * d, generator=g, device="cuda").to(ot)
    s["v"] = torch.randn(cache, kvH * d, generator=g, device="cuda").to(ot)
    return s


def rope_call(ctx, s, x_code, out_code, stream=None):
    run(ctx, "nfai_op_rope_rows", at(s["x"]), x_code, s["stride"], s["rows"], s["qH"], s["kvH"], s["d"], s["dims"], s["layout"],
        at(s["freqs"]), s["magnitude"], at(s["positions"]), at(s["slots"]), at(s["q"]), at(s["k"]), at(s["v"]), out_code, s["cache"], stream=stream)


def rope_check(s, before_k, before_v):
    """The float32 turn: the angle in half turns is rounded to float32 (2^-25 at most, pi 2^-25 of angle = 1.6 u), sine and cosine are
    good to 2 u, the magnitude, two products and their sum add 4 u: below 8 u (|a| + |b|) magnitude. Then the rounding to the output's type."""
    rows, qH, kvH, d, dims = s["rows"], s["qH"], s["kvH"], s["d"], s["dims"]
    x = torch.as_strided(s["x"], (rows, (qH + 2 * kvH) * d), (s["stride"], 1)).double().view(rows, qH + 2 * kvH, d)
    half, qk = dims // 2, qH + kvH
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if s["layout"] == 0 else (i, i + half)
    angle = s["positions"].double()[:, None, None] * s["freqs"]
    c, n = angle.cos() * s["magnitude"], angle.sin() * s["magnitude"]
    want, slack = x.clone(), torch.zeros_like(x)
    a, b = x[:, :qk][..., first], x[:, :qk][..., second]
    want[:, :qk, first], want[:, :qk, second] = a * c - b * n, a * n + b * c
    slack[:, :qk, first] = slack[:, :qk, second] = (a.abs() + b.abs()) * s["magnitude"] * 8 * U
    slack += half_step(s["ot"]) * (want.abs() + slack) + torch.finfo(s["ot"]).tiny
    slots = torch.arange(rows, device="cuda") if s["slots"] is None else s["slots"].long()
    goes = (slots >= 0) & (slots < s["cache"])
    k, v = before_k.double(), before_v.double()
    k_slack, v_slack = torch.zeros_like(k), torch.zeros_like(v)
    for cache, room, heads in ((k, k_slack, slice(qH, qk)), (v, v_slack, slice(qk, None))):
        cache[slots[goes]] = want[goes][:, heads].flatten(1)
        room[slots[goes]] = slack[goes][:, heads].flatten(1)
    for name, got, exp, room in (("q", s["q"], want[:, :qH].flatten(1), slack[:, :qH].flatten(1)), ("k", s["k"], k, k_slack), ("v", s["v"], v, v_slack)):
        off = (got.double() - exp).abs() - room
        assert off.numel() == 0 or off.max().item() <= 0, (name, off.max().item())


ROPE_SIZES = [  # rows, qH, kvH, d, dims
    (1, 32, 8, 64, 64), (5, 8, 2, 32, 32), (37, 32, 8, 128, 64), (300, 6, 2, 128, 128), (3, 1, 1, 64, 16), (4, 4, 2, 80, 48), (7, 3, 1, 6, 4),
    (9, 5, 1, 33, 10), (2, 2, 0, 64, 64), (4, 0, 2, 64, 64), (3, 2, 1, 64, 0), (2, 64, 64, 256, 256)]


@pytest.mark.parametrize("rows,qH,kvH,d,dims", ROPE_SIZES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("x,out", [("f32", "f16"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "bf16")])
def test_rope_rows(cuda_ctx, rows, qH, kvH, d, dims, layout, x, out):
    s = rope_args(rows, qH, kvH, d, dims, layout, x, out, rows + 11, rows * 131 + d)
    k, v = s["k"].clone(), s["v"].clone()
    rope_call(cuda_ctx, s, TYPES[x][1], TYPES[out][1])
    rope_check(s, k, v)


@pytest.mark.parametrize("stride,offset", [(48 * 64 + 8, 0), (48 * 64 + 3, 0), (48 * 64, 1), (48 * 64 + 24, 8)])
@pytest.mark.parametrize("layout", [0, 1])
def test_rope_rows_strides_and_alignment(cuda_ctx, stride, offset, layout):
    s = rope_args(21, 32, 8, 64, 64, layout, "f16", "f16", 40, 5, stride=stride, offset=offset)
    k, v = s["k"].clone(), s["v"].clone()
    rope_call(cuda_ctx, s, _lib.F16, _lib.F16)
    rope_check(s, k, v)


def test_rope_rows_without_slots_and_past_the_cache(cuda_ctx):
    s = rope_args(9, 4, 2, 64, 64, 0, "f32", "f16", 6, 3, slots=None)  # rows 6, 7, 8 have no place
    k, v = s["k"].clone(), s["v"].clone()
    rope_call(cuda_ctx, s, _lib.F32, _lib.F16)
    rope_check(s, k, v)


def test_rope_rows_cache_beyond_32_bits(cuda_ctx):
    """Cache rows whose offset in elements does not fit into 32 bits."""
    rows, kvH, d, cache = 4, 8, 128, (1 << 32) // 1024 + 5
    s = rope_args(rows, 0, kvH, d, d, 1, "f16", "f16", 8, 1)
    s["k"], s["v"] = (torch.empty(cache, kvH * d, device="cuda", dtype=torch.float16) for _ in range(2))
    s["cache"] = cache
    s["slots"] = torch.tensor([cache - 1, 0, cache - 4, (1 << 31) // 1024], dtype=torch.int32, device="cuda")
    for n in ("k", "v"):
        for r in s["slots"].tolist() + [1, cache - 2]:
            s[n][r] = 3.0
    rope_call(cuda_ctx, s, _lib.F16, _lib.F16)
    few = dict(s, cache=cache)
    pick = s["slots"].long()
    small = dict(few, k=s["k"][pick].clone(), v=s["v"][pick].clone(), slots=torch.arange(rows, device="cuda", dtype=torch.int32), cache=rows)
    rope_check(small, small["k"] * 0, small["v"] * 0)
    assert (s["k"][1] == 3).all() and (s["v"][cache - 2] == 3).all()


# ---- attention over shared rows --------------------------------------------------------------------------------------------
def attn_args(kind, B, qH, kvH, d, P, cap, lens, seed, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(TYPES[kind][0])
    s = dict(kind=kind, B=B, qH=qH, kvH=kvH, d=d, P=P, cap=cap, q=(spread * normal(B, qH * d).float()).to(TYPES[kind][0]), kp=normal(P, kvH * d),
             vp=normal(P, kvH * d), ko=normal(B, cap, kvH * d), vo=normal(B, cap, kvH * d))
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):  # what lies behind a sequence's rows is no number
        s["ko"][b, max(0, n):] = math.nan
        s["vo"][b, max(0, n):] = math.inf
    s["out"] = torch.full((B, qH * d), 5.0, device="cuda", dtype=TYPES[kind][0])
    need = _lib.load().nfai_op_attn_shared_scratch_bytes(TYPES[kind][1], B, qH, kvH, d, P, cap)
    s["scratch"] = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    return s


def attn_call(ctx, s, scale=0.0, stream=None):
    run(ctx, "nfai_op_attn_shared", at(s["q"]), at(s["kp"]), at(s["vp"]), s["P"], at(s["ko"]), at(s["vo"]), s["cap"], at(s["lens"]),
        TYPES[s["kind"]][1], s["B"], s["qH"], s["kvH"], s["d"], scale, at(s["out"]), at(s["scratch"]), s["scratch"].numel() - 256, stream=stream)
    if stream is None:
        assert (s["scratch"][-256:] == 0xff).all()


def attn_check(s, scale=0.0, out=None):
    """Scores are float32 sums of d products: off by at most 2 d u sum |q k| scale (twice, for sums that cut instead of rounding), and
    by 4 u of their size in the exponent; an exponential is good to 4 u more. A weight is then rounded to the caches' type (not float32), sums over n keys
    lose at most n u, and the result is rounded once. So |error| <= (2 (score errors) + 4 u + half + n u) sum w |v| + half |out|."""
    out = s["out"] if out is None else out
    B, qH, kvH, d, P = s["B"], s["qH"], s["kvH"], s["d"], s["P"]
    G, scale = qH // kvH, scale or d ** -0.5
    kind = TYPES[s["kind"]][0]
    half = half_step(kind) if kind != torch.float32 else 0.0
    kp, vp = s["kp"].double().view(P, kvH, d), s["vp"].double().view(P, kvH, d)
    worst = 0.0
    for b, n in enumerate(s["lens"].tolist()):
        got = out[b].double().view(kvH, G, d)
        if n < 0:
            assert (got == 5).all()
            continue
        n = min(n, s["cap"])
        k = torch.cat([kp, s["ko"][b, :n].double().view(n, kvH, d)]).permute(1, 2, 0)
        v = torch.cat([vp, s["vo"][b, :n].double().view(n, kvH, d)]).permute(1, 0, 2)
        if P + n == 0:
            assert (got == 0).all()
            continue
        q = s["q"][b].double().view(kvH, G, d)
        scores = (q @ k) * scale
        w = torch.softmax(scores, -1)
        want = w @ v
        off = 2 * d * U * scale * (q.abs() @ k.abs()).amax(-1, keepdim=True) + 4 * U * scores.abs().amax(-1, keepdim=True) * 1.4427
        room = (2 * off + 8 * U + half + (P + n) * U) * (w @ v.abs()) + half_step(kind) * want.abs() + torch.finfo(kind).tiny
        rest = ((got - want).abs() / room).max().item()
        worst = max(worst, rest)
        assert rest <= 1, (b, n, rest)
    return worst


ATTN_SIZES = [  # B, qH, kvH, d, P, cap, lens
    (1, 8, 2, 64, 1, 4, [0]), (1, 8, 2, 64, 0, 4, [1]), (2, 8, 2, 64, 0, 4, [0, 3]), (3, 32, 8, 64, 300, 128, [0, 128, 77]),
    (2, 32, 8, 128, 129, 70, [64, 65]), (5, 6, 2, 128, 511, 40, [-1, 40, 0, 1, 39]), (4, 16, 16, 64, 127, 33, [5, -1, 33, 12]),
    (3, 16, 1, 128, 128, 30, [30, 2, 9]), (3, 5, 1, 64, 700, 300, [300, 256, 255]), (7, 8, 2, 32, 1000, 50, [3] * 7),
    (2, 24, 8, 128, 2011, 1100, [1100, 1]), (9, 32, 8, 64, 2500, 64, [64, 0, -1, 5, 6, 7, 8, 9, 10]), (2, 3, 3, 8, 50, 20, [20, 0]),
    (2, 6, 2, 40, 90, 100, [100, 3]), (3, 10, 1, 80, 77, 10, [9, 0, 4]), (2, 4, 1, 256, 200, 90, [90, 0]), (1, 20, 1, 96, 70, 5, [5]),
    (40, 32, 8, 128, 1111, 20, [1 + b % 20 for b in range(40)]), (70, 32, 8, 64, 1300, 9, [b % 10 - 1 for b in range(70)]),
    (33, 16, 1, 128, 640, 100, [3 * b for b in range(33)]), (2, 32, 8, 64, 9000, 16, [16, 2]), (1, 8, 8, 128, 5000, 3000, [2900]),
    (20, 10, 5, 80, 600, 10, [b % 11 for b in range(20)]), (18, 4, 2, 256, 531, 4, [b % 5 - 1 for b in range(18)]), (17, 3, 3, 8, 777, 3, [b % 4 for b in range(17)]),
    (70, 8, 8, 40, 513, 2, [b % 3 for b in range(70)]), (13, 20, 4, 64, 1000, 9, [b % 10 for b in range(13)]), (6, 48, 8, 128, 900, 5, [5, 4, 3, -1, 1, 0]),
    (200, 8, 8, 40, 1513, 2, [b % 3 for b in range(200)]), (13, 20, 4, 64, 8000, 9, [b % 10 for b in range(13)]), (6, 48, 8, 128, 3900, 5, [5, 4, 3, -1, 1, 0]),
    (33, 16, 1, 128, 2000, 100, [3 * b for b in range(33)]), (80, 20, 4, 64, 1900, 130, [b * 2 % 131 for b in range(80)]), (50, 32, 8, 64, 640, 17, [-1] * 49 + [3]),
    (90, 24, 4, 128, 2100, 100, [b + 11 for b in range(90)]), (40, 20, 4, 72, 1500, 21, [b % 22 for b in range(40)]), (100, 8, 2, 8, 9000, 5, [b % 7 - 1 for b in range(100)]),
    (36, 16, 1, 120, 2500, 30, [b % 31 for b in range(36)]), (64, 8, 2, 32, 2200, 20, [b % 21 for b in range(64)]), (250, 8, 2, 32, 700, 9, [b % 10 for b in range(250)]),
    (3, 24, 8, 104, 2900, 40, [40, 0, 7]), (20, 12, 2, 136, 1500, 20, [b for b in range(20)]), (2, 8, 2, 64, 300, 0, [0, 5]), (2, 8, 2, 64, 0, 0, [3, 0]),
    (30, 8, 2, 64, 3000, 0, [0] * 29 + [-1]), (100, 16, 4, 128, 2000, 0, [b % 2 for b in range(100)])]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", range(len(ATTN_SIZES)))
def test_attention(cuda_ctx, kind, case):
    s = attn_args(kind, *ATTN_SIZES[case], seed=case)
    attn_call(cuda_ctx, s)
    attn_check(s)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,d,P", [(2, 64, 100), (24, 64, 1500), (24, 128, 1500), (3, 32, 300), (24, 64, 15000), (24, 128, 15000), (6, 64, 60000), (6, 128, 60000), (100, 64, 9000),
                                   (100, 128, 9000), (40, 32, 9000)])
def test_attention_peaked_scaled_and_repeated(cuda_ctx, kind, B, d, P):
    """Scores far apart (a few keys have all the weight, maxima grow along the walk), another scale, and twice with the same bits."""
    s = attn_args(kind, B, 8, 2, d, P, 200, [(37 * b) % 201 for b in range(B)], seed=B + d, spread=6.0)
    s["kp"] *= torch.linspace(0.2, 1.5, P, device="cuda")[:, None].to(s["kp"].dtype)
    attn_call(cuda_ctx, s, scale=0.3)
    attn_check(s, scale=0.3)
    first = s["out"].clone()
    for _ in range(3):
        attn_call(cuda_ctx, s, scale=0.3)
        assert torch.equal(first, s["out"])


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,d,P,G", [(3, 64, 200, 2), (24, 64, 1500, 2), (24, 128, 1500, 2), (3, 32, 300, 2), (80, 64, 1500, 4), (80, 128, 1500, 8), (80, 40, 3100, 8), (30, 88, 3100, 3)])
def test_attention_values_that_are_not_finite(cuda_ctx, kind, B, d, P, G):
    """Keys that are -infinity towards a query have no weight; a row with no others is not a number; neither is one that sees a NaN; and
    other rows are as they were."""
    s = attn_args(kind, B, 2 * G, 2, d, P, 60, [b % 61 for b in range(B)], seed=3)
    s["q"] = s["q"].abs() + 0.5
    clean = dict(s, out=s["out"].clone())
    attn_call(cuda_ctx, clean)
    # the second KV head's keys are -infinity everywhere: its query heads have nothing but them
    s["kp"].view(P, 2, d)[:, 1] = -math.inf
    s["ko"].view(B, 60, 2, d)[:, :, 1] = -math.inf
    # of the first one's, a few are
    s["kp"].view(P, 2, d)[P // 2:, 0] = -math.inf
    # and sequence 1 has a NaN among its own values
    s["vo"].view(B, 60, 2, d)[1, 0, 0, 3] = math.nan
    attn_call(cuda_ctx, s)
    out = s["out"].view(B, 2, G, d)
    assert out[:, 1].isnan().all()
    assert out[1, 0, :, 3].isnan().all() and out[1, 0, :, [0, 1, 2, 4]].isfinite().all()
    half = dict(clean, P=P // 2, kp=clean["kp"][:P // 2].contiguous(), vp=clean["vp"][:P // 2].contiguous(), out=s["out"].clone())
    half["out"].view(B, 2, G, d)[:, 1] = 0
    got = half["out"]
    ref = attn_args(kind, B, 2 * G, 2, d, P // 2, 60, [b % 61 for b in range(B)], seed=3)
    ref.update(q=clean["q"], kp=half["kp"], vp=half["vp"], ko=clean["ko"], vo=clean["vo"])
    attn_call(cuda_ctx, ref)
    a, b = got.view(B, 2, G, d)[2:, 0].double(), ref["out"].view(B, 2, G, d)[2:, 0].double()
    assert (a - b).abs().max() <= 8 * half_step(TYPES[kind][0]) * b.abs().max() + 1e-5


def test_attention_lengths_beyond_the_capacity_are_the_capacity(cuda_ctx):
    s = attn_args("f16", 3, 8, 2, 64, 20, 16, [16, 16, 16], seed=1)
    s["lens"] = torch.tensor([17, 2 ** 31 - 1, 16], dtype=torch.int32, device="cuda")
    attn_call(cuda_ctx, s)
    attn_check(s)


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_attention_own_rows_beyond_32_bits(cuda_ctx, kind):
    """The last sequence's rows begin behind 2^32 elements."""
    B, kvH, d = 3, 8, 128
    cap = (1 << 31) // (kvH * d) + 7
    if kind == "f32":
        B, kvH, d, cap = 2, 8, 128, (1 << 31) // (8 * 128) + 7
    s = attn_args(kind, B, 8, kvH, d, 64, 50, [50] * B, seed=2)
    wide = dict(s, cap=cap, lens=s["lens"])
    for n in ("ko", "vo"):
        wide[n] = torch.empty(B, cap, kvH * d, device="cuda", dtype=s[n].dtype)
        wide[n][:, :50] = s[n]
    need = _lib.load().nfai_op_attn_shared_scratch_bytes(TYPES[kind][1], B, 8, kvH, d, 64, cap)
    wide["scratch"] = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    wide["out"] = s["out"].clone()
    attn_call(cuda_ctx, wide)
    s["out"] = wide["out"]
    attn_check(s)


def test_attention_prefix_beyond_32_bits(cuda_ctx):
    """Shared rows whose offset in elements does not fit into 32 bits: the last ones have all the weight."""
    kvH, d, P = 16, 128, (1 << 31) // (16 * 128) * 2 + 100
    s = attn_args("f16", 2, 16, kvH, d, 1, 4, [0, 2], seed=2)
    s["P"] = P
    s["kp"] = torch.zeros(P, kvH * d, device="cuda", dtype=torch.float16)
    s["vp"] = torch.zeros(P, kvH * d, device="cuda", dtype=torch.float16)
    s["q"] = s["q"].abs() + 1
    s["kp"][P - 3:], s["vp"][P - 3:] = 4.0, torch.randn(3, kvH * d, device="cuda").half()
    need = _lib.load().nfai_op_attn_shared_scratch_bytes(_lib.F16, 2, 16, kvH, d, P, 4)
    s["scratch"] = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    attn_call(cuda_ctx, s)
    # scores of the last three are equal and at least 128 * 4 / sqrt(128) = 45 above the others': e^-45 of 2.1 million zeros is below 2^-40
    want = s["vp"][P - 3:].double().mean(0)
    got = s["out"][0].double()
    assert (got - want).abs().max() <= 2 * 2.0 ** -11 * s["vp"][P - 3:].abs().max().double()


# ---- rules on logits -------------------------------------------------------------------------------------------------------
def rules_args(rows, V, H, n_bias, n_masks, seed, offset=0):
    r = np.random.default_rng(seed)
    s = dict(rows=rows, V=V, H=H, n_bias=n_bias, n_masks=n_masks)
    s["logits"] = (3 * r.standard_normal((rows, V))).astype(np.float32)
    s["logits"][0, ::7] = -np.inf
    s["history"] = r.integers(0, min(V + 3, max(2, V // 2) + 3), (rows, H)).astype(np.uint32) if H else np.zeros((rows, 0), np.uint32)
    s["history"][:, ::5] = 0xffffffff
    s["history_len"] = r.integers(-1, H + 3, rows).astype(np.int32)
    s["rep"], s["freq"], s["pres"] = (r.uniform(a, b, rows).astype(np.float32) for a, b in ((1.0, 1.5), (-0.2, 0.5), (0.0, 1.0)))
    s["bias_start"] = np.sort(np.concatenate([[0], r.integers(0, n_bias + 1, rows - 1), [n_bias]])).astype(np.int32)
    s["bias_ids"] = r.integers(0, V + 2, n_bias).astype(np.uint32)
    s["bias_ids"][n_bias // 2:] = s["bias_ids"][:n_bias - n_bias // 2]  # listed twice
    s["bias"] = r.standard_normal(n_bias).astype(np.float32)
    s["masks"] = r.integers(0, 1 << 32, (n_masks, (V + 31) // 32), dtype=np.uint64).astype(np.uint32)
    if n_masks:
        s["masks"][0] = 0  # nothing is allowed
    s["mask_rows"] = (np.arange(rows) % (n_masks + 2) - 1).astype(np.int32)
    return s


def rules_want(s, in64=True):
    t = np.float64 if in64 else np.float32
    out = s["logits"].astype(t)
    for r in range(s["rows"]):
        h = s["history"][r, :max(0, min(s["H"], s["history_len"][r]))]
        ids, c = np.unique(h[h < s["V"]], return_counts=True)
        x = out[r, ids]
        y = np.where(x > 0, x / t(s["rep"][r]), x * t(s["rep"][r]))
        out[r, ids] = y - t(s["freq"][r]) * c.astype(t) - t(s["pres"][r])
        for i, b in dict(zip(s["bias_ids"][s["bias_start"][r]:s["bias_start"][r + 1]].tolist(), s["bias"][s["bias_start"][r]:s["bias_start"][r + 1]])).items():
            if i < s["V"]:
                out[r, i] += t(b)
        m = s["mask_rows"][r]
        if 0 <= m < s["n_masks"]:
            bits = np.unpackbits(s["masks"][m].view(np.uint8), bitorder="little")[:s["V"]]
            out[r, bits == 0] = -np.inf
    return out


def rules_dev(s, offset=0):
    dev = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in s.items() if isinstance(v, np.ndarray)}
    n = s["rows"] * s["V"]
    flat = torch.zeros(n + offset, device="cuda")
    flat[offset:] = dev["logits"].reshape(-1)
    dev["logits"], dev["out"] = flat[offset:], torch.full((n + offset + 8,), 5.0, device="cuda")[offset:]
    return dev


def rules_call(ctx, s, dev, in_place=False, stream=None):
    out = dev["logits"] if in_place else dev["out"]
    run(ctx, "nfai_op_logit_rules", at(dev["logits"]), s["rows"], s["V"], at(dev["history"]) if s["H"] else None, s["H"], at(dev["history_len"]),
        at(dev["rep"]), at(dev["freq"]), at(dev["pres"]), at(dev["bias_start"]), at(dev["bias_ids"]), at(dev["bias"]), s["n_bias"],
        at(dev["masks"]), s["n_masks"], at(dev["mask_rows"]), at(out), stream=stream)
    return out


def rules_check(s, got):
    """Four roundings of float32 follow one another (quotient, product, two differences, a sum): within 5 u of the terms' sizes."""
    want = rules_want(s)
    got = got.cpu().numpy()[:s["rows"] * s["V"]].reshape(s["rows"], s["V"]).astype(np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)) and np.array_equal(want[~fine], got[~fine])
    size = np.abs(np.where(np.isfinite(s["logits"]), s["logits"], 0)) * 1.5 + 0.5 * max(1, s["H"]) + 6.0
    assert (np.abs(got[fine] - want[fine]) <= (5 * U * size)[fine]).all()
    # no operation is done in another order or precision than float32 in the order of the definition
    same = rules_want(s, in64=False)
    assert np.array_equal(same[fine].astype(np.float64), got[fine])


RULES_SIZES = [  # rows, V, history, biases, masks
    (1, 1, 1, 1, 1), (1, 3, 2, 0, 0), (2, 5, 4, 2, 1), (3, 31, 3, 5, 2), (3, 33, 40, 9, 3), (2, 1000, 64, 0, 0), (5, 1023, 100, 30, 2), (4, 4097, 0, 7, 0),
    (3, 4099, 300, 0, 3), (7, 8197, 1000, 50, 1), (1, 128256, 64, 4, 0), (40, 128256, 700, 100, 20), (33, 100003, 3000, 1000, 5), (1, 300000, 9000, 10, 1)]


@pytest.mark.parametrize("case", range(len(RULES_SIZES)))
@pytest.mark.parametrize("offset", [0, 1])
def test_rules(cuda_ctx, case, offset):
    s = rules_args(*RULES_SIZES[case], seed=case)
    dev = rules_dev(s, offset)
    got = rules_call(cuda_ctx, s, dev)
    assert (got[s["rows"] * s["V"]:] == 5).all()
    rules_check(s, got)
    rules_check(s, rules_call(cuda_ctx, s, dev, in_place=True))


def test_rules_nothing_asked_for(cuda_ctx):
    x = torch.randn(3, 1001, device="cuda")
    x[1, 5] = math.nan
    out = torch.empty_like(x)
    run(cuda_ctx, "nfai_op_logit_rules", at(x), 3, 1001, None, 0, None, None, None, None, None, None, None, 0, None, 0, None, at(out))
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))


def test_rules_bad_starts_stay_inside(cuda_ctx):
    """Starts that are not ascending or lie outside the list: entries outside it are not read, and a row whose end is before its start has none."""
    x = torch.zeros(3, 64, device="cuda")
    out = torch.empty_like(x)
    start = torch.tensor([-5, 2, 1, 1 << 30], dtype=torch.int32, device="cuda")
    ids, bias = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda"), torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda")
    run(cuda_ctx, "nfai_op_logit_rules", at(x), 3, 64, None, 0, None, None, None, None, at(start), at(ids), at(bias), 4, None, 0, None, at(out))
    want = torch.zeros(3, 64)
    want[0, 1], want[0, 2], want[2, 2], want[2, 3], want[2, 4] = 1, 2, 2, 3, 4
    assert torch.equal(out.cpu(), want)


# ---- streams, graphs, threads, and a step ------------------------------------------------------------------------------------
def test_refusals_on_a_context(cuda_ctx):
    """What is refused without a context is refused with one, and the context goes on working."""
    s = attn_args("f16", 2, 8, 2, 64, 20, 16, [3, 4], seed=1)
    for change in ({"scratch": s["scratch"][:-512]}, {"d": 60}):
        with pytest.raises(_lib.NfaiError) as e:
            attn_call(cuda_ctx, {**s, **change})
        assert e.value.code == _lib.ERR_ARG
    attn_call(cuda_ctx, s)
    attn_check(s)


def test_on_another_stream_behind_its_work_and_captured(cuda_ctx):
    """Work on a side stream is ordered with the stream's other work; a captured step gives, replayed on new inputs, what calls give."""
    a = attn_args("bf16", 24, 32, 8, 64, 1500, 64, [b % 60 for b in range(24)], seed=4)
    r = rope_args(24, 32, 8, 64, 64, 1, "bf16", "bf16", 24 * 64, 4, slots="all")
    s = rules_args(6, 5000, 50, 10, 2, seed=4)
    dev = rules_dev(s)
    r["k"], r["v"], r["q"] = a["ko"].view(24 * 64, -1), a["vo"].view(24 * 64, -1), a["q"]
    slots = torch.arange(24, device="cuda", dtype=torch.int32) * 64 + a["lens"] - 1
    r["slots"] = torch.where(a["lens"] > 0, slots, -1)
    logits, raw = dev["logits"].clone(), r["x"].clone()

    def step(stream):
        rope_call(cuda_ctx, r, _lib.BF16, _lib.BF16, stream=stream)
        attn_call(cuda_ctx, a, stream=stream)
        rules_call(cuda_ctx, s, dev, stream=stream)

    def spoil():  # (what lies behind the last row of logits is left alone, so it is the same before every step)
        for t in (a["q"], a["out"], dev["out"]):
            t.fill_(1)
    spoil()
    step(None)
    want = [t.clone() for t in (a["q"], a["ko"], a["out"], dev["out"])]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        spoil()
        r["x"].zero_(), dev["logits"].zero_()
        r["x"].copy_(raw), dev["logits"].copy_(logits)  # the calls are ordered behind these
        step(side.cuda_stream)
        got = [t.clone() for t in (a["q"], a["ko"], a["out"], dev["out"])]
    side.synchronize()
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    r["x"].mul_(0.5), a["vp"].mul_(-1.0)
    step(None)
    want = [t.clone() for t in (a["q"], a["ko"], a["out"], dev["out"])]
    for _ in range(3):
        spoil()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((a["q"], a["ko"], a["out"], dev["out"]), want))
    # and on the default stream, by the name it has
    spoil()
    step(1)
    torch.cuda.synchronize()
    assert torch.equal(a["out"].view(torch.int16), want[2].view(torch.int16))


def test_two_calls_at_once(cuda_ctx):
    """Calls of one context on two streams, eager and as two graphs, each with its scratch: what they give one after the other."""
    jobs = [attn_args(kind, 70, 32, 8, 64, 1900, 90, [(7 * b + i) % 91 for b in range(70)], seed=i) for i, kind in enumerate(("f16", "f32"))]
    rules = rules_args(9, 50000, 500, 30, 3, seed=8)
    devs = [rules_dev(rules) for _ in jobs]
    for s, dev in zip(jobs, devs):
        attn_call(cuda_ctx, s)
        rules_call(cuda_ctx, rules, dev)
    want = [(s["out"].clone(), dev["out"].clone()) for s, dev in zip(jobs, devs)]
    streams, graphs = [torch.cuda.Stream() for _ in jobs], []

    def both(go):
        for s, dev in zip(jobs, devs):
            s["out"].fill_(5.0), dev["out"].fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(len(jobs)):
                go(i)
        torch.cuda.synchronize()
        for s, dev, (a, b) in zip(jobs, devs, want):
            assert torch.equal(s["out"], a) and torch.equal(dev["out"], b)

    def calls(i, stream):
        attn_call(cuda_ctx, jobs[i], stream=stream)
        rules_call(cuda_ctx, rules, devs[i], stream=stream)
    both(lambda i: calls(i, streams[i].cuda_stream))
    for i, s in enumerate(streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=s):
            calls(i, torch.cuda.current_stream().cuda_stream)

    def replay(i):
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    both(replay)


def test_two_contexts_from_two_threads(cuda_ctx):
    """Calls at the same time on streams of their own, each with its scratch."""
    from nfai_b200 import CudaContext
    jobs = [attn_args("f16", 24, 32, 8, 128, 3000, 90, [(7 * b + i) % 91 for b in range(24)], seed=i) for i in range(2)]
    other = CudaContext(0)
    failed = []

    def work(ctx, s):
        try:
            for _ in range(30):
                _lib.check(_lib.load().nfai_op_attn_shared(
                    ctx.handle, at(s["q"]), at(s["kp"]), at(s["vp"]), s["P"], at(s["ko"]), at(s["vo"]), s["cap"], at(s["lens"]), _lib.F16, s["B"],
                    s["qH"], s["kvH"], s["d"], 0.0, at(s["out"]), at(s["scratch"]), s["scratch"].numel() - 256, None), ctx.handle)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=a) for a in zip((cuda_ctx, other), jobs)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    other.close()
    assert not failed
    for s in jobs:
        attn_check(s)


def test_a_step_of_four_answers(cuda_ctx):
    """One layer's attention block and the choice of the next tokens for four answers behind a shared prompt, with the library's own
    products (nfai_op_gemm), against the same in 64 bits; a free place in the batch stays out of it."""
    B, H, qH, kvH, d, P, cap, V = 5, 256, 8, 2, 64, 700, 32, 4096
    g = torch.Generator(device="cuda").manual_seed(9)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    x = normal(B, H).half()
    wqkv, wo, head = (normal(n, k).half() * 0.06 for n, k in (((qH + 2 * kvH) * d, H), (H, qH * d), (V, H)))
    kp, vp, ko, vo = normal(P, kvH * d).half(), normal(P, kvH * d).half(), normal(B, cap, kvH * d).half(), normal(B, cap, kvH * d).half()
    lens = torch.tensor([3, 0, 31, 12, -1], dtype=torch.int32, device="cuda")     # own rows so far
    freqs = (C.c_double * (d // 2))()
    mag = C.c_float()
    _lib.check(_lib.load().nfai_rope_frequencies(d, 500000.0, 2, 8.0, 1.0, 4.0, 8192, freqs, C.byref(mag)))
    table = torch.tensor(list(freqs), dtype=torch.float64, device="cuda")
    before = ko.clone(), vo.clone()
    qkv, q, att = torch.empty(B, (qH + 2 * kvH) * d, device="cuda"), torch.empty(B, qH * d, device="cuda", dtype=torch.float16), torch.zeros(B, qH * d, device="cuda", dtype=torch.float16)
    free = lens < 0
    positions = (P + lens).clamp(min=0).int()
    slots = torch.where(free, -1, torch.arange(B, device="cuda", dtype=torch.int32) * cap + lens).int()
    now = torch.where(free, -1, lens + 1).int()
    torch.cuda.synchronize()
    lib, h = _lib.load(), cuda_ctx.handle
    _lib.check(lib.nfai_op_gemm(h, at(x), at(wqkv), _lib.F16, B, (qH + 2 * kvH) * d, H, at(qkv)), h)
    run(cuda_ctx, "nfai_op_rope_rows", at(qkv), _lib.F32, 0, B, qH, kvH, d, d, 0, at(table), mag.value, at(positions), at(slots), at(q), at(ko), at(vo), _lib.F16, B * cap)
    need = lib.nfai_op_attn_shared_scratch_bytes(_lib.F16, B, qH, kvH, d, P, cap)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    run(cuda_ctx, "nfai_op_attn_shared", at(q), at(kp), at(vp), P, at(ko), at(vo), cap, at(now), _lib.F16, B, qH, kvH, d, 0.0, at(att), at(scratch), need)
    hid, logits = torch.empty(B, H, device="cuda"), torch.empty(B, V, device="cuda")
    _lib.check(lib.nfai_op_gemm(h, at(att), at(wo), _lib.F16, B, H, qH * d, at(hid)), h)
    hid16 = hid.half()
    torch.cuda.synchronize()
    _lib.check(lib.nfai_op_gemm(h, at(hid16), at(head), _lib.F16, B, V, H, at(logits)), h)
    plain_logits = logits.clone()
    # every answer may only say odd tokens, and not again what it said
    mask = torch.full((1, V // 32), -0x55555556, dtype=torch.int32, device="cuda")  # bits 1, 3, 5, ...
    best = torch.where(torch.arange(V, device="cuda") % 2 == 1, logits, -math.inf).argmax(-1).int()
    pick = torch.zeros(B, dtype=torch.int32, device="cuda")
    pen = torch.full((B,), 1e4, device="cuda")
    run(cuda_ctx, "nfai_op_logit_rules", at(logits), B, V, at(best), 1, None, None, None, at(pen), None, None, None, 0, at(mask), 1, at(pick), at(logits))
    tokens = []
    for b in range(B):
        tok = torch.zeros(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        _lib.check(lib.nfai_op_sample_top_p(h, at(logits[b]), V, 0.5, 0.95, 1, 0.3, at(tok)), h)
        tokens.append(tok.item())
    # in 64 bits
    y = (x.double() @ wqkv.double().T).view(B, qH + 2 * kvH, d)
    ang = positions.double()[:, None, None] * table
    c, n = ang.cos(), ang.sin()
    turned = y.clone()
    a_, b_ = y[:, :qH + kvH, 0::2], y[:, :qH + kvH, 1::2]
    turned[:, :qH + kvH, 0::2], turned[:, :qH + kvH, 1::2] = a_ * c - b_ * n, a_ * n + b_ * c
    att64 = torch.zeros(B, qH * d, dtype=torch.float64, device="cuda")
    for b in range(B):
        if free[b]:
            assert torch.equal(ko[b], before[0][b]) and torch.equal(vo[b], before[1][b]) and (att[b] == 0).all()
            continue
        m = int(lens[b])
        k = torch.cat([kp.double(), before[0][b, :m].double(), turned[b, qH:qH + kvH].reshape(1, -1)]).view(-1, kvH, d).permute(1, 2, 0)
        v = torch.cat([vp.double(), before[1][b, :m].double(), turned[b, qH + kvH:].reshape(1, -1)]).view(-1, kvH, d).permute(1, 0, 2)
        w = torch.softmax(turned[b, :qH].view(kvH, qH // kvH, d) @ k / math.sqrt(d), -1)
        att64[b] = (w @ v).reshape(-1)
    # q, k, v, weights and the result are rounded to float16 once each, 2^-11: q and k move a score by 2 * 2^-11 |q| |k| / sqrt(d) at most
    qn, kn = turned[:, :qH].norm(dim=-1).max(), max(kp.view(-1, d).double().norm(dim=-1).max(), turned[:, qH:qH + kvH].norm(dim=-1).max())
    room = 2.0 ** -11 * (2 * 2 * qn * kn / math.sqrt(d) + 3) * max(vp.abs().max(), turned[:, qH + kvH:].abs().max(), vo.abs().max())
    assert (att.double() - att64)[~free].abs().max() <= room
    masked = plain_logits.clone()
    masked[:, 0::2] = -math.inf
    masked.scatter_(1, best.long()[:, None], -1e5)
    assert torch.equal(masked.argmax(-1)[~free], torch.tensor(tokens, device="cuda")[~free]) and all(t % 2 == 1 for t in tokens[:4])
