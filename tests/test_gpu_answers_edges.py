"""Where the operators of a step of several answers to one prompt could go wrong: weights far below a row's heaviest, infinite values,
alignment, waits that run out. The helpers and the conventions on tolerances are those of test_gpu_answers.py."""
import os
import shutil
import subprocess

import pytest

from nfai_b200 import _lib, build

from .test_gpu_answers import TYPES, U, attn_args, attn_call, half_step, rope_args, rope_call, rules_args, rules_call, rules_check, rules_dev, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def timed_in_turn(*calls):
    """The median time of 20 calls(stream) of each on the device, one after the other, in ms."""
    stream, times = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for _ in range(7):
        for call in calls:
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            with torch.cuda.stream(stream):
                torch.cuda._sleep(2_000_000)  # the calls are enqueued behind it, so that the host's time does not count
                a.record()
                for _ in range(20):
                    call(stream.cuda_stream)
                b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
    return [sorted(times[2 * len(calls) + i::len(calls)])[2] for i in range(len(calls))]


# ---- attention: weights far below the heaviest --------------------------------------------------------------------------------
def attn_want(s, scale=0.0):
    """The definition in 64 bits, sum w |v| and sum |v|: [B][qH][d] each; rows of free places are zero."""
    B, qH, kvH, d, P = s["B"], s["qH"], s["kvH"], s["d"], s["P"]
    want, size, all_v = torch.zeros(3, B, qH, d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        n = min(n, s["cap"])
        if n < 0 or P + n == 0:
            continue
        k = torch.cat([s["kp"].double(), s["ko"][b, :n].double()]).view(-1, kvH, d).permute(1, 2, 0)
        v = torch.cat([s["vp"].double(), s["vo"][b, :n].double()]).view(-1, kvH, d).permute(1, 0, 2)
        w = torch.softmax(s["q"][b].double().view(kvH, qH // kvH, d) @ k * (scale or d ** -0.5), -1)
        want[b], size[b], all_v[b] = ((x @ y).view(qH, d) for x, y in ((w, v), (w, v.abs()), (torch.ones_like(w), v.abs())))
    return want, size, all_v


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("where", ["shared", "own"])
@pytest.mark.parametrize("B,kvH,G,d,P,cap", [(1, 2, 4, 64, 2000, 900), (24, 8, 4, 64, 3000, 600), (24, 8, 4, 128, 3000, 600), (3, 8, 4, 64, 9000, 700), (9, 2, 3, 128, 6000, 300),
                                             (70, 8, 8, 40, 2500, 300), (200, 8, 4, 64, 1500, 60), (2, 2, 2, 256, 900, 300), (4, 2, 2, 32, 200, 800)])
def test_attention_many_light_keys_behind_a_heavy_one(cuda_ctx, kind, where, B, kvH, G, d, P, cap):
    """One key takes nearly all of a row's weight and has a value of zero (the first token of many models); what the row gives are the others,
    17.5 below it, a weight of 2^-25.2 of the heaviest each.

    Queries of 1 and keys of 0 and of 17.5 / sqrt(d) rounded to three bits: all scores are exact. A weight is rounded to the caches' type (not float32):
    half a step of its size, or of float16's smallest step, 2^-24 of a weight that has been multiplied by 2^7: 2^-32 of the heaviest.
    Exponentials 8 u, sums of n keys n u, one rounding of the result."""
    s = attn_args(kind, B, kvH * G, kvH, d, P, cap, [cap - b % 7 for b in range(B)], seed=B + d)
    heavy = float(torch.tensor(17.5 / d ** 0.5).to(torch.float8_e4m3fn))
    s["q"].fill_(1.0), s["kp"].zero_(), s["ko"].zero_()
    for v in (s["vp"], s["vo"]):
        v.copy_(v.float().abs().clamp(0.25, 4.0) * 8192.0)
    k, v = (s["kp"], s["vp"]) if where == "shared" else (s["ko"], s["vo"])
    if where == "shared":
        k[P // 3], v[P // 3] = heavy, 0.0
    else:
        k[:, 5], v[:, 5] = heavy, 0.0
    for b, n in enumerate(s["lens"].tolist()):  # what lies behind a sequence's rows is no number
        s["ko"][b, n:], s["vo"][b, n:] = float("nan"), float("inf")
    attn_call(cuda_ctx, s)
    want, size, all_v = attn_want(s)
    kind = TYPES[kind][0]
    n = P + cap
    half = half_step(kind) if kind != torch.float32 else 0.0
    floor = 2.0 ** -32 * all_v if kind == torch.float16 else 0.0
    room = (8 * U + half + n * U) * size + floor + half_step(kind) * want.abs() + torch.finfo(kind).tiny
    off = (s["out"].view(want.shape).double() - want).abs()
    assert (room < 0.05 * want).all()  # (what is left out would be seen)
    assert (off <= room).all(), (off / room).max().item()


# ---- attention: infinite values -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,kvH,G,d,P,cap", [(1, 2, 4, 64, 300, 70), (3, 2, 2, 32, 200, 30), (24, 8, 4, 64, 1500, 40), (24, 8, 4, 128, 1500, 40), (5, 8, 4, 64, 9000, 100),
                                             (9, 2, 3, 128, 6000, 300), (80, 2, 8, 40, 3100, 60), (200, 8, 4, 64, 1500, 60), (2, 2, 2, 256, 400, 70), (12, 2, 2, 136, 3000, 9), (2, 2, 4, 64, 0, 900)])
def test_attention_infinite_values(cuda_ctx, kind, B, kvH, G, d, P, cap):
    """An infinite value gives an infinity to every row that sees its key, however light the key is there; infinities of both signs and a NaN
    give NaN; elements without either are as they were, bit for bit."""
    s = attn_args(kind, B, kvH * G, kvH, d, P, cap, [cap - b % 7 for b in range(B)], seed=B + d)
    s["q"] = s["q"].abs() + 0.5
    own = s["vo"].view(B, cap, kvH, d)
    if P:
        # key P // 4 lies about 20 below the others: below 2^-25 of a weight, above 2^-126
        s["kp"][P // 4] = -20.0 / (1.7 * d ** 0.5)
    clean = dict(s, out=s["out"].clone())
    attn_call(cuda_ctx, clean)
    if P:
        v = s["vp"].view(P, kvH, d)
        v[P // 3, :, 1], v[P // 2, 0, 2] = float("inf"), float("-inf")
        v[P // 4, 1, 3] = float("inf")
        v[0, 0, 4], v[P - 1, 0, 4] = float("inf"), float("-inf")
        v[P // 5, 1, 5], v[P // 2, 1, 5] = float("inf"), float("nan")
    own[:, 0, 0, 6] = float("inf")
    own[B - 1, 1, 1, 7] = float("-inf")
    own[B // 2, 2, 0, d - 1], own[B // 2, 1, 0, d - 1] = float("inf"), float("-inf")
    attn_call(cuda_ctx, s)
    want = attn_want(s)[0]
    bad = ~want.isfinite()
    got = s["out"].view(want.shape).double()
    assert bad.any() and torch.equal(got[bad].nan_to_num(0.5), want[bad].nan_to_num(0.5))
    assert torch.equal(got[~bad], clean["out"].view(want.shape).double()[~bad])


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,d,P", [(1, 64, 200), (24, 64, 1500), (24, 128, 1500), (5, 64, 9000), (3, 256, 200)])
def test_attention_infinite_values_without_a_weight(cuda_ctx, kind, B, d, P):
    """A row whose scores are all -infinity, or one of them NaN, stays NaN, also where its values are infinite."""
    s = attn_args(kind, B, 8, 2, d, P, 20, [20] * B, seed=B + d)
    s["q"] = s["q"].abs() + 0.5
    s["kp"].view(P, 2, d)[:, 0] = float("-inf")
    s["ko"].view(B, 20, 2, d)[:, :, 0] = float("-inf")
    s["kp"].view(P, 2, d)[P // 2, 1] = float("nan")
    s["vp"][P // 3] = float("inf")
    attn_call(cuda_ctx, s)
    assert s["out"].isnan().all()


# ---- a wait that gave up ------------------------------------------------------------------------------------------------------
def test_a_wait_that_gave_up_is_told_by_the_next_call_that_waits(tmp_path):
    """Also with other operators in between, by nobody else, and once; what others left in their word is not taken for it. The program writes
    the words as a kernel that gave up does."""
    gxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else shutil.which("g++")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(build._nvcc())))
    lib, exe = build.build(), str(tmp_path / "answers_note")
    subprocess.run([gxx, "-std=c++17", "-I", os.path.join(root, "nfai_b200", "csrc"), "-I", os.path.join(root, "include"), "-I", os.path.join(cuda, "include"),
                    os.path.join(root, "tests", "cabi", "answers_note.cpp"), "-o", exe, "-L", os.path.dirname(lib), "-lnfai_cuda",
                    "-Wl,-rpath," + os.path.dirname(lib), "-L", os.path.join(cuda, "lib64"), "-lcudart_static", "-lpthread", "-ldl", "-lrt"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)


@pytest.mark.parametrize("d,P,kind", [(128, 8000, "bf16"), (64, 1500, "f16"), (64, 600, "f32")])
def test_attention_queries_of_free_places_may_be_anything(cuda_ctx, d, P, kind):
    """Where they are no numbers, the other rows' bits stay, and so does the time (60 % and more were lost where their sums were looked into)."""
    B = 64
    s = attn_args(kind, B, 32, 8, d, P, 40, [-1 if b % 20 == 7 else b % 41 for b in range(B)], seed=d)
    other = dict(s, q=s["q"].clone(), out=s["out"].clone())
    other["q"][s["lens"] < 0] = float("nan")
    clean_ms, other_ms = timed_in_turn(*(lambda stream, x=x: attn_call(cuda_ctx, x, stream=stream) for x in (s, other)))
    assert torch.equal(s["out"], other["out"])
    print(f"{kind} {d} {P}: {clean_ms * 50:.2f} {other_ms * 50:.2f} us")
    assert other_ms <= 1.3 * clean_ms


# ---- rotary rows: alignment ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("x,out", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("f16", "f32")])
def test_rope_rows_on_16_bytes(cuda_ctx, x, out, layout):
    """Buffers that begin on an odd multiple of 16 bytes give the same bits as others, and take no kernel that goes an element at a time: that one
    takes several times as long, here at most twice is allowed."""
    names = ("x", "q", "k", "v")
    even = rope_args(2011, 32, 8, 64, 64, layout, x, out, 2100, 7, slots="all")
    odd = dict(even)
    for n in names:
        room = torch.empty(even[n].numel() + 16, device="cuda", dtype=even[n].dtype)
        odd[n] = room[16 // room.element_size():][:even[n].numel()].view(even[n].shape)
        odd[n].copy_(even[n])
        assert odd[n].data_ptr() % 32 == 16 and even[n].data_ptr() % 32 == 0
    codes = TYPES[x][1], TYPES[out][1]
    even_ms, odd_ms = timed_in_turn(*(lambda stream, s=s: rope_call(cuda_ctx, s, *codes, stream=stream) for s in (even, odd)))
    for n in names:
        assert torch.equal(even[n], odd[n])
    print(f"{x} {out} {layout}: {even_ms * 50:.2f} {odd_ms * 50:.2f} us")
    assert odd_ms <= 2 * even_ms


@pytest.mark.parametrize("B,kvH,G,d,P,cap,kind", [(24, 8, 4, 64, 1500, 40, "f16"), (24, 8, 4, 128, 1500, 40, "bf16"), (9, 2, 3, 128, 6000, 300, "f16"), (70, 8, 8, 64, 2500, 60, "bf16"),
                                                  (40, 8, 4, 64, 100, 2000, "f16"), (300, 2, 2, 32, 90, 900, "bf16"), (200, 8, 4, 64, 1500, 60, "f16")])
def test_a_wait_that_runs_out_leaves_no_number(cuda_ctx, B, kvH, G, d, P, cap, kind):
    """With a budget of a nanosecond the kernels give up on their copies: they return, the call says so, and what a row then has is NaN, or, where
    nothing had to be waited for, what it has otherwise. Nothing is left for the next call."""
    def budget(ns):
        _lib.check(_lib.load().nfai_ctx_set_wait_ns(cuda_ctx.handle, ns), cuda_ctx.handle)
    s = attn_args(kind, B, kvH * G, kvH, d, P, cap, [cap - b % 7 for b in range(B)], seed=B + d)
    attn_call(cuda_ctx, s)
    want = s["out"].clone()

    def nan_or_right():
        heads, right = s["out"].view(-1, d), want.view(-1, d)
        gone = heads.isnan().all(-1)
        assert torch.equal(heads[~gone], right[~gone])
        return gone.float().mean().item()
    try:
        budget(1)
        for _ in range(3):
            s["out"].fill_(5.0)
            with pytest.raises(_lib.NfaiError) as e:
                attn_call(cuda_ctx, s)
            assert e.value.code == _lib.ERR_TIMEOUT
            assert nan_or_right() > 0
        attn_call(cuda_ctx, s, stream=torch.cuda.current_stream().cuda_stream or 1)  # on a stream nobody is told yet
        torch.cuda.synchronize()
        assert nan_or_right() > 0
    finally:
        budget(1_000_000_000)
    with pytest.raises(_lib.NfaiError) as e:  # the next call that waits is, and is right itself
        attn_call(cuda_ctx, s)
    assert e.value.code == _lib.ERR_TIMEOUT and torch.equal(s["out"], want)
    s["out"].fill_(5.0)
    attn_call(cuda_ctx, s)
    assert torch.equal(s["out"], want)


def test_a_wait_that_runs_out_in_the_rules(cuda_ctx):
    def budget(ns):
        _lib.check(_lib.load().nfai_ctx_set_wait_ns(cuda_ctx.handle, ns), cuda_ctx.handle)
    x = torch.randn(700, 100000, device="cuda")  # more than the L2 holds
    out = torch.empty_like(x)

    def call():  # (nothing is asked for: there is nothing to do while the logits come)
        out.fill_(5.0)
        run(cuda_ctx, "nfai_op_logit_rules", x.data_ptr(), 700, 100000, *[None, 0] + [None] * 7, 0, None, 0, None, out.data_ptr())
    try:
        budget(1)
        with pytest.raises(_lib.NfaiError) as e:
            call()
        assert e.value.code == _lib.ERR_TIMEOUT
        gone = out.isnan()
        assert gone.any() and torch.equal(out[~gone], x[~gone])
    finally:
        budget(1_000_000_000)
    call()
    assert torch.equal(out, x)


# ---- attention: scores of any size ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,spread", [("f16", 3e3), ("bf16", 1e5), ("bf16", 1e7), ("bf16", 1e9), ("bf16", 1e12), ("f32", 1e8), ("f32", 1e13)])
@pytest.mark.parametrize("B,kvH,G,d,P,cap", [(2, 8, 4, 64, 300, 60), (5, 8, 4, 64, 9000, 100), (24, 8, 4, 128, 1500, 40), (70, 2, 8, 40, 2500, 60), (200, 8, 4, 64, 1500, 30)])
def test_attention_scores_far_beyond_their_differences(cuda_ctx, kind, spread, B, kvH, G, d, P, cap):
    """Scores so large that float32 leaves few bits or none behind the point: the largest has all the weight, whatever its size. Rows whose two
    largest are nearer than float32 sums can tell (4 d u of the products' size) are left out; most remain. The result is a value of the cache: off
    by half a step where the one weight is rounded and its sum is not, by 4 u for quotient and product, and by half a step of the result."""
    s = attn_args(kind, B, kvH * G, kvH, d, P, cap, [cap - b % 7 for b in range(B)], seed=B + d, spread=spread)
    attn_call(cuda_ctx, s)
    seen = 0
    for b, n in enumerate(s["lens"].tolist()):
        k = torch.cat([s["kp"].double(), s["ko"][b, :n].double()]).view(-1, kvH, d).permute(1, 2, 0)
        v = torch.cat([s["vp"], s["vo"][b, :n]]).view(-1, kvH, d).permute(1, 0, 2)
        q = s["q"][b].double().view(kvH, G, d)
        best = (q @ k).topk(2, -1)
        room = 4 * d * U * (q.abs() @ k.abs()).amax(-1) + 200 * d ** 0.5  # (and a weight of e^-200 is 0 in float32)
        clear = best.values[..., 0] - best.values[..., 1] > room
        want = v.gather(1, best.indices[..., :1].expand(-1, -1, d))
        off = (s["out"][b].view(kvH, G, d).double() - want.double()).abs() / want.double().abs()
        assert off[clear].max().item() <= 2 * half_step(TYPES[kind][0]) + 4 * U, b
        seen += clear.float().mean().item()
    assert seen > 0.5 * B


@pytest.mark.parametrize("B,kvH,G,d,P,cap", [(2, 8, 4, 64, 300, 60), (5, 8, 4, 64, 9000, 100), (24, 8, 4, 128, 1500, 40), (70, 2, 8, 40, 2500, 60), (200, 8, 4, 64, 1500, 30), (3, 2, 2, 256, 700, 9)])
@pytest.mark.parametrize("kind,low,pick", [("bf16", -3.3895313892515355e38, 1.0), ("f32", -3.4028234663852886e38, 1.0), ("f16", -65504.0, 1.0), ("f16", -65504.0, 32768.0)])
def test_attention_rows_with_nothing_but_the_lowest_scores(cuda_ctx, kind, low, pick, B, kvH, G, d, P, cap):
    """Keys whose scores are the lowest number that the type has, as a mask leaves them (the query picks one element): where a row has nothing else
    they weigh the same, and where it has others they weigh nothing."""
    s = attn_args(kind, B, kvH * G, kvH, d, P, cap, [cap - b % 7 for b in range(B)], seed=B + d)
    s["q"].zero_()
    s["q"].view(B, kvH, G, d)[..., 3] = pick
    for k, v in ((s["kp"], s["vp"]), (s["ko"], s["vo"])):
        k.view(*k.shape[:-1], kvH, d)[..., 3] = low
        v.copy_(v.float().abs().clamp(0.25, 4.0))
    # the last KV head has a few keys with scores of their own
    s["kp"].view(P, kvH, d)[P // 3:P // 3 + 5, -1, 3] = 1.5
    s["ko"].view(B, cap, kvH, d)[:, 1, -1, 3] = 1.5
    for b, n in enumerate(s["lens"].tolist()):
        s["ko"][b, n:], s["vo"][b, n:] = float("nan"), float("inf")
    attn_call(cuda_ctx, s, scale=0.125)
    want, size, _ = attn_want(s, scale=0.125)
    half = half_step(TYPES[kind][0])
    # equal scores, so equal weights: sums of n of them n u, quotient and product 4 u, weights in two terms 2^-16, the result half a step
    room = ((P + cap + 8) * U + (2.0 ** -16 if kind != "f32" else 0.0) + half) * size
    off = (s["out"].view(want.shape).double() - want).abs()
    assert (off <= room).all(), (off / room).max().item()


# ---- rules: the end of the history --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,V,H", [(1, 5000, 4000), (3, 128256, 3000), (40, 1000, 9000)])
def test_rules_history_that_ends_with_the_last_rows_tokens(cuda_ctx, rows, V, H):
    """Nothing behind them is read: what lies there here would count, and need not be there."""
    s = rules_args(rows, V, H, 5, 0, seed=rows)
    s["history_len"][:] = H
    s["history_len"][-1] = 7
    dev = rules_dev(s)
    flat = torch.zeros(rows * H, device="cuda", dtype=torch.int32)  # token 0 behind them
    flat[:(rows - 1) * H + 7] = dev["history"].reshape(-1)[:(rows - 1) * H + 7]
    dev["history"] = flat
    rules_check(s, rules_call(cuda_ctx, s, dev))
