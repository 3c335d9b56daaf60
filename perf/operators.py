"""Several answers to one prompt, a step at a time: the operators of such a step beside the matrix products, as cases.

A host asks for n answers to one prompt (or serves n chats behind one system prompt). The prompt's keys and values are in
memory once, every answer has rows of its own behind them, and a step brings one token of each answer:

  rope    rotates the queries and keys of a batch of tokens, each at its own position, and puts keys and values into cache rows
  attend  attention of one token of every answer over the shared rows and over its own
  rules   repetition, frequency and presence penalties, biases and the tokens that a grammar allows, on the logits of every answer

Head counts and sizes are those of the framework's own models (nfai_b200/synth.py and the layer plans in perf/cases.py), or
generic ones: one key head a query head, many query heads a key head.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"f32": 0, "f16": 1, "bf16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one chat: all that counts is how long a call takes
        {"name": "rope-1", "op": "rope", "rows": 1, "qH": 32, "kvH": 8, "d": 64, "dims": 64, "layout": "pairs", "scaling": "bands",
         "far": 4000, "cache": 1024, "x": "f32", "out": "f16"},
        # a step of 37 answers far into a long context that the frequencies are stretched for; halves, a part of the head
        {"name": "rope-37-far", "op": "rope", "rows": 37, "qH": 32, "kvH": 8, "d": 128, "dims": 64, "layout": "halves",
         "scaling": "yarn", "far": 1000000, "cache": 8192, "x": "bf16", "out": "bf16"},
        # a page or two of prompt
        {"name": "rope-2011", "op": "rope", "rows": 2011, "qH": 32, "kvH": 8, "d": 64, "dims": 64, "layout": "pairs",
         "scaling": "plain", "far": 4000, "cache": 4096, "x": "f32", "out": "f16"},
        # a pass of a long document through the largest of the models
        {"name": "rope-9472", "op": "rope", "rows": 9472, "qH": 32, "kvH": 8, "d": 128, "dims": 128, "layout": "halves",
         "scaling": "linear", "far": 30000, "cache": 9472, "x": "f32", "out": "bf16"},
        # two answers to a short question
        {"name": "attend-2-300", "op": "attend", "batch": 2, "qH": 32, "kvH": 8, "d": 64, "prefix": 300, "capacity": 128, "own": 40,
         "idle": 0, "dtype": "f16"},
        # eight drafts behind a page or two, some way on
        {"name": "attend-8-2011", "op": "attend", "batch": 8, "qH": 32, "kvH": 8, "d": 128, "prefix": 2011, "capacity": 1024,
         "own": 300, "idle": 1, "dtype": "bf16"},
        # a few answers about a long document
        {"name": "attend-5-100003", "op": "attend", "batch": 5, "qH": 32, "kvH": 8, "d": 64, "prefix": 100003, "capacity": 512,
         "own": 200, "idle": 0, "dtype": "f16"},
        # a full batch behind a long document, the largest heads
        {"name": "attend-64-32768", "op": "attend", "batch": 64, "qH": 32, "kvH": 8, "d": 128, "prefix": 32768, "capacity": 1024,
         "own": 500, "idle": 3, "dtype": "bf16"},
        # many chats behind one system prompt
        {"name": "attend-256-1500", "op": "attend", "batch": 256, "qH": 32, "kvH": 8, "d": 64, "prefix": 1500, "capacity": 2048,
         "own": 500, "idle": 9, "dtype": "f16"},
        # the model that is kept in 32 bits
        {"name": "attend-9-1000-f32", "op": "attend", "batch": 9, "qH": 8, "kvH": 2, "d": 32, "prefix": 1000, "capacity": 512,
         "own": 200, "idle": 0, "dtype": "f32"},
        # one chat: a penalty over the last tokens, a few biases
        {"name": "rules-1", "op": "rules", "rows": 1, "V": 128256, "history": 64, "biases": 3, "masks": 0},
        # a batch of answers with long histories, half of them in a grammar
        {"name": "rules-48", "op": "rules", "rows": 48, "V": 128256, "history": 4000, "biases": 300, "masks": 24},
    ]


HEADS = ((32, 8, 64), (32, 8, 64), (32, 8, 128), (32, 8, 128), (8, 2, 32), (6, 2, 128), (4, 2, 64), (16, 16, 64), (32, 4, 128), (16, 1, 128))


def draw(rng):
    """The ranges of the listed cases, sizes even over their logarithm."""
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["rope", "attend", "attend", "rules"])
    qH, kvH, d = rng.choice(HEADS)
    if op == "rope":
        rows = between(1, 9472)
        return {"op": "rope", "rows": rows, "qH": qH, "kvH": kvH, "d": d, "dims": rng.choice([d, d, d // 2]),
                "layout": rng.choice(["pairs", "halves"]), "scaling": rng.choice(["plain", "linear", "bands", "yarn"]),
                "far": between(max(rows, 100), 1000000), "cache": rows + between(1, 2000), "x": rng.choice(["f32", "f32", "f16", "bf16"]),
                "out": rng.choice(["f16", "bf16", "f32"])}
    if op == "rules":
        V = between(1000, 152000)
        rows = min(between(1, 256), 48 * 128256 // V)
        return {"op": "rules", "rows": rows, "V": V, "history": between(1, 8000), "biases": rng.choice([0, between(1, 20 * rows)]),
                "masks": rng.choice([0, rows, (rows + 1) // 2])}
    dtype = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
    batch = between(1, 256)
    most = (64 * 32 * 128 * 33000 if dtype != "f32" else 9 * 32 * 64 * 8000) // (batch * qH * d)
    prefix = between(1, max(2, min(131072, most)))
    capacity = between(16, max(17, min(4096, 65536 // batch)))
    return {"op": "attend", "batch": batch, "qH": qH, "kvH": kvH, "d": d, "prefix": prefix, "capacity": capacity,
            "own": max(1, int(capacity * rng.uniform(0.1, 0.9))), "idle": rng.choice([0, 0, batch // 10]), "dtype": dtype}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def frequencies(dims, scaling):
    """Angle per position of each pair, in 64 bits, and the factor of the cosines and sines: the frequencies as a model was trained
    with, positions pressed together by 4, the long waves stretched by 8 (the bands between by degrees), or by 16 with a factor."""
    base, out, magnitude = 500000.0, [], 1.0
    for i in range(dims // 2):
        f = base ** (-2.0 * i / dims)
        if scaling == "linear":
            f /= 4.0
        elif scaling == "bands":
            wave = 2 * math.pi / f
            keep = min(1.0, max(0.0, (8192 / wave - 1.0) / (4.0 - 1.0)))
            f = keep * f + (1 - keep) * f / 8.0
        elif scaling == "yarn":
            def place(turns):
                return dims * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
            lo, hi = max(0, math.floor(place(32.0))), min(dims - 1, math.ceil(place(1.0)))
            keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = keep * f + (1 - keep) * f / 16.0
            magnitude = 0.1 * math.log(16.0) + 1.0
        out.append(f)
    return out, magnitude


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    def whole(lo, hi, *shape):  # lo .. hi - 1
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int64)

    s = dict(case)
    if case["op"] == "rope":
        rows, width = case["rows"], case["kvH"] * case["d"]
        kind = DTYPES[case["out"]]
        s["in"] = normal(rows, (case["qH"] + 2 * case["kvH"]) * case["d"]).to(DTYPES[case["x"]])
        f, s["magnitude"] = frequencies(case["dims"], case["scaling"])
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        first = whole(0, max(1, case["far"] - rows), 1)
        s["positions"] = (first + torch.arange(rows, device="cuda") if rows > 256 else whole(0, case["far"], rows)).to(torch.int32)
        s["slots"] = torch.randperm(case["cache"], generator=g, device="cuda")[:rows].to(torch.int32)
        s["k"], s["v"] = normal(case["cache"], width).to(kind), normal(case["cache"], width).to(kind)
        s["q"] = torch.zeros(rows, case["qH"] * case["d"], dtype=kind, device="cuda")
    elif case["op"] == "attend":
        B, width, kind = case["batch"], case["kvH"] * case["d"], DTYPES[case["dtype"]]
        s["q"] = (1.5 * normal(B, case["qH"] * case["d"])).to(kind)
        s["kp"], s["vp"] = normal(case["prefix"], width).to(kind), normal(case["prefix"], width).to(kind)
        s["ko"], s["vo"] = normal(B, case["capacity"], width).to(kind), normal(B, case["capacity"], width).to(kind)
        # answers go on for about as long as one another; a few have just begun, some places of the batch are free
        lens = whole(max(0, case["own"] // 2), min(case["capacity"], case["own"] + case["own"] // 2) + 1, B)
        lens = torch.where(torch.rand(B, generator=g, device="cuda") < 0.05, lens % 3, lens)
        lens[B - case["idle"]:] = -1
        s["lens"] = lens.to(torch.int32)
        s["out"] = torch.zeros(B, case["qH"] * case["d"], dtype=kind, device="cuda")
    else:
        rows, V = case["rows"], case["V"]
        s["in"] = 3.0 * normal(rows, V)
        # words come again: ranks by a power law, spread over the vocabulary
        ranks = (V ** torch.rand(rows, case["history"], generator=g, device="cuda", dtype=torch.float64)).long()
        s["history"] = (ranks * 7919 % V).to(torch.int32)
        s["lens"] = whole(case["history"] // 2, case["history"] + 1, rows).to(torch.int32)
        uniform = torch.rand(3, rows, generator=g, device="cuda", dtype=torch.float32)
        s["repetition"], s["frequency"], s["presence"] = 1.0 + 0.3 * uniform[0], 0.5 * uniform[1], 0.6 * uniform[2]
        cuts = torch.sort(whole(0, case["biases"] + 1, max(0, rows - 1))).values
        ends = torch.tensor([case["biases"]], device="cuda")
        s["bias_start"] = torch.cat([ends * 0, cuts, ends]).to(torch.int32)
        s["bias_ids"] = whole(0, V, case["biases"]).to(torch.int32)
        s["bias"] = 4.0 * normal(case["biases"])
        words = (V + 31) // 32
        bits = whole(-(1 << 31), 1 << 31, case["masks"], words)
        few = torch.rand(case["masks"], 1, generator=g, device="cuda") < 0.5  # a grammar leaves few tokens, or most
        s["masks"] = torch.where(few, bits & whole(-(1 << 31), 1 << 31, case["masks"], words) & (bits >> 3), bits | (bits >> 5)).to(torch.int32)
        picked = torch.arange(rows, device="cuda") * max(1, rows // max(1, case["masks"]))
        s["mask_rows"] = torch.where(torch.arange(rows, device="cuda") < case["masks"], picked % max(1, case["masks"]), -1).to(torch.int32)
        s["out"] = torch.zeros(rows, V, dtype=torch.float32, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
_ctx = None


def _call(name, *args):
    """A call of the library on torch's current stream (1 is how CUDA names the default stream)."""
    global _ctx
    from nfai_b200 import CudaContext, _lib
    if _ctx is None:
        _ctx = CudaContext(torch.cuda.current_device())
    stream = torch.cuda.current_stream().cuda_stream or 1
    _lib.check(getattr(_lib.load(), name)(_ctx.handle, *args, stream), _ctx.handle)


def _own_rope(s):
    _call("nfai_op_rope_rows", s["in"].data_ptr(), CODES[s["x"]], 0, s["rows"], s["qH"], s["kvH"], s["d"], s["dims"],
          0 if s["layout"] == "pairs" else 1, s["freqs"].data_ptr(), s["magnitude"], s["positions"].data_ptr(), s["slots"].data_ptr(),
          s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), CODES[s["out"]], s["cache"])
    return s["q"], s["k"], s["v"]


def _own_attend(s):
    from nfai_b200 import _lib
    sizes = (CODES[s["dtype"]], s["batch"], s["qH"], s["kvH"], s["d"])
    if "scratch" not in s:  # a program makes it once for the largest step it will run
        need = _lib.load().nfai_op_attn_shared_scratch_bytes(*sizes, s["prefix"], s["capacity"])
        s["scratch"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    _call("nfai_op_attn_shared", s["q"].data_ptr(), s["kp"].data_ptr(), s["vp"].data_ptr(), s["prefix"], s["ko"].data_ptr(),
          s["vo"].data_ptr(), s["capacity"], s["lens"].data_ptr(), *sizes, 0.0, s["out"].data_ptr(), s["scratch"].data_ptr(),
          s["scratch"].numel())
    return s["out"]


def _own_rules(s):
    _call("nfai_op_logit_rules", s["in"].data_ptr(), s["rows"], s["V"], s["history"].data_ptr(), s["history"].shape[1], s["lens"].data_ptr(),
          s["repetition"].data_ptr(), s["frequency"].data_ptr(), s["presence"].data_ptr(), s["bias_start"].data_ptr(),
          s["bias_ids"].data_ptr(), s["bias"].data_ptr(), s["bias"].numel(), s["masks"].data_ptr(), s["masks"].shape[0],
          s["mask_rows"].data_ptr(), s["out"].data_ptr())
    return s["out"]


def _rotated(x, cos, sin, dims, layout):
    """x [rows][heads][d], cos and sin [rows][1][dims / 2]; what lies behind the first `dims` elements of a head stays."""
    if layout == "pairs":
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :dims // 2], x[..., dims // 2:dims]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., dims:]], dim=-1)


def _plain_rope(s):
    qH, kvH, d, kind = s["qH"], s["kvH"], s["d"], DTYPES[s["out"]]
    x = s["in"].float().view(s["rows"], qH + 2 * kvH, d)
    angle = s["positions"].double()[:, None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    turned = _rotated(x[:, :qH + kvH], cos, sin, s["dims"], s["layout"])
    at = s["slots"].long()
    s["k"][at] = turned[:, qH:].flatten(1).to(kind)
    s["v"][at] = x[:, qH + kvH:].flatten(1).to(kind)
    return turned[:, :qH].flatten(1).to(kind), s["k"], s["v"]


def _plain_attend(s):
    B, qH, kvH, d = s["batch"], s["qH"], s["kvH"], s["d"]
    q = s["q"].float().view(B, kvH, qH // kvH, d)
    kp, vp = (s[n].float().view(-1, kvH, d) for n in ("kp", "vp"))
    ko, vo = (s[n].float().view(B, -1, kvH, d) for n in ("ko", "vo"))
    seen = (torch.arange(s["capacity"], device="cuda") < s["lens"][:, None]).view(B, 1, 1, -1)
    scores = torch.cat([torch.einsum("bkgd,pkd->bkgp", q, kp), torch.einsum("bkgd,blkd->bkgl", q, ko).masked_fill(~seen, -math.inf)], dim=-1)
    scores = scores / math.sqrt(d)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weights.sum(-1, keepdim=True)
    wp, wo = weights[..., :s["prefix"]], weights[..., s["prefix"]:]
    out = (torch.einsum("bkgp,pkd->bkgd", wp, vp) + torch.einsum("bkgl,blkd->bkgd", wo, vo)) / total
    return torch.where(s["lens"][:, None] < 0, s["out"], out.reshape(B, -1).to(s["out"].dtype))


def _plain_rules(s):
    rows, V, x = s["rows"], s["V"], s["in"]
    place = torch.arange(s["history"].shape[1], device="cuda")
    ids = torch.where(place < s["lens"][:, None], s["history"].long(), V)
    count = torch.zeros(rows, V + 1, device="cuda").scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))[:, :V]
    rep = s["repetition"][:, None]
    y = torch.where(count > 0, torch.where(x > 0, x / rep, x * rep), x)
    y = y - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    # the last of several biases for a token counts
    entry = torch.arange(s["bias"].numel(), device="cuda")
    cell = torch.searchsorted(s["bias_start"][1:].long(), entry, right=True) * V + s["bias_ids"].long()
    last = torch.full((rows * V,), -1, dtype=torch.int64, device="cuda").scatter_reduce_(0, cell, entry, "amax").view(rows, V)
    y = torch.where(last >= 0, y + torch.cat([s["bias"], x.new_zeros(1)])[last], y)
    token = torch.arange(V, device="cuda")
    words = torch.cat([s["masks"], torch.full_like(s["masks"][:1], -1) if s["masks"].shape[0] else torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")])
    allowed = (words[s["mask_rows"].long()][:, token // 32] >> (token % 32).int()) & 1
    return torch.where(allowed != 0, y, -math.inf)


def run(state):
    if own:
        return _own_rope(state) if state["op"] == "rope" else _own_attend(state) if state["op"] == "attend" else _own_rules(state)
    return _plain_rope(state) if state["op"] == "rope" else _plain_attend(state) if state["op"] == "attend" else _plain_rules(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "rope":
        values = case["rows"] * (case["qH"] + 2 * case["kvH"]) * case["d"]
        return {"bytes": values * (SIZES[case["x"]] + SIZES[case["out"]]) + case["rows"] * 8 + case["dims"] * 4,
                "flops": 3 * case["rows"] * (case["qH"] + case["kvH"]) * case["dims"]}
    if case["op"] == "attend":
        busy = case["batch"] - case["idle"]
        keys = case["prefix"] + busy * case["own"]
        return {"bytes": (2 * keys * case["kvH"] + 2 * busy * case["qH"]) * case["d"] * SIZES[case["dtype"]],
                "flops": 4 * busy * case["qH"] * case["d"] * (case["prefix"] + case["own"])}
    values = case["rows"] * case["V"]
    return {"bytes": 8 * values + min(case["masks"], case["rows"]) * ((case["V"] + 31) // 32) * 4 + 3 * case["rows"] * case["history"] + 8 * case["biases"],
            "flops": 2 * values}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        qH, kvH, d, half = s["qH"], s["kvH"], s["d"], s["dims"] // 2
        x = s["in"].double().view(s["rows"], qH + 2 * kvH, d)
        # a pair as a complex number, turned by a complex number
        turn = s["magnitude"] * torch.exp(1j * (s["positions"].double()[:, None] * s["freqs"][None, :]))
        first = torch.arange(half, device="cuda") * (2 if s["layout"] == "pairs" else 1)
        second = first + (1 if s["layout"] == "pairs" else half)
        y = x.clone()
        for h in range(qH + kvH):
            z = torch.complex(x[:, h, first], x[:, h, second]) * turn
            y[:, h, first], y[:, h, second] = z.real, z.imag
        k, v = s["k"].double(), s["v"].double()
        k[s["slots"].long()] = y[:, qH:qH + kvH].reshape(s["rows"], -1)
        v[s["slots"].long()] = x[:, qH + kvH:].reshape(s["rows"], -1)
        return y[:, :qH].reshape(s["rows"], -1), k, v
    if case["op"] == "attend":
        B, qH, kvH, d = s["batch"], s["qH"], s["kvH"], s["d"]
        out = s["out"].double()
        kp, vp = s["kp"].double(), s["vp"].double()
        for b, n in enumerate(s["lens"].tolist()):
            if n < 0:
                continue
            k = torch.cat([kp, s["ko"][b, :n].double()]).view(-1, kvH, d).permute(1, 2, 0)
            v = torch.cat([vp, s["vo"][b, :n].double()]).view(-1, kvH, d).permute(1, 0, 2)
            p = torch.matmul(s["q"][b].double().view(kvH, qH // kvH, d), k) * d ** -0.5
            out[b] = torch.matmul(torch.softmax(p, dim=-1), v).reshape(-1)
        return out
    rows, V = s["rows"], s["V"]
    out = s["in"].double()
    starts, lens, picked = s["bias_start"].tolist(), s["lens"].tolist(), s["mask_rows"].tolist()
    shifts = torch.arange(32, device="cuda")
    for r in range(rows):
        tokens, times = torch.unique(s["history"][r, :lens[r]].long(), return_counts=True)
        at, rep = out[r, tokens], s["repetition"][r].double()
        at = torch.minimum(at * rep, at / rep)  # lower it either way (the penalty is at least one)
        out[r, tokens] = at - s["frequency"][r].double() * times - s["presence"][r].double()
        wanted = dict(zip(s["bias_ids"][starts[r]:starts[r + 1]].tolist(), s["bias"][starts[r]:starts[r + 1]].tolist()))
        if wanted:
            out[r, torch.tensor(list(wanted), device="cuda")] += torch.tensor(list(wanted.values()), dtype=torch.float64, device="cuda")
        if picked[r] >= 0:
            bits = ((s["masks"][picked[r]].long()[:, None] >> shifts) & 1).reshape(-1)[:V]
            out[r, bits == 0] = -math.inf
    return out
