"""The token operators as they are measured: multi-axis rotary positions, cross attention to an encoder's states, and the AdamW step
over many tensors, each with the plain form that it has to agree with.

A case is one call as a program makes it: keypoint queries (animals x nodes) that read the feature-map tokens of a frame or of a
clip of frames, forward or with gradients, and the optimizer step over the tensors of a backbone.
"""
import math

import torch

own = False  # False: the plain forms; True: the package's operators

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 10000.0
BETA1, BETA2, EPS, DECAY, LR, STEP = 0.9, 0.999, 1e-8, 0.01, 2e-3, 100


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------
def listed():
    return [
        # 4 animals x 13 nodes of one frame at sub-pixel (x, y): the smallest rotary call, all latency
        dict(name="rope_queries", op="rope", dtype="fp16", batch=1, frames=1, rows=1, cols=52, points=True, heads=8, dim=64, sections="16,16",
             interleaved=False, ladder="axis", grad=False),
        # two clips of 8 frames, the 64 x 64 map (1024 pixels at stride 16) of each as (t, y, x) tokens
        dict(name="rope_clip", op="rope", dtype="bf16", batch=2, frames=8, rows=64, cols=64, points=False, heads=8, dim=64, sections="8,12,12",
             interleaved=False, ladder="axis", grad=False),
        # float32 features of odd maps, neighbouring pairs, part of the head left as it is; with the gradient
        dict(name="rope_odd_grad", op="rope", dtype="fp32", batch=3, frames=5, rows=37, cols=53, points=False, heads=6, dim=80,
             sections="8,15,13", interleaved=True, ladder="shared", grad=True),
        # the 52 queries of one frame read its 32 x 32 map (1024 pixels at stride 32): latency
        dict(name="attn_frame", op="attn", dtype="fp16", batch=1, queries=52, keys=1024, heads=8, kv_heads=8, dim=32, ragged="none", grad=False),
        # one new query token per video against 4 frames of 64 x 64 tokens, shared heads, clips of different lengths
        dict(name="attn_token", op="attn", dtype="bf16", batch=32, queries=1, keys=16384, heads=8, kv_heads=2, dim=128, ragged="lengths", grad=False),
        # every token of a 64 x 64 map reads a clip of 4 such maps: the largest
        dict(name="attn_clip", op="attn", dtype="bf16", batch=2, queries=4096, keys=16384, heads=8, kv_heads=8, dim=128, ragged="none", grad=False),
        # frames of different sizes padded to one batch (one of them empty), hidden tokens inside, odd everything
        dict(name="attn_ragged", op="attn", dtype="fp16", batch=6, queries=193, keys=2917, heads=12, kv_heads=4, dim=72, ragged="both", grad=False),
        # training: 8 animals x 24 nodes on the 64 x 64 map of each of 8 frames
        dict(name="attn_queries_grad", op="attn", dtype="bf16", batch=8, queries=192, keys=4096, heads=8, kv_heads=8, dim=64, ragged="none", grad=True),
        # training: a map's tokens on two maps, long both ways
        dict(name="attn_clip_grad", op="attn", dtype="bf16", batch=1, queries=4096, keys=8192, heads=8, kv_heads=8, dim=128, ragged="none", grad=True),
        # training on padded odd maps with shared heads
        dict(name="attn_ragged_grad", op="attn", dtype="fp16", batch=3, queries=417, keys=1531, heads=8, kv_heads=2, dim=40, ragged="both", grad=True),
        # the 16-filter UNet that the benchmark model is: few small tensors
        dict(name="adamw_unet", op="adamw", dtype="fp32", family="unet", width=16, depth=5, amsgrad=False),
        # 66 M parameters in 3 x 3 x 256 x 256 kernels with their normalisations, as one hourglass stack holds
        dict(name="adamw_hourglass", op="adamw", dtype="fp32", family="residual", width=256, depth=112, amsgrad=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "rope", "attn", "attn", "attn", "adamw"])
    if op == "rope":
        while True:
            c = dict(op="rope", dtype=rng.choice(["fp16", "bf16", "fp32"]), batch=_log(rng, 1, 8), frames=_log(rng, 1, 16), rows=_log(rng, 1, 96),
                     cols=_log(rng, 1, 96), points=rng.random() < 0.25, heads=rng.randint(1, 16), dim=2 * rng.randint(6, 64), sections="",
                     interleaved=rng.random() < 0.5, ladder=rng.choice(["axis", "shared"]), grad=rng.random() < 0.4)
            pairs, axes = c["dim"] // 2, 2 if c["points"] else 3
            sections = [rng.randint(1, pairs // axes) for _ in range(axes)]
            c["sections"] = ",".join(str(s) for s in sections)
            if work(c)["bytes"] <= 1.3e8:
                return c
    if op == "attn":
        while True:
            kv_heads = rng.choice([1, 2, 3, 4, 8])
            c = dict(op="attn", dtype=rng.choice(["fp16", "bf16"]), batch=_log(rng, 1, 32), queries=_log(rng, 1, 4096), keys=_log(rng, 1, 16384),
                     heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads, dim=8 * rng.randint(2, 16),
                     ragged=rng.choice(["none", "lengths", "mask", "both"]), grad=rng.random() < 0.5)
            scores = c["batch"] * c["heads"] * c["queries"] * c["keys"]
            if scores <= (2.6e8 if c["grad"] else 1.0e9) and work(c)["bytes"] <= 5e8 and work(c)["flops"] <= 5e11:
                return c
    family = rng.choice(["unet", "residual"])
    return dict(op="adamw", dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), family=family,
                width=rng.randint(5, 40) if family == "unet" else rng.randint(24, 240), depth=rng.randint(2, 5) if family == "unet" else rng.randint(3, 110),
                amsgrad=rng.random() < 0.3)


def tensor_sizes(case):
    """Element counts of the parameters of a backbone, layer by layer: kernels of 3 x 3 with their biases (a UNet of `depth` halvings
    with two convolutions a level), or `depth` square kernels with bias, gain and shift."""
    w = case["width"]
    if case["family"] == "residual":
        return [n for _ in range(case["depth"]) for n in (9 * w * w, w, w, w)]
    sizes, cin = [], 1
    for level in range(case["depth"] + 1):
        cout = w << level
        sizes += [9 * cin * cout, cout, 9 * cout * cout, cout]
        cin = cout
    for level in range(case["depth"] - 1, 1, -1):
        cout = w << level
        sizes += [9 * (cin + cout) * cout, cout, 9 * cout * cout, cout]
        cin = cout
    return sizes + [13 * cin, 13, 24 * cin, 24]


def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def work(case):
    if case["op"] == "rope":
        size = 4 if case["dtype"] == "fp32" else 2
        tokens = case["frames"] * case["rows"] * case["cols"]
        n = case["batch"] * tokens * case["heads"] * case["dim"]
        passes = 2 if case["grad"] else 1
        places = case["batch"] * tokens * 2 * 4 if case["points"] else tokens * 3 * 4
        return {"bytes": passes * 2 * n * size + places, "flops": passes * 3 * n}
    if case["op"] == "attn":
        q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
        kv = case["batch"] * case["keys"] * case["kv_heads"] * case["dim"]
        product = 2 * case["batch"] * case["heads"] * case["queries"] * case["keys"] * case["dim"]
        if case["ragged"] in ("lengths", "both"):  # lengths lie between a half and the whole; of three images and more two are as good as empty
            part = 0.75 * (case["batch"] - 2 if case["batch"] > 2 else case["batch"]) / case["batch"]
            kv, product = part * kv, part * product
        if case["grad"]:  # q, k, v and the output's gradient in; the output and three gradients out
            return {"bytes": 2 * (4 * q + 4 * kv), "flops": 7 * product}
        return {"bytes": 2 * (2 * q + 2 * kv), "flops": 2 * product}
    n = sum(tensor_sizes(case))
    size = 4 if case["dtype"] == "fp32" else 2
    states = 3 if case["amsgrad"] else 2
    return {"bytes": n * (3 * size + 8 * states), "flops": 14 * n}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if case["op"] == "rope":
        tokens = case["frames"] * case["rows"] * case["cols"]
        s["sections"] = _sections(case)
        s["x"] = normal(case["batch"], tokens, case["heads"], case["dim"])
        if case["points"]:  # a batch of keypoints: pixels of a 1024 x 1024 frame, refined below the pixel
            s["positions"] = torch.rand((case["batch"], tokens, 2), generator=g, device="cuda") * 1024
        else:  # (time, row, column); the clip starts somewhere in a long video
            start = int(torch.randint(0, 2_000_000, (1,), generator=g, device="cuda"))
            s["positions"] = torch.stack(torch.meshgrid(torch.arange(case["frames"], device="cuda") + start, torch.arange(case["rows"], device="cuda"),
                                                        torch.arange(case["cols"], device="cuda"), indexing="ij"), -1).reshape(tokens, 3).to(torch.int32)
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dout"] = normal(case["batch"], tokens, case["heads"], case["dim"])
        return s
    if case["op"] == "attn":
        B, Tq, Tk, H, K, D = (case[n] for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
        s["q"] = normal(B, Tq, H, D, scale=1.5)
        s["k"], s["v"] = normal(B, Tk, K, D), normal(B, Tk, K, D)
        s["lengths"] = s["mask"] = None
        seen = torch.ones((B, Tk), dtype=torch.bool, device="cuda")
        if case["ragged"] in ("lengths", "both"):
            n = torch.randint((Tk + 1) // 2, Tk + 1, (B,), generator=g, device="cuda")
            if B > 2:
                n[1], n[2] = 0, min(Tk, 1)  # an image without a token, and one with a single token
            s["lengths"] = n.to(torch.int32)
            seen &= torch.arange(Tk, device="cuda")[None, :] < n[:, None]
        if case["ragged"] in ("mask", "both"):
            s["mask"] = torch.rand((B, Tk), generator=g, device="cuda") < 0.8
            seen &= s["mask"]
        hidden = ~seen[:, :, None, None]
        s["k"].masked_fill_(hidden, float("nan"))  # what padding holds is nobody's business
        s["v"].masked_fill_(hidden, float("inf"))
        if case["grad"]:
            for n in "qkv":
                s[n].requires_grad_(True)
            s["dout"] = normal(B, Tq, H, D)
        return s
    sizes = tensor_sizes(case)
    starts, total = [], 0
    for n in sizes:  # each tensor begins on a line of its own, as an allocator gives it
        starts.append(total)
        total += (n + 63) // 64 * 64
    filled = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        filled[a:a + n] = True

    def flat(make):
        t = make(torch.randn(total, generator=g, device="cuda"))
        return torch.where(filled, t, torch.zeros_like(t))

    s["param"], s["grad_"] = flat(lambda t: (t * 0.05).to(dtype)), flat(lambda t: (t * 1e-2).to(dtype))
    s["exp_avg"], s["exp_avg_sq"] = flat(lambda t: t * 2e-3), flat(lambda t: (t * 1e-2).square() * 0.1)
    if case["amsgrad"]:
        s["max_exp_avg_sq"] = s["exp_avg_sq"] * 1.1
    for n in [n for n in ("param", "grad_", "exp_avg", "exp_avg_sq", "max_exp_avg_sq") if n in s]:
        s[n + "s"] = [s[n][a:a + k] for a, k in zip(starts, sizes)]
    return s


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def run(state):
    return {"rope": _rope, "attn": _attn, "adamw": _adamw}[state["op"]](state)


def _rope(s):
    if own:
        from sleap_amd import ops

        y = ops.rotary_axes(s["x"], s["positions"], s["sections"], theta=THETA, ladder=s["ladder"], interleaved=s["interleaved"])
        if not s["grad"]:
            return y
        return [y.detach(), torch.autograd.grad(y, s["x"], s["dout"])[0]]
    with torch.no_grad():
        sections, pairs = s["sections"], sum(s["sections"])
        # angles in 64 bits: a frame index of millions times a frequency of one leaves few bits of 32 for the fraction of a turn
        axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda")
        power = [i / n for n in sections for i in range(n)] if s["ladder"] == "axis" else [i / pairs for i in range(pairs)]
        turn = s["positions"].double()[..., axis] * torch.tensor([THETA ** -p for p in power], dtype=torch.float64, device="cuda")
        c, n = turn.cos().float()[..., None, :], turn.sin().float()[..., None, :]
        y = _rotated(s, s["x"], c, n, pairs)
        return [y, _rotated(s, s["dout"], c, -n, pairs)] if s["grad"] else y


def _rotated(s, x, c, n, pairs):
    y = x.float().clone()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if s["interleaved"] else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * n, b * c + a * n
    return y.to(x.dtype)


def _attn(s):
    if own:
        from sleap_amd import ops

        out = ops.cross_attention(s["q"], s["k"], s["v"], key_lengths=s["lengths"], key_mask=s["mask"])
        if not s["grad"]:
            return out
        return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])]
    with torch.no_grad():
        B, Tq, H, D = s["q"].shape
        Tk, K = s["k"].shape[1:3]
        seen = _seen(s, B, Tk)
        rows = lambda t: t.float().reshape(B, Tq, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * Tq, D)  # noqa: E731
        back = lambda t: t.reshape(B, K, H // K, Tq, D).permute(0, 3, 1, 2, 4).reshape(B, Tq, H, D).to(s["q"].dtype)  # noqa: E731
        q = rows(s["q"])
        k, v = (t.float().masked_fill(~seen[:, :, None, None], 0.0).transpose(1, 2).contiguous() for t in (s["k"], s["v"]))
        scale = 1.0 / math.sqrt(D)
        w = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(~seen[:, None, None, :], float("-inf"))
        top = w.amax(-1, keepdim=True)
        w = w.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
        total = w.sum(-1, keepdim=True)
        w = w.div_(torch.where(total == 0, torch.ones_like(total), total))
        out = torch.matmul(w, v)
        if not s["grad"]:
            return back(out)
        do = rows(s["dout"])
        dv = torch.matmul(w.transpose(2, 3), do)
        dw = torch.matmul(do, v.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(w).mul_(scale)
        dq, dk = torch.matmul(dw, k), torch.matmul(dw.transpose(2, 3), q)
        return [back(out), back(dq), dk.transpose(1, 2).to(s["k"].dtype).contiguous(), dv.transpose(1, 2).to(s["v"].dtype).contiguous()]


def _seen(s, B, Tk):
    seen = torch.ones((B, Tk), dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        seen = seen & (torch.arange(Tk, device="cuda")[None, :] < s["lengths"][:, None])
    return seen if s["mask"] is None else seen & s["mask"]


def _adamw(s):
    if own:
        from sleap_amd import ops

        ops.adamw_step(s["params"], s["grad_s"], s["exp_avgs"], s["exp_avg_sqs"], max_exp_avg_sqs=s.get("max_exp_avg_sqs"), step=STEP, lr=LR,
                       betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY)
    else:  # all tensors as the one run of values that they lie in
        g = s["grad_"].float()
        m = s["exp_avg"].mul_(BETA1).add_(g, alpha=1 - BETA1)
        v = s["exp_avg_sq"].mul_(BETA2).add_(g * g, alpha=1 - BETA2)
        if s["amsgrad"]:
            v = torch.maximum(s["max_exp_avg_sq"], v, out=s["max_exp_avg_sq"])
        down = v.sqrt().div_(math.sqrt(1 - BETA2 ** STEP)).add_(EPS)
        p = s["param"].float() * (1 - LR * DECAY) - (m / down).mul_(LR / (1 - BETA1 ** STEP))
        s["param"].copy_(p)
    return {n: s[n] for n in ("param", "exp_avg", "exp_avg_sq", "max_exp_avg_sq") if n in s}


# --------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rope":
            y = _turned(s, s["x"], 1.0)
            return [y, _turned(s, s["dout"], -1.0)] if case["grad"] else y
        if case["op"] == "attn":
            return _attention_by_heads(s)
        g, m, v = s["grad_"].double(), s["exp_avg"].double(), s["exp_avg_sq"].double()
        m, v = m + (1 - BETA1) * (g - m), v + (1 - BETA2) * (g ** 2 - v)
        got = {"exp_avg": m, "exp_avg_sq": v}
        if case["amsgrad"]:
            got["max_exp_avg_sq"] = v = torch.max(v, s["max_exp_avg_sq"].double())
        p = s["param"].double()
        got["param"] = p - LR * (DECAY * p + (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)) ** 0.5 + EPS))
        return got


def _turned(s, x, sign):
    """Each pair as a complex number, times the unit number of its axis's angle."""
    y, pair, pairs = x.double().clone(), 0, sum(s["sections"])
    for axis, n in enumerate(s["sections"]):
        for i in range(n):
            angle = sign * s["positions"][..., axis].double() * math.exp(-math.log(THETA) * (i / n if s["ladder"] == "axis" else pair / pairs))
            at = (2 * pair, 2 * pair + 1) if s["interleaved"] else (pair, pair + pairs)
            z = torch.complex(x[..., at[0]].double(), x[..., at[1]].double()) * torch.polar(torch.ones_like(angle), angle)[..., None]
            y[..., at[0]], y[..., at[1]] = z.real, z.imag
            pair += 1
    return y


def _attention_by_heads(s):
    """Each image and head by itself, over the tokens that it sees alone."""
    q, k, v = (s[n].detach().double() for n in "qkv")
    B, Tq, H, D = q.shape
    Tk, K = k.shape[1:3]
    seen = _seen(s, B, Tk)
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        at = seen[b].nonzero()[:, 0]
        if not len(at):
            continue
        for h in range(H):
            kh, vh, qh = k[b, at, h // (H // K)], v[b, at, h // (H // K)], q[b, :, h]
            w = torch.softmax(qh @ kh.T / D ** 0.5, -1)
            out[b, :, h] = w @ vh
            if s["grad"]:
                do = s["dout"][b, :, h].double()
                dw = do @ vh.T
                ds = w * (dw - (w * dw).sum(-1, keepdim=True)) / D ** 0.5
                dq[b, :, h] = ds @ kh
                dk[b, at, h // (H // K)] += ds.T @ qh
                dv[b, at, h // (H // K)] += w.T @ do
    return [out, dq, dk, dv] if s["grad"] else out
