"""Measured workloads of the multi-head attention operators: rotary positions, the per-head norm of
queries and keys with the rotation in the same pass, and softmax attention over packed sequences.

`run` with `own` false computes an operator in its plain form (elementary torch operations in 32
bits, angles and long sums in 64, one rounding at the end); with `own` true it makes the calls a
user of compare_gan_amd makes.  `exact` evaluates the definitions in 64 bits, written apart.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _rotary(name, **kw):
    case = {"name": name, "op": "rotary", "type": "bf16", "tokens": 1, "heads": 1, "dim": 64, "rot": 64,
            "layout": "half", "base": 10000.0, "scaling": "none", "factor": 1.0, "original": 4096,
            "axes": 1, "map": 0, "far": 4096, "grad": False}
    case.update(kw)
    return case


def _qk_norm(name, **kw):
    case = _rotary(name, op="qk_norm_rotary", kv_heads=1, merged=False)
    case.update(kw)
    return case


def _attention(name, **kw):
    case = {"name": name, "op": "attention", "heads": 1, "kv_heads": 1, "dim": 64, "dim_v": 64,
            "q_lengths": "1", "k_lengths": "", "capacity": 0, "causal": False, "grad": False}
    case.update(kw)
    return case


def listed():
    return [
        # the positions of one new token for each of 8 sequences, half of a 64-wide head turned:
        # the smallest call, where latency counts
        _rotary("rotary_new_tokens", tokens=8, heads=8, dim=64, rot=32, layout="interleaved"),
        # training on 64 maps of 64x64 (BigGAN-128's self-attention: batch 64, 192 channels in 3
        # heads), row and column each turning half of a head
        _rotary("rotary_maps_train", tokens=64 * 64 * 64, heads=3, dim=64, rot=64, axes=2, map=64,
                grad=True),
        # a long context in 32 bits, far beyond the length the frequencies were made for; odd counts
        _rotary("rotary_far_f32", type="f32", tokens=30011, heads=5, dim=80, rot=40, scaling="yarn",
                factor=16.0, far=131072, grad=True),
        # one new token for each of 64 sequences, 16 query heads over 4 key heads
        _qk_norm("qk_norm_new_tokens", tokens=64, heads=16, kv_heads=4, dim=128, rot=128, far=32768),
        # training on 16 maps of 64x64 with 192 channels in 6 heads, axial positions
        _qk_norm("qk_norm_maps_train", tokens=16 * 64 * 64, heads=6, kv_heads=6, dim=32, rot=32, axes=2,
                 map=64, grad=True),
        # ragged training batch: views into one merged projection, odd counts, part of the head
        _qk_norm("qk_norm_merged_train", tokens=10007, heads=12, kv_heads=4, dim=72, rot=36,
                 layout="interleaved", scaling="ntk", factor=4.0, merged=True, grad=True),
        # a batch of long prompts read in one pass
        _qk_norm("qk_norm_prompts", tokens=65536, heads=32, kv_heads=8, dim=128, rot=128,
                 scaling="linear", factor=8.0, far=65536),
        # training on 256 maps of 4x4 tokens (the smallest maps of a ResNet generator, 512 channels)
        _attention("attention_small_maps_train", heads=8, kv_heads=8, q_lengths="16*256", grad=True),
        # training on 64 maps of 64x64 tokens (BigGAN-128's self-attention with 3 heads of 64)
        _attention("attention_maps_train", heads=3, kv_heads=3, q_lengths="4096*64", grad=True),
        # one long prompt, causal, grouped heads
        _attention("attention_prompt", heads=16, kv_heads=4, dim=128, dim_v=128, q_lengths="16384",
                   causal=True),
        # training on packed sequences of different lengths (an empty one and single tokens among
        # them), causal, grouped heads, narrower values
        _attention("attention_ragged_train", heads=8, kv_heads=2, dim=96, dim_v=64, causal=True, grad=True,
                   q_lengths="2047,1,5000,333,0,64,129,4097,1,777,1500,63,2500,31,6001,1000"),
        # one new token for each of 48 sequences against a cache of 8192 rows a sequence
        _attention("attention_new_tokens", heads=32, kv_heads=8, dim=128, dim_v=128, causal=True,
                   q_lengths="1*48", capacity=8192,
                   k_lengths=",".join(str(1 + (i * 1777 + 4091) % 8192) for i in range(48))),
    ]


def _log_uniform(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rotation(rng, case, dim):
    axes = rng.choice((1, 1, 2))
    case["axes"] = axes
    most = dim // (2 * axes)
    case["rot"] = 2 * axes * (most if rng.random() < 0.5 else rng.randint(1, most))
    case["layout"] = rng.choice(("half", "interleaved"))
    case["scaling"] = rng.choice(("none", "linear", "ntk", "yarn"))
    case["factor"] = 1.0 if case["scaling"] == "none" else rng.choice((2.0, 4.0, 16.0))
    case["map"] = rng.choice((8, 33, 64)) if axes == 2 else 0
    case["far"] = _log_uniform(rng, 64, 131072)
    case["grad"] = rng.random() < 0.5


def _draw_lengths(rng, count, longest):
    return [0 if rng.random() < 0.05 else _log_uniform(rng, 1, longest) for _ in range(count)]


_MOST_PAIRS = 64 * 4096 * 4096 * 3 * 128 // 2


def draw(rng):
    kind = rng.choice(("rotary", "qk_norm_rotary", "attention", "attention"))
    if kind == "rotary":
        dim = 2 * rng.randint(4, 64)
        heads = rng.randint(1, 16)
        case = _rotary("", type=rng.choice(("bf16", "f32")), heads=heads, dim=dim,
                       tokens=_log_uniform(rng, 1, min(262144, 25000000 // (heads * dim))))
        _draw_rotation(rng, case, dim)
    elif kind == "qk_norm_rotary":
        dim = rng.choice((2 * rng.randint(4, 64), 32, 64, 128))
        kv_heads = rng.randint(1, 8)
        heads = kv_heads * rng.randint(1, 4)
        case = _qk_norm("", type=rng.choice(("bf16", "bf16", "f32")), heads=heads, kv_heads=kv_heads,
                        dim=dim, merged=rng.random() < 0.5,
                        tokens=_log_uniform(rng, 1, min(65536, 60000000 // ((heads + kv_heads) * dim))))
        _draw_rotation(rng, case, dim)
    else:
        kv_heads = rng.randint(1, 8)
        heads = kv_heads * rng.randint(1, 8)
        dim = 8 * rng.randint(1, 16)
        dim_v = dim if rng.random() < 0.5 else 8 * rng.randint(1, 16)
        form = rng.choice(("packed", "packed", "maps", "crossed", "new_tokens"))
        causal = rng.random() < 0.5
        capacity = 0
        k_lengths = ""
        if form == "maps":
            q = [rng.choice((4, 8, 12, 16, 32)) ** 2] * rng.randint(1, 64)
        elif form == "packed":
            q = _draw_lengths(rng, rng.randint(1, 24), 8192)
        else:
            count = rng.randint(1, 48)
            capacity = _log_uniform(rng, 64, 8192) if form == "new_tokens" else 0
            q = [1] * count if form == "new_tokens" else _draw_lengths(rng, count, 2048)
            k = _draw_lengths(rng, count, capacity or 4096)
            k_lengths = ",".join(str(x) for x in k)
        if not any(q):
            q[0] = 1
        k = k if k_lengths else q
        pairs = sum(a * b for a, b in zip(q, k)) * heads * (dim + dim_v)
        while pairs > _MOST_PAIRS:          # no drawn case costs more than the largest listed one
            q = [(x + 1) // 2 for x in q]
            if k_lengths:
                k = [(x + 1) // 2 for x in k]
                k_lengths = ",".join(str(x) for x in k)
            else:
                k = q
            pairs = sum(a * b for a, b in zip(q, k)) * heads * (dim + dim_v)
        case = _attention("", heads=heads, kv_heads=kv_heads, dim=dim, dim_v=dim_v, causal=causal,
                          q_lengths=",".join(str(x) for x in q), k_lengths=k_lengths,
                          capacity=capacity, grad=form != "new_tokens" and rng.random() < 0.5)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _lengths(text):
    out = []
    for part in text.split(","):
        value, _, times = part.partition("*")
        out += [int(value)] * int(times or 1)
    return out


def _attention_shape(case):
    q = _lengths(case["q_lengths"])
    k = _lengths(case["k_lengths"]) if case["k_lengths"] else list(q)
    q_starts = [sum(q[:i]) for i in range(len(q))]
    if case["capacity"]:
        k_starts = [i * case["capacity"] for i in range(len(k))]
        rows = len(k) * case["capacity"]
    else:
        k_starts = [sum(k[:i]) for i in range(len(k))]
        rows = sum(k)
    return q, k, q_starts, k_starts, sum(q), rows


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if case["op"] == "attention":
        _, _, _, _, q_rows, k_rows = _attention_shape(case)
        heads, kv_heads = case["heads"], case["kv_heads"]
        s = {"q": normal((q_rows, heads, case["dim"]), torch.bfloat16),
             "k": normal((k_rows, kv_heads, case["dim"]), torch.bfloat16),
             "v": normal((k_rows, kv_heads, case["dim_v"]), torch.bfloat16)}
        if case["grad"]:
            s["dout"] = normal((q_rows, heads, case["dim_v"]), torch.bfloat16)
        return s
    dtype = _TYPES[case["type"]]
    tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
    if case["axes"] == 2:
        side = case["map"]
        cell = torch.arange(tokens, device="cuda") % (side * side)
        shift = random.Random(seed).randrange(case["far"])
        positions = torch.stack((cell // side + shift, cell % side), 1).to(torch.int32)
    else:
        positions = torch.randint(0, case["far"], (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    s = {"positions": positions}
    if case["op"] == "rotary":
        s["x"] = normal((tokens, heads, dim), dtype)
        if case["grad"]:
            s["dy"] = normal((tokens, heads, dim), dtype)
        return s
    kv_heads = case["kv_heads"]
    if case["merged"]:
        merged = normal((tokens, heads + 2 * kv_heads, dim), dtype)
        s["q"], s["k"] = merged[:, :heads], merged[:, heads:heads + kv_heads]
    else:
        s["q"], s["k"] = normal((tokens, heads, dim), dtype), normal((tokens, kv_heads, dim), dtype)
    s["q_gain"] = 1.0 + 0.2 * normal((dim,), torch.float32)
    s["k_gain"] = 1.0 + 0.2 * normal((dim,), torch.float32)
    if case["grad"]:
        s["dq"], s["dk"] = normal((tokens, heads, dim), dtype), normal((tokens, kv_heads, dim), dtype)
    return s


_EPS = 1e-6


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "attention":
        q, k, q_starts, k_starts, _, _ = _attention_shape(case)
        state["shape"] = (q, k, q_starts, k_starts)
        if own:
            from compare_gan_amd.hip import kernels as K
            state["plan"] = K.AttentionPlan(q, k, heads=case["heads"], kv_heads=case["kv_heads"],
                                            causal=case["causal"], k_starts=k_starts, device="cuda")
        else:
            state["groups"] = _plain_groups(q, k, q_starts, k_starts)
        wanted = ("q", "k", "v")
    else:
        if own:
            from compare_gan_amd.hip import kernels as K
            state["table"] = K.RotaryTable(case["rot"], layout=case["layout"], base=case["base"],
                                           scaling=case["scaling"], factor=case["factor"],
                                           original_length=case["original"], axes=case["axes"],
                                           device="cuda")
        else:
            state["frequencies"], state["amplitude"] = _frequencies(case)
        wanted = ("x",) if case["op"] == "rotary" else ("q", "k", "q_gain", "k_gain")
    if own and case["grad"]:
        for name in wanted:
            state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if case["op"] == "rotary":
        return _own_rotary(state) if own else _plain_rotary(state)
    return _own_qk_norm(state) if own else _plain_qk_norm(state)


def _own_rotary(s):
    from compare_gan_amd.hip import functional as Fn
    if not s["case"]["grad"]:
        return {"y": Fn.rotary(s["x"], s["positions"], s["table"])}
    y = Fn.rotary(s["x"], s["positions"], s["table"])
    (dx,) = torch.autograd.grad(y, (s["x"],), s["dy"])
    return {"y": y.detach(), "dx": dx}


def _own_qk_norm(s):
    from compare_gan_amd.hip import functional as Fn
    q, k = Fn.qk_norm_rotary(s["q"], s["k"], s["q_gain"], s["k_gain"], s["positions"], s["table"], eps=_EPS)
    if not s["case"]["grad"]:
        return {"q": q, "k": k}
    dq, dk, dq_gain, dk_gain = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_gain"], s["k_gain"]),
                                                   (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dq_gain": dq_gain, "dk_gain": dk_gain}


def _own_attention(s):
    from compare_gan_amd.hip import functional as Fn
    out = Fn.packed_attention(s["q"], s["k"], s["v"], s["plan"])
    if not s["case"]["grad"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians a position for every pair of the turned part (float64), and the amplitude."""
    n = case["rot"] // 2 // case["axes"]
    i = torch.arange(n, dtype=torch.float64, device="cuda")
    base, factor, amplitude = case["base"], case["factor"], 1.0
    if case["scaling"] == "ntk" and n > 1:
        base = base * factor ** (n / (n - 1.0))
    f = base ** (-i / n)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "yarn":
        turns = case["original"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f, amplitude


def _plain_cos_sin(s):
    positions = s["positions"].reshape(s["positions"].shape[0], -1).double()
    angles = (positions[:, :, None] * s["frequencies"]).flatten(1)
    return ((torch.cos(angles) * s["amplitude"]).float()[:, None],
            (torch.sin(angles) * s["amplitude"]).float()[:, None])


def _plain_turn(x, cos, sin, case):
    """x fp32 [T, H, D] with the first `rot` entries of each head turned by the angles."""
    rot = case["rot"]
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat((first, second), -1) if case["layout"] == "half" else torch.stack(
        (first, second), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(s):
    case, x = s["case"], s["x"]
    cos, sin = _plain_cos_sin(s)
    out = {"y": _plain_turn(x.float(), cos, sin, case).to(x.dtype)}
    if case["grad"]:
        out["dx"] = _plain_turn(s["dy"].float(), cos, -sin, case).to(x.dtype)
    return out


def _plain_qk_norm(s):
    case = s["case"]
    cos, sin = _plain_cos_sin(s)
    out, grads, gains = {}, {}, {}
    for name in ("q", "k"):
        x, gain = s[name].float(), s[name + "_gain"]
        inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        unit = x * inv
        out[name] = _plain_turn(unit * gain, cos, sin, case).to(s[name].dtype)
        if case["grad"]:
            g = _plain_turn(s["d" + name].float(), cos, -sin, case)
            gains["d" + name + "_gain"] = (g * unit).double().sum((0, 1)).float()
            g = g * gain
            grads["d" + name] = (inv * (g - unit * (g * unit).mean(-1, keepdim=True))).to(s[name].dtype)
    out.update(grads)
    out.update(gains)
    return out


_MOST_SCORES = 1 << 28


def _plain_groups(q, k, q_starts, k_starts):
    """Sequences of equal lengths go through the products together: (lq, lk, rows of q, rows of k)."""
    same = {}
    for i, key in enumerate(zip(q, k)):
        if key[0]:
            same.setdefault(key, []).append(i)
    out = []
    for (lq, lk), members in same.items():
        rows_q = torch.tensor([q_starts[i] for i in members], device="cuda")[:, None] + torch.arange(
            lq, device="cuda")
        rows_k = torch.tensor([k_starts[i] for i in members], device="cuda")[:, None] + torch.arange(
            lk, device="cuda")
        out.append((lq, lk, rows_q, rows_k))
    return out


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    shared = heads // kv_heads
    scale = 1.0 / math.sqrt(case["dim"])
    out = torch.zeros((q.shape[0], heads, v.shape[2]), dtype=torch.float32, device=q.device)
    if case["grad"]:
        dq = torch.zeros_like(q, dtype=torch.float32)
        dk = torch.zeros_like(k, dtype=torch.float32)
        dv = torch.zeros_like(v, dtype=torch.float32)
    for lq, lk, all_q, all_k in s["groups"]:
        if lk == 0:
            continue
        allowed = None
        if case["causal"]:
            allowed = (torch.arange(lk, device=q.device)[None, :] <=
                       torch.arange(lq, device=q.device)[:, None] + (lk - lq))
        step = max(1, _MOST_SCORES // (heads * lq * lk))
        slices = [slice(0, kv_heads)] if heads * lq * lk <= _MOST_SCORES else [
            slice(h, h + 1) for h in range(kv_heads)]
        for at in range(0, all_q.shape[0], step):
            rows_q, rows_k = all_q[at:at + step], all_k[at:at + step]
            for part in slices:
                mine = slice(part.start * shared, part.stop * shared)
                hk = part.stop - part.start

                def queries(x):     # [n, lq, heads, d] -> [n, kv heads, shared, lq, d]
                    return x[:, :, mine].float().permute(0, 2, 1, 3).reshape(
                        rows_q.shape[0], hk, shared, lq, -1)

                def keys(x):        # [n, lk, kv heads, d] -> [n, kv heads, 1, lk, d]
                    return x[:, :, part].float().permute(0, 2, 1, 3)[:, :, None].contiguous()

                def back(x):        # queries' inverse
                    return x.reshape(rows_q.shape[0], hk * shared, lq, -1).permute(0, 2, 1, 3)

                qs, ks, vs = queries(q[rows_q]), keys(k[rows_k]), keys(v[rows_k])
                kt = ks.transpose(-1, -2).contiguous()
                p = torch.matmul(qs, kt.expand(-1, -1, shared, -1, -1)) * scale
                if allowed is not None:
                    p = p.masked_fill(~allowed, -math.inf)
                top = p.amax(-1, keepdim=True)
                top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                p = torch.exp(p - top)
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, torch.ones_like(total), total)
                out[rows_q, mine] = back(torch.matmul(p, vs.expand(-1, -1, shared, -1, -1)))
                if not case["grad"]:
                    continue
                do = queries(s["dout"][rows_q])
                dv[rows_k, part] = torch.matmul(p.transpose(-1, -2).contiguous(), do).sum(2).permute(
                    0, 2, 1, 3)
                ds = torch.matmul(do, vs.transpose(-1, -2).contiguous().expand(-1, -1, shared, -1, -1))
                ds = p * (ds - (p * ds).sum(-1, keepdim=True)) * scale
                dq[rows_q, mine] = back(torch.matmul(ds, ks.expand(-1, -1, shared, -1, -1)))
                dk[rows_k, part] = torch.matmul(ds.transpose(-1, -2).contiguous(), qs).sum(2).permute(
                    0, 2, 1, 3)
    if not case["grad"]:
        return {"out": out.to(q.dtype)}
    return {"out": out.to(q.dtype), "dq": dq.to(q.dtype), "dk": dk.to(k.dtype), "dv": dv.to(v.dtype)}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        q, k, _, _, _, _ = _attention_shape(case)
        heads, kv_heads, dim, dim_v = case["heads"], case["kv_heads"], case["dim"], case["dim_v"]
        pairs = 0
        for lq, lk in zip(q, k):
            if case["causal"]:
                whole = min(lq, lk)         # the last min(lq, lk) rows see lk - whole + 1 .. lk keys
                pairs += whole * lk - whole * (whole - 1) // 2
            else:
                pairs += lq * lk
        at_q = 2 * sum(q) * heads
        at_k = 2 * sum(b for a, b in zip(q, k) if a) * kv_heads
        size = at_q * (dim + dim_v) + at_k * (dim + dim_v)
        flops = 2 * pairs * heads * (dim + dim_v)
        if case["grad"]:                    # dout in, three gradients out; four more products
            size += at_q * (dim_v + dim) + at_k * (dim + dim_v)
            flops *= 3
        return {"bytes": size, "flops": flops}
    each = 2 if case["type"] == "bf16" else 4
    heads = case["heads"] + case.get("kv_heads", 0)
    elements = case["tokens"] * heads * case["dim"]
    size = 2 * elements * each + 4 * case["tokens"] * case["axes"]
    flops = elements * (3 if case["op"] == "rotary" else 6)
    if case["grad"]:
        size += 2 * elements * each
        flops += elements * (3 if case["op"] == "rotary" else 10)
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    pairs = case["rot"] // 2
    each = pairs // case["axes"]
    # one complex number e^{i angle} for each token and pair
    columns = []
    positions = s["positions"].reshape(case["tokens"], -1).to(torch.float64)
    amplitude = 1.0 + 0.1 * math.log(case["factor"]) if case["scaling"] == "yarn" else 1.0
    for pair in range(pairs):
        axis, i = divmod(pair, each)
        base = case["base"]
        if case["scaling"] == "ntk" and each > 1:
            base *= case["factor"] ** (each / (each - 1.0))
        f = base ** (-float(i) / each)
        if case["scaling"] == "linear":
            f /= case["factor"]
        if case["scaling"] == "yarn":
            r = case["original"] * f / (2 * math.pi)
            ramp = min(1.0, max(0.0, (r - 1.0) / (32.0 - 1.0)))
            f = (1.0 - ramp) * f / case["factor"] + ramp * f
        angle = positions[:, axis] * f
        columns.append(torch.polar(torch.full_like(angle, amplitude), angle))
    turn = torch.stack(columns, 1)[:, None]
    if case["layout"] == "half":
        first = list(range(pairs))
        second = list(range(pairs, 2 * pairs))
    else:
        first = list(range(0, 2 * pairs, 2))
        second = list(range(1, 2 * pairs, 2))

    def turned(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        y = x.clone()
        y[..., first] = z.real
        y[..., second] = z.imag
        return y

    if case["op"] == "rotary":
        out = {"y": turned(s["x"].double(), turn)}
        if case["grad"]:
            out["dx"] = turned(s["dy"].double(), turn.conj())
        return out
    values, grads, gains = {}, {}, {}
    for name in ("q", "k"):
        x, gain = s[name].double(), s[name + "_gain"].double()
        norm = torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + _EPS)
        values[name] = turned(x / norm * gain, turn)
        if case["grad"]:
            g = turned(s["d" + name].double(), turn.conj())
            gains["d" + name + "_gain"] = torch.einsum("thd,thd->d", g, x / norm)
            g = g * gain
            along = (g * x).sum(-1, keepdim=True) / (case["dim"] * norm ** 3)
            grads["d" + name] = g / norm - x * along
    values.update(grads)
    values.update(gains)
    return values


def _exact_attention(case, s):
    lens_q, lens_k, q_starts, k_starts, _, _ = _attention_shape(case)
    pairs = sum(a * b for a, b in zip(lens_q, lens_k)) * case["heads"]
    if pairs * (case["dim"] + case["dim_v"]) > 3e12 or sum(1 for a in lens_q if a) * case["heads"] > 20000:
        return None
    shared = case["heads"] // case["kv_heads"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.zeros(q.shape[:2] + v.shape[2:], dtype=torch.float64, device=q.device)
    if case["grad"]:
        do = s["dout"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for lq, lk, q0, k0 in zip(lens_q, lens_k, q_starts, k_starts):
        # row i of a causal sequence sees the keys 0 .. i + lk - lq
        first = max(0, lq - lk) if case["causal"] else 0
        if lk == 0 or first >= lq:
            continue
        rows, cols = slice(q0 + first, q0 + lq), slice(k0, k0 + lk)
        for h in range(case["heads"]):
            g = h // shared
            kk, vv = k[cols, g].contiguous(), v[cols, g].contiguous()
            qq = q[rows, h].contiguous()
            logits = qq @ kk.t().contiguous() / math.sqrt(case["dim"])
            if case["causal"]:
                last = torch.arange(first, lq, device=q.device) + (lk - lq)
                logits[torch.arange(lk, device=q.device)[None, :] > last[:, None]] = -math.inf
            prob = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
            del logits
            o = prob @ vv
            out[rows, h] = o
            if case["grad"]:
                dd = do[rows, h].contiguous()
                dv[cols, g] += prob.t().contiguous() @ dd
                inner = prob * (dd @ vv.t().contiguous() - (dd * o).sum(-1, keepdim=True))
                inner /= math.sqrt(case["dim"])
                dq[rows, h] = inner @ kk
                dk[cols, g] += inner.t().contiguous() @ qq
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["grad"] else {"out": out}
