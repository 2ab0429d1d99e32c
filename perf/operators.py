"""Operators of training a scene's association of points to superpoints, and the optimiser steps beside it.

  adamw        `adamw_step`: decoupled-decay Adam over a list of tensors at once, 32-bit moments, gradients optionally clipped by
               the norm of all of them together
  adamw8       `adamw8_step`: the same with both moments in 8 bits, blocks of 256 elements under a power of two each; the moments
               come back as the values that they stand for (`adamw8_moments`; at most four significant bits: exact in bfloat16)
  balance      `balance_loss`: softmax over the superpoints, how often each is among a point's K largest, and the loss
               M * sum(share of the choices * mean probability), with its gradient by the logits
  neighbours   `neighbour_balance`: the same loss on the neighbour weights of points that see K superpoints each

`own` says whose form `run` takes: this package's entry points, or the elementary torch operations below.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BETAS = (0.9, 0.999)
DECAY = 0.01
BLOCK = 256  # elements under one pair of scales of the 8-bit moments
# per-point parameters of a scene (columns, learning rate): positions, first and further SH coefficients, scales, rotations, opacity
POINT_GROUPS = ((3, 1.6e-4), (3, 2.5e-3), (45, 1.25e-4), (2, 5e-3), (4, 1e-3), (1, 5e-2))


def listed():
    return [
        # the deformation network and its control points after one iteration: 27 small tensors, latency counts
        {"name": "adamw_net", "kind": "adamw", "layout": "net", "dtype": "float32", "clip": False},
        # all parameters of a large captured scene, clipped
        {"name": "adamw_points_3m", "kind": "adamw", "layout": "points", "points": 3_000_000, "dtype": "float32", "clip": True},
        # a model kept in 16 bits: two dozen tensors of all sizes, none a round number
        {"name": "adamw_bf16_ragged", "kind": "adamw", "layout": "ragged", "tensors": 24, "elements": 8_000_003, "dtype": "bfloat16",
         "clip": True},
        # the network again, moments in 8 bits
        {"name": "adamw8_net", "kind": "adamw8", "layout": "net", "dtype": "float32", "clip": False},
        # the learned association of 300k points with 512 superpoints beside the points' own parameters, clipped
        {"name": "adamw8_association_300k", "kind": "adamw8", "layout": "association", "points": 300_000, "superpoints": 512,
         "dtype": "float32", "clip": True},
        {"name": "adamw8_bf16_ragged", "kind": "adamw8", "layout": "ragged", "tensors": 24, "elements": 8_000_003,
         "dtype": "bfloat16", "clip": False},
        # a small scene's association at the start of its training
        {"name": "balance_10k_512", "kind": "balance", "points": 10_000, "superpoints": 512, "choices": 1, "dtype": "float32",
         "masked": False, "train": True},
        # the benchmark scene's association, as many choices as there are neighbours
        {"name": "balance_300k_512", "kind": "balance", "points": 300_000, "superpoints": 512, "choices": 4, "dtype": "float32",
         "masked": False, "train": True},
        # few superpoints (the coarse stage), 16-bit logits, a third of the points out of the frame
        {"name": "balance_200k_64_bf16", "kind": "balance", "points": 200_001, "superpoints": 64, "choices": 2,
         "dtype": "bfloat16", "masked": True, "train": True},
        # a large scene, looked at without a gradient: how full its superpoints are
        {"name": "balance_400k_2000_view", "kind": "balance", "points": 400_000, "superpoints": 2000, "choices": 8,
         "dtype": "bfloat16", "masked": False, "train": False},
        # neighbour weights of a small dynamic scene
        {"name": "neighbours_50k", "kind": "neighbours", "points": 50_000, "superpoints": 512, "neighbours": 3, "masked": False},
        # neighbour weights of a large one
        {"name": "neighbours_3m", "kind": "neighbours", "points": 3_000_000, "superpoints": 2048, "neighbours": 8, "masked": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["adamw", "adamw8", "balance", "neighbours"])
    if kind == "neighbours":
        return {"kind": kind, "points": _log_uniform(rng, 1, 2_500_000), "superpoints": _log_uniform(rng, 8, 5000),
                "neighbours": rng.randint(1, 8), "masked": rng.random() < 0.5}
    dtype = rng.choice(["float32", "float32", "bfloat16"])
    if kind == "balance":
        superpoints = _log_uniform(rng, 8, 2500)
        return {"kind": kind, "points": _log_uniform(rng, 1, min(400_000, 150_000_000 // superpoints)),
                "superpoints": superpoints, "choices": rng.randint(1, 8), "dtype": dtype, "masked": rng.random() < 0.5,
                "train": rng.random() < 0.7}
    layout = rng.choice(["points", "ragged", "association"])
    case = {"kind": kind, "layout": layout, "dtype": dtype, "clip": rng.random() < 0.5}
    if layout == "points":
        case["points"] = _log_uniform(rng, 100, 1_500_000)
    elif layout == "association":
        case.update(points=_log_uniform(rng, 100, 200_000), superpoints=_log_uniform(rng, 16, 500))
    else:
        case.update(tensors=rng.randint(1, 27), elements=_log_uniform(rng, 300, 20_000_000))
    return case


def _tensors(case):
    """[(elements, learning rate)] of a case's parameter tensors."""
    if case["layout"] == "net":  # eight layers of 256, the 84-wide encoding again before the fifth, four heads, 512 control points
        layers = [(256, 84)] + [(256, 340 if i == 4 else 256) for i in range(7)] + [(3, 256), (4, 256), (3, 256), (4, 256)]
        return [(n, 1.6e-4) for rows, columns in layers for n in (rows * columns, rows)] + [(512 * 3, 1.6e-4)]
    if case["layout"] == "ragged":
        rng = random.Random(case["elements"])
        parts = [math.exp(rng.uniform(-9, 0)) for _ in range(case["tensors"])]
        return [(max(1, int(case["elements"] * part / sum(parts))) | 1, 3e-4) for part in parts]
    groups = [(case["points"] * columns, rate) for columns, rate in POINT_GROUPS]
    return groups if case["layout"] == "points" else groups + [(case["points"] * case["superpoints"], 1e-3)]


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device=DEVICE)


def _gradient(g, n):
    """Magnitudes over several orders, as from points near and far; a third of the points is not in the picture."""
    seen = _uniform(g, -(-n // 16)) < 0.67
    return _normal(g, n) * torch.exp(_normal(g, n) - 8) * seen.repeat_interleave(16)[:n]


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "balance":
        N, M = case["points"], case["superpoints"]
        # logits that have begun to prefer some superpoints, and some points that may not use all of them
        logits = _normal(g, N, M).mul_(2).add_(_normal(g, M))
        logits[: N // 8, : M // 4] = float("-inf")
        rows = _uniform(g, N) < 0.67 if case["masked"] else None
        return {"kind": "balance", "K": min(case["choices"], M), "rows": rows, "train": case["train"],
                "logits": logits.to(DTYPES[case["dtype"]]).requires_grad_(case["train"]), "upstream": _uniform(g, 1)[0] + 0.5}
    if case["kind"] == "neighbours":
        N, M, K = case["points"], case["superpoints"], case["neighbours"]
        # points in the order of space: neighbours of neighbouring points are near each other
        centre = torch.arange(N, device=DEVICE)[:, None] * M // N
        indices = (centre + (_normal(g, N, K) * 8).long()) % M
        weights = torch.softmax(_normal(g, N, K) * 2, dim=-1).requires_grad_(True)
        rows = _uniform(g, N) < 0.67 if case["masked"] else None
        return {"kind": "neighbours", "M": M, "indices": indices, "weights": weights, "rows": rows, "upstream": _uniform(g, 1)[0] + 0.5}

    dtype, tensors = DTYPES[case["dtype"]], _tensors(case)
    starts, total = [], 0
    for n, _ in tensors:  # tensors of one allocation, each on a boundary of its own as an allocator gives them
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    flat = {"param": torch.zeros(total, device=DEVICE, dtype=dtype), "grad": torch.zeros(total, device=DEVICE, dtype=dtype)}
    names = ["param", "grad"]
    if case["kind"] == "adamw":
        flat.update(m=torch.zeros(total, device=DEVICE), v=torch.zeros(total, device=DEVICE))
        names += ["m", "v"]
    state = {"kind": case["kind"], "flat": flat, "steps": [torch.tensor(float(40 + k % 3)) for k in range(len(tensors))],
             "rates": [rate for _, rate in tensors], "max_norm": None, "seed": seed % 1000, "states": []}
    for name in names:
        state[name] = [flat[name][at:at + n] for at, (n, _) in zip(starts, tensors)]
    for k, (n, _) in enumerate(tensors):
        state["param"][k].copy_(_normal(g, n) * 0.3)
        grad = _gradient(g, n)
        state["grad"][k].copy_(grad)
        root = torch.exp(_normal(g, n) * 0.7 - 8) + 1e-7  # of the second moment, and a first moment that may go with it
        m = root * torch.tanh(_normal(g, n))
        if case["kind"] == "adamw":
            state["m"][k].copy_(m)
            state["v"][k].copy_(root * root)
        else:
            state["states"].append(_encode(m, root * root, torch.full((n,), 0.5, device=DEVICE), torch.full((n,), 0.5, device=DEVICE)))
    if case["clip"]:  # as in training: the clipped norm is a part of what the gradients have
        state["max_norm"] = 0.3 * float(flat["grad"].double().norm())
    return state


# ---- the 8-bit moments --------------------------------------------------------------------------------------------------
# One tensor of bytes: codes of m [blocks * 256], codes of v [blocks * 256], then (m, v) exponents [blocks, 2]. A code's
# magnitude has 3 bits of fraction below 4 (m, with a sign above) or 5 (v) bits of exponent. It stands for u units: u itself below
# one binade of fractions, then (8 + fraction) << (exponent - 1). The unit is the smallest power of two for which the block's
# largest value is no larger than the highest code's. An exponent byte is that of the highest binade as float32 has it: 0 for a
# block of zeros, 255 if a value is not finite. v > 0 stays > 0.


def _mix(x):
    """32 bits made of 32 bits, each of which depends on all; on 64-bit integers."""
    x = (x ^ (x >> 16)) * 0xBB67AE85 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x3C6EF373 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _noise(n, step, seed):
    """What is added before rounding down, for m and for v: 16 bits each of a hash of the element, the step and the seed."""
    key = _mix((int(step) + seed * 0x9E3779B1) & 0xFFFFFFFF)
    h = _mix((torch.arange(n, device=DEVICE) * 0x9E3779B1 + key) & 0xFFFFFFFF)
    return (h & 0xFFFF).double() / 65536, (h >> 16).double() / 65536


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -len(x) % BLOCK)).view(-1, BLOCK)


def _codes(x, noise, bits):
    """(codes [blocks, 256], exponent bytes [blocks]) of values >= 0, `bits` bits of exponent."""
    x, noise = _blocks(x), _blocks(noise)
    top = x.amax(dim=1)
    fraction, exponent = torch.frexp(top)  # fraction in [0.5, 1)
    exponent = exponent.long() - 1 + (fraction > 1.875 / 2)
    y = x.double() * torch.exp2(((1 << bits) + 1 - exponent).double())[:, None]  # in units
    # NaN and infinities are gone with the block; what is left of them here does not matter
    y = torch.nan_to_num(y, 0.0, 0.0, 0.0)
    binade = torch.clamp(torch.frexp(y)[1].long() - 1, min=3)
    k = torch.floor(y * torch.exp2((3 - binade).double()) + noise.double()).long()
    code = torch.clamp(k + ((binade - 3) << 3), max=(8 << bits) - 1)
    scale = torch.where(torch.isfinite(top), torch.where(top > 0, torch.clamp(exponent + 127, 1, 254), 0), 255)
    return code, scale


def _encode(m, v, noise_m, noise_v):
    code, scale_m = _codes(m.abs(), noise_m, 4)
    code_m = torch.where((_blocks(m) < 0) & (code > 0), code + 128, code)
    code_v, scale_v = _codes(v, noise_v, 5)
    code_v = torch.where((code_v == 0) & (_blocks(v) > 0), 1, code_v)
    return torch.cat([code_m.view(-1), code_v.view(-1), torch.stack([scale_m, scale_v], dim=1).view(-1)]).to(torch.uint8)


def _values(code, scale, bits):
    units = torch.where(code < 8, code, (8 + (code & 7)) << torch.clamp((code >> 3) - 1, min=0))
    value = units.double() * torch.exp2((scale - 128 - (1 << bits)).double())[:, None]
    return torch.where(scale[:, None] == 255, math.nan, value)


def _decode(state, n):
    """(m, v) of a state, float32."""
    blocks = -(-n // BLOCK)
    codes, scales = state[:blocks * 512].long().view(2, blocks, BLOCK), state[blocks * 512:].long().view(blocks, 2)
    m = _values(codes[0] & 127, scales[:, 0], 4) * torch.where(codes[0] > 127, -1, 1)
    return m.view(-1)[:n].float(), _values(codes[1], scales[:, 1], 5).view(-1)[:n].float()


# ---- one pass, plain ------------------------------------------------------------------------------------------------------


def _plain_update(p, g, m, v, step, rate):
    """(parameters, moments) after a step, in float32."""
    b1, b2 = BETAS
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denominator = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + 1e-15
    return p * (1 - rate * DECAY) - rate / (1 - b1 ** step) * m / denominator, m, v


def _plain_step(s):
    norm, factor = None, 1.0
    if s["max_norm"] is not None:
        norm = sum(g.double().square().sum() for g in s["grad"]).sqrt().float()  # long sums: in 64 bits
        factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    moments = []
    for k, (p, grad, rate) in enumerate(zip(s["param"], s["grad"], s["rates"])):
        s["steps"][k] += 1
        step = float(s["steps"][k])
        g = grad.float() * factor
        if s["kind"] == "adamw":
            new, m, v = _plain_update(p.float(), g, s["m"][k], s["v"][k], step, rate)
            s["m"][k].copy_(m)
            s["v"][k].copy_(v)
        else:
            new, m, v = _plain_update(p.float(), g, *_decode(s["states"][k], len(p)), step, rate)
            s["states"][k].copy_(_encode(m, v, *_noise(len(p), step, s["seed"])))
            moments.append([x.bfloat16() for x in _decode(s["states"][k], len(p))])
        p.copy_(new)
    return norm, moments


def _plain_loss(counts, importance, superpoints):
    share = counts.float() / counts.sum().clamp(min=1)
    return superpoints * (share * importance).sum(), share


def _plain_balance(s):
    logits, rows, M = s["logits"].detach().float(), s["rows"], s["logits"].shape[1]
    on = (logits > -math.inf).any(dim=1) if rows is None else rows & (logits > -math.inf).any(dim=1)
    logits = torch.where(on[:, None], logits, 0.0)
    p = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True) * on[:, None]
    chosen = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, : s["K"]]
    counted = on[:, None] & (logits.gather(1, chosen) > -math.inf)
    counts = torch.bincount(chosen[counted], minlength=M)
    T = on.sum().clamp(min=1)
    importance = (p.sum(dim=0, dtype=torch.float64) / T).float()
    loss, share = _plain_loss(counts, importance, M)
    out = {"loss": loss, "counts": counts.to(torch.int32), "importance": importance}
    if s["train"]:
        a = s["upstream"] * M * share / T
        out["grad"] = (p * (a - (p * a).sum(dim=1, keepdim=True))).to(s["logits"].dtype)
    return out


def _plain_neighbours(s):
    weights, indices, M = s["weights"].detach(), s["indices"], s["M"]
    on = torch.ones(len(weights), dtype=torch.bool, device=DEVICE) if s["rows"] is None else s["rows"]
    counts = torch.bincount(indices.gather(1, weights.argmax(dim=1, keepdim=True))[:, 0][on], minlength=M)
    T = on.sum().clamp(min=1)
    sums = torch.zeros(M, dtype=torch.float64, device=DEVICE)
    sums.index_add_(0, indices.reshape(-1), (weights * on[:, None]).double().reshape(-1))
    importance = (sums / T).float()
    loss, share = _plain_loss(counts, importance, M)
    grad = (s["upstream"] * M * share / T)[indices] * on[:, None]
    return {"loss": loss, "counts": counts.to(torch.int32), "importance": importance, "grad": grad}


# ---- one pass ---------------------------------------------------------------------------------------------------------------


def _own_step(s):
    from fast_sp_gs_amd.adamw import adamw8_moments, adamw8_step, adamw_step
    settings = {"lr": s["rates"], "betas": BETAS, "eps": 1e-15, "weight_decay": DECAY, "max_norm": s["max_norm"]}
    if s["kind"] == "adamw":
        return adamw_step(s["param"], s["grad"], s["m"], s["v"], s["steps"], **settings), []
    norm = adamw8_step(s["param"], s["grad"], s["states"], s["steps"], seed=s["seed"], **settings)
    return norm, adamw8_moments(s["states"], s["param"], dtype=torch.bfloat16)


def _own_balance(s):
    from fast_sp_gs_amd.balance import balance_loss, neighbour_balance
    if s["kind"] == "balance":
        loss, counts, importance = balance_loss(s["logits"], s["K"], rows=s["rows"])
        of = s["logits"]
    else:
        loss, counts, importance = neighbour_balance(s["weights"], s["indices"], s["M"], rows=s["rows"])
        of = s["weights"]
    out = {"loss": loss, "counts": counts, "importance": importance}
    if of.requires_grad:
        out["grad"], = torch.autograd.grad(loss, of, s["upstream"])
    return out


def run(state):
    if state["kind"] in ("balance", "neighbours"):
        if own:
            return _own_balance(state)
        return _plain_balance(state) if state["kind"] == "balance" else _plain_neighbours(state)
    norm, moments = _own_step(state) if own else _plain_step(state)
    out = {"param": state["flat"]["param"], "norm": norm}
    if state["kind"] == "adamw":
        out.update(m=state["flat"]["m"], v=state["flat"]["v"])
    else:
        out.update(moments=[list(pair) for pair in moments])
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "balance":
        n = case["points"] * case["superpoints"]
        size, mask = (4 if case["dtype"] == "float32" else 2), case["points"] if case["masked"] else 0
        return {"bytes": n * size * (2 if case["train"] else 1) + mask + 8 * case["superpoints"],
                "flops": n * (10 if case["train"] else 5)}
    if case["kind"] == "neighbours":
        n = case["points"] * case["neighbours"]
        return {"bytes": n * (4 + 8 + 4) + (case["points"] if case["masked"] else 0) + 8 * case["superpoints"], "flops": 4 * n}
    n = sum(count for count, _ in _tensors(case))
    size = 4 if case["dtype"] == "float32" else 2
    moments = 16 if case["kind"] == "adamw" else 4 + 4  # read and written; codes read and written, and the values that come back
    return {"bytes": n * (3 * size + moments), "flops": n * (18 if case["clip"] else 15)}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------


def _exact_hash(x):
    for shift, factor in ((16, 0xBB67AE85), (15, 0x3C6EF373)):
        x = ((x ^ (x >> shift)) * factor) % (1 << 32)
    return x ^ (x >> 16)


def _exact_round(x, noise, binades):
    """Values of x >= 0 as blocks of 256 keep them, and what the smallest of their codes stands for."""
    n, blocks = len(x), (len(x) + 255) // 256
    padded = x.new_zeros(2, blocks * 256)
    padded[0, :n], padded[1, :n] = x, noise
    x, noise = padded.view(2, blocks, 256)
    largest = x.amax(dim=1, keepdim=True).clamp(min=2.0 ** -126)
    top = torch.floor(torch.log2(largest))
    top = top + (largest > 1.875 * 2.0 ** top)
    smallest = top - binades + 2  # of the exponents with a full fraction
    exponent = torch.maximum(torch.floor(torch.log2(x.clamp(min=2.0 ** -300))), smallest)
    spacing = 2.0 ** exponent / 8
    kept = torch.floor(x / spacing + noise) * spacing
    most = 2.0 ** top * (2 - 1 / 8)
    return torch.minimum(kept, most).view(-1)[:n], (2.0 ** smallest / 8).expand(-1, 256).reshape(-1)[:n]


def _exact_moments(state):
    """m and v of a state from its bytes, by tables of the 128 and 256 magnitudes."""
    blocks = len(state) // 514
    tables = []
    for binades in (16, 32):
        tables.append(torch.tensor([f if e == 0 else (8 + f) * 2.0 ** (e - 1) for e in range(binades) for f in range(8)],
                                   dtype=torch.float64, device=DEVICE) / (8 * 2.0 ** (binades - 2)))
    scale = 2.0 ** (state[512 * blocks:].double().view(blocks, 2) - 127)
    first, second = state[:256 * blocks].view(blocks, 256).long(), state[256 * blocks:512 * blocks].view(blocks, 256).long()
    m = tables[0][first % 128] * (1 - 2 * (first // 128)) * scale[:, :1]
    return m.view(-1), (tables[1][second] * scale[:, 1:]).view(-1)


def _exact_step(case, s):
    grads = [g.double() for g in s["grad"]]
    norm = torch.sqrt(torch.stack([torch.dot(g, g) for g in grads]).sum())
    clip = 1.0 if s["max_norm"] is None else min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    param, first, second = (torch.zeros_like(s["flat"]["param"], dtype=torch.float64) for _ in range(3))
    moments = []
    for k, g in enumerate(grads):
        g, t, n, rate = g * clip, float(s["steps"][k]) + 1, len(g), s["rates"][k]
        if case["kind"] == "adamw":
            m, v = s["m"][k].double(), s["v"][k].double()
        else:
            m, v = (x[:n] for x in _exact_moments(s["states"][k]))
        m, v = m + (g - m) * (1 - BETAS[0]), v + (g * g - v) * (1 - BETAS[1])
        m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
        x = s["param"][k].double()
        at = s["param"][k].storage_offset()
        param[at:at + n] = x - rate * (m_hat / (v_hat.sqrt() + 1e-15) + DECAY * x)
        if case["kind"] == "adamw":
            first[at:at + n], second[at:at + n] = m, v
        else:
            key = _exact_hash((int(t) + s["seed"] * 0x9E3779B1) % (1 << 32))
            h = _exact_hash((torch.arange(n, device=DEVICE, dtype=torch.int64) * 0x9E3779B1 + key) % (1 << 32))
            kept_m, _ = _exact_round(m.abs(), (h % 65536) / 65536.0, 16)
            kept_v, unit = _exact_round(v, (h // 65536) / 65536.0, 32)
            moments.append([torch.sign(m) * kept_m, torch.where((kept_v == 0) & (v > 0), unit, kept_v)])
    out = {"param": param, "norm": norm if s["max_norm"] is not None else None}
    out.update({"m": first, "v": second} if case["kind"] == "adamw" else {"moments": moments})
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("adamw", "adamw8"):
        return _exact_step(case, s)
    up = s["upstream"].double()
    if case["kind"] == "balance":
        M = case["superpoints"]
        x = s["logits"].detach().double()
        on = ~torch.isinf(x).all(dim=1)
        if s["rows"] is not None:
            on &= s["rows"]
        x, T = x[on], max(1, int(on.sum()))
        p = torch.softmax(x, dim=1)
        # a key for each logit that is larger for larger ones and, among equals, for the lower index
        rank = torch.argsort(torch.argsort(-x, dim=1, stable=True), dim=1)
        taken = (rank < s["K"]) & ~torch.isinf(x)
        counts = taken.sum(dim=0).double()
        importance = p.sum(dim=0) / T
        share = counts / max(1.0, float(counts.sum()))
        out = {"loss": M * torch.dot(share, importance), "counts": None, "importance": importance}
        if case["train"]:
            a = up * M * share / T
            grad = torch.zeros(len(on), M, dtype=torch.float64, device=DEVICE)
            grad[on] = p * (a - (p @ a)[:, None])
            out["grad"] = grad
        return out
    M, N = case["superpoints"], case["points"]
    on = s["rows"] if s["rows"] is not None else torch.ones(N, dtype=torch.bool, device=DEVICE)
    w, index, T = s["weights"].detach().double()[on], s["indices"][on], max(1, int(on.sum()))
    importance = torch.bincount(index.reshape(-1), weights=w.reshape(-1), minlength=M) / T
    best = index[torch.arange(len(w), device=DEVICE), torch.sort(w, dim=1, descending=True, stable=True).indices[:, 0]]
    share = torch.bincount(best, minlength=M).double() / max(1, len(w))
    grad = torch.zeros(N, case["neighbours"], dtype=torch.float64, device=DEVICE)
    grad[on] = (up * M / T * share)[index]
    return {"loss": M * torch.dot(share, importance), "counts": None, "importance": importance, "grad": grad}
