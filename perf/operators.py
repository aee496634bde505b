"""Cases of the optimiser's operators: the AdamW step with 32-bit and with 8-bit states, gradient clipping by the global norm,
and writing / reading the 8-bit state.

A case holds many parameter tensors, as a network does. They lie in one flat buffer, each at a multiple of BLOCK elements with zeros
behind it, so that the plain forms are passes over the whole buffer; the framework gets the list of tensors, as a user's program has it.
BLOCK is also the number of elements that share one scale of the 8-bit state.
"""
import math

import torch

own = False

BLOCK = 256
BETAS, EPS, LR = (0.9, 0.999), 1e-8, 1e-4
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- shapes -------------------------------------------------------------------------------------------------------------------------

def _network(start, fpn, most, stages):
    """Parameter shapes of a 3D Retina U-Net: encoder of two convolutions a stage with affine norms, laterals, transposed convolutions,
    output convolutions, and the two detection heads. (start, fpn, most, stages) = (32, 128, 320, 6) is the network of the benchmark."""
    ch = [min(start << s, most) for s in range(stages)]
    dec = [min(c, fpn) for c in ch]
    shapes, cin = [], 1
    for c in ch:
        shapes += [(c, cin, 3, 3, 3), (c,), (c,), (c, c, 3, 3, 3), (c,), (c,)]
        cin = c
    for c, d in zip(ch, dec):
        shapes += [(d, c, 1, 1, 1), (d,), (d, d, 3, 3, 3), (d,)]
    for lo, hi in zip(dec[:-1], dec[1:]):
        shapes += [(hi, lo, 2, 2, 2), (lo,)]
    for anchors in (27, 162):
        shapes += [(fpn, fpn, 3, 3, 3), (fpn,), (fpn,)] * 2 + [(anchors, fpn, 3, 3, 3), (anchors,)]
    return shapes + [()] * 4 + [(2, dec[0], 1, 1, 1), (2,)]


def _shapes(case):
    if case["net"] == "ragged":  # sizes from `least` to `most`, evenly over their logarithm
        k, a, b = case["tensors"], case["least"], case["most"]
        return [(max(1, round(a * (b / a) ** (i / max(1, k - 1)))),) for i in range(k)]
    s = _network(*(int(x) for x in case["net"].split("-")))
    return [x for x in s if len(x) < 5] if case.get("vectors_only") else s


def _sizes(case):
    return [math.prod(s) for s in _shapes(case)]


def listed():
    luna = "32-128-320-6"
    return [
        # fine-tuning of the norm layers and biases alone, convolutions frozen: some 50 tensors of 1 to 320 elements, all latency
        {"name": "adamw_vectors", "op": "adamw", "net": luna, "vectors_only": True, "dtype": "f32", "decay": 0.01},
        # the benchmark's network, no decay on vectors, gradients clipped: the ordinary training step
        {"name": "adamw_luna_clip", "op": "adamw", "net": luna, "dtype": "f32", "decay": 0.01, "clip": True},
        # the smaller plan under a loss scaler: scale and overflow flag on the device
        {"name": "adamw_toy_scaled", "op": "adamw", "net": "32-128-320-5", "dtype": "f32", "decay": 0.01, "scaled": True},
        # parameters held in 16 bits, sizes of every kind, none a multiple of anything
        {"name": "adamw_ragged_bf16", "op": "adamw", "net": "ragged", "tensors": 37, "least": 3, "most": 2900001, "dtype": "bf16", "decay": 0.1},
        # four times the channels: bandwidth and nothing else
        {"name": "adamw_wide", "op": "adamw", "net": "128-512-1280-6", "dtype": "f32", "decay": 0.01},
        # 8-bit states: the benchmark's network, odd sizes in fp16 under a loss scaler, and the wide one, clipped
        {"name": "adamw8_luna", "op": "adamw8", "net": luna, "dtype": "f32", "decay": 0.01},
        {"name": "adamw8_ragged_f16", "op": "adamw8", "net": "ragged", "tensors": 61, "least": 1, "most": 1300007, "dtype": "f16", "decay": 0.1, "scaled": True},
        {"name": "adamw8_wide_clip", "op": "adamw8", "net": "128-512-1280-6", "dtype": "f32", "decay": 0.01, "clip": True},
        # clipping in place, for any optimiser
        {"name": "clip_luna", "op": "clip", "net": luna, "dtype": "f32"},
        {"name": "clip_ragged_bf16", "op": "clip", "net": "ragged", "tensors": 150, "least": 7, "most": 1900003, "dtype": "bf16"},
        # a 32-bit checkpoint goes into 8-bit states, and 8-bit states into a 32-bit checkpoint
        {"name": "state_write_luna", "op": "write", "net": luna, "dtype": "f32"},
        {"name": "state_read_wide", "op": "read", "net": "128-512-1280-6", "dtype": "f32"},
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "clip", "write", "read"])
    case = {"op": op, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]) if op not in ("write", "read") else "f32"}
    if rng.random() < 0.3:
        start = rng.choice([8, 16, 24, 32, 48, 64])
        case["net"] = "%d-%d-%d-%d" % (start, 4 * start, start * rng.choice([6, 10, 16]), rng.choice([3, 4, 5, 6]))
    else:
        k = round(math.exp(rng.uniform(0, math.log(300))))
        most = math.exp(rng.uniform(math.log(200), math.log(6e7 / max(1, k / 6))))
        case |= {"net": "ragged", "tensors": k, "least": max(1, round(most ** rng.uniform(0, 1))), "most": round(most)}
    if op in ("adamw", "adamw8"):
        case["decay"] = rng.choice([0.0, 0.01, 0.1])
        case["clip"] = rng.random() < 0.4
        case["scaled"] = rng.random() < 0.3
        case["first"] = rng.random() < 0.15
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------------------

def _fill(gen, sizes, starts, total, spread, scale, dev):
    """Normal values, each tensor at a scale of its own (10 ** -spread .. 1, times `scale`), zeros between the tensors."""
    x = torch.randn(total, generator=gen, device=dev)
    f = (10.0 ** (-spread * torch.rand(len(sizes), generator=gen, device=dev)) * scale).tolist()
    for n, a, b, s in zip(sizes, starts, starts[1:] + [total], f):
        x[a:a + n] *= s
        x[a + n:b] = 0
    return x


def prepare(case, seed):
    dev = torch.device("cuda")
    shapes, dt = _shapes(case), DTYPES[case["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [sum(blocks[:i]) * BLOCK for i in range(len(sizes))]
    total = sum(blocks) * BLOCK
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    fill = lambda spread, scale: _fill(gen, sizes, starts, total, spread, scale, dev)  # noqa: E731
    views = lambda flat: [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]  # noqa: E731
    per_block = lambda flat: [flat[a // BLOCK:a // BLOCK + b] for a, b in zip(starts, blocks)]  # noqa: E731
    op, st = case["op"], {"op": case["op"], "blocks": total // BLOCK}
    scale = 2.0 ** 10 if case.get("scaled") else 1.0
    if op != "read" and op != "write":
        # gradients: every tensor at its own scale; some tensors get none of the loss at all (a head without positives)
        g = fill(2.5, 1e-2)
        for i in range(5, len(sizes), 11):
            g[starts[i]:starts[i] + sizes[i]] = 0
        st["grads_flat"] = (g * scale).to(dt)
        st["grads"] = views(st["grads_flat"])
    if op in ("adamw", "adamw8"):
        st["flat"] = fill(1.0, 0.3).to(dt)
        st["params"] = views(st["flat"])
        # decay on the weights, none on vectors and scalars; per block for the plain form
        st["decay"] = [case["decay"] if len(s) != 1 or case["net"] == "ragged" else 0.0 for s in shapes]
        st["decay_of_block"] = torch.tensor(st["decay"], device=dev, dtype=torch.float64).repeat_interleave(torch.tensor(blocks, device=dev)).view(-1, 1)
        st["max_norm"] = 0.3 if case.get("clip") else None
        st["grad_scale"] = torch.tensor(scale, device=dev) if case.get("scaled") else None
        st["found_inf"] = torch.tensor(0.0, device=dev) if case.get("scaled") else None
        # where each block lies in its own tensor, in pairs of elements: the dither of the 8-bit state counts them
        st["pair"] = torch.cat([torch.arange(b, dtype=torch.int32, device=dev) for b in blocks]).mul_(BLOCK // 2).view(-1, 1)
        first = bool(case.get("first"))
        st["steps"] = torch.full((len(sizes),), 0 if first else 1 + int(seed) % 4000, dtype=torch.int32, device=dev)
    if op == "clip":
        st["max_norm"] = 0.5 * math.sqrt(total) * 1e-4  # every pass clips: the limit falls a little with each
    if op != "clip":
        first = bool(case.get("first"))
        m = fill(2.5, 0.0 if first else 3e-3)
        v = (m * fill(0.5, 3.0)).square().mul_(0.1).add_(m.square())
        if op == "adamw" or op == "write":
            st["m"], st["v"] = m, v
            st["exp_avgs"], st["exp_avg_sqs"] = views(m), views(v)
        if op != "adamw":
            st["codes"], st["scales"] = [None] * 2, [None] * 2
            for k, x in enumerate((m, v.sqrt())):
                st["codes"][k], st["scales"][k] = _to8(x.view(-1, BLOCK), k == 1)
            st["state"] = (views(st["codes"][0].view(-1)), per_block(st["scales"][0].view(-1)), views(st["codes"][1].view(-1)), per_block(st["scales"][1].view(-1)))
        if op == "write":  # what is written over: a state of zeros
            st["codes"], st["scales"] = [torch.zeros_like(c) for c in st["codes"]], [torch.zeros_like(c) for c in st["scales"]]
            st["state"] = (views(st["codes"][0].view(-1)), per_block(st["scales"][0].view(-1)), views(st["codes"][1].view(-1)), per_block(st["scales"][1].view(-1)))
        if op == "read":
            st["m"], st["v"] = torch.zeros_like(m), torch.zeros_like(v)
            st["exp_avgs"], st["exp_avg_sqs"] = views(st["m"]), views(st["v"])
    return st


# ---- plain forms --------------------------------------------------------------------------------------------------------------------

def _mixed(pair, step):
    """32 well mixed bits for each pair of elements of a tensor at a step (int32 arithmetic, which wraps)."""
    x = pair + step * (0x9E3779B1 - 2 ** 32)
    x = (x ^ ((x >> 16) & 0xFFFF)) * 0x6A09E667
    x = (x ^ ((x >> 15) & 0x1FFFF)) * (0xBB67AE85 - 2 ** 32)
    return x ^ ((x >> 16) & 0xFFFF)


def _to8(x, root, pair=None, step=None):
    """Rows of BLOCK values as e4m3 codes and one fp32 scale a row: scale = max |x| / 448, codes = x / scale rounded to nearest even.
    root: the values are square roots of second moments. One that is not zero is not stored as zero (2^-9 is the least code), and a
    training step (`pair` given) rounds it up with the probability of its distance from the code below, by 16 bits an element that follow
    from its place and the step: a moving average that changes by 0.1 % a step would stand still under rounding to nearest."""
    scale = x.abs().amax(1, keepdim=True) * (1.0 / 448.0)
    scale = torch.where(scale >= 2.0 ** -110, scale, 0.0)
    y = torch.where(scale > 0, x * (1.0 / scale), 0.0)
    if not root:
        return y.to(torch.float8_e4m3fn), scale
    least = (x > 0) & (scale > 0)
    if pair is None:
        return torch.where(least, y.clamp_min(2.0 ** -9), y).to(torch.float8_e4m3fn), scale
    bits = _mixed(pair + torch.arange(BLOCK // 2, dtype=torch.int32, device=x.device), step)
    dither = torch.stack([bits & 0xFFFF, (bits >> 16) & 0xFFFF], 2).view(x.shape) * 16 + 8
    # times 2^-120 an fp32 number has e4m3's exponent field, denormals among them: the code is its bits without the low 20
    code = ((y * 2.0 ** -120).view(torch.int32) + dither) >> 20
    code = torch.maximum(code.clamp(max=0x7E), least.int())
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _from8(codes, scale):
    return codes.float() * scale


def _norm(flat, grad_scale):
    n = flat.double().square().sum().sqrt()  # a sum over all parameters
    return (n if grad_scale is None else n / grad_scale.double()).float()


def _step_plain(s, m, v):
    """One AdamW step on rows of BLOCK elements: new parameters (in their own type), moments, and the norm."""
    p, g = s["flat"].view(-1, BLOCK).float(), s["grads_flat"].view(-1, BLOCK).float()
    b1, b2 = BETAS
    norm, factor = None, torch.ones((), dtype=torch.float64, device=p.device)
    if s["grad_scale"] is not None:
        factor = factor / s["grad_scale"].double()
    if s["max_norm"] is not None:
        norm = _norm(s["grads_flat"], s["grad_scale"])
        factor = factor * (s["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0)
    if s["grad_scale"] is not None or s["max_norm"] is not None:
        g = g * factor.float()
    t = (s["steps"][0] + 1).double()
    size = (LR / (1 - b1 ** t)).float()
    unbias = (1 / (1 - b2 ** t).sqrt()).float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = v.sqrt()
    p = p * (1 - LR * s["decay_of_block"]).float() - (m / (root * unbias + EPS)) * size
    return p, m, v, root, norm


def _skip(s, new, old):
    return new if s["found_inf"] is None else torch.where(s["found_inf"] == 0, new.to(old.dtype), old)


def _adamw_plain(s):
    p, m, v, _, norm = _step_plain(s, s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK))
    s["flat"].copy_(_skip(s, p.view(-1), s["flat"]))
    s["m"].copy_(_skip(s, m.view(-1), s["m"]))
    s["v"].copy_(_skip(s, v.view(-1), s["v"]))
    s["steps"].copy_(_skip(s, s["steps"] + 1, s["steps"]))
    return norm


def _adamw8_plain(s):
    (cm, cr), (sm, sr) = s["codes"], s["scales"]
    p, m, _, root, norm = _step_plain(s, _from8(cm, sm), _from8(cr, sr).square())
    s["flat"].copy_(_skip(s, p.view(-1), s["flat"]))
    for code, scale, (nc, ns) in ((cm, sm, _to8(m, False)), (cr, sr, _to8(root, True, s["pair"], s["steps"][0] + 1))):
        code.view(torch.uint8).copy_(_skip(s, nc.view(torch.uint8), code.view(torch.uint8)))
        scale.copy_(_skip(s, ns, scale))
    s["steps"].copy_(_skip(s, s["steps"] + 1, s["steps"]))
    return norm


def _outputs(s, norm):
    op = s["op"]
    out = {} if norm is None else {"norm": norm}
    if op in ("adamw", "adamw8"):
        out |= {"params": s["flat"], "steps": s["steps"]}
    if op == "clip":
        out["grads"] = s["grads_flat"]
    if op in ("adamw", "read"):
        out |= {"exp_avg": s["m"], "exp_avg_sq": s["v"]}
    if op in ("adamw8", "write"):  # what the codes stand for: e4m3 values and their scales
        out |= {"exp_avg8": s["codes"][0], "exp_avg_scale": s["scales"][0], "root8": s["codes"][1], "root_scale": s["scales"][1]}
    return out


def run(s):
    op = s["op"]
    if op == "clip":
        s["max_norm"] *= 0.9999
    if own:
        from nndetection_amd import optim
        if op == "adamw":
            norm = optim.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["steps"], lr=LR, betas=BETAS, eps=EPS,
                                    weight_decay=s["decay"], max_norm=s["max_norm"], grad_scale=s["grad_scale"], found_inf=s["found_inf"])
        elif op == "adamw8":
            norm = optim.adamw8_step(s["params"], s["grads"], optim.AdamState8(*s["state"]), s["steps"], lr=LR, betas=BETAS, eps=EPS,
                                     weight_decay=s["decay"], max_norm=s["max_norm"], grad_scale=s["grad_scale"], found_inf=s["found_inf"])
        elif op == "clip":
            norm = optim.clip_grads_(s["grads"], s["max_norm"])
        elif op == "write":
            norm = optim.write_adam_state8(optim.AdamState8(*s["state"]), s["exp_avgs"], s["exp_avg_sqs"])
        else:
            norm = optim.read_adam_state8(optim.AdamState8(*s["state"]), s["exp_avgs"], s["exp_avg_sqs"])
    elif op == "adamw":
        norm = _adamw_plain(s)
    elif op == "adamw8":
        norm = _adamw8_plain(s)
    elif op == "clip":
        g = s["grads_flat"]
        norm = _norm(g, None)
        g.copy_((g.float() * (s["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()))
    else:
        norm = None
        if op == "write":
            for k, x in enumerate((s["m"], s["v"].sqrt())):
                code, scale = _to8(x.view(-1, BLOCK), k == 1)
                s["codes"][k].copy_(code)
                s["scales"][k].copy_(scale)
        else:
            s["m"].copy_(_from8(s["codes"][0], s["scales"][0]).view(-1))
            s["v"].copy_(_from8(s["codes"][1], s["scales"][1]).square().view(-1))
    return _outputs(s, norm)


# ---- what a pass cannot do without, and the definition in 64 bits -------------------------------------------------------------------

def work(case):
    sizes = _sizes(case)
    n, e = sum(sizes), 4 if case["dtype"] == "f32" else 2
    codes = 2 * n + 8 * sum(-(-k // BLOCK) for k in sizes)  # both moments in 8 bits, with their scales
    move = {"adamw": n * (3 * e + 16), "adamw8": n * 3 * e + 2 * codes, "clip": 2 * n * e, "write": 8 * n + codes, "read": 8 * n + codes}[case["op"]]
    return {"bytes": move, "flops": n * {"adamw": 16, "adamw8": 30, "clip": 3, "write": 6, "read": 3}[case["op"]]}


def _grid8(y, up=None):
    """y in 64 bits on the e4m3 values, whose steps are 2^(e-3) for 2^e <= |y| and 2^-9 below 2^-6: to the nearest (ties to even), or down
    after `up` of a step is added."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) if up is None else torch.floor(y / step + up)).mul(step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    rows = lambda x: x.double().view(-1, BLOCK)  # noqa: E731

    def codes(x, root, t=None):
        top = x.abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, top / 448, top)
        y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
        up = None
        if t is not None:  # the same bits for the same element and step
            i = s["pair"].long() + torch.arange(BLOCK // 2, device=x.device)
            bits = (i + t * 0x9E3779B1) % 2 ** 32
            for shift, factor in ((16, 0x6A09E667), (15, 0xBB67AE85), (16, 1)):
                bits = torch.bitwise_xor(bits, bits // 2 ** shift)
                bits = ((bits % 2 ** 16) * factor + (((bits // 2 ** 16) * factor) % 2 ** 16) * 2 ** 16) % 2 ** 32
            up = (torch.stack([bits % 2 ** 16, bits // 2 ** 16], 2).view(x.shape).double() + 0.5) / 2 ** 16
        y = _grid8(y, up)
        if root:
            y = torch.where((x > 0) & (y == 0), torch.full_like(y, 2.0 ** -9), y)
        return y, scale

    if op == "clip":
        g = s["grads_flat"].double()
        norm = torch.linalg.vector_norm(g)
        limit = s["max_norm"] * 0.9999
        return {"norm": norm, "grads": g * min(1.0, limit / (float(norm) + 1e-6))}
    if op == "read":
        return {"exp_avg": (rows(s["codes"][0].float()) * s["scales"][0].double()).view(-1),
                "exp_avg_sq": (rows(s["codes"][1].float()) * s["scales"][1].double()).pow(2).view(-1)}
    if op == "write":
        (cm, sm), (cr, sr) = codes(rows(s["m"]), False), codes(rows(s["v"]).pow(0.5), True)
        return {"exp_avg8": cm, "exp_avg_scale": sm, "root8": cr, "root_scale": sr}
    m0, v0 = ((rows(s["m"]), rows(s["v"])) if op == "adamw" else
              (rows(s["codes"][0].float()) * s["scales"][0].double(), (rows(s["codes"][1].float()) * s["scales"][1].double()) ** 2))
    g = rows(s["grads_flat"])
    if s["grad_scale"] is not None:
        g = g / float(s["grad_scale"])
    out = {}
    if s["max_norm"] is not None:
        norm = torch.linalg.vector_norm(g)
        out["norm"] = norm
        g = g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    t = int(s["steps"][0]) + 1
    m = torch.lerp(m0, g, 1 - BETAS[0])
    v = torch.lerp(v0, g * g, 1 - BETAS[1])
    m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    p = rows(s["flat"])
    out |= {"params": (p - LR * s["decay_of_block"] * p - LR * m_hat / (v_hat.sqrt() + EPS)).view(-1), "steps": s["steps"] + 1}
    if op == "adamw":
        return out | {"exp_avg": m.view(-1), "exp_avg_sq": v.view(-1)}
    (cm, sm), (cr, sr) = codes(m, False), codes(v.sqrt(), True, t)
    return out | {"exp_avg8": cm, "exp_avg_scale": sm, "root8": cr, "root_scale": sr}
