"""The optimizer operators and what they are measured on: the global norm of the gradients of many
tensors, and the AdamW step over many tensors with 32-bit and with 8-bit states.

Every tensor's first element lies at a multiple of 64 in the flat state, as in the framework's
parameter arenas.  8-bit states hold blocks of 64 elements: a sign and a 7-bit magnitude for the
first moment, an 8-bit magnitude for the root of the second, both small floats with 4 exponent
bits whose unit is a power of two for each block, so the values they stand for are exact in bf16.
"""
import math
import random

import torch

own = False

HYPER = {"lr": 1e-3, "beta_1": 0.9, "beta_2": 0.999, "epsilon": 1e-7, "weight_decay": 0.01, "grad_scale": 0.5}
ALIGN = 64  # elements between the places where tensors may start in an arena
STEP_WORDS = 1024  # the step counter's copies
# the dither's hash (step, position) -> 32 bits
HASH_STEP, HASH_HIGH, HASH_1, HASH_2 = 0x632BE5AB, 0x27D4A62F, 0x6E7A3B15, 0x35D2C1A7
M_BITS, ROOT_BITS = 3, 4  # mantissa bits of the two codes


def listed():
    return [
        # the head that trains over a frozen DenseNet-121: one kernel and one bias, where latency counts
        {"name": "adamw head", "op": "adamw", "bits": 32, "tensors": 2, "params": 1025, "grad": "f32", "layout": "arena",
         "clip": 0.0, "decay": "all", "step": 0},
        # the secure-FL tiny CNN
        {"name": "adamw8 tiny", "op": "adamw", "bits": 8, "tensors": 6, "params": 1937, "grad": "f32", "layout": "arena",
         "clip": 0.0, "decay": "all", "step": 12},
        {"name": "norm tiny", "op": "norm", "tensors": 6, "params": 1937, "grad": "f32", "layout": "arena"},
        # MobileNetV2's trainable weights in the arena that Model.compile makes
        {"name": "adamw mobilenet", "op": "adamw", "bits": 32, "tensors": 158, "params": 2225153, "grad": "f32",
         "layout": "arena", "clip": 0.0, "decay": "matrices", "step": 999},
        # DenseNet-121 trained whole, clipped, no decay of BatchNorm weights and biases
        {"name": "adamw8 densenet", "op": "adamw", "bits": 8, "tensors": 364, "params": 6954881, "grad": "f32",
         "layout": "arena", "clip": 1.0, "decay": "matrices", "step": 400},
        {"name": "norm densenet", "op": "norm", "tensors": 364, "params": 6954881, "grad": "f32", "layout": "arena"},
        # VGG16: tensors of their own, outside an arena
        {"name": "adamw8 vgg", "op": "adamw", "bits": 8, "tensors": 28, "params": 14715201, "grad": "f32",
         "layout": "separate", "clip": 0.0, "decay": "all", "step": 7000},
        # DenseNet-201, clipped
        {"name": "adamw densenet201", "op": "adamw", "bits": 32, "tensors": 604, "params": 18102533, "grad": "f32",
         "layout": "arena", "clip": 1.0, "decay": "matrices", "step": 50},
        # several federated clients' or a larger model's tensors, gradients as a bf16 all-reduce leaves them
        {"name": "adamw large bf16", "op": "adamw", "bits": 32, "tensors": 40, "params": 120000007, "grad": "bf16",
         "layout": "separate", "clip": 0.0, "decay": "all", "step": 3000},
        {"name": "adamw8 large bf16", "op": "adamw", "bits": 8, "tensors": 48, "params": 120000007, "grad": "bf16",
         "layout": "separate", "clip": 1.0, "decay": "matrices", "step": 3000},
        {"name": "adamw8 large", "op": "adamw", "bits": 8, "tensors": 300, "params": 120000007, "grad": "f32",
         "layout": "arena", "clip": 0.0, "decay": "all", "step": 20000},
        {"name": "norm large bf16", "op": "norm", "tensors": 48, "params": 120000007, "grad": "bf16", "layout": "separate"},
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw", "norm"])
    params = int(round(math.exp(rng.uniform(math.log(1.0), math.log(1.2e8)))))
    layout = rng.choice(["arena", "separate"])
    tensors = int(round(math.exp(rng.uniform(0.0, math.log(48.0 if layout == "separate" else 600.0)))))
    case = {"op": op, "tensors": min(tensors, params), "params": params, "grad": rng.choice(["f32", "bf16"]), "layout": layout}
    if op == "adamw":
        case.update(bits=rng.choice([8, 32]), clip=rng.choice([0.0, 1.0]), decay=rng.choice(["all", "matrices"]),
                    step=int(round(math.exp(rng.uniform(0.0, math.log(1e5))))) - 1)
    return case


def sizes_of(case):
    """The tensors' sizes: every second one is small (a bias, a BatchNorm weight), the others share
    the rest unevenly, odd sizes among them."""
    n, total = case["tensors"], case["params"]
    r = random.Random(n * 1000003 + total)
    share = [(0.002 if i % 2 else 1.0) * math.exp(r.uniform(-1.5, 1.5)) for i in range(n)]
    scale = (total - n) / sum(share)
    sizes = [1 + int(s * scale) for s in share]
    sizes[0] += total - sum(sizes)
    return sizes


def padded(n):
    return -(-n // ALIGN) * ALIGN


# ----------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    sizes = sizes_of(case)
    offsets = [0]
    for n in sizes:
        offsets.append(offsets[-1] + padded(n))
    numel = offsets[-1]
    lens = torch.tensor(sizes, device=dev)
    spans = torch.tensor([b - a for a, b in zip(offsets, offsets[1:])], device=dev)
    first = torch.tensor(offsets[:-1], device=dev)
    tensor_of = torch.repeat_interleave(torch.arange(len(sizes), device=dev), spans, output_size=numel)
    real = (torch.arange(numel, device=dev) - first[tensor_of]) < lens[tensor_of]

    def normal():
        return torch.randn(numel, device=dev, generator=gen)

    def uniform():
        return torch.rand(numel, device=dev, generator=gen)

    # gradients differ in size from tensor to tensor and from element to element; some are zero
    size = torch.exp(torch.rand(len(sizes), device=dev, generator=gen) * math.log(1e3) + math.log(1e-5))[tensor_of]
    grad = normal() * size * (uniform() > 0.05) * real
    grad_type = torch.float32 if case["grad"] == "f32" else torch.bfloat16
    grad = grad.to(grad_type)

    def split(flat):
        """Views of an arena, or tensors of their own."""
        views = [flat[o:o + n] for o, n in zip(offsets, sizes)]
        return views if case["layout"] == "arena" else [v.clone() for v in views]

    state = {"case": case, "sizes": sizes, "offsets": offsets, "numel": numel, "grads": split(grad),
             "grad": grad if case["layout"] == "arena" else None}
    if case["layout"] == "separate":
        state["pads"] = [torch.zeros(padded(n) - n, device=dev) for n in sizes]
        state["grad_pads"] = [p.to(grad_type) for p in state["pads"]]
    if case["op"] == "adamw":
        data = normal() * 0.05 * real
        state["params"] = split(data)
        state["data"] = data if case["layout"] == "arena" else None
        fresh = case["step"] == 0
        m = (normal() * size * 0.3 * real) * (0.0 if fresh else 1.0)
        v = (size * size * (0.02 + uniform() * 2.0) * real) * (0.0 if fresh else 1.0)
        # every second tensor (the kernels) decays, or all of them
        state["decay"] = [case["decay"] == "all" or i % 2 == 0 for i in range(len(sizes))]
        state["mask"] = torch.tensor(state["decay"], device=dev, dtype=torch.float32)[tensor_of]
        state["step"] = torch.full((STEP_WORDS,), case["step"], dtype=torch.int32, device=dev)
        if case["bits"] == 8:
            mid = torch.full((numel,), 1 << 15, device=dev, dtype=torch.int32)  # to nearest
            state["m"], ms = encode(m, M_BITS, mid)
            state["v"], vs = encode(torch.sqrt(v), ROOT_BITS, mid)
            state["scales"] = torch.stack([ms, vs], 1)
            state["index"] = torch.arange(numel, device=dev)
        else:
            state["m"], state["v"] = m, v
    if own:
        from idc_models_amd.ops import optim
        if case["op"] == "norm":
            state["table"] = optim.TensorTable(state["grads"])
        else:
            state["table"] = optim.TensorTable(state["grads"], state["params"], decay=state["decay"])
            st = optim.AdamWState(state["table"], bits=case["bits"])
            st.m.copy_(state["m"])
            st.v.copy_(state["v"])
            if case["bits"] == 8:
                st.scales.copy_(state["scales"])
            st.step.copy_(state["step"])
            state["adamw"] = st
    return state


# ----------------------------------------------------------------------------------- the 8-bit codes
def dither(index, step):
    """Two times 16 bits from an element's place in the state and the step's number."""
    x = ((index & 0xFFFFFFFF) + (index >> 32) * HASH_HIGH + step.long() * HASH_STEP) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * HASH_1) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * HASH_2) & 0xFFFFFFFF
    x = x ^ (x >> 16)
    return (x & 0xFFFF).to(torch.int32), (x >> 16).to(torch.int32)


def power_of_two(exponent):
    """2 ** exponent as fp32 (exponent: -126 ... 127)."""
    return ((exponent + 127) << 23).view(torch.float32)


def encode(x, mantissa, bits16):
    """(codes, scale bytes): the codes' magnitudes are floats of `mantissa` bits; 16 random bits say
    whether one is rounded up.  A block's unit is the smallest power of two whose codes reach its
    largest value; a root (4 bits, no sign) that is not zero keeps a code that is not zero."""
    one = 1 << mantissa  # the first code with an implicit one
    a = x.abs().view(-1, ALIGN)
    top = a.amax(1)
    drop = 23 - mantissa
    last = ((2 * one - 1) << drop) - (1 << 23)  # the mantissa of the largest code
    scale = ((top.view(torch.int32) + (0x7FFFFF - last)) >> 23) - (14 + mantissa)
    bad = ~torch.isfinite(top)
    scale = torch.where(bad, torch.full_like(scale, 255), scale.clamp(min=1))
    y = (a * power_of_two(torch.where(bad, torch.zeros_like(scale), 127 - scale))[:, None]).view(-1)
    low = y < one
    t = torch.where(low, y + one, y)
    first = (127 + mantissa - 1) << 23  # the bits of fp32's `one`, less the exponent that codes from `one` on have
    part = t.view(torch.int32) - (low.to(torch.int32) << 23) - first
    code = (part + ((bits16 << (drop - 16)) + (1 << (drop - 17)))) >> drop
    if mantissa == ROOT_BITS:
        code = torch.maximum(code, (x > 0).to(torch.int32))
    else:
        code = code | ((x < 0).to(torch.int32) << 7)
    code = (code.view(-1, ALIGN) * (~bad).to(torch.int32)[:, None]).view(-1)
    return code.to(torch.uint8), scale.to(torch.uint8)


def decode(codes, scales, mantissa):
    """The values in fp32: NaN where the block's scale is 255."""
    one = 1 << mantissa
    c = codes.to(torch.int32)
    sign = 1.0
    if mantissa == M_BITS:
        sign = 1.0 - 2.0 * (c >> 7)
        c = c & 127
    low = c < one
    bits = (c << (23 - mantissa)) + (low.to(torch.int32) << 23) + ((127 + mantissa - 1) << 23)
    value = bits.view(torch.float32)
    value = (value - low * float(one)) * sign
    s = scales.to(torch.int32)
    unit = torch.where(s == 0, torch.zeros_like(s), s << 23).view(torch.float32)
    unit = torch.where(s == 255, torch.full_like(unit, float("nan")), unit)
    return (value.view(-1, ALIGN) * unit[:, None]).view(-1)


# ----------------------------------------------------------------------------------- one pass
def flat(tensors, pads):
    return torch.cat([t for pair in zip(tensors, pads) for t in pair])


def norm_of(grad):
    g = grad.float()
    return torch.sqrt((g * g).sum(dtype=torch.float64)).float()


def run(state):
    case = state["case"]
    if own:
        from idc_models_amd.ops import optim
        if case["op"] == "norm":
            return {"norm": optim.global_norm(state["table"])}
        st = state["adamw"]
        optim.adamw_(state["table"], st, HYPER["lr"], HYPER["beta_1"], HYPER["beta_2"], HYPER["epsilon"],
                     HYPER["weight_decay"], HYPER["grad_scale"], clip_norm=case["clip"])
        m, v = st.decode(torch.bfloat16) if case["bits"] == 8 else (st.m, st.v)
        step, norm = st.step, st.norm
    else:
        arena = case["layout"] == "arena"
        grad = state["grad"] if arena else flat(state["grads"], state["grad_pads"])
        if case["op"] == "norm":
            return {"norm": norm_of(grad)}
        w = state["data"] if arena else flat(state["params"], state["pads"])
        g = grad.float() * HYPER["grad_scale"]
        norm = None
        if case["clip"]:
            norm = norm_of(grad)
            scaled = norm * HYPER["grad_scale"]
            g = g * (case["clip"] / torch.clamp(scaled, min=case["clip"]))
        b1, b2 = HYPER["beta_1"], HYPER["beta_2"]
        m, v = state["m"], state["v"]
        if case["bits"] == 8:
            m = decode(m, state["scales"][:, 0], M_BITS)
            v = decode(v, state["scales"][:, 1], ROOT_BITS)
            v = v * v
        m = b1 * m + (1.0 - b1) * g
        v = b2 * v + (1.0 - b2) * (g * g)
        step = state["step"]
        step += 1
        t = step[0].double()
        alpha = (HYPER["lr"] * torch.sqrt(1.0 - b2 ** t) / (1.0 - b1 ** t)).float()
        root = torch.sqrt(v)
        w_new = w - (HYPER["lr"] * HYPER["weight_decay"] * state["mask"] * w + alpha * (m / (root + HYPER["epsilon"])))
        if arena:
            w.copy_(w_new)
        else:
            [p.copy_(w_new[o:o + n]) for p, o, n in zip(state["params"], state["offsets"], state["sizes"])]
        if case["bits"] == 8:
            low, high = dither(state["index"], step[0])
            state["m"], ms = encode(m, M_BITS, low)
            state["v"], vs = encode(root, ROOT_BITS, high)
            state["scales"] = torch.stack([ms, vs], 1)
            m = decode(state["m"], ms, M_BITS).to(torch.bfloat16)
            v = decode(state["v"], vs, ROOT_BITS).to(torch.bfloat16)
        else:
            state["m"], state["v"] = m, v
    # of an 8-bit state, "v" is the root of the second moment, which is what its codes stand for
    out = {"w": state["data"] if case["layout"] == "arena" else state["params"], "m": m, "v": v, "step": step}
    if case["clip"]:
        out["norm"] = norm
    return out


def work(case):
    n, g = case["params"], 4 if case["grad"] == "f32" else 2
    if case["op"] == "norm":
        return {"bytes": n * g + 4, "flops": 2 * n}
    if case["bits"] == 32:
        return {"bytes": n * (g + 24), "flops": 15 * n}
    # codes read and written, a scale byte for 64 of them, and the values that are given back
    return {"bytes": n * (g + 8 + 4 + 4) + n // 16, "flops": 30 * n}


# ----------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definition: the same update with doubles, and the codes by their values (which of
    the two neighbours, by the fraction between them) instead of by bits of fp32 numbers."""
    s = prepare(case, seed)
    arena = case["layout"] == "arena"
    n = s["numel"]
    g = (s["grad"] if arena else flat(s["grads"], s["grad_pads"])).double()
    norm = g.square().sum().sqrt()
    if case["op"] == "norm":
        return {"norm": norm}
    w = (s["data"] if arena else flat(s["params"], s["pads"])).double()
    h = HYPER
    factor = h["grad_scale"]
    if case["clip"] and float(norm) * factor > case["clip"]:
        factor = case["clip"] / float(norm)
    g = g * factor

    def values(column, mantissa):
        c = s["m" if column == 0 else "v"].double()
        sign = torch.ones_like(c)
        if column == 0:
            sign = torch.where(c >= 128, -sign, sign)
            c = torch.where(c >= 128, c - 128, c)
        one = 2.0 ** mantissa
        e = torch.floor(c / one)
        f = c - e * one
        value = sign * torch.where(e == 0, f, (one + f) * torch.exp2(e - 1))
        k = s["scales"][:, column].double()
        unit = torch.where(k == 0, torch.zeros_like(k), torch.exp2(k - 127.0))
        return value * unit.repeat_interleave(ALIGN)

    if case["bits"] == 8:
        m, v = values(0, M_BITS), values(1, ROOT_BITS).square()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = h["beta_1"] * m + (1.0 - h["beta_1"]) * g
    v = h["beta_2"] * v + (1.0 - h["beta_2"]) * g.square()
    t = case["step"] + 1
    alpha = h["lr"] * math.sqrt(1.0 - h["beta_2"] ** t) / (1.0 - h["beta_1"] ** t)
    root = v.sqrt()
    w = w * (1.0 - h["lr"] * h["weight_decay"] * s["mask"].double()) - alpha * m / (root + h["epsilon"])

    def rounded(x, mantissa, random_bits):
        one = 2.0 ** mantissa
        a = x.abs().view(-1, ALIGN)
        top = a.amax(1)
        largest = (2.0 * one - 1.0) * 2.0 ** 14
        k = torch.ceil(torch.log2(torch.clamp(top, min=1e-37) / largest))
        unit = torch.exp2(torch.clamp(k, min=-126.0)).repeat_interleave(ALIGN)
        y = a.view(-1) / unit
        e = torch.clamp(torch.floor(torch.log2(torch.clamp(y, min=1.0))) - mantissa, min=0.0)
        quantum = torch.exp2(e)
        c = torch.floor(y / quantum + (random_bits.double() + 0.5) / 65536.0) * quantum
        if mantissa == ROOT_BITS:
            c = torch.where((x > 0) & (c < 1.0), torch.ones_like(c), c)
        return torch.sign(x) * c * unit

    if case["bits"] == 8:
        low, high = dither(s["index"], torch.tensor(t, device=w.device))
        m, v = rounded(m, M_BITS, low), rounded(root, ROOT_BITS, high)
    if not arena:
        w = [w[o:o + k] for o, k in zip(s["offsets"], s["sizes"])]
    out = {"w": w, "m": m, "v": v, "step": None}
    if case["clip"]:
        out["norm"] = norm
    return out
