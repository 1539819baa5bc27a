"""What the optimiser step of a Gaussian map is measured on: the gradients' norm over all tensors, the AdamW step over many tensors
with its moments in 32 bits or in 8, and the eviction of the splats with the least accumulated compositing weight.  `run` computes
them in plain torch (`own = False`) or through gs_localization_amd.map_optimizer (`own = True`)."""
import math

import torch

if torch.cuda.is_available():
    DEV = torch.device("cuda")
else:
    DEV = torch.device("cpu")
own = False

# train.py's learning rates of the six tensors of a map (arguments/__init__.py:75-82), and the pose loop's one rate
MAP_LR = [1.6e-4, 2.5e-3, 1.25e-4, 5e-2, 5e-3, 1e-3]
POSE_LR = 1e-3
BLOCK = 256                 # elements that share one window of the 8-bit second moment
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    # P: splats; degree: of the spherical harmonics (1: train.py's --sh_degree here, 3: the localisation maps); step: the optimiser's
    base = dict(kind="map", degree=1, type="f32", grad="f32", clip=False, decay=0.0, step=1000)
    return [
        # the norm behind a clipped step: a small scene, and train.py's garden at its final size
        dict(base, name="norm 2k sh3", op="norm", P=2000, degree=3),
        dict(base, name="norm 1.5M sh1", op="norm", P=1_500_000),
        # the pose loop's own optimiser: eight numbers in four tensors, where only latency counts
        dict(base, name="adamw32 pose", op="adamw32", kind="pose", P=1, step=3),
        # train.py's garden when it starts and when it ends
        dict(base, name="adamw32 200k sh1 clip", op="adamw32", P=200_000, clip=True),
        dict(base, name="adamw32 1.5M sh1", op="adamw32", P=1_500_000),
        # a map held in half precision, an odd number of splats, decay
        dict(base, name="adamw32 100003 sh3 bf16", op="adamw32", P=100_003, degree=3, type="bf16", grad="bf16", decay=0.01, step=1),
        # 8-bit moments: an object, the chess map, the KingsCollege map
        dict(base, name="adamw8 2001 sh1", op="adamw8", P=2001, clip=True),
        dict(base, name="adamw8 800k sh3", op="adamw8", P=800_000, degree=3),
        dict(base, name="adamw8 3M sh3", op="adamw8", P=3_000_000, degree=3, decay=0.01),
        # pruning to a budget: an object, the garden with 32-bit moments, the garden with 8-bit moments
        dict(op="evict", name="evict 2k sh3", P=2000, degree=3, share=0.75, recent=100, views=1, states="32", forget=1.0),
        dict(op="evict", name="evict 1.5M sh1", P=1_500_000, degree=1, share=0.9, recent=50_000, views=4, states="32", forget=1.0),
        dict(op="evict", name="evict 1.5M sh1 8-bit", P=1_500_000, degree=1, share=0.6, recent=0, views=16, states="8", forget=0.5),
    ]


def draw(rng):
    op = rng.choice(["norm", "adamw32", "adamw32", "adamw8", "adamw8", "evict", "evict"])
    P = int(round(math.exp(rng.uniform(0.0, math.log(2_500_000)))))
    P = max(1, P - rng.randrange(0, 2))
    degree = rng.choice([0, 1, 2, 3])
    if op == "evict":
        return dict(op=op, P=min(P, 1_500_000), degree=degree, share=rng.choice([rng.uniform(0.02, 1.0), rng.uniform(0.5, 0.99)]),
                    recent=rng.choice([0, 1, P // 30, P // 7]), views=rng.choice([0, 1, 3, 16]), states=rng.choice(["none", "32", "8"]),
                    forget=rng.choice([1.0, 0.9, rng.uniform(0.0, 1.0)]))
    type_ = rng.choice(["f32", "f32", "f32", "bf16", "f16"])
    grad = rng.choice([type_, "f32"]) if op != "norm" else type_
    return dict(op=op, kind="pose" if op == "adamw32" and rng.random() < 0.2 else "map", P=P, degree=degree, type=type_, grad=grad, clip=rng.random() < 0.5,
                decay=rng.choice([0.0, 0.0, 0.01, rng.uniform(0.0, 0.1)]), step=rng.choice([0, 1, rng.randrange(2, 50), rng.randrange(50, 30000)]))


def _shapes(case):
    if case.get("kind") == "pose":
        return [(3,), (3,), (1,), (1,)]
    P, rest = case["P"], (case["degree"] + 1) ** 2 - 1
    return [(P, 3), (P, 1, 3), (P, rest, 3), (P, 1), (P, 3), (P, 4)]


def _numel(shape):
    return math.prod(shape)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _codes(n, gen):
    """8-bit moments of n elements as training leaves them: a window per block, a code per root of the second moment, a ratio."""
    window = torch.randint(80, 100, (_blocks(n),), generator=gen, device=DEV, dtype=torch.uint8)
    rms = torch.randint(1, 256, (n,), generator=gen, device=DEV, dtype=torch.int16).to(torch.uint8)
    never = torch.rand(n, generator=gen, device=DEV) < 0.1                        # splats that no view has shown yet
    ratio = (torch.randn(n, generator=gen, device=DEV) * 8).clamp_(-127, 127).to(torch.int8)
    return rms.masked_fill_(never, 0), ratio.masked_fill_(never, 0), window


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    randn = lambda s, k=1.0: torch.randn(s, generator=gen, device=DEV) * k                                        # noqa: E731
    rand = lambda s: torch.rand(s, generator=gen, device=DEV)                                                     # noqa: E731
    shapes, s = _shapes(case), dict(case=case)
    if case["op"] == "evict":
        P = case["P"]
        s["keep"], s["recent"] = _keep(case)
        s["tensors"] = [randn(x) for x in shapes]
        if case["states"] == "32":
            s["tensors"] += [randn(x, 1e-5) for x in shapes] + [randn(x, 1e-5).square() for x in shapes]
        s["rms"], s["ratio"] = [], []
        if case["states"] == "8":
            for x in shapes:
                rms, ratio, window = _codes(_numel(x), gen)
                s["rms"].append((rms.reshape(x), window))
                s["ratio"].append(ratio.reshape(x))
        s["tensors"] += [rand(P) * 20, torch.randint(0, 2, (P,), generator=gen, device=DEV).bool()]               # max_radii2D, a flag
        # most splats get little weight, many none (hidden in every view): ties at zero
        weigh = lambda x: torch.exp(randn(x, 2.0)) * (rand(x) < 0.7)                                              # noqa: E731
        s["scores"] = weigh((P,)) * (rand((P,)) < 0.8)
        s["weights"] = weigh((case["views"], P)) if case["views"] else None
        return s
    n = len(shapes)
    s["lr"] = [POSE_LR] * n if case["kind"] == "pose" else MAP_LR
    s["eps"] = 1e-8 if case["kind"] == "pose" else 1e-15                     # torch's default; train.py's
    s["betas"], s["dither"] = (0.9, 0.999), seed & 0x7FFFFFFF
    t = case["step"]
    s["clip"] = torch.tensor([1.7, 1.0 / 1.7], device=DEV) if case["clip"] else None
    s["clock"] = [torch.tensor([0.9 ** t, 0.999 ** t, float(t), 0.0], dtype=torch.float64, device=DEV) for _ in range(n)]
    half, ghalf = TYPES[case["type"]], TYPES[case["grad"]]
    s["params"], s["grads"], s["m"], s["v"], s["rms"], s["ratio"], s["window"] = [], [], [], [], [], [], []
    for x in shapes:
        rows = (x[0],) + (1,) * (len(x) - 1)
        s["params"].append(randn(x).to(half))
        # 40 % of the splats are out of the view: no gradient; the others' spread over four decades
        mag = torch.pow(10.0, rand(rows) * 4.0 - (4.0 if ghalf == torch.float16 else 7.0)) * (rand(rows) < 0.6)
        g = randn(x)
        if case["op"] == "adamw32" and t > 0:
            u = mag * (0.2 + rand(x))
            s["m"].append(u * randn(x, 0.4))
            s["v"].append(u.square_())
        elif case["op"] == "adamw32":
            s["m"].append(torch.zeros(x, device=DEV))
            s["v"].append(torch.zeros(x, device=DEV))
        elif case["op"] == "adamw8":
            k = _numel(x)
            rms, ratio, window = _codes(k, gen)
            if t == 0:
                rms, ratio, window = (torch.zeros_like(y) for y in (rms, ratio, window))
            else:           # gradients of the size that the second moment has seen
                g = g * torch.exp2(window.float() - 122.0).repeat_interleave(BLOCK)[:k].reshape(x)
                if ghalf == torch.float16:
                    window += 20
                    g = g * 2.0 ** 20
            if t == 0 or k == 0:
                g = g * mag
            else:
                g = g * (rand(rows) < 0.6)
            s["rms"].append(rms.reshape(x))
            s["ratio"].append(ratio.reshape(x))
            s["window"].append(window)
        s["grads"].append((g if case["op"] == "adamw8" else g * mag).to(ghalf))
    return s


def _keep(case):
    P = case["P"]
    recent = min(case["recent"], P)
    return max(recent, min(P, int(round(case["share"] * P)))), recent


# ---- the plain forms --------------------------------------------------------------------------------------------------------------

def _plain_norm(grads):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for g in grads:
        total = total + g.double().square().sum()
    norm = total.sqrt().float()
    return torch.stack((norm, (1.0 / (norm + 1e-6)).clamp(max=1.0)))


def _rates(clock, lr, betas, decay):
    """The step's scalars, in 64 bits on the device; advances the clock."""
    b1, b2 = clock[0] * betas[0], clock[1] * betas[1]
    clock[0], clock[1], clock[2] = b1, b2, clock[2] + 1.0
    return float(1.0 - lr * decay), (lr / (1.0 - b1)).float(), (1.0 / (1.0 - b2).sqrt()).float()


def _moments(m, v, g, betas):
    return m * betas[0] + g * (1.0 - betas[0]), v * betas[1] + (g * g) * (1.0 - betas[1])


def _plain_adamw32(s):
    case, out = s["case"], {"params": [], "exp_avg": [], "exp_avg_sq": [], "clock": []}
    for p, g, m, v, clock, lr in zip(s["params"], s["grads"], s["m"], s["v"], s["clock"], s["lr"]):
        shrink, rate, unbias = _rates(clock, lr, s["betas"], case["decay"])
        g = g.float() if s["clip"] is None else g.float() * s["clip"][1]
        m1, v1 = _moments(m, v, g, s["betas"])
        p.copy_(p.float() * shrink - m1 / (v1.sqrt() * unbias + s["eps"]) * rate)
        m.copy_(m1)
        v.copy_(v1)
        out["params"].append(p)
        out["exp_avg"].append(m)
        out["exp_avg_sq"].append(v)
        out["clock"].append(clock[:3])
    return out


def _range(betas):
    """The largest |m| / sqrt(v) that gradients can bring about (Cauchy-Schwarz over both exponential sums)."""
    return (1.0 - betas[0]) / math.sqrt((1.0 - betas[1]) * (1.0 - betas[0] ** 2 / betas[1]))


def _shift(x, k):
    return (x >> k) & ((1 << (32 - k)) - 1)


def _int32(x):
    x &= 0xFFFFFFFF
    return x - (1 << 32) if x >> 31 else x


def _mix(x):
    x = (x ^ _shift(x, 16)) * _int32(0x6C8E9CF5)
    x = (x ^ _shift(x, 15)) * _int32(0x2F7A5D1B)
    return x ^ _shift(x, 16)


def _dither(n, seed, place, step):
    """Random bits of n elements from the seed, the tensor's place in the list and the step: 19 for the root, 13 for the ratio."""
    key = _mix(step.to(torch.int32) + _int32(seed * 0x9E3779B1 + (place + 1) * 0x85EBCA77))
    quad = torch.arange((n + 3) // 4, dtype=torch.int32, device=DEV)
    h = _mix((quad * _int32(0x9E3779B1)) ^ key)
    r = h[:, None] * torch.tensor([_int32(k) for k in (0x00000001, 0xB5297A4D, 0x68E31DA5, 0x1B56C4E9)], dtype=torch.int32, device=DEV)
    r = r.reshape(-1)[:n]
    r = r ^ _shift(r, 15)
    return _shift(r, 13), r & 8191


def _in_blocks(x):
    return torch.cat((x, x.new_zeros(-x.numel() % BLOCK))).reshape(-1, BLOCK)


def _decode(rms, window):
    """A code c > 0 of a block with window w stands for the float whose upper 13 bits are c + 16 w + 1; 0 stands for 0."""
    top = (rms.reshape(-1).int() + (window.int() * 16 + 1).repeat_interleave(BLOCK)[: rms.numel()]) << 19
    return torch.where(rms.reshape(-1) > 0, top, 0).view(torch.float32)


def _window_of(bits):
    """The window that holds a block's largest value: sixteen binades, the largest value's own the last but one."""
    return ((_in_blocks(bits).amax(1) >> 23) - 15).clamp_(min=0)


def _plain_adamw8(s):
    case, span = s["case"], _range(s["betas"])
    out = {"params": [], "exp_avg": [], "rms": [], "clock": []}
    for i, (p, g, rms, ratio, window, clock, lr) in enumerate(zip(s["params"], s["grads"], s["rms"], s["ratio"], s["window"], s["clock"], s["lr"])):
        n = p.numel()
        shrink, rate, unbias = _rates(clock, lr, s["betas"], case["decay"])
        if n == 0:
            out["params"].append(p)
            out["exp_avg"].append(p.to(torch.bfloat16))
            out["rms"].append(p.to(torch.bfloat16))
            out["clock"].append(clock[:3])
            continue
        g = g.reshape(-1).float() if s["clip"] is None else g.reshape(-1).float() * s["clip"][1]
        u = _decode(rms, window)
        m1, v1 = _moments((ratio.reshape(-1).float() * (span / 127.0)) * u, u * u, g, s["betas"])
        u1 = v1.sqrt()
        p.copy_((p.reshape(-1).float() * shrink - m1 / (u1 * unbias + s["eps"]) * rate).reshape(p.shape))
        du, dr = _dither(n, s["dither"], i, clock[2])
        bits = u1.view(torch.int32)
        window.copy_(_window_of(bits).to(torch.uint8))
        code = ((bits + du) >> 19) - (window.int() * 16 + 1).repeat_interleave(BLOCK)[:n]
        rms.copy_(torch.where(bits > 0, code.clamp_(1, 255), 0).to(torch.uint8).reshape(p.shape))
        u = _decode(rms, window)
        r = torch.floor((m1 / u) * (127.0 / span) + dr.float() * (1.0 / 8192.0)).clamp_(-127.0, 127.0)
        ratio.copy_(torch.where(u > 0, r, 0.0).to(torch.int8).reshape(p.shape))
        out["params"].append(p)
        # the values that the codes stand for: the root's five bits are exact in bfloat16
        out["exp_avg"].append(((ratio.reshape(-1).float() * (span / 127.0)) * u).to(torch.bfloat16).reshape(p.shape))
        out["rms"].append(u.to(torch.bfloat16).reshape(p.shape))
        out["clock"].append(clock[:3])
    return out


def _plain_evict(s):
    case, keep, recent = s["case"], s["keep"], s["recent"]
    total = s["scores"].double() * case["forget"]
    if s["weights"] is not None:
        total = total + s["weights"].double().sum(0)
    scores = total.float()
    old = scores.numel() - recent
    best = torch.sort(torch.where(scores[:old].isnan(), -math.inf, scores[:old]), descending=True, stable=True).indices[: keep - recent]
    kept = torch.cat((torch.sort(best).values, torch.arange(old, scores.numel(), device=DEV)))
    out = {"kept": kept, "scores": scores[kept], "rows": [x[kept] for x in s["tensors"]], "exp_avg": [], "rms": []}
    span = _range((0.9, 0.999))
    for (rms, window), ratio in zip(s["rms"], s["ratio"]):
        u = _decode(rms, window).reshape(rms.shape)[kept]
        ratio, flat = ratio[kept], u.reshape(-1)
        if flat.numel():
            bits = flat.view(torch.int32)
            base = (_window_of(bits) * 16 + 1).repeat_interleave(BLOCK)[: flat.numel()]
            code = torch.where(bits > 0, ((bits >> 19) - base).clamp_(1, 255), 0)
            u = torch.where(code > 0, (code + base) << 19, 0).view(torch.float32).reshape(u.shape)
        out["rms"].append(u.to(torch.bfloat16))
        out["exp_avg"].append(((ratio.float() * (span / 127.0)) * u).to(torch.bfloat16))
    return out


def run(s):
    op = s["case"]["op"]
    if not own:
        if op == "norm":
            return _plain_norm(s["grads"])
        return _plain_adamw32(s) if op == "adamw32" else _plain_adamw8(s) if op == "adamw8" else _plain_evict(s)
    from gs_localization_amd import map_optimizer as MO
    if op == "norm":
        return MO.grad_norm(s["grads"], max_norm=1.0)
    if op == "adamw32":
        MO.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["clock"], lr=s["lr"], betas=s["betas"], eps=s["eps"],
                      weight_decay=s["case"]["decay"], clip=s["clip"])
        return {"params": s["params"], "exp_avg": s["m"], "exp_avg_sq": s["v"], "clock": [c[:3] for c in s["clock"]]}
    if op == "adamw8":
        MO.adamw_step_8bit(s["params"], s["grads"], s["rms"], s["ratio"], s["window"], s["clock"], lr=s["lr"], betas=s["betas"],
                           eps=s["eps"], weight_decay=s["case"]["decay"], clip=s["clip"], seed=s["dither"])
        exp_avg, rms = MO.moments_8bit(s["rms"], s["ratio"], s["window"], betas=s["betas"], dtype=torch.bfloat16)
        return {"params": s["params"], "exp_avg": exp_avg, "rms": rms, "clock": [c[:3] for c in s["clock"]]}
    kept, scores, rows, pairs = MO.evict_rows(s["scores"], s["keep"], s["tensors"] + s["ratio"], recent=s["recent"], weights=s["weights"],
                                              decay=s["case"]["forget"], rms=s["rms"])
    ratio = rows[len(s["tensors"]):]
    exp_avg, rms = MO.moments_8bit([c for c, _ in pairs], ratio, [w for _, w in pairs], dtype=torch.bfloat16) if pairs else ([], [])
    return {"kept": kept, "scores": scores, "rows": rows[: len(s["tensors"])], "exp_avg": exp_avg, "rms": rms}


def work(case):
    elements = sum(_numel(x) for x in _shapes(case))
    if case["op"] == "evict":
        keep, P = _keep(case)[0], case["P"]
        row = (elements // P) * {"none": 4, "32": 12, "8": 4}[case["states"]] + 5
        coded = (elements // P) * {"none": 0, "32": 0, "8": 6}[case["states"]]            # two codes read, two values of 16 bits written
        return {"bytes": 4 * P * (1 + case["views"]) + keep * (2 * row + coded + 12), "flops": P * (1 + case["views"])}
    size, gsize = (4 if case[k] == "f32" else 2 for k in ("type", "grad"))
    if case["op"] == "norm":
        return {"bytes": elements * gsize + 8, "flops": 2 * elements}
    if case["op"] == "adamw32":
        return {"bytes": elements * (2 * size + gsize + 16), "flops": 14 * elements}
    return {"bytes": elements * (2 * size + gsize + 4 + 4) + elements // 64, "flops": 30 * elements}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------------

def _exact_roots(rms, window):
    """code -> value by its binade and its sixteenth in it; denormals have the first binade's spacing."""
    place = rms.reshape(-1).double() + 16.0 * window.double().repeat_interleave(BLOCK)[: rms.numel()] + 1.0
    binade = torch.floor(place / 16.0)
    value = torch.where(binade > 0, (1.0 + (place / 16.0 - binade)) * torch.exp2(binade - 127.0), place / 16.0 * 2.0 ** -126)
    return torch.where(rms.reshape(-1) > 0, value, 0.0)


def _exact_store(u, bits):
    """A root as the 8-bit window stores it: to a sixteenth of its binade by the random bits, not under the window's lowest value."""
    top = torch.cat((u, u.new_zeros(-u.numel() % BLOCK))).reshape(-1, BLOCK).amax(1)
    top = torch.floor(torch.log2(top.clamp(min=1e-300))).clamp(min=-112.0)
    low = (1.125 * torch.exp2(top - 15.0)).repeat_interleave(BLOCK)[: u.numel()]
    step = torch.exp2(torch.floor(torch.log2(u.clamp(min=2.0 ** -126))) - 4.0)
    down = torch.floor(u / step)
    up = (u / step - down) + bits.double() / 2 ** 19 >= 1.0
    return torch.where(u > 0, torch.maximum((down + up.double()) * step, low), 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        norm = torch.sqrt(sum((g.double() ** 2).sum() for g in s["grads"]))
        return torch.stack((norm, torch.minimum(1.0 / (norm + 1e-6), torch.ones_like(norm))))
    if case["op"] == "evict":
        total = case["forget"] * s["scores"].double()
        for v in range(case["views"]):
            total = total + s["weights"][v].double()
        # the lowest is evicted first, of equal ones the last: by pairs (score, place)
        old = case["P"] - s["recent"]
        single = total[:old].float()
        order = torch.argsort(torch.flip(single, (0,)), stable=True)
        alive = torch.ones(case["P"], dtype=torch.bool, device=DEV)
        alive[old - 1 - order[: case["P"] - s["keep"]]] = False
        out = {"kept": None, "scores": total[alive], "rows": [x[alive].double() if x.is_floating_point() else None for x in s["tensors"]],
               "exp_avg": [], "rms": []}
        for (rms, window), ratio in zip(s["rms"], s["ratio"]):
            u = _exact_roots(rms, window).reshape(rms.shape)[alive]
            u = _exact_store(u.reshape(-1), torch.zeros_like(u.reshape(-1))).reshape(u.shape)
            out["rms"].append(u)
            out["exp_avg"].append(ratio[alive].double() / 127.0 * _range((0.9, 0.999)) * u)
        return out
    b1, b2, t = 0.9, 0.999, case["step"] + 1
    out = {"params": [], "exp_avg": [], "exp_avg_sq" if case["op"] == "adamw32" else "rms": [], "clock": []}
    for i, (p, g, lr) in enumerate(zip(s["params"], s["grads"], s["lr"])):
        out["clock"].append(torch.tensor([b1 ** t, b2 ** t, t], dtype=torch.float64, device=DEV))
        g = g.double().reshape(-1) * (1.0 if s["clip"] is None else float(s["clip"][1]))
        if case["op"] == "adamw32":
            m, v = s["m"][i].double().reshape(-1), s["v"][i].double().reshape(-1)
        else:
            u = _exact_roots(s["rms"][i], s["window"][i])
            m, v = s["ratio"][i].double().reshape(-1) / 127.0 * _range((b1, b2)) * u, u ** 2
        m = m + (1.0 - b1) * (g - m)
        v = v + (1.0 - b2) * (g ** 2 - v)
        step = (m / (1.0 - b1 ** t)) / (torch.sqrt(v / (1.0 - b2 ** t)) + s["eps"])
        x = p.double().reshape(-1)
        out["params"].append((x - lr * case["decay"] * x - lr * step).reshape(p.shape))
        if case["op"] == "adamw32":
            out["exp_avg"].append(m.reshape(p.shape))
            out["exp_avg_sq"].append(v.reshape(p.shape))
        elif p.numel():
            du, dr = _dither(p.numel(), s["dither"], i, torch.tensor(float(t), device=DEV))
            u = _exact_store(torch.sqrt(v), du)
            r = torch.floor(127.0 * m / (_range((b1, b2)) * u.clamp(min=1e-300)) + dr.double() / 8192.0).clamp(-127.0, 127.0)
            out["rms"].append(u.reshape(p.shape))
            out["exp_avg"].append((r / 127.0 * _range((b1, b2)) * u).reshape(p.shape))
        else:
            out["rms"].append(p.double())
            out["exp_avg"].append(p.double())
    return out
