"""Cases of the optimizer's operators: the AdamW step over many tensors at once, with states in 32 or in 8
bits, and the global gradient norm with clipping and loss scaling that goes before it.

Where ``own`` is false they run in plain form, as elementary torch operations; where it is true, as calls of
sodkit.  Both work on the same data: parameters and gradients are flat storages, cut into the tensors of an
encoder-decoder network, as the gradient reducer's buckets are.

The step, in float32 with every operation rounded by itself, t counting the steps from one:

    g = float(grad) * grad_scale * scale_t
    m = b1*m + (1-b1)*g                         v = b2*v + ((1-b2)*g)*g
    w = w*(1-lr*wd) - (lr/(1-b1^t)) * (m / (sqrt(v)/sqrt(1-b2^t) + eps))

In 8 bits a tensor is cut into blocks of 256 elements; a block has two scales, its largest |m| and sqrt(v).
m is a sign and 7 bits, 8 code steps an octave below the scale; sqrt(v) is 8 bits, 16 steps an octave, and
never zero unless v is.  Both are rounded stochastically, by the halves of a 32-bit hash of seed, step,
tensor and element.  The values that the codes stand for are handed out in bfloat16.
"""

import math

import torch

own = False

BLOCK = 256                     # elements of an 8-bit block; tensors start at multiples of it in the states
BUCKET = 25 * (1 << 20)         # bytes of a gradient bucket
GROWTH = 500                    # good steps before the loss scale doubles
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # the affine parameters of a small network's norms, tuned alone: many vectors, all latency
        {"name": "norm_vectors", "op": "norm", "dtype": "fp32", "base": 16, "blocks": "2222", "convs": False,
         "buckets": False, "clip": 1.0, "scaler": False},
        # the gradient buckets of a 25M network in bfloat16, clipped
        {"name": "norm_r50_buckets", "op": "norm", "dtype": "bf16", "base": 64, "blocks": "3463", "convs": True,
         "buckets": True, "clip": 0.5, "scaler": False},
        # a deep float16 network's gradients tensor by tensor, odd sizes, with the dynamic loss scale
        {"name": "norm_odd_scaler", "op": "norm", "dtype": "fp16", "base": 61, "blocks": "34N3", "convs": True,
         "buckets": False, "clip": 0.0, "scaler": True},
        # 1.5G gradients: far more than the caches hold
        {"name": "norm_large", "op": "norm", "dtype": "bf16", "base": 512, "blocks": "3463", "convs": True,
         "buckets": True, "clip": 1.0, "scaler": False},
        # the same vectors' step
        {"name": "adamw_vectors", "op": "adamw", "dtype": "fp32", "base": 16, "blocks": "2222", "convs": False,
         "step": 0, "mult": 0.0, "lr_on_device": False},
        # the 25M network in bfloat16, clipped, the learning rate on the device as in a captured step
        {"name": "adamw_r50", "op": "adamw", "dtype": "bf16", "base": 64, "blocks": "3463", "convs": True,
         "step": 1000, "mult": 0.7, "lr_on_device": True},
        # float16, deep, odd sizes: gradients that start at any two bytes of their bucket, a loss scale to take out
        {"name": "adamw_odd", "op": "adamw", "dtype": "fp16", "base": 61, "blocks": "34N3", "convs": True,
         "step": 17, "mult": 0.0009765625, "lr_on_device": True},
        # 377M parameters in float32, without a copy of their own
        {"name": "adamw_large", "op": "adamw", "dtype": "fp32", "base": 256, "blocks": "3463", "convs": True,
         "step": 100000, "mult": 0.0, "lr_on_device": False},
        # the four again with states in 8 bits
        {"name": "adamw8_vectors", "op": "adamw8", "dtype": "fp32", "base": 16, "blocks": "2222", "convs": False,
         "step": 0, "mult": 0.0, "lr_on_device": False},
        {"name": "adamw8_r50", "op": "adamw8", "dtype": "bf16", "base": 64, "blocks": "3463", "convs": True,
         "step": 1000, "mult": 0.7, "lr_on_device": True},
        {"name": "adamw8_odd", "op": "adamw8", "dtype": "fp16", "base": 61, "blocks": "34N3", "convs": True,
         "step": 17, "mult": 0.0009765625, "lr_on_device": True},
        {"name": "adamw8_large", "op": "adamw8", "dtype": "bf16", "base": 256, "blocks": "3463", "convs": True,
         "step": 100000, "mult": 0.0, "lr_on_device": False},
    ]


def draw(rng):
    op = rng.choice(["norm", "adamw", "adamw8"])
    top = 400 if op == "norm" else 180
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "base": int(round(math.exp(rng.uniform(math.log(5), math.log(top))))),
            "blocks": "".join(str(rng.randint(1, 6)) for _ in range(4)), "convs": rng.random() < 0.85}
    if op == "norm":
        case |= {"buckets": rng.random() < 0.5, "clip": rng.choice([0.0, 0.1, 1.0, 100.0]),
                 "scaler": rng.random() < 0.5}
    else:
        case |= {"step": rng.choice([0, 1, 7, 300, 20000]), "mult": rng.choice([0.0, 0.3, 2.0 ** -10]),
                 "lr_on_device": rng.random() < 0.5}
    return case


# ---------------------------------------------------------------------------------------------- the tensors

def shapes(case):
    """(convolution weights, vectors) of a network with bottleneck stages and a decoder of `base` channels:
    [cout, r, s, cin] each, and scale and shift of every convolution's norm.  "N" stands for 23 blocks."""
    b = case["base"]
    convs, cin, outs = [(b, 7, 7, 3)], b, [b]
    for s, n in enumerate(case["blocks"]):
        w = b << s
        for i in range(23 if n == "N" else int(n)):
            convs += [(w, 1, 1, cin), (w, 3, 3, w), (4 * w, 1, 1, w)]
            if i == 0:
                convs.append((4 * w, 1, 1, cin))
            cin = 4 * w
        outs.append(cin)
    convs += [(b, 1, 1, c) for c in outs] + [(b, 3, 3, b)] * 20 + [(b // 2, 3, 3, b)]
    vectors = [(c[0],) for c in convs for _ in range(2)] + [(1,)]
    convs.append((1, 1, 1, b // 2))
    return (convs if case["convs"] else []), vectors


def sizes(case):
    return [[math.prod(s) for s in group] for group in shapes(case)]


def padded(n):
    return -(-n // BLOCK) * BLOCK


def layout(numels, device):
    """Where tensors that lie end to end lie in the states, where each starts at a multiple of BLOCK: the place
    of every element (`dst`), the element of every place (`src`, the number of elements for a gap), and of
    every block its tensor and its first element."""
    n = torch.tensor(numels, dtype=torch.int64, device=device)
    p = (n + BLOCK - 1) // BLOCK * BLOCK
    start, tight = p.cumsum(0) - p, n.cumsum(0) - n
    total, places = int(n.sum()), int(p.sum())
    dst = torch.repeat_interleave(start - tight, n) + torch.arange(total, device=device)
    src = torch.full((places,), total, dtype=torch.int64, device=device)
    src[dst] = torch.arange(total, device=device)
    tensor = torch.repeat_interleave(torch.arange(len(numels), device=device), p // BLOCK)
    first = torch.arange(places // BLOCK, device=device) * BLOCK - start[tensor]
    return {"dst": dst, "src": src, "tensor": tensor, "first": first, "places": places}


def views(flat, group):
    out, at = [], 0
    for s in group:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += n
    return out


# ---------------------------------------------------------------------------------------------- preparing

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    convs, vectors = shapes(case)
    nc, nv = sizes(case)
    dtype = DTYPES[case["dtype"]]
    # gradients differ in size from tensor to tensor far more than within one
    spread = torch.exp(1.5 * normal(len(nc) + len(nv))) * 1e-3
    each = torch.tensor(nc + nv, dtype=torch.int64, device=dev)
    size = torch.repeat_interleave(spread, each)
    loss_scale = 1024.0 if case["dtype"] == "fp16" else 1.0
    grad = normal(size.numel()).mul_(size).mul_(loss_scale)
    gc, gv = grad[:sum(nc)].to(dtype), grad[sum(nc):].clone()
    st = {"case": case, "gc": gc, "gv": gv}
    if case["op"] == "norm":
        flats = [f for f in (gc, gv) if f.numel()]
        if case["buckets"]:
            st["grads"] = [b for f in flats for b in f.split(BUCKET // f.element_size())]
        else:
            st["grads"] = views(gc, convs) + views(gv, vectors)
        st["flats"] = flats
        if case["dtype"] == "fp16" or case["scaler"]:
            st["loss_scale"] = torch.tensor(loss_scale, device=dev)
        if case["scaler"]:
            st["good"] = torch.tensor(GROWTH - 2.0, device=dev)
            st["skips"] = torch.tensor(3.0, device=dev)
        return st

    w = normal(size.numel()) * 0.05
    st |= {"pc": w[:sum(nc)].to(dtype), "pv": w[sum(nc):].clone(), "t": case["step"], "seed": 1234 + seed % 1000,
           "betas": (0.9, 0.999), "eps": 1e-8, "wd": 0.05, "grad_scale": 0.125}
    lr = 1e-3
    st["lr"] = torch.tensor(lr, device=dev) if case["lr_on_device"] else lr
    st["mult"] = torch.tensor(case["mult"], device=dev) if case["mult"] else None
    lay = layout(nc + nv, dev)
    st["lay"], st["lc"] = lay, sum(padded(n) for n in nc)
    live = lay["src"] < size.numel()
    here = torch.cat([size, size.new_zeros(1)])[lay["src"]] * 0.1
    if case["op"] == "adamw":
        st["m"] = normal(lay["places"]) * here
        st["v"] = (normal(lay["places"]) * 3 * here).square_()
    else:
        # codes of a run under way: signs and sizes of every kind, gaps zero
        st["m"] = torch.randint(1, 256, (lay["places"],), device=dev, generator=gen, dtype=torch.uint8)
        st["m"][(st["m"] == 128) | ~live] = 0
        st["r"] = torch.randint(1, 256, (lay["places"],), device=dev, generator=gen, dtype=torch.uint8)
        st["r"][~live] = 0
        top = here.view(-1, BLOCK).amax(1)
        st["scales"] = torch.stack([top, 3 * top], 1).contiguous()
    if dtype != torch.float32:
        st["master"] = torch.cat([st["pc"], st["pc"].new_zeros(1)])[
            torch.where(lay["src"][:st["lc"]] < sum(nc), lay["src"][:st["lc"]], sum(nc))].float()
    if own:
        # what a training program keeps: its parameters, their gradients' places and the optimizer
        from sodkit.ops import SodAdamW
        pc = [torch.nn.Parameter(p) for p in views(st["pc"], convs)]
        pv = [torch.nn.Parameter(p) for p in views(st["pv"], vectors)]
        for p, g in zip(pc + pv, views(gc, convs) + views(gv, vectors)):
            p.grad = g
        opt = SodAdamW([{"params": pc, "weight_decay": st["wd"]}, {"params": pv, "weight_decay": 0.0}],
                       betas=st["betas"], eps=st["eps"], state_bits=32 if case["op"] == "adamw" else 8,
                       seed=st["seed"])
        if case["op"] == "adamw":
            opt.exp_avg.copy_(st["m"])
            opt.exp_avg_sq.copy_(st["v"])
        else:
            opt.code_m.copy_(st["m"])
            opt.code_r.copy_(st["r"])
            opt.scales.copy_(st["scales"])
        opt.set_step(st["t"])
        st["opt"] = opt
    return st


# ---------------------------------------------------------------------------------------------- running

def run(st):
    op = st["case"]["op"]
    if op == "norm":
        return _own_norm(st) if own else _plain_norm(st)
    return _own_step(st) if own else _plain_step(st, op == "adamw8")


def _own_norm(st):
    from sodkit import ops
    norm, mult = ops.grad_norm(st["grads"], prescale=0.125, max_norm=st["case"]["clip"],
                               loss_scale=st.get("loss_scale"), good_steps=st.get("good"), skips=st.get("skips"),
                               growth_interval=GROWTH)
    return {"norm": norm, "mult": mult, **{k: st[k] for k in ("loss_scale", "good", "skips") if k in st}}


def _own_step(st):
    opt = st["opt"]
    opt.step(st["lr"], st["grad_scale"], scale_t=st["mult"])
    m, v = opt.moments()
    return _outputs(st, m, v, opt.master)


def _outputs(st, m, v, master):
    out = {"vectors": st["pv"], "m": m, "v": v}
    if st["pc"].numel():
        out["convs"] = st["pc"]
    if "master" in st and st["pc"].numel():
        out["master"] = master
    return out


def _plain_norm(st):
    case = st["case"]
    total = sum(f.double().square().sum() for f in st["flats"])
    scale = st["loss_scale"].double() if "loss_scale" in st else torch.ones_like(total)
    norm = (total.sqrt() * 0.125 / scale).float()
    fine = norm.isfinite()
    clip = (case["clip"] / (norm.double() + 1e-6)).clamp(max=1.0) if case["clip"] > 0 else torch.ones_like(total)
    tiny = torch.finfo(torch.float32).tiny
    mult = torch.where(fine, (clip / scale).float().clamp(min=tiny), torch.zeros_like(norm))
    out = {"norm": norm, "mult": mult}
    if case["scaler"]:
        good = torch.where(fine, st["good"] + 1, torch.zeros_like(norm))
        grow = good >= GROWTH
        up = torch.where(grow, (st["loss_scale"] * 2).clamp(max=65536.0), st["loss_scale"])
        st["loss_scale"].copy_(torch.where(fine, up, (st["loss_scale"] * 0.5).clamp(min=1.0)))
        st["good"].copy_(torch.where(grow, torch.zeros_like(good), good))
        st["skips"].add_((~fine).float())
    return {**out, **{k: st[k] for k in ("loss_scale", "good", "skips") if k in st}}


def _mix(h):
    """The finalizer of MurmurHash3 (Appleby, public domain), on int64 that hold 32 bits."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & M32
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & M32
    return h ^ (h >> 16)


def _grid(code, bias, shift):
    """The value at or below one that a code stands for, before its block's scale."""
    return torch.where(code > 0, ((code + bias) << shift).view(torch.float32), torch.zeros((), device=code.device))


def _code(x, top, noise, bias, shift):
    """Codes of x, 0 <= x <= top, rounded up with the chance that `noise` (16 bits) gives."""
    inv = 1.0 / top.clamp(min=2.0 ** -100)
    bits = (x * inv).view(torch.int32).clamp(max=0x3F800000)
    return ((bits + (noise << (shift - 16))) >> shift) - bias


def _plain_step(st, eight):
    (b1, b2), eps, lr, lay, lc = st["betas"], st["eps"], st["lr"], st["lay"], st["lc"]
    st["t"] += 1
    t = st["t"]
    lr64 = lr.double() if torch.is_tensor(lr) else lr
    rate = lr64 / (1 - b1 ** t)
    keep = 1 - lr64 * st["wd"]
    if torch.is_tensor(lr):
        rate, keep = rate.float(), keep.float()
    src, nc = lay["src"], st["pc"].numel()
    none = torch.zeros(1, device=src.device)
    # gradients and weights in the states' places, gaps zero
    g = torch.cat([st["gc"].float(), st["gv"], none])[src]
    g = g * (st["mult"] * st["grad_scale"] if st["mult"] is not None else st["grad_scale"])
    w = torch.cat([st["pc"].float(), st["pv"], none])[src]
    if "master" in st:
        w[:lc] = st["master"]
    if eight:
        cm, cr = st["m"].int(), st["r"].int()
        sm, sr = st["scales"][:, :1], st["scales"][:, 1:]
        m = (_grid(cm & 127, 889, 20).view(-1, BLOCK) * sm).view(-1)
        m = torch.where(cm > 127, -m, m)
        r = (_grid(cr, 1777, 19).view(-1, BLOCK) * sr).view(-1)
        v = r * r
    else:
        m, v = st["m"], st["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    r = v.sqrt()
    w[:lc] = w[:lc] * keep
    w = w - (m / (r * (1 / math.sqrt(1 - b2 ** t)) + eps)) * rate
    if eight:
        key = _mix(torch.full((), (st["seed"] + t * 0x9E3779B9) & M32, dtype=torch.int64, device=src.device))
        key = _mix((_mix((key + lay["tensor"]) & M32) + (lay["first"] >> 32)) & M32)
        i = (lay["first"] & M32).view(-1, 1) + torch.arange(BLOCK, device=src.device)
        h = _mix((i + key.view(-1, 1)) & M32)
        a, r2 = m.abs().view(-1, BLOCK), r.view(-1, BLOCK)
        sm, sr = a.amax(1, keepdim=True), r2.amax(1, keepdim=True)
        cm = _code(a, sm, (h >> 16).int(), 889, 20).clamp(min=0)
        cr = torch.where(r2 > 0, _code(r2, sr, (h & 0xFFFF).int(), 1777, 19).clamp(min=1), 0)
        neg = (m.view(-1, BLOCK) < 0) & (cm > 0)
        st["m"] = (cm + 128 * neg).to(torch.uint8).view(-1)
        st["r"] = cr.to(torch.uint8).view(-1)
        st["scales"] = torch.cat([sm, sr], 1)
        m = (torch.where(neg, -_grid(cm, 889, 20), _grid(cm, 889, 20)) * sm).view(-1).bfloat16()
        r = _grid(cr, 1777, 19) * sr
        v = (r * r).view(-1).bfloat16()
    else:
        st["m"], st["v"] = m, v
    new = w[lay["dst"]]
    big = torch.finfo(st["pc"].dtype).max
    st["pc"].copy_(new[:nc].clamp(-big, big))
    st["pv"].copy_(new[nc:])
    if "master" in st:
        st["master"] = w[:lc]
    return _outputs(st, m, v, st.get("master"))


# ---------------------------------------------------------------------------------------------- accounting

def work(case):
    nc, nv = sizes(case)
    c, v = sum(nc), sum(nv)
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        return {"bytes": c * e + v * 4, "flops": 2 * (c + v)}
    # weight in and out; a gradient in and a parameter out of 16 bits each, or a gradient of 32
    weights = (c + v) * 12
    if case["op"] == "adamw":
        return {"bytes": weights + (c + v) * 16, "flops": 15 * (c + v)}
    places = sum(padded(n) for n in nc + nv)
    # one byte each in and out, the blocks' scales, and the values that the codes stand for
    return {"bytes": weights + (c + v) * 4 + places // BLOCK * 16 + places * 4, "flops": 40 * (c + v)}


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """From the definition, tensor by tensor and in float64.  A code whose rounding lies on a border may come out
    one step away from a computation in 32 bits."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return _exact_norm(st) if case["op"] == "norm" else _exact_step(st, case["op"] == "adamw8")


def _exact_norm(st):
    case = st["case"]
    s = 0.0
    for f in st["flats"]:
        for part in f.split(1 << 26):
            s += float((part.double() ** 2).sum())
    scale = float(st["loss_scale"]) if "loss_scale" in st else 1.0
    norm = math.sqrt(s) / 8 / scale
    if not math.isfinite(norm) or norm > 3.4028235677973366e38:
        norm, mult = math.inf, 0.0
    else:
        mult = (min(1.0, case["clip"] / (norm + 1e-6)) if case["clip"] > 0 else 1.0) / scale
    out = {"norm": norm, "mult": mult}
    if "loss_scale" in st:
        out["loss_scale"] = scale
    if case["scaler"]:
        good = float(st["good"]) + 1 if math.isfinite(norm) else 0.0
        if not math.isfinite(norm):
            out["loss_scale"] = max(scale / 2, 1.0)
        elif good >= GROWTH:
            out["loss_scale"], good = min(scale * 2, 65536.0), 0.0
        out |= {"good": good, "skips": float(st["skips"]) + (not math.isfinite(norm))}
    return {k: torch.tensor(x, dtype=torch.float64, device="cuda") for k, x in out.items()}


def _hash32(x):
    for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35), (16, None)):
        x = x ^ (x >> shift)
        if factor is not None:
            x = (x * factor) % (1 << 32)
    return x


def _level(c, top, steps):
    """The value of code c where `top` stands for one and an octave has `steps`."""
    down = top - c.double()
    octave = torch.ceil(down / steps)
    return torch.where(c > 0, torch.exp2(-octave) * (1 + (octave * steps - down) / steps), 0.0)


def _rounded(x, top, steps, chance):
    """Codes of 0 <= x <= 1, rounded up where the part past the lower code and `chance` make one."""
    frac, e = torch.frexp(x)
    up = top - steps * (1 - e.double()) + (2 * frac - 1) * steps
    return torch.where(x > 0, torch.floor(up + chance), -1.0)


def _exact_step(st, eight):
    (b1, b2), eps, t = st["betas"], st["eps"], st["t"] + 1
    lr = float(st["lr"])
    scale = st["grad_scale"] * (float(st["mult"]) if st["mult"] is not None else 1.0)
    nc, nv = sizes(st["case"])
    lc, convs = st["lc"], sum(nc)
    places = st["lay"]["places"]
    m_out = torch.zeros(places, dtype=torch.float64, device="cuda")
    v_out = torch.zeros_like(m_out)
    w_out = torch.zeros_like(m_out)
    tight = torch.zeros(convs + sum(nv), dtype=torch.float64, device="cuda")
    at = place = 0
    for k, n in enumerate(nc + nv):
        conv = k < len(nc)
        g = (st["gc"][at:at + n] if conv else st["gv"][at - convs:at - convs + n]).double() * scale
        if conv and "master" in st:
            w = st["master"][place:place + n].double()
        else:
            w = (st["pc"][at:at + n] if conv else st["pv"][at - convs:at - convs + n]).double()
        here = slice(place, place + n)
        if eight:
            blocks = torch.arange(n, device="cuda") // BLOCK
            s = st["scales"][place // BLOCK:place // BLOCK + -(-n // BLOCK)].double()
            cm, cr = st["m"][here], st["r"][here]
            m = _level(cm % 128, 127, 8) * s[blocks, 0] * torch.where(cm >= 128, -1.0, 1.0)
            v = (_level(cr, 255, 16) * s[blocks, 1]) ** 2
        else:
            m, v = st["m"][here].double(), st["v"][here].double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        w = w * (1 - lr * (st["wd"] if conv else 0.0))
        w = w - lr / (1 - b1 ** t) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + eps)
        if eight:
            i = torch.arange(n, device="cuda")
            key = _hash32((st["seed"] + t * 0x9E3779B9) % (1 << 32))
            key = _hash32((_hash32((key + k) % (1 << 32)) + (i >> 32)) % (1 << 32))
            h = _hash32((i + key) % (1 << 32))
            r = torch.sqrt(v)
            full = -(-n // BLOCK) * BLOCK
            sm, sr = (torch.nn.functional.pad(x, (0, full - n)).view(-1, BLOCK).amax(1)[blocks] for x in (m.abs(), r))
            cm = _rounded(m.abs() / sm.clamp(min=2.0 ** -100), 127, 8, (h >> 16).double() / 65536).clamp(min=0)
            cr = _rounded(r / sr.clamp(min=2.0 ** -100), 255, 16, (h % 65536).double() / 65536).clamp(min=1)
            m = _level(cm, 127, 8) * sm * m.sign()
            v = torch.where(r > 0, _level(cr, 255, 16) * sr, 0.0) ** 2
        m_out[here], v_out[here], w_out[here], tight[at:at + n] = m, v, w, w
        at, place = at + n, place + full if eight else place + padded(n)
    out = {"vectors": tight[convs:], "m": m_out, "v": v_out}
    if convs:
        out["convs"] = tight[:convs]
        if "master" in st:
            out["master"] = w_out[:lc]
    return out
