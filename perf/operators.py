"""Optimizer operators over many tensors at once: what is timed, and on which sizes.

Four operators of ``superresolution_amd.optim``, each with its plain form beside it:

* ``step``, 32 bits: one AdamW step of a list of parameters, moments in fp32 (with the total gradient norm and the clip
  coefficient in front where ``clip`` is set);
* ``step``, 8 bits: the same with both moments in 8 bits, an e4m3 value for each element and a power of two for each block
  of 32 -- of the first moment, and of the second moment's square root;
* ``norm``: the L2 norm of a list of gradients;
* ``pack`` / ``unpack``: moments written to 8 bits and read back.

``own = False`` computes them from elementary torch operations, ``own = True`` calls the package.

A parameter list's moments lie in one buffer, the part of each tensor padded to whole blocks of 32 elements; the position in
that buffer is what the random bits of the stochastic rounding are drawn from:

    key  = mix(mix(seed) + step * G)        h = mix((lo32(j) + hi32(j) * G) ^ key)         (32-bit arithmetic)
    first moment: h & 0xffff    square root of the second: h >> 16    bf16 parameter: mix(h + G) >> 16
"""
import math
import random

import torch

own = False

LR, BETA1, BETA2, EPS, WD = 1e-4, 0.9, 0.999, 1e-8, 0.01           # the training loops' AdamW
BLOCK = 32
STEP0 = 99                                                         # steps taken before the timed ones
M32, G, MIX_A, MIX_B = 0xFFFFFFFF, 0x9E3779B9, 0x5340508D, 0x7495C5A5


# ---- parameter lists ---------------------------------------------------------------------------------------------------
def _generator_sizes():
    """Element counts of the generator's 167 parameters (16 residual blocks of 96 channels)."""
    conv = 96 * 96 * 9
    sizes = [96 * 3 * 81, 96, 1]
    for i in range(16):
        sizes += [conv, 96, 96, 96, 96, conv, 96, 96, 96]
        if i in (7, 15):
            sizes += [12 * 96, 12, 96 * 12, 96]
    return sizes + [conv, 96, 96, 96, 4 * conv, 384, 1, conv, 96, 1, 3 * 96 * 81, 3]


def _discriminator_sizes():
    """Element counts of the PatchGAN discriminator's 20 parameters."""
    sizes = []
    for cin, cout in ((3, 64), (64, 64), (64, 128), (128, 128), (128, 256), (256, 256), (256, 512), (512, 512), (512, 256), (256, 1)):
        sizes += [9 * cin * cout, cout]
    return sizes


def _ragged_sizes(count, total):
    """``count`` odd and even sizes with ``total`` elements, spread over several powers of ten as a model's weights and
    biases are."""
    if count == 1:
        return [total]
    r = random.Random(1000003 * count + total)
    w = [math.exp(r.uniform(0.0, 9.0)) for _ in range(count)]
    sizes = [1 + int((total - count) * x / sum(w)) for x in w]
    sizes[sizes.index(max(sizes))] += total - sum(sizes)
    return sizes


def _sizes(case):
    if case["sizes"] == "generator":
        return _generator_sizes()
    if case["sizes"] == "discriminator":
        return _discriminator_sizes()
    return _ragged_sizes(case["count"], case["total"])


def _padded(n):
    return -(-n // BLOCK) * BLOCK


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of slopes and biases fine-tuned alone: launch latency
        dict(name="step32 one small tensor", kind="step", bits=32, dtype="fp32", sizes="ragged", count=1, total=4099, clip=0.0),
        # the generator's own step in the training loop, gradient clipping included
        dict(name="step32 generator clipped", kind="step", bits=32, dtype="fp32", sizes="generator", count=167, total=3214974, clip=0.5),
        # a bf16 network of some hundred layers
        dict(name="step32 bf16 300 tensors", kind="step", bits=32, dtype="bf16", sizes="ragged", count=300, total=40000003, clip=0.0),
        # one flat buffer of a large network
        dict(name="step32 one large tensor", kind="step", bits=32, dtype="fp32", sizes="ragged", count=1, total=268435456, clip=0.0),
        # a few small tensors, moments in 8 bits: latency
        dict(name="step8 five small tensors", kind="step", bits=8, dtype="fp32", sizes="ragged", count=5, total=10007, clip=0.0),
        # the discriminator's step with small state
        dict(name="step8 discriminator", kind="step", bits=8, dtype="fp32", sizes="discriminator", count=20, total=5867585, clip=0.0),
        # a large fp32 network with clipping
        dict(name="step8 400 tensors clipped", kind="step", bits=8, dtype="fp32", sizes="ragged", count=400, total=100000007, clip=1.0),
        # the least memory a large bf16 network trains in
        dict(name="step8 bf16 large tensor", kind="step", bits=8, dtype="bf16", sizes="ragged", count=1, total=268435493, clip=0.0),
        # the training loop's logged gradient norm
        dict(name="norm generator", kind="norm", bits=32, dtype="fp32", sizes="generator", count=167, total=3214974, clip=0.0),
        # the norm of a large bf16 network's gradients
        dict(name="norm bf16 500 tensors", kind="norm", bits=32, dtype="bf16", sizes="ragged", count=500, total=120000001, clip=0.0),
        # a checkpoint's moments of the generator, taken into 8 bits
        dict(name="pack generator", kind="pack", bits=8, dtype="fp32", sizes="ragged", count=1, total=3214974, clip=0.0),
        # the moments of a large network read back for a checkpoint
        dict(name="unpack large", kind="unpack", bits=8, dtype="fp32", sizes="ragged", count=1, total=60000011, clip=0.0),
    ]


def draw(rng):
    kind = rng.choice(("step", "step", "step", "step", "norm", "pack", "unpack"))
    total = int(2.0 ** rng.uniform(8.0, 27.0)) | rng.randint(0, 1)
    count = 1 if kind in ("pack", "unpack") else min(int(2.0 ** rng.uniform(0.0, 9.0)), max(1, total // 8))
    return dict(kind=kind, bits=rng.choice((8, 32)) if kind == "step" else 32 if kind == "norm" else 8,
                dtype=rng.choice(("fp32", "bf16")) if kind in ("step", "norm") else "fp32", sizes="ragged", count=count, total=total,
                clip=rng.choice((0.0, 0.5, 1e6)) if kind == "step" else 0.0)


def work(case):
    n = case["total"]
    w = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        return {"bytes": n * w + 4, "flops": 2 * n}
    moments8 = 2 * n + 2 * -(-n // BLOCK)                             # a byte for each moment, a byte for each block's scale
    if case["kind"] in ("pack", "unpack"):
        return {"bytes": 8 * n + moments8, "flops": 8 * n}
    moments = 8 * n if case["bits"] == 32 else moments8
    # gradient read, parameter and moments read and written; clipping needs the gradients a second time
    return {"bytes": 3 * n * w + 2 * moments + (n * w if case["clip"] else 0), "flops": (16 if case["bits"] == 32 else 60) * n}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    sizes = _sizes(case)
    dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    starts, n = [], 0
    for k in sizes:
        starts.append(n)
        n += _padded(k)
    s = {"case": dict(case), "sizes": sizes, "starts": starts, "n": n, "seed": seed & 0x7FFFFFFF, "t": STEP0}
    # gradients of one scale for each tensor, some of them exactly zero, one after another as a backward pass leaves them
    scale = (torch.randn(len(sizes), generator=gen, device=dev) * 1.5).exp_() * 1e-3
    per = scale.repeat_interleave(torch.tensor(sizes, device=dev), output_size=sum(sizes))
    flat_g = torch.randn(sum(sizes), generator=gen, device=dev).mul_(per)
    flat_g.mul_(torch.rand(flat_g.shape, generator=gen, device=dev).gt_(0.03))
    if case["kind"] == "norm":
        s["grads"] = list(flat_g.to(dtype).split(sizes))
        return s
    # moments as some steps of such gradients leave them, in the padded layout
    m = torch.zeros(n, device=dev)
    v = torch.zeros(n, device=dev)
    m0 = torch.randn(flat_g.shape, generator=gen, device=dev).mul_(per).mul_(0.3)
    v0 = torch.randn(flat_g.shape, generator=gen, device=dev).square_().add_(0.05).mul_(per).mul_(per)
    for k, a, b, c in zip(sizes, starts, m0.split(sizes), v0.split(sizes)):
        m[a:a + k], v[a:a + k] = b, c
    del m0, v0, per
    if case["kind"] == "pack":
        s["m"], s["v"] = m[:case["total"]], v[:case["total"]]
        return s
    if case["bits"] == 8:
        s["m8"], s["me"] = _encode(m, torch.full((n,), 0x8000, device=dev), False)
        s["r8"], s["re"] = _encode(_root(v), torch.full((n,), 0x8000, device=dev), True)
        if case["kind"] == "unpack":
            return s
        m, v = _decode(s["m8"], s["me"]), _decode(s["r8"], s["re"]).square()
    else:
        s["m"], s["v"] = m, v
    s["flat_p"] = torch.zeros(n, device=dev, dtype=dtype)
    s["params"] = [torch.nn.Parameter(s["flat_p"][a:a + k]) for a, k in zip(starts, sizes)]
    for p in s["params"]:
        p.data.normal_(0.0, 0.05, generator=gen)
    s["flat_g"] = flat_g.to(dtype)
    for p, g in zip(s["params"], s["flat_g"].split(sizes)):
        p.grad = g
    if own:
        from superresolution_amd import optim
        s["opt"] = optim.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=WD, state_bits=case["bits"],
                               max_grad_norm=case["clip"] or None, seed=s["seed"])
        sd = s["opt"].state_dict()
        sd["state"] = {i: {"step": torch.tensor(float(STEP0)), "exp_avg": m[a:a + k], "exp_avg_sq": v[a:a + k]}
                       for i, (a, k) in enumerate(zip(starts, sizes))}
        s["opt"].load_state_dict(sd)
        if case["bits"] == 32:
            del s["m"], s["v"]
        else:
            del s["m8"], s["me"], s["r8"], s["re"]
    return s


# ---- the operators -----------------------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "norm":
        return {"norm": torch.cat([g.reshape(-1) for g in s["grads"]]).double().square().sum().sqrt().float()}
    if kind == "pack":
        n = s["m"].numel()
        pad = torch.zeros(_padded(n) - n, device=s["m"].device)
        half = torch.full((_padded(n),), 0x8000, device=s["m"].device)
        m8, me = _encode(torch.cat([s["m"], pad]), half, False)
        r8, re = _encode(_root(torch.cat([s["v"], pad])), half, True)
        return {"m": m8, "m_scale": me, "r": r8, "r_scale": re}
    if kind == "unpack":
        n = s["case"]["total"]
        return {"m": _decode(s["m8"], s["me"])[:n], "v": _decode(s["r8"], s["re"])[:n].square()}
    return _plain_step(s)


def _run_own(s, kind):
    from superresolution_amd import optim
    if kind == "norm":
        return {"norm": optim.total_norm(s["grads"])}
    if kind == "pack":
        m8, me, r8, re = optim.pack_moments(s["m"], s["v"])
        return {"m": m8, "m_scale": me, "r": r8, "r_scale": re}
    if kind == "unpack":
        m, v = optim.unpack_moments(s["m8"], s["me"], s["r8"], s["re"], s["case"]["total"])
        return {"m": m, "v": v}
    opt = s["opt"]
    opt.step()
    mo = opt.moments[0]
    out = {"p": s["flat_p"], "norm": opt.last_grad_norm if s["case"]["clip"] else None}
    if s["case"]["bits"] == 32:
        return {**out, "m": mo.exp_avg, "v": mo.exp_avg_sq}
    return {**out, "m": mo.exp_avg, "m_scale": mo.exp_avg_scale, "r": mo.root, "r_scale": mo.root_scale}


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _mix(x):
    x = x ^ (x >> 16)
    x = (x * MIX_A) & M32
    x = x ^ (x >> 15)
    x = (x * MIX_B) & M32
    return x ^ (x >> 16)


def _hash(n, seed, step, dev):
    key = _mix((_mix(seed & M32) + step * G) & M32)
    j = torch.arange(n, device=dev)
    return _mix(((((j & M32) + (j >> 32) * G) & M32) ^ key))


def _encode(x, rnd, positive):
    """e4m3 values and their blocks' powers of two of the fp32 ``x`` (whole blocks).  The scale is the power of two that puts
    the block's largest magnitude at the top of e4m3's range; ``rnd`` (16 bits) is added under the last bit that is kept,
    and what lies below is cut off.  Not finite: NaN, beside the block's maximum.  ``positive``: what is not zero is not
    stored as zero."""
    bits = x.view(torch.int32) & 0x7FFFFFFF
    bad = bits >= 0x7F800000
    top = bits.masked_fill(bad, 0).view(-1, BLOCK).amax(1)
    e = ((top + 0x1FFFFF) >> 23).clamp_(min=9) - 8                    # the largest is at most 1.75 * 2^8 in units of 2^(e - 127)
    unit = ((127 - e + 1023).to(torch.int64) << 52).view(torch.float64)  # 2^(127 - e)
    y = (x.double().abs().view(-1, BLOCK) * unit[:, None]).view(-1)
    normal = ((y.float().view(torch.int32) + (rnd << 4)) >> 20) - (120 << 3)
    small = ((y * 2.0 ** 25).nan_to_num(posinf=0.0).to(torch.int64) + rnd) >> 16
    code = torch.where(y < 2.0 ** -6, small, normal)
    code = torch.where((x > 0) & (code == 0), 1, code) if positive else code
    code = code.masked_fill(bad, 0x7F) | torch.where(x.view(torch.int32) < 0, 0x80, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _decode(code, scale):
    return (code.float().view(-1, BLOCK) * scale.float()[:, None]).view(-1)


def _root(v):
    """The square root to the nearest fp32."""
    return v.double().sqrt().float()


def _gather(tensors):
    """The tensors one after another, each padded to whole blocks, in fp32."""
    zeros = torch.zeros(BLOCK, device=tensors[0].device, dtype=tensors[0].dtype)
    return torch.cat([x for t in tensors for x in (t.reshape(-1), zeros[:_padded(t.numel()) - t.numel()])]).float()


def _plain_step(s):
    c = s["case"]
    s["t"] += 1
    t = s["t"]
    params = [p.detach() for p in s["params"]]
    g = _gather([p.grad for p in s["params"]])
    p = _gather(params)
    out = {"p": s["flat_p"], "norm": None}
    coef = None
    if c["clip"]:
        out["norm"] = g.double().square().sum().sqrt().float()
        coef = (c["clip"] / (out["norm"].double() + 1e-6)).clamp(max=1.0).float()
    if c["bits"] == 32:
        if coef is not None:
            g = g * coef
        m = s["m"].mul_(BETA1).add_(g, alpha=1.0 - BETA1)
        v = s["v"].mul_(BETA2).addcmul_(g, g, value=1.0 - BETA2)
        r = v.sqrt()
        out.update(m=m, v=v)
    else:
        # the rounded moments lie on a border now and then: evaluated in 64 bits, rounded to 32, and from there to 8
        g = g.double()
        if coef is not None:
            g = g * coef.double()
        m = _decode(s["m8"], s["me"]).double().mul_(BETA1).add_(g, alpha=1.0 - BETA1).float()
        r = _decode(s["r8"], s["re"]).double().square_().mul_(BETA2).addcmul_(g, g, value=1.0 - BETA2).float()
        r = _root(r)
    p = p * (1.0 - LR * WD) - (LR / (1.0 - BETA1 ** t)) * (m / (r / math.sqrt(1.0 - BETA2 ** t) + EPS))
    h = _hash(s["n"], s["seed"], t, p.device) if c["bits"] == 8 or c["dtype"] == "bf16" else None
    if c["bits"] == 8:
        m8, me = _encode(m, h & 0xFFFF, False)
        r8, re = _encode(r, h >> 16, True)
        s["m8"].copy_(m8), s["me"].copy_(me), s["r8"].copy_(r8), s["re"].copy_(re)
        out.update(m=s["m8"], m_scale=s["me"], r=s["r8"], r_scale=s["re"])
    if c["dtype"] == "bf16":                                            # stochastic rounding: random bits under the kept ones
        rnd = (_mix((h + G) & M32) >> 16).to(torch.int32)
        p = (p.view(torch.int32) + rnd).bitwise_and_(-65536).view(torch.float32).to(torch.bfloat16)
    torch._foreach_copy_(params, [p[a:a + k] for a, k in zip(s["starts"], s["sizes"])])
    return out


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _power(e):
    """2^e, exactly (torch.ldexp goes through pow)."""
    return torch.bitwise_left_shift(e.long() + 1023, 52).view(torch.float64)


def _exact_e4m3(x, u, positive):
    """Multiples of e4m3's step at |x| / scale: floor(value / step + u), u in [0, 1)."""
    a = x.abs().view(-1, BLOCK)
    top = a.amax(1, keepdim=True)
    f, e = torch.frexp(top.clamp(min=2.0 ** -117))                     # top = f * 2^e, f in [0.5, 1)
    e = e - 9 + (f > 0.875)                                            # 2^8 <= top / 2^e <= 1.75 * 2^8 or just under 2^8
    e = e.clamp(min=-126)
    y = a * _power(-e)
    _, ey = torch.frexp(y)
    step = _power((ey - 1).clamp(min=-6) - 3)
    k = torch.floor(y / step + u.view(-1, BLOCK))
    if positive:
        k = torch.where((a > 0) & (k == 0), torch.ones_like(k), k)
    return (k * step).view(-1) * torch.sign(x), _power(e).view(-1)


def _exact_hash(n, seed, step, dev):
    def mix(x):
        x = x ^ torch.div(x, 65536, rounding_mode="floor")
        x = (x * MIX_A).remainder(2 ** 32)
        x = x ^ torch.div(x, 32768, rounding_mode="floor")
        x = (x * MIX_B).remainder(2 ** 32)
        return x ^ torch.div(x, 65536, rounding_mode="floor")

    def wide(v):
        return torch.tensor(v, dtype=torch.int64, device=dev)

    key = mix((mix(wide(seed)) + step * G).remainder(2 ** 32))
    h = mix(torch.arange(n, device=dev) ^ key)                          # (n < 2^32)
    return h, mix((h + G).remainder(2 ** 32))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return {"norm": torch.stack([g.double().norm() for g in s["grads"]]).norm()}
    dev = torch.device("cuda")
    if kind == "pack":
        n = case["total"]
        half = torch.full((_padded(n),), 0.5, dtype=torch.float64, device=dev)
        m, v = (torch.nn.functional.pad(x.double(), (0, _padded(n) - n)) for x in (s["m"], s["v"]))
        m8, me = _exact_e4m3(m, half, False)
        r8, re = _exact_e4m3(v.sqrt().float().double(), half, True)
        return {"m": m8, "m_scale": me, "r": r8, "r_scale": re}
    if case["bits"] == 8:
        m, r = (c.double() * e.double().repeat_interleave(BLOCK) for c, e in ((s["m8"], s["me"]), (s["r8"], s["re"])))
        v = r * r
        if kind == "unpack":
            return {"m": m[:case["total"]], "v": v[:case["total"]]}
    else:
        m, v = s["m"].double(), s["v"].double()
    g, t = torch.zeros(s["n"], dtype=torch.float64, device=dev), STEP0 + 1
    for a, k, x in zip(s["starts"], s["sizes"], s["flat_g"].split(s["sizes"])):
        g[a:a + k] = x.double()
    out = {"norm": None}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g *= torch.tensor(min(1.0, case["clip"] / (out["norm"].float().item() + 1e-6))).float().item()
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    out.update(m=m, v=v)
    h, h2 = _exact_hash(s["n"], s["seed"], t, dev)
    if case["bits"] == 8:                                               # the 8-bit state rounds the moments of the 32-bit one
        m, r = m.float().double(), v.float().double().sqrt().float().double()
        m8, me = _exact_e4m3(m, (h % 65536).double() / 65536, False)
        r8, re = _exact_e4m3(r, torch.div(h, 65536, rounding_mode="floor").double() / 65536, True)
        out = {"norm": out["norm"], "m": m8, "m_scale": me, "r": r8, "r_scale": re}
    else:
        r = v.sqrt()
    p = s["flat_p"].double()
    p = (1.0 - LR * WD) * p - LR / (1.0 - BETA1 ** t) * m / (r / (1.0 - BETA2 ** t) ** 0.5 + EPS)
    if case["dtype"] == "bf16":
        a = p.float().double().abs()
        _, e = torch.frexp(a)
        step = _power((e - 1).clamp(min=-126) - 7)
        p = torch.sign(p) * step * torch.floor(a / step + torch.div(h2, 65536, rounding_mode="floor").double() / 65536)
    out["p"] = p
    return out
