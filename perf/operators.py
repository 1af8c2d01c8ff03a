"""What is measured of the first-order steps over the tensors of a model: the AdamW step with its moments in 32 bits, the same step
with its moments in 8 bits, and the norm over all gradients that clips them.

Every case is a model: `layers` blocks of four width x width and three width x ffn matrices and two vectors of width, a table of
vocab x width and a last vector; with layers = 0 it is one vector of `width` elements, what the quasi-Newton optimisers work on.
Tensors lie one after the other in one buffer, each from a multiple of 128 elements on; what lies between them is zero and stays so.

`run` gives the operators in elementary torch operations over the whole buffers, or, with `own`, by the calls of stochqn_amd.
"""
import math

import torch

own = False

BLOCK = 128                                     # elements that share the scale of an 8-bit moment, and the grain of the layout
BETA1, BETA2, EPS, DECAY = 0.9, 0.999, 1e-8, 0.01
STEP_SIZE, MAX_NORM = 1e-4, 1.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
GOLDEN = 0x9E3779B97F4A7C15                     # of the counter-based generator: 2^64 / golden ratio ...
STEP_KEY = 0xD1B54A32D192ED03                   # ... and what a step's number is multiplied with
LANE = 0x9E3779B9                               # between the eight elements of a group


def model(op, layers, width, ffn, vocab, **kw):
    return dict(dict(op=op, layers=layers, width=width, ffn=ffn, vocab=vocab, param="f32", grad="f32", master=False, bits=32,
                     stochastic=False), **kw)


def listed():
    return [
        # one vector of 1e3 variables: what a call costs
        model("step", 0, 1000, 0, 0, name="step 1e3 vector"),
        # the 1e8 variables of the framework's headline configuration, all in 32 bits
        model("step", 0, 100_000_000, 0, 0, name="step 1e8 vector"),
        # a small model of odd sizes, trained in bf16 with 32-bit weights beside it
        model("step", 6, 321, 853, 1009, param="bf16", grad="bf16", master=True, name="step odd layers"),
        # a large model, trained in bf16 with 32-bit weights beside it
        model("step", 24, 2048, 5504, 32000, param="bf16", grad="bf16", master=True, name="step layers"),
        # the smallest model, moments in 8 bits: what a call costs
        model("step", 2, 64, 172, 257, bits=8, name="step8 small"),
        # a small model of odd sizes whose weights are bf16 alone
        model("step", 6, 321, 853, 1009, param="bf16", grad="bf16", bits=8, stochastic=True, name="step8 odd layers"),
        # the headline configuration's vector, moments in 8 bits
        model("step", 0, 100_000_000, 0, 0, bits=8, name="step8 1e8 vector"),
        # a large model whose weights are bf16 alone: the least memory that it can be trained in
        model("step", 24, 2048, 5504, 32000, param="bf16", grad="bf16", bits=8, stochastic=True, name="step8 layers"),
        # a small model's norm: what the calls cost
        model("norm", 6, 321, 853, 1009, grad="bf16", name="norm odd layers"),
        # the headline configuration's vector
        model("norm", 0, 100_000_000, 0, 0, name="norm 1e8 vector"),
        # a large model's
        model("norm", 24, 2048, 5504, 32000, grad="bf16", name="norm layers"),
        # a whole step in f16 with loss scaling: the norm, its coefficient, the step that takes it from the device
        model("clipped", 12, 1024, 2816, 50001, param="f16", grad="f16", master=True, bits=8, name="clipped step8 layers"),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["step", "step", "step8", "step8", "norm", "clipped"])
    grad = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        kw = dict(grad=grad)
    else:
        param = rng.choice(["f32", "bf16", "f16"]) if grad == "f32" else grad
        master = param == "f16" or (param == "bf16" and rng.random() < 0.5)
        kw = dict(grad=grad, param=param, master=master, bits=8 if op == "step8" or (op == "clipped" and rng.random() < 0.5) else 32,
                  stochastic=param == "bf16" and not master)
    op = "step" if op == "step8" else op
    if rng.random() < 0.25:
        return model(op, 0, log(1000, 200_000_000), 0, 0, **kw)
    width = log(64, 2048)
    return model(op, rng.randint(1, 24), width, int(width * rng.uniform(2, 4)), log(257, 50_001) if width < 1500 else log(257, 32_000), **kw)


def layout(c):
    """(sizes, offsets, elements in all) of a case's tensors."""
    d, f = c["width"], c["ffn"]
    sizes = ([d * d] * 4 + [d * f] * 3 + [d] * 2) * c["layers"] + ([c["vocab"] * d] if c["vocab"] else []) + [d]
    offsets, at = [], 0
    for s in sizes:
        offsets.append(at)
        at += -(-s // BLOCK) * BLOCK
    return sizes, offsets, at


def work(case):
    sizes, _, total = layout(case)
    n, grad = sum(sizes), SIZE[case["grad"]]
    if case["op"] == "norm":
        return {"bytes": n * grad, "flops": 2 * n}
    weights = 8 if case["param"] == "f32" else 2 + 8 if case["master"] else 4
    moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK       # a byte of scale for each block and moment, read and written
    return {"bytes": n * (grad + weights + moments), "flops": n * (18 if case["op"] == "step" else 20)}


def prepare(case, seed):
    sizes, offsets, total = layout(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(n):
        return torch.randn(n, device="cuda", generator=gen)

    def hole(flat):                                             # nothing between the tensors
        for n, at in zip(sizes, offsets):
            if n % BLOCK:
                flat[at + n:at + -(-n // BLOCK) * BLOCK] = 0
        return flat

    # gradients whose size differs from one row of a matrix to the next, and rows that nothing has touched (a table's unseen words)
    row = 10 ** normal(total // BLOCK).mul_(0.5).sub_(3.5)
    row = torch.where(torch.rand(total // BLOCK, device="cuda", generator=gen) < 0.05, torch.zeros_like(row), row)
    grad = hole((normal(total).view(-1, BLOCK) * row[:, None]).view(-1))
    s = {"case": dict(case), "seed": 7 + int(seed)}
    if case["op"] != "step":                                    # by a loss scale of 1024, so that small ones do not fall out of f16
        s["loss_scale"] = 1024.0
        grad.mul_(1024.0)
    s["grad"] = grad.to(TYPES[case["grad"]])
    del grad
    if case["op"] != "norm":
        w = hole(normal(total).mul_(0.02))
        s["param"] = w.to(TYPES[case["param"]])
        s["master"] = w.clone() if case["master"] else None
        del w
        m = hole((normal(total).view(-1, BLOCK) * row[:, None] * 0.3).view(-1))
        v = hole((torch.rand(total, device="cuda", generator=gen).add_(0.5).view(-1, BLOCK) * (row * row)[:, None]).view(-1))
        s["count"] = torch.tensor([100 + int(seed) % 1000, 0], dtype=torch.int64, device="cuda")
        if case["bits"] == 32:
            s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
        else:
            half = torch.full((), 0.5, dtype=torch.float64, device="cuda")
            s["m"], s["m_scale"] = to_codes(m, half, 7, 3, -6, torch.float8_e4m3fn)
            s["v"], s["v_scale"] = to_codes(v, half, 14, 2, -14, torch.float8_e5m2)
        del m, v
    if own:
        import stochqn_amd

        def tensors(flat):
            return [flat[at:at + n] for n, at in zip(sizes, offsets)]
        s["grads"] = stochqn_amd.TensorList(tensors(s["grad"]))
        if case["op"] != "norm":
            opt = stochqn_amd.AdamW_free(tensors(s["param"]), beta1=BETA1, beta2=BETA2, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                         master=case["master"], stochastic=case["stochastic"], seed=s["seed"])
            for name in ("m", "v", "m_scale", "v_scale", "master", "count"):
                if s[name] is not None:
                    getattr(opt, name).copy_(s[name])
                    s[name] = getattr(opt, name)
            opt.update_gradient(s["grads"])
            s["opt"] = opt
    return s


def run(s):
    c = s["case"]
    if own:
        if c["op"] == "norm":
            return s["grads"].norm(max_norm=MAX_NORM, grad_scale=1 / s["loss_scale"])
        if c["op"] == "clipped":
            clip = s["grads"].norm(max_norm=MAX_NORM, grad_scale=1 / s["loss_scale"])
            s["opt"].run_optimizer(STEP_SIZE, grad_scale=clip[1:])
        else:
            clip = None
            s["opt"].run_optimizer(STEP_SIZE)
    else:
        clip = None if c["op"] == "step" else plain_norm(s["grad"], 1 / s["loss_scale"])
        if c["op"] == "norm":
            return clip
        plain_step(s, None if clip is None else clip[1])
    return {"param": s["param"], "master": s["master"], "m": s["m"], "v": s["v"], "m_scale": s["m_scale"], "v_scale": s["v_scale"],
            "count": s["count"][:1], "clip": clip}


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------
def plain_norm(grad, grad_scale):
    """The norm of all gradients times grad_scale, and what they are to be multiplied with so that it is at most MAX_NORM."""
    norm = grad.double().square().sum().sqrt() * grad_scale
    return torch.stack([norm, grad_scale * torch.clamp(MAX_NORM / norm, max=1.0)]).float()


def finalise(z):
    """A bijection of 64 bits (in int64: products and sums modulo 2^64, logical shifts)."""
    z = (z ^ ((z >> 30) & (1 << 34) - 1)) * (0xBF58476D1CE4E5B9 - (1 << 64))
    z = (z ^ ((z >> 27) & (1 << 37) - 1)) * (0x94D049BB133111EB - (1 << 64))
    return z ^ ((z >> 31) & (1 << 33) - 1)


def uniform(total, seed, t):
    """Two words of 32 bits for every element: of each group of eight one word of 64 bits, its halves advanced by a golden step."""
    key = finalise(seed ^ (t * (STEP_KEY - (1 << 64))))
    word = finalise(key + torch.arange(total // 8, device="cuda") * (GOLDEN - (1 << 64)))
    lane = torch.arange(8, device="cuda") * LANE
    return [((half[:, None] + lane) & 0xFFFFFFFF).view(-1) for half in (word, word >> 32)]


def to_codes(x, u, top, mantissa, least, kind):
    """Blocks of x over a scale that is a power of two and brings the largest of them to 2^top .. 2^(top + 1), each value to one of its two
    neighbours in the 8-bit type, away from zero where the rest plus u (0 <= u < 1) reaches a whole step."""
    x = x.view(-1, BLOCK)
    _, e = torch.frexp(x.abs().amax(1).clamp(min=2.0 ** -126))
    scale = torch.ldexp(torch.ones((), dtype=torch.float64, device="cuda"), (e - 1 - top).clamp(min=-126))
    x = x.double() / scale[:, None]
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones((), dtype=torch.float64, device="cuda"), (e - 1).clamp(min=least) - mantissa)
    q = torch.floor(x.abs() / step + u.view(-1, BLOCK) if u.dim() else x.abs() / step + u) * step
    if kind == torch.float8_e5m2:                               # a second moment above zero stays above zero
        q = torch.where(x > 0, q.clamp(min=2.0 ** (least - mantissa)), q)
    return torch.copysign(q, x).float().to(kind).view(-1), scale.float().to(torch.float8_e8m0fnu)


def from_codes(code, scale):
    return (code.float().view(-1, BLOCK) * scale.float()[:, None]).view(-1)


def plain_step(s, scale):
    c = s["case"]
    t = s["count"][0] + 1
    g = s["grad"].float() if scale is None else s["grad"].float() * scale
    m = s["m"] if c["bits"] == 32 else from_codes(s["m"], s["m_scale"])
    v = s["v"] if c["bits"] == 32 else from_codes(s["v"], s["v_scale"])
    p = s["master"] if c["master"] else s["param"].float()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    one = 1 - BETA1 ** t.double(), torch.sqrt(1 - BETA2 ** t.double())
    p = p * (1 - STEP_SIZE * DECAY) - (STEP_SIZE / one[0]).float() * (m / (torch.sqrt(v) * (1 / one[1]).float() + EPS))
    if c["bits"] == 8 or c["stochastic"]:
        um, uv = uniform(m.numel(), s["seed"], t)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        for name, x, u, kind in (("m", m, um, (7, 3, -6, torch.float8_e4m3fn)), ("v", v, uv, (14, 2, -14, torch.float8_e5m2))):
            code, by = to_codes(x, u * 2.0 ** -32, *kind)
            s[name].copy_(code)
            s[name + "_scale"].copy_(by)
    if c["master"]:
        s["master"].copy_(p)
    if c["stochastic"]:                                         # to one of the two bf16 beside it, by the low half of the first word
        p = ((p.view(torch.int32) + (um & 0xFFFF).int()) & -0x10000).view(torch.float32)
    s["param"].copy_(p)
    s["count"][0] += 1


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    f64 = torch.float64
    g = s["grad"].to(f64)
    clip = None
    if case["op"] != "step":
        norm = torch.linalg.vector_norm(g) / s["loss_scale"]
        clip = torch.stack([norm, min(1.0, MAX_NORM / norm.item()) / s["loss_scale"] * torch.ones_like(norm)])
        if case["op"] == "norm":
            return clip
        g *= clip[1]
    n, t = g.numel(), int(s["count"][0]) + 1
    states = []
    for name in ("m", "v"):
        x = s.pop(name).to(f64)
        by = s.pop(name + "_scale")
        states.append(x if by is None else x * by.to(f64).repeat_interleave(BLOCK))
    m = torch.lerp(g, states.pop(0), BETA1)
    v = torch.lerp(g.square_(), states.pop(0), BETA2)
    del g, x
    p = (s["master"] if case["master"] else s["param"]).to(f64)
    p -= STEP_SIZE * (DECAY * p + (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt_() + EPS))
    out = {"param": p, "master": p if case["master"] else None, "m": m, "v": v, "m_scale": None, "v_scale": None, "count": None, "clip": clip}
    if case["bits"] == 8 or case["stochastic"]:
        first, second = words(n, s["seed"], t)
    if case["bits"] == 8:
        out["m"], out["m_scale"] = rounded(m, first, 2.0 ** 8, 3, 2.0 ** -6, 0.0)
        out["v"], out["v_scale"] = rounded(v, second, 2.0 ** 15, 2, 2.0 ** -14, 2.0 ** -16)
    if case["stochastic"]:
        step = 2.0 ** (torch.floor(torch.log2(p.float().abs().clamp(min=2.0 ** -126))).to(f64) - 7)
        low = (first % 65536).to(f64) / 65536
        out["param"] = torch.sign(p) * torch.floor((p.float().to(f64) / step).abs() + low) * step
    elif case["param"] != "f32":
        out["param"] = p.to(TYPES[case["param"]]).to(f64)
    return out


def words(n, seed, t):
    """The words that stochastic rounding adds, from Python's whole numbers for the key and from 16-bit limbs for the groups."""
    def whole(z):
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) % 2 ** 64
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) % 2 ** 64
        return z ^ (z >> 31)

    def times(hi, lo, c):                                       # (hi, lo) of 32 bits each times a constant of 64, modulo 2^64
        ch, cl = c >> 32, c & 0xFFFFFFFF
        a, b = lo & 0xFFFF, lo >> 16
        low = a * (cl & 0xFFFF)
        mid = a * (cl >> 16) + b * (cl & 0xFFFF) + (low >> 16)
        top = (b * (cl >> 16) + (mid >> 16)) + (lo & 0xFFFF) * (ch & 0xFFFF)
        top = top + (((lo >> 16) * (ch & 0xFFFF) + (lo & 0xFFFF) * (ch >> 16)) & 0xFFFF) * 65536
        top = top + (hi & 0xFFFF) * (cl & 0xFFFF) + ((((hi >> 16) * (cl & 0xFFFF) + (hi & 0xFFFF) * (cl >> 16)) & 0xFFFF) << 16)
        return top & 0xFFFFFFFF, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    def shifted(hi, lo, k):
        return hi ^ (hi >> k), lo ^ ((lo >> k) | ((hi << (32 - k)) & 0xFFFFFFFF))

    key = whole((seed ^ (t * STEP_KEY)) % 2 ** 64)
    group = torch.arange(n // 8, device="cuda")
    hi, lo = times(group >> 32, group & 0xFFFFFFFF, GOLDEN)
    lo = lo + (key & 0xFFFFFFFF)
    hi = (hi + (key >> 32) + (lo >> 32)) & 0xFFFFFFFF
    lo = lo & 0xFFFFFFFF
    hi, lo = times(*shifted(hi, lo, 30), 0xBF58476D1CE4E5B9)
    hi, lo = times(*shifted(hi, lo, 27), 0x94D049BB133111EB)
    hi, lo = shifted(hi, lo, 31)
    at = torch.tensor([j * LANE for j in range(8)], device="cuda")
    return [torch.remainder(torch.add(half.unsqueeze(1), at), 2 ** 32).flatten() for half in (lo, hi)]


def rounded(x, word, over, mantissa, normal, least):
    """x as multiples of a block's scale in the 8-bit type, and the scale."""
    top = x.float().abs().unflatten(0, (-1, BLOCK)).max(dim=1).values.to(torch.float64)
    scale = 2.0 ** (torch.floor(torch.log2(top.clamp(min=2.0 ** -126))) + 1) / over
    scale = scale.clamp(min=2.0 ** -126)
    x = x / scale.repeat_interleave(BLOCK)
    size = x.abs()
    step = 2.0 ** (torch.floor(torch.log2(size.clamp(min=normal))) - mantissa)
    whole = torch.floor(size / step + word.to(torch.float64) / 2 ** 32) * step
    return torch.sign(x) * torch.where(size > 0, whole.clamp(min=least), whole), scale
