"""The AdamW step over many tensors and the norm of their gradients, on the GPU, against the formula in 64 bits (tests/adamw_reference.py)."""
import ctypes as C
import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import adamw_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}                   # half a step relative to the value
SIZES = [1, 0, 7, 8, 127, 128, 129, 2047, 2048, 2049, 5003]
LR = 0.01


def stochqn():
    import stochqn_amd
    assert stochqn_amd.cdll().stochqn_hip_available() == 1
    return stochqn_amd


class Model:
    """Tensors of given sizes inside one buffer each for weights and gradients, `gap` elements of a canary between them."""

    def __init__(self, sizes, ptype, gtype, gap=1, seed=0, grad_size=1e-2):
        self.sizes, self.gap = list(sizes), gap
        self.ptypes = ptype if isinstance(ptype, list) else [ptype] * len(sizes)
        self.gtypes = gtype if isinstance(gtype, list) else [gtype] * len(sizes)
        self.rng = np.random.default_rng(seed)
        self.grad_size = grad_size
        self.pbuf, self.params = self.place(self.ptypes)
        self.gbuf, self.grads = self.place(self.gtypes)
        for p in self.params:
            p.copy_(torch.as_tensor(self.rng.standard_normal(p.numel()).astype(np.float32)))
        self.new_grads()

    def place(self, types):
        bufs, views = [], []
        for n, t in zip(self.sizes, types):
            buf = torch.full((n + 2 * self.gap,), 77.0, dtype=t, device="cuda")
            bufs.append(buf)
            views.append(buf[self.gap:self.gap + n])
        return bufs, views

    def new_grads(self):
        for g in self.grads:
            x = self.rng.standard_normal(g.numel()) * self.grad_size * 10 ** self.rng.uniform(-2, 1)
            x[self.rng.random(g.numel()) < 0.05] = 0
            g.copy_(torch.as_tensor(x.astype(np.float32)))

    def whole(self):
        """No canary was touched."""
        for b in self.pbuf + self.gbuf:
            if self.gap:
                assert (b[:self.gap] == 77).all() and (b[-self.gap:] == 77).all()


def host(t):
    return t.detach().float().cpu().numpy().reshape(-1)


def codes(t):
    return t.view(torch.uint8).cpu().numpy()


def check_step(model, opt, lr=LR, scale=1.0, decay=None, **run):
    """One step of `opt`, every array of it held to the reference from the state before."""
    b1, b2, eps, wd, t = opt.beta1, opt.beta2, opt.eps, opt.weight_decay, int(opt.count[0]) + 1
    before = {}
    for i, n in enumerate(model.sizes):
        at = opt.offsets[i]
        pad = at + -(-n // 128) * 128
        w = opt.master[at:at + n] if opt.master is not None and model.ptypes[i] != F32 else model.params[i]
        if opt.state_bits == 8:
            m, v = [ref.decode(codes(x[at:pad]), codes(s[at // 128:pad // 128]), k) for x, s, k in ((opt.m, opt.m_scale, "m"), (opt.v, opt.v_scale, "v"))]
        else:
            m, v = (host(x[at:pad]) for x in (opt.m, opt.v))
        before[i] = host(w), m, v, host(model.grads[i]), pad
    opt.run_optimizer(run.get("step_size", lr), grad_scale=run.get("grad_scale"))
    torch.cuda.synchronize()
    assert int(opt.count[0]) == t and int(opt.count[1]) == 0
    for i, n in enumerate(model.sizes):
        w, m, v, g, pad = before[i]
        at = opt.offsets[i]
        d = wd if decay is None or decay[i] else 0.0
        w64, m64, v64, w_tol, m_tol, v_tol = ref.step64(w, m[:n], v[:n], g, scale, t, lr, b1, b2, eps, d)
        word = ref.words(at, pad - at, opt.seed, t)
        m32, v32 = ref.moments32(m, v, np.pad(g, (0, pad - at - n)), scale, b1, b2)
        assert (np.abs(m32[:n] - m64) <= m_tol).all() and (np.abs(v32[:n] - v64) <= v_tol).all()        # the emulation itself
        if opt.state_bits == 32:
            for x, x64, tol in ((opt.m, m64, m_tol), (opt.v, v64, v_tol)):
                x = host(x[at:pad])
                assert (np.abs(x[:n] - x64) <= tol).all(), (i, n)
                assert not x[n:].any()
        else:
            for x, s, x32, k in ((opt.m, opt.m_scale, m32, "m"), (opt.v, opt.v_scale, v32, "v")):
                code, byte = ref.encode(x32, word[0 if k == "m" else 1], k)
                assert (codes(s[at // 128:pad // 128]) == byte).all(), (i, n, k)
                assert (codes(x[at:pad]) == code).all(), (i, n, k)
        new = host(model.params[i])
        if model.ptypes[i] == F32:
            assert (np.abs(new - w64) <= w_tol).all(), (i, n, np.max(np.abs(new - w64) / w_tol))
        elif opt.master is not None:
            mast = host(opt.master[at:at + n])
            assert (np.abs(mast - w64) <= w_tol).all(), (i, n)
            assert (torch.as_tensor(mast).to(model.ptypes[i]).float().numpy() == new).all()
        elif opt.stochastic:
            # rounded from an f32 value within w_tol of w64; for one word the rounding is monotone (the word is added to the magnitude's bits
            # before the cut), so the result lies between what the ends of that interval give
            lo, hi = (ref.bf16_stochastic(x.astype(np.float32), word[0][:n]) for x in (w64 - 1.01 * w_tol, w64 + 1.01 * w_tol))
            assert ((lo <= new) & (new <= hi)).all(), (i, n)
            assert (lo == hi).mean() > 0.95 if n > 1000 else True
        else:
            assert (np.abs(new - w64) <= w_tol + HALF[model.ptypes[i]] * (np.abs(w64) + w_tol) + (2.0 ** -25 if model.ptypes[i] == F16 else 0)).all(), (i, n)
    model.whole()


KINDS = [(F32, F32, {}), (F32, BF16, {}), (BF16, BF16, {}), (BF16, F32, {}), (F16, F16, {}), (BF16, BF16, dict(master=True)), (F16, F16, dict(master=True)),
         (F16, F32, dict(master=True)), (BF16, BF16, dict(stochastic=True)), (BF16, F16, dict(stochastic=True))]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("gap", [0, 1, 3])
def test_steps_against_the_formula(bits, kind, gap):
    ptype, gtype, kw = KINDS[kind]
    model = Model(SIZES, ptype, gtype, gap=gap, seed=kind)
    opt = stochqn().AdamW_free(model.params, state_bits=bits, seed=2 ** 63 + kind, **kw)
    assert opt.offsets[3] == 256 and opt.m.numel() == sum(-(-n // 128) * 128 for n in SIZES)
    for _ in range(3):
        model.new_grads()
        opt.update_gradient(model.grads)
        check_step(model, opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_decay_flags_and_other_numbers(bits):
    sizes = [300, 5, 2100, 64, 4096]
    model = Model(sizes, [F32, BF16, F16, F32, BF16], [BF16, BF16, F32, F32, F16], seed=3)
    decay = [True, False, True, False, True]
    opt = stochqn().AdamW_free(model.params, beta1=0.0, beta2=0.5, eps=1e-6, weight_decay=0.3, state_bits=bits, master=True, decay=decay, seed=9)
    opt.update_gradient(model.grads)
    for lr in (0.1, 0.0, -0.02):
        model.new_grads()
        check_step(model, opt, lr=lr, decay=decay)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [111, 112, 113, 300])
def test_more_tensors_than_a_launch_takes(bits, count):
    rng = np.random.default_rng(count)
    sizes = [int(n) for n in rng.integers(0, 300, count)]
    sizes[count // 2] = 30000
    model = Model(sizes, BF16, BF16, seed=count)
    opt = stochqn().AdamW_free(model.params, state_bits=bits, stochastic=True)
    opt.update_gradient(model.grads)
    for _ in range(2):
        model.new_grads()
        check_step(model, opt)
    got = opt.gradient.norm()
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in model.grads))
    assert abs(float(got[0]) - want) <= 2.0 ** -23 * want


class Large:
    """A list of tensors of given sizes and types, made on the GPU, for `places`."""

    def __init__(self, sizes, ptypes, gtypes, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.sizes, self.ptypes, self.gtypes = sizes, ptypes, gtypes
        self.pbuf = [torch.full((n + 2,), 77.0, dtype=t, device="cuda") for n, t in zip(sizes, ptypes)]
        self.gbuf = [torch.full((n + 2,), 77.0, dtype=t, device="cuda") for n, t in zip(sizes, gtypes)]
        self.params, self.grads = [b[1:-1] for b in self.pbuf], [b[1:-1] for b in self.gbuf]
        for k, (p, g) in enumerate(zip(self.params, self.grads)):
            p.copy_(torch.randn(p.numel(), device="cuda", generator=gen))
            g.copy_(torch.randn(g.numel(), device="cuda", generator=gen) * 10.0 ** -(k % 5))

    def whole(self):
        for b in self.pbuf + self.gbuf:
            assert b[0] == 77 and b[-1] == 77


def places(n, tile):
    """Elements of the first and the last block of 128 of every tile of a tensor, blocks whole."""
    blocks = -(-n // 128)
    per = tile // 128
    first = np.arange(0, blocks, per)
    pick = np.unique(np.concatenate([first, np.minimum(first + per - 1, blocks - 1)])) if blocks else first
    return (pick[:, None] * 128 + np.arange(128)).reshape(-1)


def check_large_step(model, opt, tile, decay):
    """One step, its results at `places` held to the reference from the state before: every tile of every tensor is looked at, at both its ends."""
    b1, b2, eps, wd, t = opt.beta1, opt.beta2, opt.eps, opt.weight_decay, int(opt.count[0]) + 1
    eight, before = opt.state_bits == 8, []
    at = [torch.as_tensor(places(n, tile)).cuda() for n in model.sizes]

    def state(x, scale, i, k):
        e = at[i] + opt.offsets[i]
        if not eight:
            return x[e].cpu().numpy()
        return ref.decode(codes(x.view(torch.uint8)[e]), codes(scale.view(torch.uint8)[e[::128] // 128]), k)

    def values(x, i):
        got = np.zeros(at[i].numel(), dtype=np.float32)
        real = (at[i] < model.sizes[i]).cpu().numpy()
        got[real] = host(x[at[i][at[i] < model.sizes[i]]])
        return got, real

    for i, n in enumerate(model.sizes):
        master = opt.master is not None and model.ptypes[i] != F32
        w = opt.master[opt.offsets[i]:opt.offsets[i] + n] if master else model.params[i]
        before.append((values(w, i), values(model.grads[i], i)[0], state(opt.m, opt.m_scale, i, "m"), state(opt.v, opt.v_scale, i, "v")))
    opt.run_optimizer(LR)
    torch.cuda.synchronize()
    assert opt.count.tolist() == [t, 0]
    for i, n in enumerate(model.sizes):
        (w, real), g, m, v = before[i]
        if not n:
            continue
        w64, m64, v64, w_tol, m_tol, v_tol = ref.step64(w, m, v, g, 1.0, t, LR, b1, b2, eps, wd if decay[i] else 0.0)
        e = at[i].cpu().numpy().astype(np.uint64) + np.uint64(opt.offsets[i])
        with np.errstate(over="ignore"):
            key = ref.finalise(np.uint64((opt.seed ^ (t * ref.STEP_KEY)) & ref.M64))
            word = ref.finalise(key + (e >> np.uint64(3)) * np.uint64(ref.GOLDEN))
        lane = (e & np.uint64(7)) * np.uint64(ref.LANE)
        low, high = (((h + lane) & np.uint64(0xFFFFFFFF)).astype(np.uint32) for h in (word & np.uint64(0xFFFFFFFF), word >> np.uint64(32)))
        assert (low[:128] == ref.words(int(e[0]), 128, opt.seed, t)[0]).all()
        if eight:
            m32, v32 = ref.moments32(m, v, g, 1.0, b1, b2)
            place = at[i] + opt.offsets[i]
            for x, scale, x32, k, u in ((opt.m, opt.m_scale, m32, "m", low), (opt.v, opt.v_scale, v32, "v", high)):
                code, byte = ref.encode(x32, u, k)
                assert (codes(x.view(torch.uint8)[place]) == code).all() and (codes(scale.view(torch.uint8)[place[::128] // 128]) == byte).all(), (i, k)
        else:
            for x, x64, tol in ((state(opt.m, None, i, "m"), m64, m_tol), (state(opt.v, None, i, "v"), v64, v_tol)):
                assert (np.abs(x - x64) <= tol)[real].all() and not x[~real].any(), i
        new = values(model.params[i], i)[0][real]
        w64, w_tol = w64[real], w_tol[real]
        if model.ptypes[i] == F32:
            assert (np.abs(new - w64) <= w_tol).all(), i
        elif opt.master is not None:
            mast = values(opt.master[opt.offsets[i]:opt.offsets[i] + n], i)[0][real]
            assert (np.abs(mast - w64) <= w_tol).all() and (torch.as_tensor(mast).to(model.ptypes[i]).float().numpy() == new).all(), i
        else:
            lo, hi = (ref.bf16_stochastic(x.astype(np.float32), low[real]) for x in (w64 - 1.01 * w_tol, w64 + 1.01 * w_tol))
            assert ((lo <= new) & (new <= hi)).all(), i
    model.whole()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kw", [dict(master=True), dict(stochastic=True)], ids=["master", "stochastic"])
@pytest.mark.parametrize("tile", [2048, "large"])
def test_large_lists_of_several_tensors(bits, kw, tile):
    """Lists on both sides of the threshold of the large tiles (64 and 32 of them for each compute unit), with more tiles than workgroups, so that a
    workgroup goes on from one tensor to another of other types, flags and places."""
    units = torch.cuda.get_device_properties(0).multi_processor_count
    large, few, workgroups = (4096, 64, 16 * units) if bits == 32 else (8192, 32, 32 * units)
    tiles = workgroups * 5 // 4 if tile == 2048 else units * few * 9 // 8
    tile = large if tile == "large" else tile
    assert tiles > workgroups and (tiles * tile // large >= few * units) == (tile == large)
    part = tiles * tile
    half = F16 if "master" in kw else BF16
    sizes = [int(part * 0.31) + 1, 33, 0, int(part * 0.27) + 129, 2047, int(part * 0.24) - 1, 127, int(part * 0.18) + 3]
    ptypes, gtypes = [F32, BF16, F32, BF16, F32, half, BF16, BF16], [F32, F32, BF16, BF16, BF16, F32, F16, F16]
    decay = [True, False, True, False, False, True, True, False]
    assert sum(-(-n // tile) for n in sizes) >= tiles and (sum(-(-n // large) for n in sizes) >= few * units) == (tile == large)
    model = Large(sizes, ptypes, gtypes, seed=bits)
    opt = stochqn().AdamW_free(model.params, state_bits=bits, decay=decay, weight_decay=0.3, seed=5, **kw)
    opt.update_gradient(model.grads)
    for _ in range(2):
        check_large_step(model, opt, tile, decay)


@pytest.mark.parametrize("types", [[F32], [BF16], [F16], [F32, BF16, F16]], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("tiles", [600, 1100, 2500])
def test_norm_of_large_lists(types, tiles):
    """Past each threshold of the norm's tiles (256 compute units: 512 of 8192 elements, 1024 of 16384), and with more tiles than workgroups (2048)."""
    assert torch.cuda.get_device_properties(0).multi_processor_count == 256
    part = tiles * (8192 if tiles < 1024 else 16384)
    sizes = [int(part * 0.4) + 1, 5, int(part * 0.35) - 1, 0, 2049, int(part * 0.25) + 7]
    kinds = [types[k % len(types)] for k in range(len(sizes))]
    model = Large(sizes, kinds, kinds, seed=tiles)
    grads = stochqn().TensorList(model.grads)
    for k in range(2):
        want = math.sqrt(sum(float(g.double().square().sum()) for g in model.grads))
        out = grads.norm(max_norm=1.0)
        # f64 sums in two orders, in each of which an element goes through fewer than 1e4 additions (1e4 * 2^-53 is nothing beside a hundredth of 2^-24),
        # then one rounding to f32 each
        assert abs(float(out[0]) - want) <= 1.01 * 2.0 ** -24 * want and abs(float(out[1]) - 1 / want) <= 1.01 * 2.0 ** -24 / want
        assert torch.equal(grads.norm(max_norm=1.0), out)
        model.grads[0][-1] = 1e4                            # the last element of a tensor counts
        model.grads[-1][-1] = 3e4
    model.whole()


def test_only_empty_tensors():
    model = Model([0, 0], F32, F32)
    opt = stochqn().AdamW_free(model.params)
    opt.update_gradient(model.grads)
    opt.run_optimizer(LR)
    assert opt.count.tolist() == [1, 0]
    assert opt.gradient.norm(max_norm=1.0).tolist() == [0.0, 1.0]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_scale_from_the_device_and_a_rejected_step(bits):
    model = Model([1000, 77], BF16, BF16, seed=5)
    opt = stochqn().AdamW_free(model.params, state_bits=bits, master=True)
    opt.update_gradient(model.grads)
    scale = torch.tensor([0.25], device="cuda")
    check_step(model, opt, scale=0.25, grad_scale=scale)
    rate = torch.tensor(0.03, device="cuda")
    check_step(model, opt, lr=float(rate), scale=0.25, grad_scale=scale, step_size=rate)
    kept = [opt.m, opt.v, opt.master, opt.count] + model.params + ([opt.m_scale, opt.v_scale] if bits == 8 else [])
    was = [t.view(torch.uint8).clone() for t in kept]
    for bad in (math.nan, math.inf, -math.inf):
        scale.fill_(bad)
        opt.run_optimizer(LR, grad_scale=scale)
        assert all((t.view(torch.uint8) == w).all() for t, w in zip(kept, was)), bad
    scale.fill_(1.0)
    for bad in (math.nan, math.inf):
        rate.fill_(bad)
        opt.run_optimizer(rate, grad_scale=scale)
        assert all((t.view(torch.uint8) == w).all() for t, w in zip(kept, was)), bad
    check_step(model, opt, grad_scale=scale)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_whose_numbers_are_past_f32_is_rejected(bits):
    """A step size that is finite, but not as the f32 numbers that the step is taken with: step_size / (1 - beta1^t) and 1 - step_size * weight_decay."""
    model = Model([1000, 77], F32, F32, seed=5)
    for decay, rates in ((0.0, (1e39, -1e39, 1e300, 3.5e37, -3.5e37, torch.tensor(3.5e37, device="cuda"))), (1e30, (1e9, -1e9, torch.tensor(1e9, device="cuda")))):
        opt = stochqn().AdamW_free(model.params, state_bits=bits, weight_decay=decay)
        opt.update_gradient(model.grads)
        kept = [opt.m, opt.v, opt.count] + model.params + ([opt.m_scale, opt.v_scale] if bits == 8 else [])
        was = [t.view(torch.uint8).clone() for t in kept]
        for rate in rates:
            opt.run_optimizer(rate)
            assert all((t.view(torch.uint8) == w).all() for t, w in zip(kept, was)), rate
        opt.run_optimizer(3.3e37 if not decay else 3.3e8)   # (divided by 0.1, times 1e30: 3.3e38, within f32)
        assert opt.count.tolist() == [1, 0]
        for p in model.params:
            p.zero_()


def test_eight_bit_blocks_with_nothing_tiny_huge_and_not_finite():
    n = 128 * 12 + 40
    model = Model([n], F32, F32, seed=1)
    g = torch.randn(n, generator=torch.Generator().manual_seed(1)) * 1e-3
    g[:128] = 0                                             # nothing
    g[128:256] = 0
    g[200] = 3e-5                                           # one element
    g[256:384] *= 1e-30                                     # squares below f32's least
    g[384:512] *= 1e-18                                     # ... and in its subnormals
    g[512:640] *= 1e20                                      # squares near its greatest
    g[640:768] *= 10.0 ** -torch.linspace(0, 12, 128)       # over the whole range of the codes, and past it
    g[768:896] = 2.0 ** -10                                 # at the edge of a binade
    model.grads[0].copy_(g)
    opt = stochqn().AdamW_free(model.params, state_bits=8)
    opt.update_gradient(model.grads)
    for _ in range(3):
        check_step(model, opt)
    m, v = opt.moments(0)
    assert not m[:128].any() and not v[:128].any() and torch.isfinite(v).all()
    moved = model.grads[0][512:].abs() > 1e-15
    assert (v[512:][moved] > 0).all()                       # a second moment above zero is held above zero
    # what is not finite reads as NaN, its block alone
    model.grads[0][900] = math.nan
    model.grads[0][1100] = math.inf
    model.grads[0][1300] = 1e25                             # its square is past f32
    opt.run_optimizer(LR)
    m, v = opt.moments(0)
    for block in range(n // 128 + 1):
        part = slice(block * 128, min(n, block * 128 + 128))
        # (block 10 holds 1300: v is past f32 there, m is not)
        assert v[part].isnan().all().item() == (block in (7, 8, 10)) and m[part].isnan().all().item() == (block in (7, 8)), block
        assert v[part].isnan().any().item() == (block in (7, 8, 10)) and m[part].isnan().any().item() == (block in (7, 8)), block
    assert int(model.params[0].isnan().sum()) == 2          # 900 and 1100 (inf / inf); 1300's update is 0
    opt.run_optimizer(LR)
    assert model.params[0][7 * 128:9 * 128].isnan().all()


def test_eight_bit_codes_of_subnormal_moments():
    """Blocks whose moments lie among the subnormals of 32 bits, where the scale's exponent has reached its least: the codes are still the ones of
    the emulation, for each moment at each size."""
    n = 128 * 40
    model = Model([n], F32, F32, seed=2)
    base = np.random.default_rng(7).standard_normal(n).reshape(40, 128)
    for scale in (10.0 ** -np.linspace(14, 23, 40), 10.0 ** -np.linspace(33, 44, 40)):
        opt = stochqn().AdamW_free(model.params, state_bits=8, seed=11)
        opt.update_gradient(model.grads)
        for _ in range(3):
            model.grads[0].copy_(torch.as_tensor((base * scale[:, None]).astype(np.float32).reshape(-1)))
            check_step(model, opt)
            base = np.roll(base, 1, axis=1)


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_gradients_beside_a_tiny_eps(bits):
    """Second moments among the subnormals of 32 bits, eps below their roots: with beta1 = 0, beta2 = 0.5 the first step is lr * g / (|g| + eps).

    v = g^2 / 2 carries three roundings of at most half of 2^-149 each there (square, product, sum), or 6 u relative: its root half of that
    relative, to first order, 0.6 of it up to a tenth; the other roundings of the update are 10 u (2 root, 1 q, 1 sum, 1 eps, 3 quotient, 1 r,
    1 last sum)."""
    g = np.array([s * m * 10.0 ** -e for e in range(13, 22) for m in (1.0, 1.7, 3.3, 7.1) for s in (1, -1)], dtype=np.float32)
    w = torch.zeros(g.size, device="cuda")
    opt = stochqn().AdamW_free([w], beta1=0.0, beta2=0.5, eps=1e-30, weight_decay=0.0, state_bits=bits)
    opt.update_gradient([torch.as_tensor(g).cuda()])
    opt.run_optimizer(1.0)
    g = g.astype(np.float64)
    v = g * g / 2
    off = np.maximum(6 * 2.0 ** -24, 3 * 2.0 ** -150 / v)
    sure = off < 0.1
    assert sure.sum() > 50 and (v[sure] < 2.0 ** -126).sum() >= 10
    want = -g / (np.abs(g) + 1e-30)
    assert (np.abs(host(w) - want)[sure] <= ((0.6 * off + 10 * 2.0 ** -24) * np.abs(want))[sure]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_the_largest_eps(bits):
    """eps = 2^126, whose reciprocal is the least normal number: the update against the formula; a larger one is refused (its reciprocal is among the
    subnormals, which the hardware's takes for zero)."""
    model = Model([300], F32, F32, grad_size=1e18)
    model.params[0].zero_()
    opt = stochqn().AdamW_free(model.params, eps=2.0 ** 126, weight_decay=0.0, state_bits=bits)
    opt.update_gradient(model.grads)
    check_step(model, opt, lr=1e30)
    assert model.params[0].abs().max() > 1e6
    with pytest.raises(AssertionError):
        stochqn().AdamW_free(model.params, eps=2.0 ** 126 * (1 + 2.0 ** -23))


def test_autograd_knows_that_the_weights_were_written():
    w = torch.randn(100, device="cuda", requires_grad=True)
    x = torch.ones(100, device="cuda")
    opt = stochqn().AdamW_free([w])
    loss = (w * w * x).sum()
    loss.backward(retain_graph=True)
    opt.update_gradient([w.grad])
    opt.run_optimizer(LR)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()                                     # the saved weights are not the ones that the loss was computed from


def test_stochastic_rounding_keeps_the_mean_and_moves_what_nearest_leaves():
    """v from a constant gradient: after k steps E v = (1 - b2^k) g^2.  One step moves v by at most a hundredth of a step of e5m2 at the end, so that
    rounding to nearest would stop; the mean over 2^16 elements has to be within five standard errors, measured from the elements."""
    n, k = 1 << 16, 400
    model = Model([n], F32, F32, gap=0)
    model.grads[0].fill_(0.7)
    opt = stochqn().AdamW_free(model.params, state_bits=8, seed=4)
    opt.update_gradient(model.grads)
    for _ in range(k):
        opt.run_optimizer(0.0)
    m, v = (x.double() for x in opt.moments(0))
    g = np.float64(np.float32(0.7))
    for x, want in ((m, (1 - 0.9 ** k) * g), (v, (1 - 0.999 ** k) * g * g)):
        off = float(x.mean()) - want
        # the words' own grain: a value is rounded up too seldom by at most 2^-20 of a step, and a step is at most a quarter of it
        assert abs(off) <= 5 * float(x.std()) / math.sqrt(n) + k * 2.0 ** -22 * want, (off, float(x.std()))
    # bf16 weights without others beside them: a step far below half a bf16 step moves their mean
    w = torch.ones(n, dtype=BF16, device="cuda")
    opt = stochqn().AdamW_free([w], weight_decay=0.0, stochastic=True, beta1=0.0, beta2=0.0, eps=1e-30)
    opt.update_gradient([torch.full((n,), 1.0, dtype=BF16, device="cuda")])
    for _ in range(10):
        opt.run_optimizer(1e-4)                             # half a step of bf16 below 1 is 2^-9
    off = float(w.double().mean()) - (1 - 10 * 1e-4)
    assert abs(off) <= 5 * float(w.double().std()) / math.sqrt(n) + 10 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [2048], [2049], SIZES, [3_000_001, 17, 999_999]])
@pytest.mark.parametrize("gap", [0, 1])
def test_norm(dtype, sizes, gap):
    model = Model(sizes, dtype, dtype, gap=gap, seed=len(sizes))
    grads = stochqn().TensorList(model.grads)
    x = np.concatenate([host(g) for g in model.grads]).astype(np.float64)
    for grad_scale, max_norm in ((1.0, None), (0.5, 1e-3), (1.0, 1e6), (-2.0, 1e-2)):
        norm = abs(grad_scale) * math.sqrt((x * x).sum())
        coef = grad_scale * (1.0 if max_norm is None or norm <= max_norm else max_norm / norm)
        out = grads.norm(max_norm=max_norm, grad_scale=grad_scale)
        # the sum in f64 loses at most 2^-53 per addition of a lane's chain and the tree; then one rounding to f32 each
        assert abs(float(out[0]) - norm) <= 1.001 * 2.0 ** -24 * norm, (out, norm)
        assert abs(float(out[1]) - coef) <= 1.001 * 2.0 ** -24 * abs(coef)
        again = grads.norm(max_norm=max_norm, grad_scale=grad_scale, out=torch.empty(2, device="cuda"))
        assert (again == out).all()                         # the same bits: no order that changes
    model.whole()


def test_norm_of_what_is_not_finite_zero_and_huge():
    sq = stochqn()
    for n in (5, 100_000):
        g = torch.zeros(n, device="cuda")
        grads = sq.TensorList([g])
        assert grads.norm(max_norm=1.0, grad_scale=0.5).tolist() == [0.0, 0.5]
        g.fill_(1e30)                                       # squares past f32
        out = grads.norm(max_norm=1.0)
        want = float(np.float32(1e30)) * math.sqrt(n)
        assert abs(float(out[0]) - want) <= 2.0 ** -23 * want and abs(float(out[1]) * want - 1) <= 2.0 ** -23
        for bad in (math.inf, -math.inf, math.nan):
            g[n // 2] = bad
            out = grads.norm(max_norm=1.0)
            assert not math.isfinite(float(out[0])) and math.isnan(float(out[1]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 100_000])
def test_norm_at_the_end_of_the_range(dtype, n):
    """The norm that the caller sees is f32: past its range it is infinite, and the coefficient says so too, though the sum in f64 is finite."""
    g = torch.zeros(n, dtype=dtype, device="cuda")
    grads = stochqn().TensorList([g])
    g[n // 2] = 3e38
    x = float(g[n // 2])
    for max_norm in (None, 1.0):
        out = grads.norm(max_norm=max_norm).tolist()
        assert out[0] == np.float32(x) and out[1] == (1.0 if max_norm is None else np.float32(1.0 / x))
    g[0] = 3e38                                             # the norm is 4.2e38
    for max_norm in (None, 1.0, 1e300):
        out = grads.norm(max_norm=max_norm).tolist()
        assert out[0] == math.inf and math.isnan(out[1])
    for scale, ok in ((0.5, True), (-0.5, True), (2.0, False), (1e-300, True)):
        out = grads.norm(max_norm=1e-3, grad_scale=scale).tolist()
        want = abs(scale) * math.sqrt(2.0) * x
        assert math.isfinite(out[0]) == math.isfinite(out[1]) == ok, scale
        # one rounding of each to f32, or half its least subnormal, beside the f64 ones
        coef = scale * min(1.0, 1e-3 / want)
        assert not ok or (abs(out[0] - want) <= 1.001 * 2.0 ** -24 * want + 2.0 ** -150 and abs(out[1] - coef) <= 1.001 * 2.0 ** -24 * abs(coef) + 2.0 ** -150)


def test_a_clipped_step_with_a_loss_scale_and_a_schedule():
    """norm -> step, the coefficient never on the host: as a training loop would, four steps, one of them with an overflowed gradient."""
    model = Model([4000, 129, 1000], F16, F16, seed=8, grad_size=30.0)
    opt = stochqn().AdamW_free(model.params, state_bits=8, master=True)
    grads = stochqn().TensorList(model.grads)
    opt.update_gradient(grads)
    for k in range(4):
        model.new_grads()
        if k == 2:
            model.grads[0][17] = math.inf
        clip = grads.norm(max_norm=1.0, grad_scale=1 / 1024)
        if k == 2:
            was = opt.master.clone()
            opt.run_optimizer(LR, grad_scale=clip[1:])
            assert (opt.master == was).all() and int(opt.count[0]) == 2
        else:
            check_step(model, opt, scale=float(clip[1]), grad_scale=clip[1:])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_into_a_graph(bits):
    """norm and step replayed from a graph, with eager work between the replays, against eager calls from the same state."""
    sq = stochqn()
    a, b = Model([70_000, 33], BF16, BF16, seed=2), Model([70_000, 33], BF16, BF16, seed=2)
    opts, rates, lists = [], [], []
    for model in (a, b):
        opt = sq.AdamW_free(model.params, state_bits=bits, stochastic=True, seed=1)
        lists.append(sq.TensorList(model.grads))
        opt.update_gradient(lists[-1])
        opts.append(opt)
        rates.append(torch.tensor([LR], device="cuda"))

    def once(i):
        clip = lists[i].norm(max_norm=0.1)
        opts[i].run_optimizer(rates[i], grad_scale=clip[1:])
        return clip

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        once(0)
    torch.cuda.current_stream().wait_stream(stream)
    once(1)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        clip = once(0)
    with torch.cuda.graph(second):
        clip2 = once(0)
    for k in range(6):
        for model in (a, b):
            model.new_grads()
        for r in rates:
            r.mul_(0.9)
        if k == 4:
            for model in (a, b):
                model.grads[0][0] = math.nan                # a rejected step inside the graph
        (graph if k % 2 == 0 else second).replay()
        torch.cuda.synchronize()
        want = once(1)
        assert torch.equal((clip if k % 2 == 0 else clip2).nan_to_num(-1), want.nan_to_num(-1))
        for name in ("m", "v", "count"):
            assert (getattr(opts[0], name).view(torch.uint8) == getattr(opts[1], name).view(torch.uint8)).all(), (k, name)
        assert all((p == q).all() for p, q in zip(a.params, b.params))
        if k == 2:                                          # an eager step of the captured optimizer between two replays
            once(0)
            once(1)
    assert int(opts[0].count[0]) == 1 + 6 - 1 + 1


def test_on_another_stream_and_from_two_threads():
    sq = stochqn()
    models = [Model([50_000 + k, 9], F32, F32, seed=k) for k in range(2)]
    twins = [Model([50_000 + k, 9], F32, F32, seed=k) for k in range(2)]
    opts = [[sq.AdamW_free(m.params, state_bits=8, seed=k) for k, m in enumerate(ms)] for ms in (models, twins)]
    for ms, os_ in zip((models, twins), opts):
        for m, o in zip(ms, os_):
            o.update_gradient(m.grads)
    torch.cuda.synchronize()

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                clip = opts[0][k].gradient.norm(max_norm=0.5)
                opts[0][k].run_optimizer(LR, grad_scale=clip[1:])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(2):
        for _ in range(50):
            clip = opts[1][k].gradient.norm(max_norm=0.5)
            opts[1][k].run_optimizer(LR, grad_scale=clip[1:])
        assert all((p == q).all() for p, q in zip(models[k].params, twins[k].params))


def test_the_state_outlives_the_work_of_every_stream_that_used_it():
    """An object made on one stream, used on another and dropped at once: its memory must not come back while the step is still running.  The second
    stream is kept busy in front of the step; what is allocated and filled after the drop is then looked at."""
    sq = stochqn()
    n = 1 << 20
    w, g = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    opt = sq.AdamW_free([w])
    opt.update_gradient([g])
    size = opt.m.numel()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(200):
            big = big @ big
            big = big / big.abs().max()
        opt.run_optimizer(LR)
    del opt
    fresh = [torch.full((size,), 7.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert all((f == 7).all() for f in fresh)
    want = -LR * 1.0 / (1.0 + 1e-8)
    assert (w.double() - want).abs().max() <= 13 * 2.0 ** -24 * LR


def test_the_state_outlives_a_stream_that_was_first_used_in_a_capture():
    """As above, the second stream's first use a capture, whose work is not run: the eager step behind it is the one that must not outlive the memory."""
    sq = stochqn()
    n = 1 << 20
    w, g = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    opt = sq.AdamW_free([w])
    opt.update_gradient([g])
    size = opt.m.numel()
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.run_optimizer(LR)
    del graph                                               # (never replayed)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(200):
            big = big @ big
            big = big / big.abs().max()
        opt.run_optimizer(LR)
    del opt
    fresh = [torch.full((size,), 7.0, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert all((f == 7).all() for f in fresh)
    want = -LR * 1.0 / (1.0 + 1e-8)
    assert (w.double() - want).abs().max() <= 13 * 2.0 ** -24 * LR


def test_copies_are_refused():
    import copy
    import pickle
    sq = stochqn()
    opt = sq.AdamW_free([torch.zeros(4, device="cuda")])
    for thing in (opt, opt.params):
        for how in (copy.copy, copy.deepcopy, pickle.dumps):
            with pytest.raises(TypeError):
                how(thing)


def test_rebinding_gradients_and_state_dicts():
    sq = stochqn()
    model = Model([3000, 40], F32, F32, seed=6)
    opt = sq.AdamW_free(model.params, state_bits=8)
    for _ in range(2):                                      # other tensors every step, as after set_to_none
        model.gbuf, model.grads = model.place(model.gtypes)
        model.new_grads()
        opt.update_gradient(model.grads)
        check_step(model, opt)
    twin = [p.clone() for p in model.params]
    other = sq.AdamW_free(twin, state_bits=8)
    other.load_state_dict(opt.state_dict())
    other.update_gradient(model.grads)
    check_step(model, opt)
    other.run_optimizer(LR)
    assert all((p == q).all() for p, q in zip(twin, model.params))
    with pytest.raises(ValueError):
        sq.AdamW_free(twin, state_bits=8, seed=1).load_state_dict(opt.state_dict())
    # a list of the caller's is never rebound behind its back, and rebinding the parameters' list does not move the optimizer
    mine = sq.TensorList(model.grads)
    opt.update_gradient(mine)
    opt.update_gradient([g.clone() for g in model.grads])
    assert mine.tensors[0] is model.grads[0]
    opt.params.rebind([p.clone() for p in model.params])
    opt.update_gradient(mine)
    check_step(model, opt)


def test_a_tensor_of_more_than_2_31_elements():
    """Offsets past 32 bits: weights, gradients and codes at the end of a tensor of 2^31 + 12 345 elements."""
    n = 2 ** 31 + 12_345
    w = torch.zeros(n, dtype=BF16, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    at = [0, 2 ** 31 - 2048, n - 5000]
    rng = np.random.default_rng(0)
    for a in at:
        w[a:a + 5000] = torch.as_tensor(rng.standard_normal(5000).astype(np.float32)).to(BF16).cuda()
        g[a:a + 5000] = torch.as_tensor(rng.standard_normal(5000).astype(np.float32)).to(BF16).cuda()
    sq = stochqn()
    opt = sq.AdamW_free([w], state_bits=8, stochastic=True, seed=3)
    opt.update_gradient([g])
    was = [host(w[a // 128 * 128:min(n, a + 5000)]) for a in at]
    want = math.sqrt(sum(float((g[a:a + 5000].double() ** 2).sum()) for a in at))
    assert abs(float(opt.gradient.norm()[0]) - want) <= 2.0 ** -23 * want
    opt.run_optimizer(LR)
    for a, w0 in zip(at, was):
        first, upto = a // 128 * 128, min(n, a + 5000)
        k = -(-upto // 128) * 128 - first
        gs = np.pad(host(g[first:upto]), (0, k - (upto - first)))
        word = ref.words(first, k, 3, 1)
        m32, v32 = ref.moments32(np.zeros(k), np.zeros(k), gs, 1.0, 0.9, 0.999)
        for x, s, x32, kind in ((opt.m, opt.m_scale, m32, "m"), (opt.v, opt.v_scale, v32, "v")):
            code, byte = ref.encode(x32, word[0 if kind == "m" else 1], kind)
            full = (upto - first) // 128 * 128 if upto < n else k        # a block cut off by the slice has other neighbours
            assert (codes(x[first:first + full]) == code[:full]).all() and (codes(s[first // 128:(first + full) // 128]) == byte[:full // 128]).all()
        c = upto - first
        w64, _, _, tol, _, _ = ref.step64(w0, np.zeros(c), np.zeros(c), gs[:c], 1.0, 1, LR, 0.9, 0.999, 1e-8, 0.01)
        lo, hi = (ref.bf16_stochastic(x.astype(np.float32), word[0][:c]) for x in (w64 - 1.01 * tol, w64 + 1.01 * tol))
        new = host(w[first:upto])
        assert ((lo <= new) & (new <= hi)).all()
    assert not w[5000:2 ** 31 - 3000].any()


def test_the_first_steps_with_adamw_the_rest_with_sqn():
    """A run of them together: a noisy quadratic over a flat vector that is also seen as tensors -- clipped AdamW steps first, SQN from where
    they end.  Held to the same loop in 64 bits for AdamW; SQN then has to run on the vector that was left."""
    sq = stochqn()
    rng = np.random.default_rng(0)
    sizes, n = [640, 256, 104], 1000
    d = torch.as_tensor(0.5 + rng.random(n)).cuda()
    x = torch.as_tensor(rng.standard_normal(n)).cuda()                      # the quasi-Newton vector, 64 bits
    flat = x.float().clone()
    parts = list(torch.split(flat, sizes))
    grad = torch.zeros(n, device="cuda")
    grads = sq.TensorList(torch.split(grad, sizes))
    opt = sq.AdamW_free(parts, weight_decay=0.0)
    opt.update_gradient(grads)
    w, m, v = (a.astype(np.float64) for a in (host(flat), np.zeros(n), np.zeros(n)))
    dd = d.cpu().numpy()
    for t in range(1, 41):
        grad.copy_(flat * d.float())
        clip = grads.norm(max_norm=1.0)
        opt.run_optimizer(0.02, grad_scale=clip[1:])
        g = w * dd
        scale = min(1.0, 1.0 / np.sqrt((g * g).sum()))
        w, m, v, *_ = ref.step64(w, m, v, g, scale, t, 0.02, 0.9, 0.999, 1e-8, 0.0)
    # 40 contracting steps of 0.02 each: errors of 2^-24 relative per step, divided where |m| / sqrt(v) is ill-conditioned by no more than 1e3
    assert np.abs(host(flat) - w).max() <= 40 * 1e3 * 2.0 ** -24 * 0.02 + 40 * 3 * 2.0 ** -24 * np.abs(w).max()
    x.copy_(flat)
    loss = [float((d * x * x).sum())]
    qn = sq.SQN_free(mem_size=5, bfgs_upd_freq=3, space="device")
    r = qn.run_optimizer(x, 0.1)
    for _ in range(60):
        on = r["requested_on"]
        if r["task"] == "calc_hess_vec":
            qn.update_hess_vec(d * on[1])
        else:
            qn.update_gradient(d * on)
        r = qn.run_optimizer(x, 0.1)
    assert torch.isfinite(x).all() and float((d * x * x).sum()) < loss[0]


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_on_a_problem_then_sqn(bits):
    """A noisy quadratic: clipped steps whose gradients follow from the weights, each held to the reference, then SQN on the vector that they leave."""
    sq = stochqn()
    rng = np.random.default_rng(1)
    sizes, n = [640, 256, 104], 1000
    d = torch.as_tensor(0.5 + rng.random(n)).float().cuda()
    model = Model(sizes, F32, F32, gap=0, seed=4)
    cuts = list(zip(torch.split(d, sizes), model.params, model.grads))
    opt = sq.AdamW_free(model.params, state_bits=bits, seed=8)
    grads = sq.TensorList(model.grads)
    opt.update_gradient(grads)
    for _ in range(60):
        for part, p, g in cuts:
            g.copy_(part * p + 0.1 * torch.as_tensor(rng.standard_normal(p.numel())).float().cuda())
        clip = grads.norm(max_norm=1.0)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in model.grads))
        assert abs(float(clip[1]) - min(1.0, 1.0 / want)) <= 1.01 * 2.0 ** -24
        check_step(model, opt, scale=float(clip[1]), grad_scale=clip[1:])
    x = torch.cat(model.params).double()
    was = x.clone()
    qn = sq.SQN_free(mem_size=5, bfgs_upd_freq=3, space="device")
    r = qn.run_optimizer(x, 0.1)
    for _ in range(60):
        on = r["requested_on"]
        if r["task"] == "calc_hess_vec":
            qn.update_hess_vec(d.double() * on[1])
        else:
            qn.update_gradient(d.double() * on)
        r = qn.run_optimizer(x, 0.1)
    assert torch.isfinite(x).all() and not x.eq(was).any()


def test_memory_that_a_step_or_a_norm_both_reads_and_writes_is_refused():
    sq = stochqn()
    one, p = torch.ones(1, device="cuda"), torch.ones(300, device="cuda")
    g = torch.ones(300, device="cuda")
    opt = sq.AdamW_free([p, one], state_bits=8, master=True)
    grads = sq.TensorList([g, torch.ones(1, device="cuda")])
    opt.update_gradient(grads)
    for scalar in (one, p[7:8], opt.master[3:4], opt.m[:4].view(torch.float32), opt.count.view(torch.float32)[1:2]):
        with pytest.raises(RuntimeError):
            opt.run_optimizer(LR, grad_scale=scalar)
        with pytest.raises(RuntimeError):
            opt.run_optimizer(scalar)
    with pytest.raises(RuntimeError):
        grads.norm(out=g[:2])
    assert opt.count.tolist() == [0, 0] and p.eq(1).all() and one.item() == 1 and g.eq(1).all()
    opt.run_optimizer(g[:1], grad_scale=g[1:2])             # the step only reads gradients
    assert opt.count.tolist() == [1, 0]


def test_tensors_that_an_address_does_not_tell_are_refused():
    sq = stochqn()
    opt = sq.AdamW_free([torch.ones(300, device="cuda")])
    i = torch.tensor([[3]], device="cuda")
    for bad in (torch._neg_view(torch.ones(300, device="cuda")), torch.sparse_coo_tensor(i, torch.ones(1, device="cuda"), (300,)), None):
        with pytest.raises(ValueError):
            sq.TensorList([bad])
        with pytest.raises(ValueError):
            opt.update_gradient([bad])
    opt.update_gradient([torch.ones(300, device="cuda")])
    for bad in (torch._neg_view(torch.ones(300, device="cuda")), None):
        with pytest.raises(ValueError):
            opt.gradient.rebind([bad])
    with pytest.raises(ValueError):
        opt.run_optimizer(LR, grad_scale=torch._neg_view(torch.ones(1, device="cuda")))
    assert opt.count.tolist() == [0, 0]


def test_an_output_that_an_address_does_not_tell_is_refused():
    """A view that negates would read back the opposite of what was written; a tensor that autograd records would not know that it was."""
    sq = stochqn()
    grads = sq.TensorList([torch.ones(300, device="cuda")])
    for bad in (torch._neg_view(torch.zeros(2, device="cuda")), torch.zeros(2, device="cuda", requires_grad=True), [0.0, 0.0]):
        with pytest.raises(ValueError):
            grads.norm(out=bad)
    out = torch.zeros(2, device="cuda")
    x = torch.ones(2, device="cuda", requires_grad=True)
    y = (x * out).sum()                                     # saves out for x's gradient
    grads.norm(out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_parameter_that_is_given_other_memory():
    """The old memory stays until the optimizer goes, so nothing is written where others may be by now; the next gradient is refused."""
    sq = stochqn()
    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    opt = sq.AdamW_free([p], weight_decay=0.0)
    g = torch.ones(1000, device="cuda")
    opt.update_gradient([g])
    p.data = torch.full((1000,), 7.0, device="cuda")
    others = [torch.zeros(1000, device="cuda") for _ in range(50)]
    opt.run_optimizer(LR)
    torch.cuda.synchronize()
    assert not any(o.any() for o in others) and p.eq(7).all()
    with pytest.raises(ValueError):
        opt.update_gradient([g])
    with pytest.raises(ValueError):
        opt.update_gradient(sq.TensorList([g]))
    again = sq.AdamW_free([p], weight_decay=0.0)
    again.load_state_dict(opt.state_dict())
    again.update_gradient([g])
    again.run_optimizer(LR)
    assert again.count.tolist() == [2, 0] and p.lt(7).all()
    grad = torch.ones(1000, device="cuda")                  # the same of a gradient: the list's memory stays
    held = sq.TensorList([grad])
    grad.data = torch.zeros(1, device="cuda")
    others += [torch.zeros(1000, device="cuda") for _ in range(50)]
    assert held.norm()[0].item() == pytest.approx(math.sqrt(1000), rel=torch.finfo(torch.float32).eps)


def test_the_training_loop_of_the_documentation():
    """The loop as it is printed there, run on three batches: the weights and moments of a loop that takes each batch's own gradients."""
    import os
    import re
    sq = stochqn()
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    code = re.search(r"## Models of many tensors.*?```python\n(.*?)```", text, re.S).group(1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    first = [torch.randn(64, 40, generator=gen, device="cuda").half(), torch.randn(40, generator=gen, device="cuda").half()]
    data = [torch.randn(8, 64, generator=gen, device="cuda").half() for _ in range(3)]
    params = [torch.nn.Parameter(p.clone()) for p in first]
    loss = lambda batch, p=None: ((batch @ (p or params)[0] + (p or params)[1]).float() ** 2).mean()
    names = dict(params=params, data=data, loss=loss, lr=LR)
    exec(code, names)
    mine = [p.clone() for p in first]
    opt = sq.AdamW_free(mine, weight_decay=0.1, state_bits=8, master=True, decay=[p.ndim > 1 for p in mine])
    for batch in data:
        leaves = [p.detach().clone().requires_grad_() for p in mine]
        grads = sq.TensorList(torch.autograd.grad(loss(batch, leaves) * 1024, leaves))
        opt.update_gradient(grads)
        opt.run_optimizer(LR, grad_scale=grads.norm(max_norm=1.0, grad_scale=1 / 1024)[1:])
    assert names["opt"].count.tolist() == [3, 0] and all(p.ne(q).any() for p, q in zip(params, first))
    for a, b in zip(params + [names["opt"].m, names["opt"].v, names["opt"].master], mine + [opt.m, opt.v, opt.master]):
        assert (a.detach().view(torch.uint8) == b.view(torch.uint8)).all()


def test_gradients_are_let_go():
    """Between two steps nothing of the last gradients has to stay: their memory is free for the next backward pass."""
    sq = stochqn()
    n = 1 << 20
    p = torch.nn.Parameter(torch.ones(n, device="cuda"))
    opt = sq.AdamW_free([p])
    held = []
    for how in ("update_gradient", "attribute", "update_gradient"):
        before = torch.cuda.memory_allocated()
        (p * p).sum().backward()
        opt.update_gradient([p.grad])
        opt.run_optimizer(LR)
        p.grad = None
        held.append(torch.cuda.memory_allocated() - before)
        if how == "attribute":
            opt.gradient = None
        else:
            opt.update_gradient(None)
        assert torch.cuda.memory_allocated() == before, how
        assert opt.gradient is None
        with pytest.raises(ValueError):
            opt.run_optimizer(LR)
    assert min(held) >= 4 * n and opt.count.tolist() == [3, 0]
    mine = sq.TensorList([torch.ones(n, device="cuda")])    # a list of the caller's is the caller's to drop
    opt.update_gradient(mine)
    opt.update_gradient(None)
    assert abs(float(mine.norm()[0]) - 1024) <= 2.0 ** -24 * 1024
    opt.update_gradient([torch.ones(n, device="cuda")])
    opt.run_optimizer(LR)
    assert opt.count.tolist() == [4, 0] and mine.tensors[0].eq(1).all()


def test_refusals():
    sq = stochqn()
    p = torch.zeros(300, device="cuda")
    for bad in ([], [torch.zeros(3)], [torch.zeros(3, dtype=torch.float64, device="cuda")], [torch.zeros(4, 6, device="cuda").t()],
                [torch.zeros(1, device="cuda").expand(5)], [p, torch.zeros(3)]):
        with pytest.raises(ValueError):
            sq.TensorList(bad)
    for bad in ([p, p], [p[:200], p[199:]]):                # the same weights twice
        with pytest.raises(ValueError):
            sq.AdamW_free(bad)
    for kw in (dict(beta1=1.0), dict(beta2=-0.1), dict(eps=0.0), dict(eps=1e-39), dict(state_bits=16), dict(master=True, stochastic=True),
               dict(weight_decay=math.nan)):
        with pytest.raises(AssertionError):
            sq.AdamW_free([p], **kw)
    with pytest.raises(AssertionError):
        sq.AdamW_free([p.half()], stochastic=True)
    for bad in ([], [True, False]):
        with pytest.raises(ValueError):
            sq.AdamW_free([p], decay=bad)
    opt = sq.AdamW_free([p])
    with pytest.raises(ValueError):
        opt.run_optimizer(LR)                               # no gradient
    for bad in ([torch.zeros(299, device="cuda")], [torch.zeros(300)], [torch.zeros(300, device="cuda")] * 2, [torch.zeros(600, device="cuda")[::2]]):
        with pytest.raises(ValueError):
            opt.update_gradient(bad)
    with pytest.raises(ValueError):
        opt.update_gradient([None])                         # a parameter that has no gradient yet
    opt.update_gradient([torch.zeros(300, device="cuda")])
    with pytest.raises(ValueError):
        opt.update_gradient([None])
    opt.update_gradient([p])                                # the gradient is the weights themselves
    with pytest.raises(RuntimeError):
        opt.run_optimizer(LR)
    opt.update_gradient([opt.m[:300]])
    with pytest.raises(RuntimeError):
        opt.run_optimizer(LR)
    opt.update_gradient([torch.zeros(300, device="cuda")])
    for bad in (math.nan, math.inf):
        with pytest.raises(ValueError):
            opt.run_optimizer(bad)
    for bad in (torch.ones(1), torch.ones(2, device="cuda"), torch.ones(1, device="cuda", dtype=torch.float64), 1.0):
        with pytest.raises(ValueError):
            opt.run_optimizer(LR, grad_scale=bad)
    for kw in (dict(max_norm=0.0), dict(max_norm=math.nan), dict(grad_scale=math.inf), dict(out=torch.empty(2)), dict(out=torch.empty(3, device="cuda"))):
        with pytest.raises(ValueError):
            opt.gradient.norm(**kw)
    with pytest.raises(ValueError):
        opt.gradient.rebind([torch.zeros(300, device="cuda", dtype=BF16)])
    assert not p.any() and opt.count.tolist() == [0, 0]


def test_refusals_of_the_c_entries(capfd):
    """Host pointers, misaligned ones, ranges past their allocation, arrays that overlap: a message and NULL / -1000, nothing launched."""
    from stochqn_amd.adamw import _Setup, _library
    lib = _library()
    n = 1000
    p = torch.zeros(n, device="cuda")
    st = [torch.zeros(1024, device="cuda") for _ in range(3)]
    count, work = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(512, dtype=torch.int64, device="cuda")
    one = lambda ptr, size=n, type=0: lib.stochqn_hip_tensors_create(1, (C.c_void_p * 1)(ptr), (C.c_size_t * 1)(size), (C.c_int * 1)(type))
    hostmem = np.zeros(n, dtype=np.float32)
    for bad in (dict(ptr=hostmem.ctypes.data), dict(ptr=None), dict(ptr=p.data_ptr() + 2), dict(ptr=p.data_ptr(), size=2 ** 40), dict(ptr=p.data_ptr(), size=2 ** 42),
                dict(ptr=p.data_ptr(), type=3), dict(ptr=p.data_ptr(), type=-1)):
        assert not one(**bad), bad
    assert lib.stochqn_hip_tensors_create(1, None, None, None) is None and lib.stochqn_hip_tensors_create(-1, None, None, None) is None
    params = one(p.data_ptr())
    grads = one(st[2].data_ptr())
    good = dict(beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, state_bits=32, stochastic=0, seed=0, m=st[0].data_ptr(), v=st[1].data_ptr(),
                count=count.data_ptr(), work=work.data_ptr())

    def make(**kw):
        s = _Setup(**dict(good, **kw))
        return lib.stochqn_hip_adamw_create(params, C.byref(s))
    for bad in (dict(beta1=1.0), dict(eps=0.0), dict(eps=math.inf), dict(weight_decay=math.inf), dict(state_bits=4), dict(state_bits=8), dict(m=None),
                dict(m=st[0].data_ptr() + 4), dict(m=hostmem.ctypes.data), dict(v=st[0].data_ptr()), dict(m=p.data_ptr()), dict(count=None), dict(work=None), dict(work=count.data_ptr()),
                dict(count=st[0].data_ptr() + 8), dict(m_scale=st[2].data_ptr()), dict(stochastic=1, master=st[2].data_ptr())):
        assert not make(**bad), bad
    opt = make()
    assert opt
    assert lib.stochqn_hip_adamw_step(opt, None, LR, None, None, None) == -1000
    assert lib.stochqn_hip_adamw_step(None, grads, LR, None, None, None) == -1000
    assert lib.stochqn_hip_adamw_step(opt, grads, math.nan, None, None, None) == -1000
    assert lib.stochqn_hip_adamw_step(opt, grads, LR, None, hostmem.ctypes.data, None) == -1000
    assert lib.stochqn_hip_adamw_step(opt, params, LR, None, None, None) == -1000            # gradients that are the weights
    assert lib.stochqn_hip_tensors_rebind(grads, (C.c_void_p * 1)(hostmem.ctypes.data)) == -1000
    assert lib.stochqn_hip_tensors_norm(grads, 1.0, 0.0, st[2].data_ptr(), st[2].data_ptr(), None) == -1000
    assert lib.stochqn_hip_tensors_norm(grads, 1.0, 1.0, hostmem.ctypes.data, st[2].data_ptr(), None) == -1000
    assert lib.stochqn_hip_adamw_step(opt, grads, LR, None, None, None) == 0
    torch.cuda.synchronize()
    assert count.tolist() == [1, 0]
    err = capfd.readouterr().err
    for word in ("not device memory", "past the end", "not aligned", "overlap", "state_bits", "unknown type"):
        assert word in err, word
    lib.stochqn_hip_adamw_destroy(opt)
    lib.stochqn_hip_tensors_destroy(params)
    lib.stochqn_hip_tensors_destroy(grads)
    lib.stochqn_hip_tensors_destroy(None)


def test_the_norm_over_the_ranks_of_a_reducer():
    """Two host threads, each with half of the gradients, over the loop-back reducer: both get the norm of the whole."""
    sq = stochqn()
    lib = sq.cdll()
    rng = np.random.default_rng(0)
    halves = [torch.as_tensor(rng.standard_normal(k).astype(np.float32)).cuda() for k in (3000, 500_000)]
    want = math.sqrt(sum(float((h.double() ** 2).sum()) for h in halves))
    lists = [sq.TensorList([h]) for h in halves]
    out = [None, None]
    assert lib.stochqn_hip_loopback_init(2) == 0
    torch.cuda.synchronize()
    try:
        def work(rank):
            assert lib.stochqn_hip_loopback_join(rank) == 0
            with torch.cuda.stream(torch.cuda.Stream()):
                r = lists[rank].norm(max_norm=1.0)
                torch.cuda.current_stream().synchronize()
                out[rank] = r.tolist()
        threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        lib.stochqn_hip_loopback_finalize()
    assert out[0] == out[1]
    assert abs(out[0][0] - want) <= 2.0 ** -23 * want and abs(out[0][1] * want - 1) <= 2.0 ** -23


def test_the_norm_over_a_host_side_reducer_is_refused_in_a_capture():
    """The refused call leaves the capture as it was: what else is captured is replayed."""
    sq = stochqn()
    lib = sq.cdll()
    g = torch.full((1000,), 2.0, device="cuda")
    grads, x, out = sq.TensorList([g]), torch.zeros(5, device="cuda"), []
    assert lib.stochqn_hip_loopback_init(2) == 0
    try:
        def work():
            assert lib.stochqn_hip_loopback_join(0) == 0
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                x.add_(1)
                try:
                    grads.norm()
                except RuntimeError as e:
                    out.append(e)
                x.add_(1)
            graph.replay()
            graph.replay()
            torch.cuda.synchronize()
        t = threading.Thread(target=work)
        t.start()
        t.join()
    finally:
        lib.stochqn_hip_loopback_finalize()
    assert len(out) == 1 and x.eq(4).all()
    assert abs(float(grads.norm()[0]) - 2 * math.sqrt(1000)) <= 2.0 ** -23 * 64     # this thread has no reducer
