"""AdamW and its roundings for the tests, in numpy: the formula in 64 bits, the moments in 32 bits operation by operation (what the 8-bit
codes are rounded from), the 8-bit codes and the stochastic words from Python's and numpy's whole numbers.  Shares nothing with the library."""
import numpy as np

GOLDEN, STEP_KEY, LANE = 0x9E3779B97F4A7C15, 0xD1B54A32D192ED03, 0x9E3779B9
M64 = 2 ** 64 - 1


def finalise(z):
    """splitmix64's finaliser (Steele, Lea, Flood 2014) on uint64 arrays."""
    z = np.asarray(z, dtype=np.uint64)
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def words(first, n, seed, t):
    """The two 32-bit words of elements first .. first + n - 1 of the state."""
    with np.errstate(over="ignore"):
        at = np.arange(first, first + n, dtype=np.uint64)
        key = finalise(np.uint64((seed ^ (t * STEP_KEY)) & M64))
        w = finalise(key + (at >> np.uint64(3)) * np.uint64(GOLDEN))
    j = (at & np.uint64(7)).astype(np.uint64) * np.uint64(LANE)
    low, high = w & np.uint64(0xFFFFFFFF), w >> np.uint64(32)
    return [((h + j) & np.uint64(0xFFFFFFFF)).astype(np.uint32) for h in (low, high)]


def moments32(m, v, g, scale, beta1, beta2):
    """m and v as the library forms them: products and sums in f32, each rounded by itself."""
    f = np.float32
    with np.errstate(all="ignore"):
        g = (g.astype(f) * f(scale)).astype(f)
        m = (m.astype(f) * f(beta1)).astype(f) + (g * f(1 - beta1)).astype(f)
        v = (v.astype(f) * f(beta2)).astype(f) + ((g * g).astype(f) * f(1 - beta2)).astype(f)
    return m.astype(f), v.astype(f)


def step64(w, m, v, g, scale, t, lr, beta1, beta2, eps, decay):
    """The definition in 64 bits: (w, m, v) and what their errors in 32 bits may be.

    m: four roundings (the scaled gradient, two coefficients and products count as one each per term, the sum): 4 u (|b1 m| + |a1 g|), u = 2^-24.
    v: g^2 carries the scaled gradient's twice: 6 u (b2 v + a2 g^2), all terms >= 0, so 6 u v relative.
    update r m / (sqrt(v) q + eps): m's error over the denominator; v's 3 u, sqrt u (as 2 u: not required to be exact), q u, the sum u,
    eps's own rounding u, the quotient 2 u, r u, their product in the last sum: 12 u of its size.
    w (1 - lr wd): the coefficient u, the product u, the last sum u: 3 u |w|, and the last sum's u of the update: in the 13 u.
    2^-140 beside it where subnormals of 32 bits lose more than a relative u."""
    w, m, v, g = (np.asarray(x, dtype=np.float64) for x in (w, m, v, g))
    u = 2.0 ** -24
    g = g * float(scale)
    m_tol = 4 * u * (np.abs(beta1 * m) + np.abs((1 - beta1) * g)) + 2.0 ** -140
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    v_tol = 6 * u * v + 2.0 ** -140
    rate = lr / (1 - beta1 ** t)
    d = np.sqrt(v / (1 - beta2 ** t)) + eps
    up = rate * m / d
    w_tol = 3 * u * np.abs(w) + 13 * u * np.abs(up) + abs(rate) * m_tol / d + 2.0 ** -140
    return w * (1 - lr * decay) - up, m, v, w_tol, m_tol, v_tol


FORMATS = {"m": (3, 7, 4, 7), "v": (2, 15, 5, 14)}          # mantissa bits, bias, exponent bits, where the largest of a block is brought


def decode(code, byte, which):
    """Values (f64) of 8-bit codes over their blocks' exponent bytes."""
    mant, bias, ebits, _ = FORMATS[which]
    c = np.asarray(code, dtype=np.int64)
    sign = np.where(c & 128, -1.0, 1.0)
    e, f = (c & 127) >> mant, c & ((1 << mant) - 1)
    x = sign * np.where(e > 0, (1 + f / 2.0 ** mant) * 2.0 ** (e - bias), f / 2.0 ** mant * 2.0 ** (1 - bias))
    nan = (c & 127) == 127 if which == "m" else (c & 127) > 124
    x = np.where(nan, np.nan, x)
    b = np.repeat(np.asarray(byte, dtype=np.int64), 128)
    return np.where(b == 255, np.nan, x * 2.0 ** (b - 127.0))


def encode(x, word, which):
    """(codes, exponent bytes) of f32 values, a multiple of 128 of them, rounded by 32-bit words."""
    mant, bias, ebits, top = FORMATS[which]
    x = np.asarray(x, dtype=np.float32)
    blocks = np.abs(x).reshape(-1, 128)
    with np.errstate(invalid="ignore"):
        bad = ~np.isfinite(blocks).all(1)
        big = np.where(bad, 0, blocks.max(1)).astype(np.float32)
    byte = np.maximum((big.view(np.uint32) >> 23).astype(np.int64) - top, 1)
    byte = np.where(bad, 255, byte)
    y = x.astype(np.float64) * 2.0 ** (127.0 - np.repeat(np.where(bad, 127, byte), 128))
    y = np.where(np.repeat(bad, 128), 0.0, y)
    if which == "v":
        y = np.where(y > 0, np.maximum(y, 2.0 ** -16), y)
    a = np.abs(y)
    _, e = np.frexp(a)
    e = np.maximum(e - 1, 1 - bias)
    q = np.floor(a / 2.0 ** (e - mant) + word / 2.0 ** 32).astype(np.int64)
    code = np.where(q < 1 << mant, q, (((e + bias) << mant) - (1 << mant)) + q)
    return (code | np.where(np.signbit(y), 128, 0)).astype(np.uint8), byte.astype(np.uint8)


def bf16_stochastic(w, word):
    """f32 values to bf16 (as f32) by the low 16 bits of their words; what is not finite stays so."""
    b = np.asarray(w, dtype=np.float32).view(np.uint32)
    with np.errstate(over="ignore"):
        r = ((b + (word & np.uint32(0xFFFF))) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isfinite(w), r, w)
