"""One AdamW step over many tensors: 32-bit states bit for bit against fmlh_adamw_update, 8-bit states
against a restatement of the format in numpy (the same fp32 operations in the same order, so
codes and parameters are equal) and against the formula in 64 bits.
"""
import numpy as np
import pytest

import freeml_amd as fh
from graphs import Captured

F = np.float32
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.99, 1e-8, 0.1
SIZES = [1, 255, 256, 257, 1023, 1024, 1025, 4096, 70001, 0, 3]


def powers(t):
    return F(F(B1) ** t), F(F(B2) ** t)


def mix32(h):
    h = np.asarray(h, np.uint64)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def bits(seed, tensor, n):
    key = mix32((seed & 0xFFFFFFFF) ^ 0x9E3779B9)
    key = mix32(key ^ np.uint64((tensor + (seed >> 32)) & 0xFFFFFFFF))
    return mix32(np.arange(n, dtype=np.uint64) ^ key)


def decode(code, E):
    c = code.astype(np.int64)
    ex, ma = (c >> 3) & 15, c & 7
    v = np.where(ex > 0, np.ldexp(8.0 + ma, ex - 10), np.ldexp(ma.astype(np.float64), -9))
    v = np.where((c & 127) == 127, np.nan, np.where(c > 127, -v, v))
    E = np.repeat(E.astype(np.int64), 256)[:len(c)]
    return np.where(v == 0, v, np.ldexp(v, E - 127)).astype(F)


def encode(x, rnd, square=False):
    """fp32 values and 16 random bits each -> codes and the blocks' E."""
    n = len(x)
    blocks = -(-n // 256)
    a = np.zeros(blocks * 256, F)
    a[:n] = np.where(np.isfinite(x), np.abs(x), 0)
    E = np.maximum((a.reshape(blocks, 256).max(1).view(np.int32) >> 23) - 7, 1)
    unit = ((254 - np.repeat(E, 256)[:n]).astype(np.int32) << 23).view(F)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.abs(x) * unit
        ok = y < 256
        y = np.where(ok, y, F(0))
        e = np.where(y > 0, np.maximum(np.frexp(y)[1] - 1, -6), -6)  # y's exponent, or the smallest codes'
        gap = np.ldexp(F(1), e - 3).astype(F)
        n_low = np.floor(y / gap)
        low = (n_low * gap).astype(F)
        high, rest = low + gap, y - low
        if square:
            gap, rest = gap * (high + low), rest * (y + low)
        up = rnd.astype(F) * F(2.0**-16) * gap < rest
    code = (np.maximum(e + 6, 0) * 8 + n_low + up).astype(np.int64)
    code = np.where(ok, code, 127)
    return (code | np.where(x < 0, 128, 0)).astype(np.uint8), E.astype(np.uint8)


def step(p, g, m, v, t):
    p1, p2 = powers(t)
    lr = F(LR)
    with np.errstate(invalid="ignore", over="ignore"):
        m = F(B1) * m + (F(1) - F(B1)) * g
        v = F(B2) * v + (F(1) - F(B2)) * g * g
        update = lr * (m / (F(1) - p1)) / (np.sqrt(v / (F(1) - p2)) + F(EPS))
        return p + update - lr * F(WD) * p, m, v


def step8(p, g, m, me, v, ve, t, seed, tensor):
    r = decode(v, ve)
    p, m, v = step(p, g, decode(m, me), r * r, t)
    rnd, r = bits(seed, tensor, len(p)), np.sqrt(v)
    m, me = encode(m, rnd & np.uint64(0xFFFF))
    code, ve = encode(r, rnd >> np.uint64(16), True)
    return p, m, me, np.where(r > 0, np.maximum(code, 1), code).astype(np.uint8), ve


class Arena:
    """Tensors at any 4-byte alignment in device buffers, marked between."""

    def __init__(self, arrays, gap):
        self.at, n = [], 0
        for a in arrays:
            self.at.append(n)
            n += a.size + gap
        self.dtype = arrays[0].dtype
        self.mark = self.dtype.type(99)
        host = np.full(n + 8, self.mark, self.dtype)
        for o, a in zip(self.at, arrays):
            host[o:o + a.size] = a
        self.sizes, self.d = [a.size for a in arrays], fh.DeviceArray.from_host(host)

    def ptrs(self):
        return [self.d.at(o) for o in self.at]

    def read(self):
        host = self.d.numpy()
        got = [host[o:o + n].copy() for o, n in zip(self.at, self.sizes)]
        for o, n in zip(self.at, self.sizes):
            host[o:o + n] = self.mark
        assert np.all(host == self.mark)  # nothing between the tensors changed
        return got


def make(seed, sizes=SIZES, zero=False):
    r = np.random.default_rng(seed)
    f = lambda n, s: (s * r.standard_normal(n)).astype(F)  # noqa: E731
    scale = [10.0 ** r.uniform(-6, 1) for _ in sizes]
    p, g = [f(n, 0.1) for n in sizes], [f(n, s) for n, s in zip(sizes, scale)]
    m = [f(n, 0 if zero else 0.3 * s) for n, s in zip(sizes, scale)]
    v = [f(n, 0 if zero else s) ** 2 for n, s in zip(sizes, scale)]
    return p, g, m, v


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 1, 4])
@pytest.mark.parametrize("count", [1, 11, 150])
def test_32_bit_states_equal_the_single_update(gap, count):
    sizes = (SIZES * 14)[:count]
    p, g, m, v = make(count, sizes)
    arenas = [Arena(x, gap) for x in (p, g, m, v)]
    ptrs = [a.ptrs() for a in arenas]
    table = fh.adamw_tensors([(*x, n) for *x, n in zip(*ptrs, sizes)])
    single = [[fh.DeviceArray.from_host(x) for x in group] for group in zip(p, g, m, v)]
    for t in (1, 2, 3):
        fh.adamw_update_multi(table, 32, LR, B1, B2, *powers(t), EPS, WD)
        for (dp, dg, dm, dv), n in zip(single, sizes):
            if n:
                fh.adamw_update(dp.ptr, dg.ptr, dm.ptr, dv.ptr, n, LR, B1, B2, *powers(t), EPS, WD)
    got = [a.read() for a in arenas]
    for i, n in enumerate(sizes):
        if n:
            for k in range(4):
                np.testing.assert_array_equal(got[k][i], single[i][k].numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 1, 4])
@pytest.mark.parametrize("seed", [0, 5, 2**40 + 17])
def test_8_bit_states(gap, seed):
    p, g, m, v = make(3)
    blocks = [-(-n // 256) for n in SIZES]
    zero = lambda ns: [np.zeros(n, np.uint8) for n in ns]  # noqa: E731
    mc, vc, me, ve = zero(SIZES), zero(SIZES), zero(blocks), zero(blocks)
    arenas = [Arena(x, gap) for x in (p, g, mc, vc, me, ve)]
    P, G, M, V, ME, VE = (a.ptrs() for a in arenas)
    table = fh.adamw_tensors([(P[i], G[i], M[i], V[i], n, ME[i], VE[i]) for i, n in enumerate(SIZES)])
    for t in range(1, 5):
        fh.adamw_update_multi(table, 8, LR, B1, B2, *powers(t), EPS, WD, seed + t)
        for i, n in enumerate(SIZES):
            if n:
                p[i], mc[i], me[i], vc[i], ve[i] = step8(p[i], g[i], mc[i], me[i], vc[i], ve[i], t, seed + t, i)
        got = [a.read() for a in arenas]
        for i, n in enumerate(SIZES):
            for k, ref in enumerate((p, g, mc, vc, me, ve)):
                np.testing.assert_array_equal(got[k][i], ref[i], err_msg=f"step {t}, tensor {i} of {n}, buffer {k}")


@pytest.mark.gpu
def test_quotients_and_roots_of_every_mantissa():
    """The quick forms of the update's divisions and root against the single update's, for every mantissa of v of an
    even and an odd exponent: with beta 1 and powers 0 the states stay, and p takes lr m / (sqrt(v) + eps)."""
    n = 1 << 24
    v = (np.arange(n, dtype=np.uint32) + (np.uint32(120) << np.uint32(23))).view(F)
    m = np.random.default_rng(0).standard_normal(n).astype(F)
    zero = np.zeros(n, F)
    d = [[fh.DeviceArray.from_host(x) for x in (zero, zero, m, v)] for _ in range(2)]
    fh.adamw_update_multi(fh.adamw_tensors([(*(x.ptr for x in d[0]), n)]), 32, LR, 1.0, 1.0, 0.0, 0.0, 2.0**-48, 0.0)
    fh.adamw_update(*(x.ptr for x in d[1]), n, LR, 1.0, 1.0, 0.0, 0.0, 2.0**-48, 0.0)
    for a, b in zip(*d):
        np.testing.assert_array_equal(a.numpy(), b.numpy())
    # Divisors that are not 1: every mantissa of m and v against an arbitrary 1 - beta^t.
    m2 = np.where(np.arange(n) % 2 == 0, v, -v).astype(F)
    d = [[fh.DeviceArray.from_host(x) for x in (zero, zero, m2, v)] for _ in range(2)]
    for p1, p2 in ((0.9, 0.999), (0.1234, 0.77)):
        fh.adamw_update_multi(fh.adamw_tensors([(*(x.ptr for x in d[0]), n)]), 32, LR, 1.0, 1.0, p1, p2, EPS, 0.0)
        fh.adamw_update(*(x.ptr for x in d[1]), n, LR, 1.0, 1.0, p1, p2, EPS, 0.0)
        np.testing.assert_array_equal(d[0][0].numpy(), d[1][0].numpy())


@pytest.mark.gpu
def test_8_bit_update_against_64_bits():
    """One step from states of zero: m and v are exact before they are rounded, so p is off by the
    formula's own roundings, six of them at most half a step each, relative to the update, and one of p."""
    p, g, _, _ = make(7, [5000], zero=True)
    p, g = p[0], g[0]
    dp, dg = fh.DeviceArray.from_host(p), fh.DeviceArray.from_host(g)
    st = [fh.DeviceArray.from_host(np.zeros(n, np.uint8)) for n in (5000, 5000, 20, 20)]
    fh.adamw_update_multi(fh.adamw_tensors([(dp.ptr, dg.ptr, st[0].ptr, st[1].ptr, 5000, st[2].ptr, st[3].ptr)]), 8, LR, B1, B2, *powers(1), EPS, WD, 1)
    d = np.float64
    p1, p2 = (1 - d(x) for x in powers(1))
    m, v = (1 - d(F(B1))) * g.astype(d), (1 - d(F(B2))) * g.astype(d) ** 2
    up = d(F(LR)) * (m / p1) / (np.sqrt(v / p2) + d(F(EPS)))
    ref = p + up - d(F(LR)) * d(F(WD)) * p
    assert np.all(np.abs(dp.numpy() - ref) <= 8 * 2.0**-24 * (np.abs(up) + np.abs(p) * LR) + 2 * 2.0**-24 * np.abs(ref) + 2.0**-24 * np.abs(p))
    # The stored states: within a code's step of the states (three mantissa bits: 1/8 of the value, or 2^-9 of the unit).
    for x, c, e in ((m, st[0], st[2]), (np.sqrt(v), st[1], st[3])):
        E = e.numpy()
        unit = np.ldexp(1.0, np.repeat(E.astype(int), 256)[:5000] - 127)
        assert np.all(np.abs(decode(c.numpy(), E) - x) <= np.maximum(np.abs(x) / 8, unit * 2.0**-9) * (1 + 2.0**-20))


@pytest.mark.gpu
def test_8_bit_states_follow_on_average():
    """Rounding at random keeps m and v on average: after 400 steps of one gradient sqrt(v) has come from 4 to near
    1, where rounding to nearest would have left it.  A step that moves v by d adds a variance of at most d times
    the codes' gap g = v / 4, forgotten with 1 - beta2 = 0.01: with d = 0.01 |1 - v| a variance of g / 2 at most,
    1/8 of v squared; the mean over 4096 elements is off by 0.35 / 64 = 0.55% (one sigma), bounded here by 9 of them."""
    n = 4096
    codes, E = encode(np.full(n, 4.0, F), np.zeros(n, np.uint64))
    dv, de = fh.DeviceArray.from_host(codes), fh.DeviceArray.from_host(E)
    dm, dme = fh.DeviceArray.from_host(np.zeros(n, np.uint8)), fh.DeviceArray.from_host(np.zeros(16, np.uint8))
    dp, dg = fh.DeviceArray.from_host(np.zeros(n, F)), fh.DeviceArray.from_host(np.ones(n, F))
    table = fh.adamw_tensors([(dp.ptr, dg.ptr, dm.ptr, dv.ptr, n, dme.ptr, de.ptr)])
    for t in range(1, 401):
        fh.adamw_update_multi(table, 8, LR, B1, B2, *powers(t), EPS, 0.0, 1000 + t)
    exact = 1 + 15 * F(B2).astype(float) ** 400
    got = np.mean(decode(dv.numpy(), de.numpy()).astype(float) ** 2)
    assert abs(got / exact - 1) < 0.05, (got, exact)
    assert abs(np.mean(decode(dm.numpy(), dme.numpy())) - 1) < 0.02


@pytest.mark.gpu
def test_8_bit_extremes():
    """Blocks of zeros, of the smallest and largest numbers, with infinities and NaN: codes as restated; a
    positive sqrt(v) never becomes zero."""
    g = np.zeros(256 * 6, F)
    g[256:512] = 1e-38
    g[512:768] = 1e18
    g[768:1024] = np.geomspace(1e-12, 1e3, 256)
    g[1024:1280] = 1.0
    g[1030], g[1040], g[1050] = np.inf, np.nan, -np.inf
    g[1280:] = np.float32(1e-45)
    n = g.size
    dp, dg = fh.DeviceArray.from_host(np.zeros(n, F)), fh.DeviceArray.from_host(g)
    st = [fh.DeviceArray.from_host(np.zeros(k, np.uint8)) for k in (n, n, 6, 6)]
    table = fh.adamw_tensors([(dp.ptr, dg.ptr, st[0].ptr, st[1].ptr, n, st[2].ptr, st[3].ptr)])
    ref = (np.zeros(n, F), np.zeros(n, np.uint8), np.zeros(6, np.uint8), np.zeros(n, np.uint8), np.zeros(6, np.uint8))
    for t in (1, 2):
        fh.adamw_update_multi(table, 8, LR, B1, B2, *powers(t), EPS, WD, t)
        ref = step8(ref[0], g, *ref[1:], t, t, 0)
    ref = dict(zip(("p", "m", "me", "v", "ve"), ref))
    np.testing.assert_array_equal(dp.numpy(), ref["p"])
    for d, name in zip(st, ("m", "v", "me", "ve")):
        got = d.numpy()
        np.testing.assert_array_equal(got & 127 if name == "m" else got, ref[name] & 127 if name == "m" else ref[name], err_msg=name)
    assert np.all(st[1].numpy()[768:1024] > 0)


@pytest.mark.gpu
def test_captured_and_replayed():
    p, g, m, v = make(9)
    arenas = [Arena(x, 0) for x in (p, g, m, v)]
    again = [Arena(x, 0) for x in (p, g, m, v)]
    tables = [fh.adamw_tensors([(*x, n) for *x, n in zip(*(a.ptrs() for a in ar), SIZES)]) for ar in (arenas, again)]
    graph = Captured(lambda: fh.adamw_update_multi(tables[0], 32, LR, B1, B2, *powers(5), EPS, WD))
    for _ in range(4):
        graph.replay()
        fh.adamw_update_multi(tables[1], 32, LR, B1, B2, *powers(5), EPS, WD)
        for a, b in zip(arenas, again):
            for x, y in zip(a.read(), b.read()):
                np.testing.assert_array_equal(x, y)


# ---- refusals (no device needed) -----------------------------------------------------------------

def call(tensors, state_bits=32):
    fh.adamw_update_multi(fh.adamw_tensors(tensors), state_bits, LR, B1, B2, 0.9, 0.99, EPS, WD)


A = 1 << 20


@pytest.mark.parametrize("tensors,state_bits", [
    ([(0, A, 2 * A, 3 * A, 8)], 32), ([(A, 0, 2 * A, 3 * A, 8)], 32), ([(A, 2 * A, 0, 3 * A, 8)], 32), ([(A, 2 * A, 3 * A, 0, 8)], 32),
    ([(A, 2 * A, 3 * A, 4 * A, 8)], 16), ([(A, 2 * A, 3 * A, 4 * A, 8)], 8), ([(A, 2 * A, 3 * A, 4 * A, 8, 5 * A, 0)], 8),
    ([(A, 2 * A, 3 * A, 4 * A, 2**33 + 1)], 32),
    # the same tensor twice, one inside another, states or scales in common, a gradient that is another's parameter
    ([(A, 2 * A, 3 * A, 4 * A, 8)] * 2, 32), ([(A, 2 * A, 3 * A, 4 * A, 8), (A + 28, 5 * A, 6 * A, 7 * A, 8)], 32),
    ([(A, 2 * A, 3 * A, 4 * A, 8), (5 * A, 6 * A, 3 * A, 7 * A, 8)], 32), ([(A, 2 * A, 3 * A, 3 * A, 8)], 32), ([(A, A, 3 * A, 4 * A, 8)], 32),
    ([(A, 2 * A, 3 * A, 4 * A, 8), (5 * A, A, 6 * A, 7 * A, 8)], 32),
    ([(A, 2 * A, 3 * A, 4 * A, 8, 5 * A, 5 * A)], 8)])
def test_refusals(tensors, state_bits):
    with pytest.raises(fh.FreeMLHipError) as e:
        call(tensors, state_bits)
    assert e.value.code == -1


def test_null_list_is_refused():
    with pytest.raises(fh.FreeMLHipError) as e:
        fh.call("fmlh_adamw_update_multi", None, 1, 32, LR, B1, B2, 0.9, 0.99, EPS, WD, 0)
    assert e.value.code == -1
