"""AdamW with 8-bit moments (gt_adamw8_*, AdamWHip(state_bits=8)) against the definition in 64 bits.

A state is a code c of OCP e4m3 times 2^e with one e per 256 elements: the smallest with |value| <= 448 * 2^e over the block. Its code is
floor(|value| / step + b / 65536) steps, b the element's 16 random bits, which the test forms again. In 32 bits |value| carries at
most six half-steps of 2^-24 (three products, a sum, the root, the clip's scale) of the terms it is the sum of: m is b1 m0 + (1 - b1) g, and
where the two cancel it is as far off as they are large. So the floor can come out otherwise only within 6 * 2^-24 * (|b1 m0| +
|(1 - b1) g|) / step of a whole number (without cancellation: below 16 steps, 6 * 16 * 2^-24 < 1e-5), and such an element is held
to the next code. An exponent can differ only where the block's largest moment is within 1e-5 of
448 * 2^e (the gradients are drawn afresh each step and do not cancel a block's largest moment to less than a tenth of its terms:
60 * 2^-24 < 1e-5)."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import mod

U = 2.0 ** -24
BLK = 256
B1, B2, AEPS = 0.9, 0.999, 1e-8
NEAR = 1e-5

E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)])
E4M3[127] = np.nan
E4M3 = np.concatenate([E4M3, -E4M3])


def mix(x, rounds):
    x = np.asarray(x, np.uint64)
    for c in (0x21F0AAAD, 0x735A2D97)[:rounds]:
        x = x ^ (x >> np.uint64(16)) if c == 0x21F0AAAD else x
        x = (x * np.uint64(c)) & np.uint64(0xFFFFFFFF)
        x = x ^ (x >> np.uint64(15))
    return x


def random_words(seed, first_block, size):
    """The 32 bits of every element of a tensor whose first block has that number in its group."""
    key = mix((seed & 0xFFFFFFFF) ^ int(mix((seed >> 32) + 0x9E3779B9 & 0xFFFFFFFF, 2)), 2)
    nb = -(-size // BLK)
    block = mix((np.arange(nb, dtype=np.uint64) + np.uint64(first_block)) ^ key, 2)
    inside = (np.arange(BLK, dtype=np.uint64) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)
    return mix((block[:, None] + inside) & np.uint64(0xFFFFFFFF), 1).reshape(-1)[:size]


def blocks_of(a):
    n = -(-a.size // BLK) * BLK
    return np.concatenate([a, np.zeros(n - a.size)]).reshape(-1, BLK)


def decode(codes, e):
    return (E4M3[blocks_of(codes.astype(np.float64)).astype(int)] * 2.0 ** e.astype(np.float64)[:, None]).reshape(-1)[:codes.size]


def check_state(x, codes, e, bits16, keep, what, size=None):
    """codes and exponents of the values x (64 bits, finite ones only); keep: a value that is there has a code that is. size: the sum of the
    absolute terms of each value, where that is more than the value."""
    top = np.abs(blocks_of(np.where(np.isfinite(x), x, 0))).max(axis=1)
    with np.errstate(divide="ignore"):
        want = np.where(top > 0, np.ceil(np.log2(top / 448)), -126).clip(-126)
    edge = top / (448 * 2.0 ** want)
    off = e != want
    near = (np.abs(edge - 1) < NEAR) | (np.abs(edge - 0.5) < NEAR)
    assert np.all(~off | near), f"{what}: exponents"
    ee = np.repeat(e.astype(np.float64), BLK)[:x.size]
    ok = np.isfinite(x)
    assert np.all((codes[~ok] & 0x7F) == 0x7F), f"{what}: a value that is not finite is not held as NaN"
    y = np.abs(x[ok]) / 2.0 ** ee[ok]
    with np.errstate(divide="ignore"):
        step = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    raw = y / step + bits16[ok] / 65536
    got = E4M3[codes[ok] & 0x7F]
    near = np.maximum(NEAR, 0 if size is None else 6 * U * size[ok] / 2.0 ** ee[ok] / step)
    low, high = np.floor(raw - near) * step, np.floor(raw + near) * step
    if keep:
        low, high = np.where(x[ok] > 0, np.maximum(low, 2.0 ** -9), 0), np.where(x[ok] > 0, np.maximum(high, 2.0 ** -9), 0)
    bad = (got != low) & (got != high)
    assert not bad.any(), f"{what}: {bad.sum()} codes, first at {np.argmax(bad)}: {got[bad][0]} for {y[bad][0]} + {bits16[ok][bad][0]}/65536"
    assert np.all(((codes[ok] >> 7 == 1) == np.signbit(x[ok])) | (got == 0)), f"{what}: signs"


class Group:
    """A raw group over device buffers of its own."""

    def __init__(self, gpu, arrays, clip=1.0, wd=0.1, b2=B2, shift=(0, 0)):
        self.gpu, self.L, self.clip, self.wd, self.b2 = gpu, mod("lib"), clip, wd, b2
        self.sizes = [a.size for a in arrays]
        self.raw = []
        put = lambda n, s: self.raw.append(gpu.create_state_buffer(n + 64)) or self.raw[-1] + s  # noqa: E731
        self.w = [put(4 * n, shift[0]) for n in self.sizes]
        self.g = [put(4 * n, shift[0]) for n in self.sizes]
        self.m = [put(n, shift[1]) for n in self.sizes]
        self.r = [put(n, shift[1]) for n in self.sizes]
        self.e = [put(2 * -(-n // BLK), 0) for n in self.sizes]
        for b, a in zip(self.w, arrays):
            gpu.write_state_buffer(b, a)
        self.first = np.concatenate([[0], np.cumsum([-(-n // BLK) for n in self.sizes])])
        n = len(arrays)
        t = lambda v: (self.L.buf * max(1, n))(*v)  # noqa: E731
        self.h = C.c_void_p()
        self.check(self.L.lib.gt_adamw8_create(gpu.ctx, n, t(self.w), t(self.g), t(self.m), t(self.r), t(self.e), (C.c_int64 * max(1, n))(*self.sizes),
                                               B1, b2, AEPS, wd, clip, C.byref(self.h)))

    def check(self, rc):
        self.L.check(self.gpu.ctx, rc, "adamw8")

    def grads(self, arrays):
        for b, a in zip(self.g, arrays):
            self.gpu.write_state_buffer(b, a.astype(np.float32))

    def step(self, t, lr=1e-3, seed=None):
        self.check(self.L.lib.gt_adamw8_step(self.gpu.ctx, self.h, lr, 1 - B1 ** t, 1 - self.b2 ** t, t if seed is None else seed))

    def states(self, i):
        """(codes of m, of r, exponents of m, of r)"""
        n = self.sizes[i]
        e = self.gpu.read_state_buffer(self.e[i], 2 * -(-n // BLK), np.int8).reshape(-1, 2)
        return self.gpu.read_state_buffer(self.m[i], n, np.uint8), self.gpu.read_state_buffer(self.r[i], n, np.uint8), e[:, 0], e[:, 1]

    def weights(self, i):
        return self.gpu.read_state_buffer(self.w[i], self.sizes[i])

    def free(self):
        self.check(self.L.lib.gt_adamw_destroy(self.gpu.ctx, self.h))
        for b in self.raw:
            self.gpu.free_state_buffer(b)


def gradients(rs, sizes, scale):
    """Blocks of very different size, elements that are exactly zero and whole blocks of them."""
    out = []
    for n in sizes:
        nb = -(-n // BLK)
        s = np.repeat(np.exp(2 * rs.standard_normal(nb)) * (rs.rand(nb) > 0.2), BLK)[:n]
        g = scale * s * rs.standard_normal(n) * np.exp(rs.standard_normal(n))
        out.append(np.where(rs.rand(n) < 0.05, 0, g).astype(np.float32))
    return out


def step_and_check(G, grads, t, lr, seed):
    before = [(G.weights(i), *G.states(i)) for i in range(len(G.sizes))]
    G.grads(grads)
    G.step(t, lr, seed)
    norm = np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads))
    sc = G.clip / (norm + 1e-12) if G.clip > 0 and norm > G.clip else 1.0
    for i, (w, mc, rc, em, er) in enumerate(before):
        g = grads[i].astype(np.float64) * sc
        m0, v0 = decode(mc, em), decode(rc, er) ** 2
        m, v = B1 * m0 + (1 - B1) * g, G.b2 * v0 + (1 - G.b2) * g * g
        den = np.sqrt(v / (1 - G.b2 ** t)) + AEPS
        want = w - lr * (m / (1 - B1 ** t) / den + G.wd * w)
        size = lr * ((B1 * np.abs(m0) + (1 - B1) * np.abs(g)) / (1 - B1 ** t) / den + G.wd * np.abs(w))
        got = G.weights(i)
        # the update passes at most sixteen roundings, the weight two more (its own and the product with lr)
        far = np.abs(got - want) - (16 * U * size + 2 * U * (np.abs(w) + np.abs(want)))
        assert far.max(initial=-1) <= 0, f"tensor {i}: weights {far.max():.3g} past the bound"
        mc, rc, em, er = G.states(i)
        words = random_words(seed, G.first[i], w.size)
        check_state(m, mc, em, (words & np.uint64(0xFFFF)).astype(np.float64), False, f"tensor {i} m",
                    B1 * np.abs(m0) + (1 - B1) * np.abs(g))
        check_state(np.sqrt(v), rc, er, (words >> np.uint64(16)).astype(np.float64), True, f"tensor {i} r")
    return norm


@pytest.mark.gpu
@pytest.mark.parametrize("clip,wd,b2", [(1.0, 0.1, 0.95), (0.0, 0.0, 0.999), (0.5, 0.01, 0.999)])
@pytest.mark.parametrize("sizes", [[1], [255], [256], [257], [4096], [4097, 3], [5, 300, 1024, 70001, 256, 1], [0, 7, 0]], ids=str)
def test_steps(gpu, sizes, clip, wd, b2):
    rs = np.random.RandomState(sum(sizes))
    G = Group(gpu, [rs.standard_normal(n).astype(np.float32) for n in sizes], clip, wd, b2)
    try:
        for t, scale, seed in ((1, 1.0, 1), (2, 1e-3, 77), (3, 1e-2, (5 << 32) + 4000000000)):
            norm = step_and_check(G, gradients(rs, sizes, scale), t, 1e-3, seed)
            if clip > 0:
                got = C.c_float()
                G.check(G.L.lib.gt_adamw_grad_norm(gpu.ctx, G.h, C.byref(got)))
                assert abs(got.value - norm) <= 2 * U * norm
    finally:
        G.free()


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [(4, 0), (0, 1), (8, 2), (4, 3)])
def test_alignment_changes_no_bit(gpu, shift):
    sizes = [1000, 4096, 5000]
    out = []
    for s in ((0, 0), shift):
        rs = np.random.RandomState(1)
        G = Group(gpu, [rs.standard_normal(n).astype(np.float32) for n in sizes], clip=0.0, shift=s)
        for t in (1, 2):
            G.grads(gradients(rs, sizes, 0.1))
            G.step(t)
        out.append([a for i in range(3) for a in (G.weights(i), *G.states(i))])
        G.free()
    assert all(np.array_equal(a, b) for a, b in zip(*out))


@pytest.mark.gpu
def test_extreme_gradients(gpu):
    """The smallest and largest finite values, denormals among them; blocks of one value; a lone large one among small."""
    n = 8 * BLK
    g = np.zeros(n, np.float32)
    g[:BLK] = 1e-45
    g[BLK:2 * BLK] = 3e-23
    g[2 * BLK:3 * BLK] = 1.5e19                                     # its square times (1 - b2) is finite
    g[3 * BLK] = -1e4
    g[3 * BLK + 1:4 * BLK] = 1e-9
    g[4 * BLK:5 * BLK] = np.float32(448.0) * 2.0 ** np.arange(-100, 28).repeat(2)
    g[5 * BLK:6 * BLK] = -1e-30
    G = Group(gpu, [np.ones(n, np.float32)], clip=0.0, wd=0.0)
    try:
        G.grads([g])
        G.step(1)
        mc, rc, em, er = G.states(0)
        words = random_words(1, 0, n)
        # the moments as 32 bits hold them: below 2^-126 a product keeps fewer bits than the bound on its roundings counts
        m = ((np.float32(1 - B1) * g).astype(np.float32)).astype(np.float64)
        v = ((np.float32(1 - B2) * g).astype(np.float32) * g).astype(np.float32).astype(np.float64)
        check_state(m, mc, em, (words & np.uint64(0xFFFF)).astype(np.float64), False, "m")
        check_state(np.sqrt(v).astype(np.float32).astype(np.float64), rc, er, (words >> np.uint64(16)).astype(np.float64), True, "r")
        assert np.all(rc[3 * BLK + 1:4 * BLK] >= 1), "a second moment that is there was rounded away"
        assert np.all(np.isfinite(G.weights(0)))
    finally:
        G.free()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_where_they_are(gpu):
    n = 3 * BLK + 17
    rs = np.random.RandomState(2)
    w, g = rs.standard_normal(n).astype(np.float32), rs.standard_normal(n).astype(np.float32)
    bad = {5: np.nan, BLK + 3: np.inf, BLK + 200: -np.inf, 3 * BLK + 16: np.nan, 2 * BLK: 3e38}      # 3e38: m finite, v not
    out = []
    for dirty in (False, True):
        G = Group(gpu, [w], clip=0.0)
        h = g.copy()
        for i, x in bad.items():
            h[i] = x if dirty else 0.0
        G.grads([h])
        G.step(1)
        out.append((G.weights(0), *G.states(0)))
        G.step(2)
        out.append((G.weights(0), *G.states(0)))
        G.free()
    keep = np.ones(n, bool)
    keep[list(bad)] = False
    keep[2 * BLK:3 * BLK] = False                                     # 3e38's m is finite: its block's exponent is another
    for a, b in ((out[0], out[2]), (out[1], out[3])):
        for x, y in zip(a[:3], b[:3]):
            assert np.array_equal(x[keep], y[keep])
    w1, mc, rc, em, er = out[2]
    assert all(np.isnan(w1[i]) for i in (5, BLK + 3, BLK + 200, 3 * BLK + 16))
    assert all(mc[i] & 0x7F == 0x7F and rc[i] & 0x7F == 0x7F for i in (5, BLK + 3, BLK + 200, 3 * BLK + 16))
    assert mc[2 * BLK] & 0x7F != 0x7F and rc[2 * BLK] & 0x7F == 0x7F
    assert np.all(np.isfinite(w1[keep]))


@pytest.mark.gpu
def test_rounding_is_unbiased_where_rounding_to_nearest_stands_still(gpu):
    """A constant gradient, b2 = 0.999: a step moves r by less than a thousandth of itself, an e4m3 step is 6 to 12 percent. The mean of v over
    32768 elements follows g^2 (1 - b2^t). Rounding r without bias adds its variance to v: at most step * move <= r/8 * 0.0005 |g^2/v - 1| r
    a step against a pull of 0.001 |g^2 - v|, a sixteenth of the distance that is left, 6 percent at most; the mean's own
    spread is below 0.3 / sqrt(32768). m's mean, whose rounding is unbiased as it stands, follows g (1 - b1^t) to that spread."""
    n, g = 32768, 0.37
    G = Group(gpu, [np.zeros(n, np.float32)], clip=0.0, wd=0.0)
    try:
        G.grads([np.full(n, g, np.float32)])
        bm, bv = gpu.create_state_buffer(4 * n), gpu.create_state_buffer(4 * n)
        for t in range(1, 1501):
            G.step(t)
            if t in (30, 300, 1500):
                G.check(G.L.lib.gt_adamw8_read(gpu.ctx, G.h, 0, bm, bv))
                m, v = (gpu.read_state_buffer(b, n).astype(np.float64).mean() for b in (bm, bv))
                assert abs(m / (g * (1 - B1 ** t)) - 1) < 0.005
                assert -0.01 < v / (g * g * (1 - B2 ** t)) - 1 < 0.0625 + 0.01
        for b in (bm, bv):
            gpu.free_state_buffer(b)
    finally:
        G.free()


@pytest.mark.gpu
def test_seeds(gpu):
    rs = np.random.RandomState(3)
    w, g = rs.standard_normal(5000).astype(np.float32), rs.standard_normal(5000)
    out = []
    for seed in (9, 9, 10, 9 + (1 << 32)):
        G = Group(gpu, [w], clip=1.0)
        G.grads([g])
        G.step(1, seed=seed)
        out.append((G.weights(0), *G.states(0)))
        G.free()
    assert all(np.array_equal(a, b) for a, b in zip(out[0], out[1]))
    for other in out[2:]:
        assert np.array_equal(out[0][0], other[0])                        # the update does not depend on the rounding
        assert np.mean(out[0][1] != other[1]) > 0.1 and np.mean(out[0][2] != other[2]) > 0.1


@pytest.mark.gpu
def test_two_groups_on_two_contexts_at_once(gpu):
    """Groups of two contexts (two streams) stepped in turn without waiting: each does what it does alone."""
    hb = mod("hip_backend")
    sizes = [300000, 5000, 17]
    other = hb.HipBackend(0, streams=1)
    try:
        def groups(a, b):
            rs = np.random.RandomState(6)
            w = [rs.standard_normal(n).astype(np.float32) for n in sizes]
            G = [Group(be, w, clip=1.0) for be in (a, b)]
            for i, x in enumerate(G):
                x.grads([rs.standard_normal(n) * (i + 1) for n in sizes])
            return G
        A, B = groups(gpu, other)
        for t in range(1, 6):
            A.step(t)
            B.step(t)
        other.sync([])
        both = [[a for i in range(3) for a in (x.weights(i), *x.states(i))] for x in (A, B)]
        A.free()
        B.free()
        C_, D = groups(gpu, gpu)
        for x in (C_, D):
            for t in range(1, 6):
                x.step(t)
        alone = [[a for i in range(3) for a in (x.weights(i), *x.states(i))] for x in (C_, D)]
        C_.free()
        D.free()
        assert all(np.array_equal(a, b) for p, q in zip(both, alone) for a, b in zip(p, q))
    finally:
        other.destroy()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 300, 70001])
def test_moments_out_and_in_again(gpu, n):
    """What read gives, write takes back without a change; other values come in rounded to the nearest."""
    rs = np.random.RandomState(4)
    G = Group(gpu, [rs.standard_normal(9).astype(np.float32), rs.standard_normal(n).astype(np.float32)], clip=1.0)
    bm, bv, cm, cv = (gpu.create_state_buffer(4 * n) for _ in range(4))
    read = lambda m, v: G.check(G.L.lib.gt_adamw8_read(gpu.ctx, G.h, 1, m, v))  # noqa: E731
    try:
        for t in (1, 2):
            G.grads(gradients(rs, G.sizes, 0.3))
            G.step(t)
        read(bm, bv)
        m, v = gpu.read_state_buffer(bm, n), gpu.read_state_buffer(bv, n)
        mc, rc, em, er = G.states(1)
        assert np.array_equal(m, decode(mc, em).astype(np.float32)) and np.array_equal(v, (decode(rc, er) ** 2).astype(np.float32))
        G.check(G.L.lib.gt_adamw8_write(gpu.ctx, G.h, 1, bm, bv))
        read(cm, 0)
        read(0, cv)
        assert np.array_equal(gpu.read_state_buffer(cm, n), m) and np.array_equal(gpu.read_state_buffer(cv, n), v)
        m, v = (0.1 * rs.standard_normal(n)).astype(np.float32), (rs.standard_normal(n) ** 2).astype(np.float32)
        v[::7] = 0
        gpu.write_state_buffer(bm, m)
        gpu.write_state_buffer(bv, v)
        G.check(G.L.lib.gt_adamw8_write(gpu.ctx, G.h, 1, bm, bv))
        mc, rc, em, er = G.states(1)
        half = np.full(n, 32768.0)
        check_state(m.astype(np.float64), mc, em, half, False, "m")
        check_state(np.sqrt(v.astype(np.float64)), rc, er, half, True, "r")
        # second moments that are none: below zero and not finite are held as NaN and leave their neighbours' exponent alone, -0 is 0
        if n > 260:
            v2 = v.copy()
            v2[[1, 5, 258]] = -4e4, np.inf, -0.0
            gpu.write_state_buffer(bv, v2)
            G.check(G.L.lib.gt_adamw8_write(gpu.ctx, G.h, 1, bm, bv))
            _, rc2, _, er2 = G.states(1)
            assert rc2[1] & 0x7F == 0x7F and rc2[5] & 0x7F == 0x7F and rc2[258] == 0
            same = np.ones(n, bool)
            same[[1, 5, 258]] = False
            if er2[0] == er[0] and er2[1] == er[1]:
                assert np.array_equal(rc2[same], rc[same])
            assert np.all(E4M3[rc2[same] & 0x7F] <= 448)
        # half an e4m3 step is 2^-4 of the value, or 2^-10 units where e4m3 is denormal
        got = decode(mc, em)
        assert np.all(np.abs(got - m) <= np.maximum(2.0 ** -4 * np.abs(m), 2.0 ** -10 * 2.0 ** np.repeat(em.astype(float), BLK)[:n]) * (1 + 8 * U))
    finally:
        for b in (bm, bv, cm, cv):
            gpu.free_state_buffer(b)
        G.free()


@pytest.mark.gpu
def test_a_tensor_past_32_bits(gpu):
    """More than 2^32 elements: the last ones are stepped like the first."""
    n = (1 << 32) + 300
    L = mod("lib")
    raw = []
    try:
        new = lambda nbytes: raw.append(gpu.create_state_buffer(nbytes)) or raw[-1]  # noqa: E731
        w, g, m, r, e = new(4 * n), new(4 * n), new(n), new(n), new(2 * -(-n // BLK))
        tail = np.random.RandomState(5).standard_normal(300).astype(np.float32)
        gpu.write_state_buffer(g + 4 * (n - 300), tail)
        gpu.write_state_buffer(g, tail)
        h = C.c_void_p()
        one = lambda b: (L.buf * 1)(b)  # noqa: E731
        L.check(gpu.ctx, L.lib.gt_adamw8_create(gpu.ctx, 1, one(w), one(g), one(m), one(r), one(e), (C.c_int64 * 1)(n), B1, B2, AEPS, 0.0, 1.0, C.byref(h)), "create")
        L.check(gpu.ctx, L.lib.gt_adamw8_step(gpu.ctx, h, 1e-3, 1 - B1, 1 - B2, 1), "step")
        norm = np.sqrt(2 * (tail.astype(np.float64) ** 2).sum())
        got = C.c_float()
        L.check(gpu.ctx, L.lib.gt_adamw_grad_norm(gpu.ctx, h, C.byref(got)), "norm")
        assert abs(got.value - norm) <= 2 * U * norm
        first, last = gpu.read_state_buffer(w, 300), gpu.read_state_buffer(w + 4 * (n - 300), 300)
        # the first step of a weight is lr * g / (|g| + eps): eps is less than a hundredth of every clipped gradient here
        assert np.abs(tail).min() / norm > 100 * AEPS
        assert np.array_equal(first, last) and np.all(np.abs(first + 1e-3 * np.sign(tail)) < 1.1e-5)
        mc = gpu.read_state_buffer(m + n - 300, 300, np.uint8)
        ee = gpu.read_state_buffer(e + 2 * (-(-n // BLK) - 2), 4, np.int8).reshape(2, 2)
        x = (1 - B1) * tail.astype(np.float64) / (norm + 1e-12)
        check_state(x, mc, ee[:, 0], (random_words(1, (1 << 32) // BLK, 300) & np.uint64(0xFFFF)).astype(np.float64), False, "m of the last block")
        L.check(gpu.ctx, L.lib.gt_adamw_destroy(gpu.ctx, h), "destroy")
    finally:
        for b in raw:
            gpu.free_state_buffer(b)


@pytest.mark.gpu
def test_refusals(gpu):
    L = mod("lib")
    lib = L.lib
    b = gpu.create_state_buffer(4096)
    one = lambda v: (L.buf * 1)(v)  # noqa: E731
    h = C.c_void_p()

    def create(w=b, g=b + 1024, m=b + 2048, r=b + 2304, e=b + 3072, size=4):
        L.check(gpu.ctx, lib.gt_adamw8_create(gpu.ctx, 1, one(w), one(g), one(m), one(r), one(e), (C.c_int64 * 1)(size), B1, B2, AEPS, 0.0, 1.0, C.byref(h)), "create")
    for kw, match in ((dict(w=0), "null buffer"), (dict(e=0), "null buffer"), (dict(size=-1), "negative"), (dict(size=(1 << 40) + 1), "more than 2.40"), (dict(g=b + 2), "not aligned"), (dict(e=b + 1), "not aligned")):
        with pytest.raises(L.HipError, match=match):
            create(**kw)
    for kw in (dict(m=b + 8), dict(r=b + 2050), dict(e=b + 2048), dict(w=b + 2048)):
        with pytest.raises(L.HipError, match="overlap"):
            create(**kw)
    two = (L.buf * 2)(b, b)
    assert lib.gt_adamw8_create(gpu.ctx, 2, two, two, (L.buf * 2)(b + 64, b + 128), (L.buf * 2)(b + 192, b + 256), (L.buf * 2)(b + 320, b + 384), (C.c_int64 * 2)(4, 4),
                                B1, B2, AEPS, 0.0, 1.0, C.byref(h)) != 0 and "overlap" in lib.gt_last_error(gpu.ctx).decode()
    assert lib.gt_adamw8_create(gpu.ctx, 1, None, one(b), one(b), one(b), one(b), (C.c_int64 * 1)(4), B1, B2, AEPS, 0.0, 1.0, C.byref(h)) != 0
    create()
    refused = lambda rc, match: (rc != 0 and match in lib.gt_last_error(gpu.ctx).decode()) or pytest.fail(match)  # noqa: E731
    refused(lib.gt_adamw_step(gpu.ctx, h, 1e-3, 0.1, 0.1), "use gt_adamw8_step")
    refused(lib.gt_adamw8_step(gpu.ctx, h, 1e-3, 0.0, 0.1, 1), "must be positive")
    refused(lib.gt_adamw8_step(gpu.ctx, None, 1e-3, 0.1, 0.1, 1), "not an optimizer")
    refused(lib.gt_adamw8_read(gpu.ctx, h, 1, b, b), "tensor 1 of 1")
    refused(lib.gt_adamw8_read(gpu.ctx, h, -1, b, b), "tensor -1 of 1")
    refused(lib.gt_adamw8_read(gpu.ctx, h, 0, b + 2, b), "not aligned")
    refused(lib.gt_adamw8_write(gpu.ctx, h, 0, b, 0), "missing")
    L.check(gpu.ctx, lib.gt_adamw_destroy(gpu.ctx, h), "destroy")
    refused(lib.gt_adamw8_step(gpu.ctx, h, 1e-3, 0.1, 0.1, 1), "not an optimizer")
    refused(lib.gt_adamw_destroy(gpu.ctx, h), "not an optimizer")
    h32 = C.c_void_p()
    L.check(gpu.ctx, lib.gt_adamw_create(gpu.ctx, 1, one(b), one(b), one(b), one(b), (C.c_int64 * 1)(4), B1, B2, AEPS, 0.0, 1.0, C.byref(h32)), "create")
    refused(lib.gt_adamw8_step(gpu.ctx, h32, 1e-3, 0.1, 0.1, 1), "use gt_adamw_step")
    refused(lib.gt_adamw8_read(gpu.ctx, h32, 0, b, b), "held in 32 bits")
    L.check(gpu.ctx, lib.gt_adamw_destroy(gpu.ctx, h32), "destroy")
    with pytest.raises(ValueError, match="state_bits must be 8 or 32"):
        mod("optim").AdamWHip(gpu, [], lr=1e-3, state_bits=16)
    gpu.free_state_buffer(b)


# ---- a training loop with both operators ---------------------------------------------------------------------------------


def train(gpu, ref, arch, steps, which="adamw", resume_at=None):
    from test_gpu_model import SMALL, batches, build_pair
    optim, tr = mod("optim"), mod("train")
    kw = SMALL[arch]
    seqs = batches(ref, kw["vocab"], 21, 2 * steps, seed=10)
    _, model = build_pair(ref, kw, seed=6, std=0.1)

    def make(m):
        if which == "adamw":
            return optim.AdamWHip(gpu, m.params(), lr=1e-3, beta2=0.95, weight_decay=0.1, state_bits=8)
        mu, aux = m.param_groups()
        return optim.MuonHip(gpu, mu, aux, lr=0.01, aux={"lr": 3e-3, "state_bits": 8})
    opt = make(model)
    losses = []
    if resume_at:
        losses += tr.train_lm_hip_resident(model, gpu, opt, seqs[:2 * resume_at], resume_at, 2, 21)
        state = opt.export_state()
        if which != "adamw":
            state = optim.deserialize_opt_state(optim.serialize_opt_state(state))
        weights = {n: p.data.copy() for n, p in model.named_params()}
        opt.destroy()
        model = mod("arch").Model(model.cfg, weights)
        opt = make(model)
        opt.import_state(state)
        losses += tr.train_lm_hip_resident(model, gpu, opt, seqs[2 * resume_at:], steps - resume_at, 2, 21)
    else:
        losses += tr.train_lm_hip_resident(model, gpu, opt, seqs, steps, 2, 21)
    state = opt.export_state()
    opt.destroy()
    return losses, {n: p.data.copy() for n, p in model.named_params()}, state


@pytest.mark.gpu
@pytest.mark.parametrize("arch,which", [("qwen3", "adamw"), ("gemma3", "muon")])
def test_a_training_loop_and_its_resumption(gpu, ref, arch, which):
    """The device-resident loop with the fused QK-norm and 8-bit moments: a run that is exported after two steps and taken up again by a new
    optimizer repeats the uninterrupted one bit for bit."""
    gpu.fuse_qk_norm_rope = True
    try:
        losses, w, s = train(gpu, ref, arch, 4, which)
        again, w2, s2 = train(gpu, ref, arch, 4, which, resume_at=2)
    finally:
        gpu.fuse_qk_norm_rope = False
    assert all(np.isfinite(x) for x in losses)
    assert losses == again
    assert all(np.array_equal(w[n], w2[n]) for n in w)
    for k in s:
        assert np.array_equal(s[k], s2[k]) if k in ("t", "adamT") else all(np.array_equal(a, b) for a, b in zip(s[k], s2[k])), k


@pytest.mark.gpu
def test_import_checks_sizes(gpu):
    ag, optim = mod("autograd"), mod("optim")
    p = ag.Tensor(np.ones(300, np.float32), [300], True)
    opt = optim.AdamWHip(gpu, [p], lr=1e-3, state_bits=8)
    with pytest.raises(ValueError, match="size mismatch"):
        opt.import_state({"m": [np.zeros(299)], "v": [np.zeros(300)], "t": 1})
    with pytest.raises(ValueError, match="count mismatch"):
        opt.import_state({"m": [], "v": [], "t": 1})
    assert opt.export_state()["t"] == 0
    opt.destroy()
