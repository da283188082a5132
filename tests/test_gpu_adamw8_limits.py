"""AdamW with 8-bit moments where FP32 ends: second moments that are denormal, vanish or overflow; what is read, written and read again; buffers
that may not share memory. The states are held to the definition of test_gpu_adamw8.py, formed here from the second moments as FP32 holds them."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import mod
from test_gpu_adamw8 import B1, BLK, E4M3, NEAR, Group, U, blocks_of, check_state, decode, random_words

F = np.float32


class Moments:
    """Read and write access to tensor i of a group."""

    def __init__(self, gpu, G, i=0):
        self.gpu, self.G, self.i, self.n = gpu, G, i, G.sizes[i]
        self.b = [gpu.create_state_buffer(4 * self.n) for _ in range(2)]

    def read(self):
        self.G.check(self.G.L.lib.gt_adamw8_read(self.gpu.ctx, self.G.h, self.i, *self.b))
        return tuple(self.gpu.read_state_buffer(b, self.n) for b in self.b)

    def write(self, m, v):
        for b, a in zip(self.b, (m, v)):
            self.gpu.write_state_buffer(b, np.asarray(a, F))
        self.G.check(self.G.L.lib.gt_adamw8_write(self.gpu.ctx, self.G.h, self.i, *self.b))

    def free(self):
        for b in self.b:
            self.gpu.free_state_buffer(b)


def same(a, b):
    return all(np.array_equal(x, y, equal_nan=True) for x, y in zip(a, b))


def check_roots(x, codes, e, bits16):
    """Codes of the roots x at the block's exponent: no element leaves e4m3's range, no exponent is more than it takes (or than the least that is
    held), and a code is off by a step only where what is rounded lies within NEAR of a whole number of steps."""
    top = blocks_of(x).max(axis=1)
    with np.errstate(divide="ignore"):
        need = np.where(top > 0, np.ceil(np.log2(top / 448)), -126).clip(-126)
    assert np.all(e >= need) and np.all(e <= np.maximum(need, -65)), (e, need)
    y = x / 2.0 ** np.repeat(e.astype(np.float64), BLK)[:x.size]
    step = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    raw = y / step + bits16 / 65536
    low, high = (np.where(x > 0, np.maximum(np.floor(raw + d) * step, 2.0 ** -9), 0) for d in (-NEAR, NEAR))
    got = E4M3[codes]
    bad = (got != low) & (got != high)
    assert not bad.any(), f"{bad.sum()} codes, first at {np.argmax(bad)}: {got[bad][0]} for {y[bad][0]} + {bits16[bad][0]}/65536"


def roots_of(rs, powers, spread):
    """One block for each power: values of e4m3's four bits, the largest 15/8 * 2^power, down to 2^-spread of it, some zero."""
    out = []
    for p in powers:
        r = (8 + rs.randint(0, 8, BLK)) / 8 * 2.0 ** (p - rs.randint(0, spread + 1, BLK))
        r[rs.rand(BLK) < 0.1] = 0
        r[0] = 15 / 8 * 2.0 ** p
        out.append(r)
    return np.concatenate(out)


@pytest.mark.gpu
def test_denormal_second_moments_out_and_in_again(gpu):
    """v from 2^-120 down to where FP32 ends. Every r here is a multiple of 2^-74 of at most four bits, so its square is an FP32 number, and v, its root
    and its code are exact whatever is added for the rounding."""
    rs = np.random.RandomState(71)
    r = roots_of(rs, (-60, -61, -62, -63, -64, -65, -67, -68), 3)
    r[-BLK:] = roots_of(rs, (-71,), 0)
    v, m = (r * r).astype(F), (1e-9 * rs.standard_normal(r.size)).astype(F)
    assert np.array_equal(v.astype(np.float64), r * r) and v[v > 0].min() < 2.0 ** -140
    G = Group(gpu, [np.zeros(r.size, F)])
    M = Moments(gpu, G)
    try:
        M.write(m, v)
        first = M.read()
        assert np.array_equal(first[1], v)
        mc, rc, em, er = G.states(0)
        check_roots(r, rc, er, np.full(r.size, 32768.0))
        M.write(*first)
        assert same(M.read(), first)
    finally:
        M.free()
        G.free()


@pytest.mark.gpu
@pytest.mark.parametrize("b2", [0.95, 0.999])
def test_a_step_on_denormal_second_moments(gpu, b2):
    """Without a gradient a step leaves v b2, rounded to FP32 once. Its root is within 2^-22 of itself, the weight's update as the module's text in
    test_gpu_adamw8.py derives it."""
    rs = np.random.RandomState(72)
    r = roots_of(rs, (-58, -60, -62, -63, -64, -65, -66, -67), 3)
    v, m = (r * r).astype(F), (2.0 ** -70 * rs.standard_normal(r.size)).astype(F)
    w = (2.0 ** -12 * rs.standard_normal(r.size)).astype(F)
    G = Group(gpu, [w], clip=0.0, wd=0.0, b2=b2)
    M = Moments(gpu, G)
    try:
        M.write(m, v)
        m0 = decode(*(lambda s: (s[0], s[2]))(G.states(0)))
        G.step(5, lr=1e-3, seed=99)
        want = ((r * r).astype(F) * F(b2)).astype(F).astype(np.float64)
        words = random_words(99, 0, r.size)
        mc, rc, em, er = G.states(0)
        check_roots(np.sqrt(want), rc, er, (words >> np.uint64(16)).astype(np.float64))
        m1 = B1 * m0
        upd = 1e-3 * m1 / (1 - B1 ** 5) / (np.sqrt(want / (1 - b2 ** 5)) + 1e-8)
        assert np.all(np.abs(G.weights(0) - (w - upd)) <= 16 * U * np.abs(upd) + 2 * U * (np.abs(w) + np.abs(w - upd)))
    finally:
        M.free()
        G.free()


@pytest.mark.gpu
@pytest.mark.parametrize("b2", [0.5, 0.95])
def test_second_moments_that_decay_for_good(gpu, b2):
    """Blocks that get no gradient any more (embedding rows that no batch names). Their second moments stop at 2^-148, the square of the least root that
    is held: one that is there stays there, and at every step read and write give back what was held and a run that goes through them
    does what one without them does."""
    rs = np.random.RandomState(73)
    r = roots_of(rs, (-55, -58, -62, -66), 3)
    v, m = (r * r).astype(F), (2.0 ** -70 * rs.standard_normal(r.size)).astype(F)
    G = [Group(gpu, [np.zeros(r.size, F)], clip=0.0, wd=0.0, b2=b2) for _ in range(2)]
    M = [Moments(gpu, g) for g in G]
    try:
        for x in M:
            x.write(m, v)
        floors = 0
        for t in range(1, 61 if b2 < 0.9 else 501):
            for g in G:
                g.step(t)
            if t % 20 and t < 40:
                continue
            held = M[1].read()
            M[1].write(*held)
            again = M[1].read()
            assert same(held, again) and same(held, M[0].read()), t
            assert np.array_equal(held[1] > 0, r > 0), t
            floors += np.all(held[1][r > 0] < 2.0 ** -140)
        assert floors > 0                                                    # they got there
        assert np.array_equal(G[0].weights(0), G[1].weights(0))
    finally:
        for x in M + G:
            x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_second_moments_that_overflow(gpu, wd):
    """A gradient whose square leaves FP32 while the first moment does not: the weight is left to its decay, in this step and in all later ones, as it is
    with moments of 32 bits (m / infinity). The block's other elements are stepped as without it, and the moments come back as infinities."""
    n, at, t0 = 3 * BLK + 5, (7, 2 * BLK + 1, 3 * BLK + 4), 1
    rs = np.random.RandomState(74)
    w, g = rs.standard_normal(n).astype(F), rs.standard_normal(n).astype(F)
    big = g.copy()
    for i, x in zip(at, (6e20, -1e30, 3e38)):
        big[i] = x
    zero = g.copy()
    zero[list(at)] = 0
    G = Group(gpu, [w], clip=0.0, wd=wd)
    H = Group(gpu, [w], clip=0.0, wd=wd)
    M = Moments(gpu, G)
    L = mod("lib")
    b32 = [gpu.create_state_buffer(4 * n) for _ in range(4)]
    h32 = C.c_void_p()
    one = lambda b: (L.buf * 1)(b)  # noqa: E731
    L.check(gpu.ctx, L.lib.gt_adamw_create(gpu.ctx, 1, *[one(b) for b in b32], (C.c_int64 * 1)(n), B1, 0.999, 1e-8, wd, 0.0, C.byref(h32)), "create")
    gpu.write_state_buffer(b32[0], w)
    try:
        other = np.ones(n, bool)
        other[list(at)] = False
        for t, (a, b) in enumerate(((big, zero), (g, zero), (zero, zero), (g, zero)), t0):
            G.grads([a])
            H.grads([b])
            gpu.write_state_buffer(b32[1], a)
            for x in (G, H):
                x.step(t)
            L.check(gpu.ctx, L.lib.gt_adamw_step(gpu.ctx, h32, 1e-3, 1 - B1 ** t, 1 - 0.999 ** t), "step")
            got, alone, full = G.weights(0), H.weights(0), gpu.read_state_buffer(b32[0], n)
            # both sides round the decay three times, lr, wd and the product with w, and the weight once
            assert np.all(np.abs(got[list(at)] - full[list(at)]) <= t * (8 * U * 1e-3 * wd + 2 * U) * np.abs(w[list(at)])), (got[list(at)], full[list(at)])
            if t == 1:
                assert np.array_equal(got[other], alone[other])              # the update does not depend on what the block's exponent rounds
            m, v = M.read()
            assert np.all(np.isposinf(v[list(at)])) and np.all(np.isfinite(v[other])) and np.all(np.isfinite(m)) and np.all(np.isfinite(got))
            M.write(m, v)
            assert same(M.read(), (m, v))
    finally:
        L.check(gpu.ctx, L.lib.gt_adamw_destroy(gpu.ctx, h32), "destroy")
        for b in b32:
            gpu.free_state_buffer(b)
        M.free()
        G.free()
        H.free()


@pytest.mark.gpu
def test_moments_that_are_no_numbers(gpu):
    """A first moment that is infinite or NaN takes its weight with it, as in 32 bits. A second moment that is NaN or negative comes back as NaN, takes its
    weight with it and stays; none of them touches a neighbour."""
    n = 2 * BLK + 9
    rs = np.random.RandomState(75)
    w, g = rs.standard_normal(n).astype(F), rs.standard_normal(n).astype(F)
    m, v = rs.standard_normal(n).astype(F), (rs.standard_normal(n) ** 2).astype(F)
    bad_m, bad_v = {3: np.inf, BLK + 9: np.nan, 2 * BLK + 8: -np.inf}, {5: np.nan, BLK + 1: -1.0, 2 * BLK: -np.inf, BLK + 77: -1e-42}
    inf_v = {8: np.inf, 2 * BLK + 3: np.inf}
    G, H = Group(gpu, [w], clip=0.0, wd=0.1), Group(gpu, [w], clip=0.0, wd=0.1)
    M, K = Moments(gpu, G), Moments(gpu, H)
    try:
        mm, vv = m.copy(), v.copy()
        for d, a, z in ((bad_m, mm, m), (bad_v, vv, v), (inf_v, vv, v)):
            for i, x in d.items():
                a[i], z[i] = x, 0
        M.write(mm, vv)
        K.write(m, v)
        fine = np.ones(n, bool)
        fine[[*bad_m, *bad_v, *inf_v]] = False
        for t in (3, 4):
            a, b = M.read(), K.read()
            assert all(np.array_equal(x[fine], y[fine]) for x, y in zip(a, b))
            assert np.all(np.isnan(a[0][list(bad_m)])) and np.all(np.isnan(a[1][list(bad_v)])) and np.all(np.isposinf(a[1][list(inf_v)]))
            M.write(*a)
            assert same(M.read(), a)
            for x in (G, H):
                x.grads([g])
                x.step(t)
            ga, gb = G.weights(0), H.weights(0)
            assert np.array_equal(ga[fine], gb[fine])
            assert np.all(np.isnan(ga[[*bad_m, *bad_v]])) and np.all(np.isfinite(ga[list(inf_v)]))
    finally:
        for x in (M, K, G, H):
            x.free()


@pytest.mark.gpu
def test_the_largest_second_moments_stay_finite(gpu):
    """Up to FP32's largest number: a root that is rounded up has a square that is still finite, in a step, when written and when read again."""
    n = 4 * BLK
    rs = np.random.RandomState(76)
    v = (np.float64(np.finfo(F).max) * np.exp(-0.3 * rs.rand(n))).astype(F)
    v[:4] = np.finfo(F).max, F(2.9907e38), F(3.1e38), F(3.2e38)
    G = Group(gpu, [np.ones(n, F)], clip=0.0, wd=0.0)
    M = Moments(gpu, G)
    try:
        M.write(np.ones(n), v)
        for t in range(5, 25):
            m, got = M.read()
            assert np.all(np.isfinite(got)) and got.max() > 2.9e38, t
            M.write(m, got)
            assert same(M.read(), (m, got))
            g = np.where(rs.rand(n) < 0.5, 5.8e20, 5.5e20).astype(F)    # with (1 - b2) g^2 finite the sum with b2 v is past FP32 or just not
            M.write(m, np.minimum(got, F(2.9e38)) * F(0.02))
            _, old = M.read()
            G.grads([g])
            G.step(t)
            with np.errstate(over="ignore"):
                want = old * F(0.999) + (g * F(1 - 0.999)) * g
            _, got = M.read()
            assert np.array_equal(np.isfinite(got), np.isfinite(want)) and np.any(np.isfinite(want) & (want > 2.9908e38)), t
            assert np.all(np.isfinite(G.weights(0)))
            M.write(m, v)
    finally:
        M.free()
        G.free()


@pytest.mark.gpu
def test_the_largest_first_moments_stay_finite(gpu):
    n = 2 * BLK
    rs = np.random.RandomState(77)
    m = (np.float64(np.finfo(F).max) * np.exp(-0.3 * rs.rand(n)) * np.sign(rs.standard_normal(n))).astype(F)
    m[:4] = np.finfo(F).max, -np.finfo(F).max, F(3.2e38), F(-3.3e38)
    G = Group(gpu, [np.ones(n, F)], clip=0.0, wd=0.0)
    M = Moments(gpu, G)
    try:
        for t in range(30, 50):
            M.write(m, np.full(n, F(1e38)))
            got = M.read()
            assert np.all(np.isfinite(got[0])) and np.all(np.sign(got[0]) == np.sign(m)) and np.abs(got[0]).max() > 3.1e38, t
            M.write(*got)
            assert same(M.read(), got)
            G.grads([(m / 2).astype(F)])                                # its square is past FP32: v is infinite, m is not
            G.step(t)
            assert np.all(np.isfinite(M.read()[0])) and np.all(np.isfinite(G.weights(0))), t
            G.gpu.write_state_buffer(G.w[0], np.ones(n, F))
    finally:
        M.free()
        G.free()


@pytest.mark.gpu
def test_gradients_and_moment_buffers_that_overlap_are_refused(gpu):
    """A step writes weights and states while other workgroups still read gradients; read and write of the moments go through all of a tensor at once."""
    L = mod("lib")
    lib = L.lib
    n = 1000
    b = {m: gpu.create_state_buffer(s) for m, s in dict(w=4 * n, g=4 * n, m=n, r=n, e=8, w2=4 * n, g2=4 * n, m2=n, r2=n, e2=8, x=4 * n, y=4 * n).items()}
    h = C.c_void_p()

    def create(**kw):
        a = {**b, **kw}
        t = lambda *v: (L.buf * 2)(*v)  # noqa: E731
        L.check(gpu.ctx, lib.gt_adamw8_create(gpu.ctx, 2, t(a["w"], a["w2"]), t(a["g"], a["g2"]), t(a["m"], a["m2"]), t(a["r"], a["r2"]), t(a["e"], a["e2"]),
                                              (C.c_int64 * 2)(n, n), B1, 0.999, 1e-8, 0.0, 0.0, C.byref(h)), "create")
    try:
        for kw in (dict(g=b["w"]), dict(g=b["w2"]), dict(g2=b["w"] + 4 * n - 4), dict(g=b["m"] - 4 * n + 4), dict(g2=b["r"]), dict(g=b["e2"]), dict(g2=b["e"])):
            with pytest.raises(L.HipError, match="overlap"):
                create(**kw)
        create(g2=b["g"] + 8)                                             # gradients are only read: they may share memory
        L.check(gpu.ctx, lib.gt_adamw8_step(gpu.ctx, h, 1e-3, 0.1, 0.1, 1), "step")
        for call, args in ((lib.gt_adamw8_read, ((b["x"], b["x"]), (b["x"], b["x"] + 4 * n - 4), (b["m"] - b["m"] % 4, 0), (0, b["r"] - b["r"] % 4), (b["e"] - b["e"] % 4, b["y"]))),
                           (lib.gt_adamw8_write, ((b["m"], b["y"]), (b["x"], b["r"]), (b["x"], b["e"])))):
            for m, v in args:
                assert call(gpu.ctx, h, 0, m, v) != 0 and "overlap" in lib.gt_last_error(gpu.ctx).decode(), (m, v)
        L.check(gpu.ctx, lib.gt_adamw8_read(gpu.ctx, h, 0, b["x"], b["y"]), "read")
        L.check(gpu.ctx, lib.gt_adamw8_write(gpu.ctx, h, 0, b["x"], b["x"]), "write")       # both only read
        L.check(gpu.ctx, lib.gt_adamw_destroy(gpu.ctx, h), "destroy")
    finally:
        for x in b.values():
            gpu.free_state_buffer(x)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 2 * BLK + 9])
def test_written_moments_that_are_none_leave_their_neighbours_exponent_alone(gpu, n):
    """Second moments below zero, infinite or NaN and larger than all others in their block, first moments likewise: exponents and codes go by the rest."""
    rs = np.random.RandomState(78)
    m, v = (0.1 * rs.standard_normal(n)).astype(F), (rs.standard_normal(n) ** 2).astype(F)
    G = Group(gpu, [np.zeros(n, F)])
    M = Moments(gpu, G)
    half = np.full(n, 32768.0)
    try:
        at = [1, 5, 130, n - 1]
        vv, mm = v.copy(), m.copy()
        vv[at] = -4e4, np.inf, np.nan, -np.inf
        mm[[2, 6, 131, n - 2]] = np.inf, -np.inf, np.nan, np.inf
        M.write(mm, vv)
        mc, rc, em, er = G.states(0)
        assert np.all(rc[at] & 0x7F == 0x7F)
        x = np.where(np.isfinite(vv) & (vv >= 0), vv, 0).astype(np.float64)
        rest = rc.copy()
        rest[at] = 0
        check_state(np.sqrt(x), rest, er, half, True, "r")
        check_state(mm.astype(np.float64), mc, em, half, False, "m")
        M.write(np.where(np.isfinite(mm), mm, 0), x)
        assert all(np.array_equal(a, b) for a, b in zip(G.states(0)[2:], (em, er)))
    finally:
        M.free()
        G.free()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["adamw", "muon"])
def test_a_refused_group_keeps_no_memory(gpu, which):
    """A parameter listed twice has two sets of states that a step would write at once; what was made for them goes back."""
    ag, optim, L = mod("autograd"), mod("optim"), mod("lib")
    p = ag.Tensor(np.ones(3000, F), [3000], True)
    gpu.buffers_for(p)
    before = gpu.resident_bytes()
    for _ in range(3):
        with pytest.raises(L.HipError, match="overlap"):
            if which == "adamw":
                optim.AdamWHip(gpu, [p, p], lr=1e-3, state_bits=8)
            else:
                optim.MuonHip(gpu, [], [p, p], lr=0.01, aux={"lr": 1e-3, "state_bits": 8})
    assert gpu.resident_bytes() == before
    opt = optim.AdamWHip(gpu, [p], lr=1e-3, state_bits=8)
    opt.destroy()
    assert gpu.resident_bytes() == before
