"""QK-norm and rotation in one pass (gt_qk_norm_rope_*, ag.qk_norm_rope) against the formulas in 64 bits.

Bounds, from the number of roundings in 32 bits (u = 2^-24, half a step): a row's sum of squares passes at most 20 of them (squares, a
lane's own sum of up to 16 products, six exchanges), mean, eps, root and reciprocal five more, of which the root halves the
first: r is off by at most 15 u, y = x r w by 17 u, cos and sin by two each, a rotated element by 24 u (|y_j| + |y_{j+h}|). The
backward's first term w g r takes the rotation's 4 and r's 15: 24 u; its second, x r^3 S / hd, 3 * 15 from r^3 and at most 20
from S: 72 u of the sum of absolute products. A gain sum is at most 20 u per term, a lane's chain of at most H terms, 64 lane
groups, and 1024 partial rows summed as 64 by 16: (20 + H + 64 + 64 + 16) u of the sum of absolute terms."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import backward_from, mod

U = 2.0 ** -24
EPS = 1e-6


def angles(rows, T, hd, base, pos, places=None):
    p = np.asarray(places, np.float64) if places is not None else (np.arange(rows) % T + pos).astype(np.float64)
    a = p[:, None] * base ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(a)[:, None, :], np.sin(a)[:, None, :]


def ref_fwd(x, w, cs, eps=EPS):
    """x [rows, H, hd] -> (rotated, |y_j| + |y_{j+h}| at both places)."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    h = x.shape[2] // 2
    y = x / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps) * w
    c, s = cs
    size = np.abs(y[..., :h]) + np.abs(y[..., h:])
    return np.concatenate([y[..., :h] * c - y[..., h:] * s, y[..., :h] * s + y[..., h:] * c], axis=2), np.concatenate([size, size], axis=2)


def ref_bwd(x, w, g, cs, rot, eps=EPS):
    """(dx, dw, bound on dx's rounding, bound on dw's per unit of its own count) as the module's text derives them."""
    x, w, g = x.astype(np.float64), w.astype(np.float64), g.astype(np.float64)
    h, hd = x.shape[2] // 2, x.shape[2]
    size = np.abs(g)
    if rot:
        c, s = cs
        size = np.tile(np.abs(g[..., :h]) + np.abs(g[..., h:]), 2)
        g = np.concatenate([g[..., :h] * c + g[..., h:] * s, g[..., h:] * c - g[..., :h] * s], axis=2)
    r = 1 / np.sqrt((x * x).mean(axis=2, keepdims=True) + eps)
    S = (g * w * x).sum(axis=2, keepdims=True)
    dx = r * w * g - x * r ** 3 * S / hd
    off = 24 * U * np.abs(w) * size * r + 72 * U * np.abs(x) * r ** 3 * (size * np.abs(w * x)).sum(axis=2, keepdims=True) / hd
    H = x.shape[1]
    return dx, (g * x * r).sum(axis=(0, 1)), off, (164 + H) * U * (size * np.abs(x) * r).sum(axis=(0, 1))


def test_reference_gradient_equals_differences():
    """The 64-bit formula the device is held to, against central differences of the 64-bit forward: their error is h^2 / 6 times a
    third derivative of order one plus 2^-53 / h, both below 1e-8 for h = 1e-5 with values of order one."""
    rs = np.random.RandomState(0)
    rows, H, hd = 3, 2, 6
    x, w, g = rs.standard_normal((rows, H, hd)), 1 + 0.3 * rs.standard_normal(hd), rs.standard_normal((rows, H, hd))
    cs = angles(rows, rows, hd, 100.0, 5)
    dx, dw, _, _ = ref_bwd(x, w, g, cs, True)
    loss = lambda x_, w_: float((ref_fwd(x_, w_, cs)[0] * g).sum())  # noqa: E731
    h = 1e-5
    for i in np.ndindex(*x.shape):
        d = np.zeros_like(x)
        d[i] = h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - dx[i]) < 1e-7
    for j in range(hd):
        d = np.zeros_like(w)
        d[j] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - dw[j]) < 1e-7


# ---- refusals above the library, on the CPU ---------------------------------------------------------------------------

class _Composed:
    """A backend without the op."""

    def __init__(self):
        self.calls = []

    def rms_norm_heads(self, x, w, *a):
        self.calls.append("norm")
        return x

    def rope(self, x, *a):
        self.calls.append("rope")
        return x


class _Stub(_Composed):
    def qk_norm_rope(self, *a):
        self.calls.append("fused")
        return a[0], a[1]


def test_host_checks_and_what_takes_the_composed_form():
    ag = mod("autograd")
    be = _Stub()
    t = lambda *s: ag.Tensor(np.zeros(s, np.float32), list(s), True)  # noqa: E731
    q, k, wq, wk = t(6, 32), t(6, 16), t(8), t(8)
    call = lambda *a, **kw: ag.qk_norm_rope(*a, **kw)  # noqa: E731
    ag.set_ops_backend(be)
    try:
        call(q, k, wq, wk, 3, 4, 2, 8, EPS, 1e4)
        assert be.calls == ["fused"]
        for bad, match in (((q, k, wq, wk, 4, 4, 2, 8, EPS, 1e4), "whole number of sequences"),
                           ((q, k, wq, wk, 3, 3, 2, 8, EPS, 1e4), "q is .6, 32."),
                           ((q, k, wq, t(7), 3, 4, 2, 8, EPS, 1e4), "k is .6, 16. with a gain of 7"),
                           ((q, t(5, 16), wq, wk, 3, 4, 2, 8, EPS, 1e4), "6 rows and k 5")):
            with pytest.raises(ValueError, match=match):
                call(*bad)
        with pytest.raises(ValueError, match="5 positions for 6 rows"):
            call(q, k, wq, wk, 1, 4, 2, 8, EPS, 1e4, positions=[0] * 5)
        with pytest.raises(ValueError, match="does not fit 32 bits"):
            call(q, k, wq, wk, 1, 4, 2, 8, EPS, 1e4, positions=[0, 0, 0, 0, 0, 2 ** 31])
        with pytest.raises(ValueError, match="not an integer"):
            call(q, k, wq, wk, 1, 4, 2, 8, EPS, 1e4, positions=[0, 0, 0, 0, 0, 0.5])
        # the same tensor or gain twice, and a backend that has no such op, take the four calls
        for a in ((q, q, wq, wk, 3, 4, 4, 8), (q, k, wq, wq, 3, 4, 2, 8)):
            be.calls.clear()
            call(*a, EPS, 1e4)
            assert be.calls == ["norm", "norm", "rope", "rope"]
        be = _Composed()
        ag.set_ops_backend(be)
        call(q, k, wq, wk, 3, 4, 2, 8, EPS, 1e4)
        assert be.calls == ["norm", "norm", "rope", "rope"]
        with pytest.raises(ValueError, match="positions need the fused op"):
            call(q, k, wq, wk, 3, 4, 2, 8, EPS, 1e4, positions=[0] * 6)
    finally:
        ag.set_ops_backend(None)


# ---- on the device ----------------------------------------------------------------------------------------------------


class Bufs:
    """Device copies of host arrays, given back at the end of a test."""

    def __init__(self, gpu):
        self.gpu, self.all = gpu, []

    def raw(self, nbytes):
        b = self.gpu.create_state_buffer(nbytes)
        self.all.append(b)
        return b

    def put(self, a, shift=0):
        a = np.ascontiguousarray(a)
        b = self.raw(a.nbytes + shift + 64) + shift
        self.gpu.write_state_buffer(b, a)
        return b

    def free(self):
        for b in self.all:
            self.gpu.free_state_buffer(b)


@pytest.fixture
def bufs(gpu):
    b = Bufs(gpu)
    yield b
    b.free()


def wide(a, pad, fill=7.0):
    """[rows, H, hd] as rows of H * hd + pad elements."""
    rows = a.shape[0]
    return np.concatenate([a.reshape(rows, -1), np.full((rows, pad), fill, np.float32)], axis=1).astype(np.float32)


def inputs(rows, Hq, Hkv, hd, seed):
    rs = np.random.RandomState(seed)
    n = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    return n(rows, Hq, hd) * np.exp(n(rows, 1, 1)), n(rows, Hkv, hd), 1 + 0.3 * n(hd), 1 + 0.3 * n(hd), n(rows, Hq, hd), n(rows, Hkv, hd)


# rows, T, Hq, Hkv, hd, pos: every lane count of the vector kernels, head sizes that leave lanes idle, generic sizes, one token and far ones
SHAPES = [(1, 1, 1, 1, 2, 0), (5, 5, 3, 1, 6, 0), (7, 7, 2, 2, 10, 3), (300, 100, 5, 5, 8, 0), (9, 9, 2, 1, 16, 1), (66, 33, 4, 4, 24, 0),
          (130, 65, 4, 4, 48, 0), (127, 127, 10, 2, 64, 0), (12, 4, 4, 2, 80, 7), (66, 33, 9, 3, 96, 0), (1, 1, 16, 8, 128, 100000),
          (1030, 515, 16, 8, 128, 0), (20, 10, 4, 2, 160, 0), (40, 20, 8, 4, 256, 0), (6, 3, 2, 1, 512, 0), (4, 2, 3, 1, 514, 0), (3, 3, 1, 1, 1024, 11),
          (2, 1, 7, 1, 4, 16000000), (3, 3, 32768, 5, 8, 0), (2, 2, 1, 1001, 16, 0), (5, 5, 333, 20000, 6, 0)]


def run_fwd(gpu, bufs, shape, seed, pad=(0, 0), shift=0, places=None, base=1e6):
    rows, T, Hq, Hkv, hd, pos = shape
    L = mod("lib")
    q, k, wq, wk, _, _ = inputs(rows, Hq, Hkv, hd, seed)
    ins = [bufs.put(wide(a, pad[0]), shift) for a in (q, k)]
    outs = [bufs.put(wide(np.zeros_like(a), pad[1]), shift) for a in (q, k)]
    gains = [bufs.put(w, shift) for w in (wq, wk)]
    at = bufs.put(np.asarray(places, np.int32)) if places is not None else 0
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, rows, T, Hq, Hkv, hd, EPS, base, pos, at,
                                               ins[0], Hq * hd + pad[0], gains[0], outs[0], Hq * hd + pad[1],
                                               ins[1], Hkv * hd + pad[0], gains[1], outs[1], Hkv * hd + pad[1]), "fwd")
    cs = angles(rows, T, hd, base, pos, places)
    got = []
    for x, w, H, o in ((q, wq, Hq, outs[0]), (k, wk, Hkv, outs[1])):
        a = gpu.read_state_buffer(o, rows * (H * hd + pad[1])).reshape(rows, -1)
        assert np.all(a[:, H * hd:] == 7.0), "the space between the rows was written"
        a = a[:, :H * hd].reshape(rows, H, hd)
        want, size = ref_fwd(x, w, cs)
        far = np.abs(a - want) - 24 * U * size
        assert np.all(np.isfinite(a)) and far.max() <= 0, f"off by {np.abs(a - want).max():.3g}, {far.max():.3g} more than the bound"
        got.append(a)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(gpu, bufs, shape):
    run_fwd(gpu, bufs, shape, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,pad,shift", [((12, 4, 4, 2, 64, 0), (64, 8), 0), ((12, 4, 4, 2, 64, 0), (3, 0), 0), ((12, 4, 4, 2, 64, 0), (0, 5), 0),
                                             ((12, 4, 4, 2, 64, 0), (0, 0), 4), ((5, 5, 2, 1, 96, 2), (96, 4), 8), ((5, 5, 3, 2, 10, 2), (1, 2), 4)])
def test_forward_strides_and_alignment(gpu, bufs, shape, pad, shift):
    run_fwd(gpu, bufs, shape, 2, pad, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 96, 10])
def test_forward_with_a_position_for_each_row(gpu, bufs, hd):
    places = [0, 1, -5, 131071, 16777216, 3, 3, 999999, 12, 65536, 2]
    run_fwd(gpu, bufs, (11, 1, 4, 2, hd, 0), 3, places=places)
    # T and pos are not read: any T does, and rows in sequence give what (row mod T) + pos gives, bit for bit
    a = run_fwd(gpu, bufs, (11, 7, 4, 2, hd, 9), 3, places=[(r % 11) + 40 for r in range(11)])
    b = run_fwd(gpu, bufs, (11, 11, 4, 2, hd, 40), 3)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    # the ends of the range leave finite rows
    L = mod("lib")
    q, k, wq, wk, _, _ = inputs(2, 1, 1, hd, 4)
    o = [bufs.raw(2 * hd * 4) for _ in range(2)]
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, 2, 1, 1, 1, hd, EPS, 1e6, 0, bufs.put(np.array([2 ** 31 - 1, -2 ** 31], np.int32)), bufs.put(q), hd,
                                               bufs.put(wq), o[0], hd, bufs.put(k), hd, bufs.put(wk), o[1], hd), "fwd")
    assert all(np.all(np.isfinite(gpu.read_state_buffer(b, 2 * hd))) for b in o)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 6])
def test_forward_in_place_and_rows_apart(gpu, bufs, hd):
    """In place; a row with a NaN, an infinity or only zeros affects no other head."""
    rows, Hq, Hkv = 9, 3, 2
    L = mod("lib")
    q, k, wq, wk, _, _ = inputs(rows, Hq, Hkv, hd, 5)
    q[2, 1, 3], q[4, 0, 0], k[5, 1, 1] = np.nan, np.inf, -np.inf
    q[7, 2], k[1, 0] = 0, 0
    bq, bk = bufs.put(q), bufs.put(k)
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, rows, rows, Hq, Hkv, hd, EPS, 1e4, 0, 0, bq, Hq * hd, bufs.put(wq), bq, Hq * hd,
                                               bk, Hkv * hd, bufs.put(wk), bk, Hkv * hd), "fwd")
    cs = angles(rows, rows, hd, 1e4, 0)
    for x, w, H, b, bad in ((q, wq, Hq, bq, [(2, 1), (4, 0)]), (k, wk, Hkv, bk, [(5, 1)])):
        got = gpu.read_state_buffer(b, rows * H * hd).reshape(rows, H, hd)
        ok = np.ones((rows, H), bool)
        for i in bad:
            ok[i] = False
            assert not np.all(np.isfinite(got[i]))
        with np.errstate(invalid="ignore"):
            want, size = ref_fwd(x, w, cs)
        assert np.all(np.abs(got - want)[ok] <= 24 * U * size[ok])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256, 6])
def test_rows_too_small_for_their_squares(gpu, bufs, hd):
    """Without an eps, rows whose mean square is a denormal: each square is off by at most 2^-150, and they are above 1e-41 on the average,
    so r is off by less than 2^-150 / 1e-41 / 2 < 4e-5 of itself."""
    L = mod("lib")
    q, k, wq, wk, _, _ = inputs(4, 2, 1, hd, 18)
    q, k = (1e-20 * q / np.sqrt((q * q).mean(axis=2, keepdims=True))).astype(np.float32), (3e-20 * k / np.sqrt((k * k).mean(axis=2, keepdims=True))).astype(np.float32)
    oq, ok = bufs.raw(q.nbytes), bufs.raw(k.nbytes)
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, 4, 4, 2, 1, hd, 0.0, 1e4, 0, 0, bufs.put(q), 2 * hd, bufs.put(wq), oq, 2 * hd, bufs.put(k), hd, bufs.put(wk), ok, hd),
            "fwd")
    cs = angles(4, 4, hd, 1e4, 0)
    for x, w, b, n in ((q, wq, oq, 2), (k, wk, ok, 1)):
        want, size = ref_fwd(x, w, cs, 0.0)
        assert np.all(np.abs(gpu.read_state_buffer(b, x.size).reshape(4, n, hd) - want) <= (4e-5 + 24 * U) * size)


def run_bwd(gpu, bufs, shape, seed, rot=(1, 1), acc=(0, 0), accw=(0, 0), want=("dq", "dwq", "dk", "dwk"), pad=(0, 0), shift=0, places=None, base=1e6,
            check=True):
    rows, T, Hq, Hkv, hd, pos = shape
    L = mod("lib")
    q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, seed)
    rs = np.random.RandomState(seed + 1)
    at = bufs.put(np.asarray(places, np.int32)) if places is not None else 0
    side, args = {}, []
    for i, (n, x, w, g, H) in enumerate((("q", q, wq, gq, Hq), ("k", k, wk, gk, Hkv))):
        dx0, dw0 = rs.standard_normal(x.shape).astype(np.float32), rs.standard_normal(hd).astype(np.float32)
        dx = bufs.put(wide(dx0, pad[0]), shift) if "d" + n in want else 0
        dw = bufs.put(dw0, shift) if "dw" + n in want else 0
        side[n] = (x, w, g, H, dx0, dw0, dx, dw, rot[i], acc[i], accw[i])
        args += [bufs.put(wide(x, pad[0]), shift), H * hd + pad[0], bufs.put(w, shift), bufs.put(wide(g, pad[1]), shift), H * hd + pad[1], rot[i], dx, acc[i],
                 dw, accw[i]]
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, rows, T, Hq, Hkv, hd, EPS, base, pos, at, *args), "bwd")
    cs = angles(rows, T, hd, base, pos, places)
    out = {}
    for n, (x, w, g, H, dx0, dw0, dx, dw, ro, ac, aw) in side.items():
        wdx, wdw, odx, odw = ref_bwd(x, w, g, cs, ro)
        if dx:
            a = gpu.read_state_buffer(dx, rows * (H * hd + pad[0])).reshape(rows, -1)
            assert np.all(a[:, H * hd:] == 7.0), "the space between the rows was written"
            a = out["d" + n] = a[:, :H * hd].reshape(rows, H, hd)
            full = wdx + (dx0 if ac else 0)
            far = np.abs(a - full) - odx - 2 * U * (np.abs(full) + ac * np.abs(dx0))
            assert not check or far.max() <= 0, f"d{n} off by {np.abs(a - full).max():.3g}, {far.max():.3g} more than the bound"
        if dw:
            a = out["dw" + n] = gpu.read_state_buffer(dw, hd)
            full = wdw + (dw0 if aw else 0)
            far = np.abs(a - full) - odw - 2 * U * (np.abs(full) + aw * np.abs(dw0))
            assert not check or far.max() <= 0, f"dw{n} off by {np.abs(a - full).max():.3g}, {far.max():.3g} more than the bound"
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("rot", [(1, 1), (0, 0)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(gpu, bufs, shape, rot):
    run_bwd(gpu, bufs, shape, 10, rot)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 96, 14])
def test_backward_flags(gpu, bufs, hd):
    shape = (22, 11, 4, 2, hd, 3)
    full = run_bwd(gpu, bufs, shape, 11)
    for rot in ((1, 0), (0, 1)):
        run_bwd(gpu, bufs, shape, 11, rot)
    for acc, accw in (((1, 0), (0, 1)), ((0, 1), (1, 0)), ((1, 1), (1, 1))):
        run_bwd(gpu, bufs, shape, 11, (1, 1), acc, accw)
    # a destination left out changes nothing of the others
    for want in (("dq",), ("dk", "dwq"), ("dwk",), ("dq", "dk"), ()):
        some = run_bwd(gpu, bufs, shape, 11, want=want)
        assert set(some) == set(want) and all(np.array_equal(some[n], full[n]) for n in want)
    run_bwd(gpu, bufs, (11, 4, 4, 2, hd, 0), 12, places=[5, 0, -1, 100000, 7, 7, 2, 1, 1000000, 3, 4])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,pad,shift", [((22, 11, 4, 2, 64, 0), (64, 8), 0), ((22, 11, 4, 2, 64, 0), (3, 5), 0), ((22, 11, 4, 2, 64, 0), (0, 0), 4),
                                             ((22, 11, 2, 1, 96, 0), (4, 0), 0), ((22, 11, 2, 2, 6, 0), (1, 3), 8)])
def test_backward_strides_and_alignment(gpu, bufs, shape, pad, shift):
    run_bwd(gpu, bufs, shape, 13, pad=pad, shift=shift, acc=(1, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(9000, 3000, 10, 2, 64, 0), (4500, 1500, 4, 2, 128, 0), (2200, 1100, 2, 1, 30, 0)], ids=str)
def test_more_rows_than_workgroups_and_the_same_bits_twice(gpu, bufs, shape):
    """A workgroup goes through several groups of rows; results do not depend on timing. The gain sums' chains are longer than the
    module's bound counts, so dw is held to sqrt-free n u: (164 + terms of a lane) u."""
    a = run_bwd(gpu, bufs, shape, 14, check=False)
    b = run_bwd(gpu, bufs, shape, 14, check=False)
    assert all(np.array_equal(a[n], b[n]) for n in a)
    rows, T, Hq, Hkv, hd, pos = shape
    q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, 14)
    cs = angles(rows, T, hd, 1e6, pos)
    for n, x, w, g, H in (("q", q, wq, gq, Hq), ("k", k, wk, gk, Hkv)):
        dx, dw, odx, odw = ref_bwd(x, w, g, cs, 1)
        assert np.all(np.abs(a["d" + n] - dx) <= odx + 2 * U * np.abs(dx))
        longer = 1 + (rows // 1024 + 1) * (Hq + Hkv) / (164 + H)       # a lane's terms: every row of its workgroup's share at most
        assert np.all(np.abs(a["dw" + n] - dw) <= odw * longer + 2 * U * np.abs(dw))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 80, 10])
def test_partial_rows_and_column_sums_give_the_same_bits(gpu, bufs, hd):
    rows, Hq, Hkv = 700, 3, 2
    shape = (rows, 350, Hq, Hkv, hd, 0)
    whole = run_bwd(gpu, bufs, shape, 15)
    L = mod("lib")
    q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, 15)
    n = C.c_int(0)
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_parts_rows(gpu.ctx, rows, Hq, Hkv, hd, C.byref(n)), "rows")
    assert n.value >= 1
    pq, pk = bufs.raw(n.value * hd * 4), bufs.raw(n.value * hd * 4)
    dq, dk, dwq, dwk = bufs.raw(q.nbytes), bufs.raw(k.nbytes), bufs.raw(hd * 4), bufs.raw(hd * 4)
    bq, bk, bwq, bwk, bgq, bgk = (bufs.put(a) for a in (q, k, wq, wk, gq, gk))
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd_parts(gpu.ctx, rows, 350, Hq, Hkv, hd, EPS, 1e6, 0, 0, bq, Hq * hd, bwq, bgq, Hq * hd, 1, dq, 0, pq,
                                                     bk, Hkv * hd, bwk, bgk, Hkv * hd, 1, dk, 0, pk), "parts")
    two = (L.buf * 2)
    L.check(gpu.ctx, L.lib.gt_colsum_group(gpu.ctx, 2, two(pq, pk), (C.c_int * 2)(n.value, n.value), (C.c_int * 2)(hd, hd), two(dwq, dwk), (C.c_int * 2)(0, 0)), "sum")
    for name, b, size in (("dq", dq, q.size), ("dk", dk, k.size), ("dwq", dwq, hd), ("dwk", dwk, hd)):
        assert np.array_equal(gpu.read_state_buffer(b, size), whole[name].reshape(-1)), name


@pytest.mark.gpu
def test_two_contexts_at_once(gpu, bufs):
    """Calls on two contexts (two streams) overlap; each has its own workspace for the gain sums. The second one's inputs are made on the
    first one's stream, which it waits for on the device."""
    L, hb = mod("lib"), mod("hip_backend")
    rows, Hq, Hkv, hd = 6000, 4, 2, 64
    q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, 19)
    ins = [bufs.put(a) for a in (q, k, wq, wk, gq, gk)]
    other = hb.HipBackend(0, streams=1)
    try:
        out = [[bufs.raw(n) for n in (q.nbytes, k.nbytes, hd * 4, hd * 4)] for _ in range(2)]
        L.check(gpu.ctx, L.lib.gt_stream_mark(gpu.ctx), "mark")
        L.check(other.ctx, L.lib.gt_stream_wait(other.ctx, gpu.ctx), "wait")
        bq, bk, bwq, bwk, bgq, bgk = ins
        for _ in range(3):
            for c, (dq, dk, dwq, dwk) in ((gpu.ctx, out[0]), (other.ctx, out[1])):
                L.check(c, L.lib.gt_qk_norm_rope_bwd(c, rows, 2000, Hq, Hkv, hd, EPS, 1e6, 0, 0, bq, Hq * hd, bwq, bgq, Hq * hd, 1, dq, 0, dwq, 0,
                                                     bk, Hkv * hd, bwk, bgk, Hkv * hd, 1, dk, 0, dwk, 0), "bwd")
        L.check(other.ctx, L.lib.gt_sync(other.ctx), "sync")
        for a, b, n in zip(*out, (q.size, k.size, hd, hd)):
            assert np.array_equal(gpu.read_state_buffer(a, n), gpu.read_state_buffer(b, n))
        cs = angles(rows, 2000, hd, 1e6, 0)
        dx, _, off, _ = ref_bwd(q, wq, gq, cs, 1)
        assert np.all(np.abs(gpu.read_state_buffer(out[1][0], q.size).reshape(rows, Hq, hd) - dx) <= off + 2 * U * np.abs(dx))
    finally:
        other.destroy()


@pytest.mark.gpu
def test_no_rows(gpu, bufs):
    L = mod("lib")
    b, d = bufs.put(np.ones(64, np.float32)), bufs.put(np.ones(64, np.float32))
    dwq, dwk = bufs.put(np.ones(64, np.float32)), bufs.put(np.ones(64, np.float32))
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, 0, 1, 1, 1, 64, EPS, 1e4, 0, 0, b, 64, b, b, 64, b, 64, b, d, 64), "fwd")
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, 0, 1, 1, 1, 64, EPS, 1e4, 0, 0, b, 64, b, b, 64, 1, b, 0, dwq, 0, b, 64, b, b, 64, 1, d, 0, dwk, 1), "bwd")
    assert np.all(gpu.read_state_buffer(b, 64) == 1) and np.all(gpu.read_state_buffer(d, 64) == 1) and np.all(gpu.read_state_buffer(dwq, 64) == 0) and np.all(gpu.read_state_buffer(dwk, 64) == 1)


@pytest.mark.gpu
def test_offsets_past_32_bits(gpu, bufs):
    """Three rows 2^30 elements apart: the last one starts past element 2^31."""
    L = mod("lib")
    hd, rows = 64, 3
    q, k, wq, wk, gq, gk = inputs(rows, 1, 1, hd, 16)
    ld = (1 << 30) + 4
    big, bk, bwq, bwk, ok = bufs.raw((2 * ld + hd) * 4), bufs.put(k), bufs.put(wq), bufs.put(wk), bufs.raw(k.nbytes)
    for r in range(rows):
        gpu.write_state_buffer(big + r * ld * 4, q[r])
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, rows, rows, 1, 1, hd, EPS, 1e4, 0, 0, big, ld, bwq, big, ld, bk, hd, bwk, ok, hd), "fwd")
    got = np.stack([gpu.read_state_buffer(big + r * ld * 4, hd) for r in range(rows)])[:, None]
    want, size = ref_fwd(q, wq, angles(rows, rows, hd, 1e4, 0))
    assert np.all(np.abs(got - want) <= 24 * U * size)
    for r in range(rows):
        gpu.write_state_buffer(big + r * ld * 4, q[r])
    # dq over gq, with q compact
    gbig = bufs.raw((2 * ld + hd) * 4)
    for r in range(rows):
        gpu.write_state_buffer(gbig + r * ld * 4, gq[r])
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, rows, rows, 1, 1, hd, EPS, 1e4, 0, 0, big, ld, bwq, gbig, ld, 1, gbig, 0, 0, 0, bk, hd, bwk, bufs.put(gk), hd,
                                               1, 0, 0, 0, 0), "bwd")
    got = np.stack([gpu.read_state_buffer(gbig + r * ld * 4, hd) for r in range(rows)])[:, None]
    dx, _, off, _ = ref_bwd(q, wq, gq, angles(rows, rows, hd, 1e4, 0), 1)
    assert np.all(np.abs(got - dx) <= off + 2 * U * np.abs(dx))


@pytest.mark.gpu
def test_more_workgroups_than_one_launch_takes(gpu, bufs):
    """A row to a workgroup and more rows than 2^22: the second launch goes on where the first ended."""
    L = mod("lib")
    Hq, hd, rows = 48, 64, (1 << 22) + 5
    ld = Hq * hd
    big, bk = bufs.raw(rows * ld * 4), bufs.raw(rows * hd * 4)
    at = [0, 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, rows - 1]
    q, k, wq, wk, _, _ = inputs(len(at), Hq, 1, hd, 17)
    for i, r in enumerate(at):
        gpu.write_state_buffer(big + r * ld * 4, q[i])
        gpu.write_state_buffer(bk + r * hd * 4, k[i])
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, rows, rows, Hq, 1, hd, EPS, 1e4, 0, 0, big, ld, bufs.put(wq), big, ld, bk, hd, bufs.put(wk), bk, hd), "fwd")
    cs = angles(len(at), 1, hd, 1e4, 0, places=at)
    for x, w, b, n in ((q, wq, big, Hq), (k, wk, bk, 1)):
        want, size = ref_fwd(x, w, cs)
        got = np.stack([gpu.read_state_buffer(b + r * n * hd * 4, n * hd).reshape(n, hd) for r in at])
        assert np.all(np.abs(got - want) <= 24 * U * size)


@pytest.mark.gpu
def test_refusals(gpu, bufs):
    L = mod("lib")
    b = bufs.put(np.ones(4096, np.float32))
    ok = dict(rows=4, T=2, Hq=2, Hkv=1, hd=8, eps=EPS, base=1e4, pos=0, places=0, q=b, ldq=16, wq=b, qo=b, ldqo=16, k=b, ldk=8, wk=b, ko=b + 1024, ldko=8)
    fwd = lambda **kw: L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, *{**ok, **kw}.values()), "fwd")  # noqa: E731
    for kw, match in ((dict(rows=-1), "bad arguments"), (dict(T=0), "bad arguments"), (dict(Hq=0), "bad arguments"), (dict(Hkv=0), "bad arguments"),
                      (dict(q=0), "bad arguments"), (dict(wk=0), "bad arguments"), (dict(hd=7), "head size 7"), (dict(hd=0), "head size 0"),
                      (dict(hd=1026, ldq=4096, ldk=4096, ldqo=4096, ldko=4096), "even number up to 1024"), (dict(base=0.0), "base must be positive"), (dict(base=float("inf")), "positive and finite"), (dict(base=float("nan")), "positive and finite"),
                      (dict(ko=b), "same buffer"), (dict(Hq=32769, ldq=1 << 20, ldqo=1 << 20), "heads are more than 32768"),
                      (dict(qo=b, ldqo=20), "strides have to be the same"),
                      (dict(T=3), "whole number of sequences"), (dict(ldq=15), "row stride"), (dict(ldko=7), "row stride"), (dict(ldk=-8), "row stride"),
                      (dict(k=b + 2), "aligned to its elements"), (dict(qo=0), "an output is missing"), (dict(ko=b + 1025), "an output is missing or not aligned"),
                      (dict(places=b + 2), "aligned to its elements")):
        with pytest.raises(L.HipError, match=match):
            fwd(**kw)
    okb = dict(rows=4, T=2, Hq=2, Hkv=1, hd=8, eps=EPS, base=1e4, pos=0, places=0, q=b, ldq=16, wq=b, gq=b, ldgq=16, rot_q=1, dq=b, acc_q=0, dwq=b, acc_wq=0,
               k=b, ldk=8, wk=b, gk=b, ldgk=8, rot_k=1, dk=b + 1024, acc_k=0, dwk=b + 256, acc_wk=0)
    bwd = lambda **kw: L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, *{**okb, **kw}.values()), "bwd")  # noqa: E731
    for kw, match in ((dict(gq=0), "a gradient is missing"), (dict(gk=b + 2), "a gradient is missing or not aligned"), (dict(dwk=b), "one and the same"), (dict(dk=b), "dq and dk are the same"),
                      (dict(ldgq=20), "strides have to be the same"),
                      (dict(ldgk=4), "row stride"), (dict(hd=9), "head size 9"), (dict(T=3), "whole number of sequences")):
        with pytest.raises(L.HipError, match=match):
            bwd(**kw)
    okp = {n: v for n, v in okb.items() if n not in ("dwq", "acc_wq", "dwk", "acc_wk")}
    names = list(okp)
    parts = lambda pq, pk, **kw: L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd_parts(  # noqa: E731
        gpu.ctx, *[{**okp, **kw}[n] for n in names[:names.index("acc_q") + 1]], pq, *[{**okp, **kw}[n] for n in names[names.index("k"):]], pk), "parts")
    for a, match in (((0, 0), "bad arguments"), ((b + 4, 0), "16-byte aligned")):
        with pytest.raises(L.HipError, match=match):
            parts(*a)
    with pytest.raises(L.HipError, match="rows 0"):
        parts(b, b, rows=0)
    assert L.lib.gt_qk_norm_rope_parts_rows(gpu.ctx, 4, 2, 1, 8, None) != 0
    gpu.sync([])                                     # nothing above was launched: the stream is fine


# ---- through the autograd surface --------------------------------------------------------------------------------------


def graph(gpu, fused, T, B, Hq, Hkv, hd, seed, attend=True, frozen=(), positions=None):
    """q, k (and v) leaves -> norm and rotation (-> attention); outputs and every leaf's gradient."""
    ag = mod("autograd")
    rs = np.random.RandomState(seed)
    n = lambda *s: rs.standard_normal(s).astype(np.float32)  # noqa: E731
    rows = B * T
    arrays = dict(q=n(rows, Hq * hd), k=n(rows, Hkv * hd), v=n(rows, Hkv * hd), wq=1 + 0.3 * n(hd), wk=1 + 0.3 * n(hd))
    up = n(rows, Hq * hd)
    ts = {m: ag.Tensor(a, list(a.shape), m not in frozen) for m, a in arrays.items()}
    gpu.install()
    try:
        if fused:
            qo, ko = ag.qk_norm_rope(ts["q"], ts["k"], ts["wq"], ts["wk"], T, Hq, Hkv, hd, EPS, 1e4, 3, positions)
        else:
            qo = ag.rope(ag.rms_norm_heads(ts["q"], ts["wq"], rows, Hq, hd, EPS), T, Hq, hd, 1e4, 3)
            ko = ag.rope(ag.rms_norm_heads(ts["k"], ts["wk"], rows, Hkv, hd, EPS), T, Hkv, hd, 1e4, 3)
        out = ag.attention(qo, ko, ts["v"], T, Hq, Hkv, hd) if attend else ag.add(qo, ag.scale(qo, 0.5))
        backward_from(gpu, ag, out, up)
        gpu.sync([out, qo, ko])
    finally:
        gpu.uninstall()
    return dict(out=out.data.copy(), qo=qo.data.copy(), ko=ko.data.copy(), **{"d" + m: t.grad.copy() for m, t in ts.items() if m not in frozen})


@pytest.mark.gpu
@pytest.mark.parametrize("T,B,Hq,Hkv,hd", [(128, 2, 4, 2, 64), (256, 1, 2, 1, 128), (37, 3, 4, 2, 64), (16, 2, 3, 1, 32), (9, 1, 2, 2, 6)])
def test_one_op_equals_the_four_calls(gpu, T, B, Hq, Hkv, hd):
    """With the rotation undone by the attention's backward (kept scores: T a multiple of 128, head sizes 64 and 128) and without. Both
    sides round each of some 60 operations differently: 1e-6 relative is sixteen half-steps on every element's root mean square."""
    a, b = (graph(gpu, f, T, B, Hq, Hkv, hd, 20) for f in (True, False))
    for n in b:
        rel = np.linalg.norm(a[n].astype(np.float64) - b[n]) / np.linalg.norm(b[n])
        assert rel <= 1e-6, (n, rel)


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hkv,hd", [(9, 2, 1, 16), (7, 2, 2, 6)])
def test_device_gradients_equal_device_differences(gpu, ref, T, Hq, Hkv, hd):
    """The recipe (and its bounds) that every op of the backend goes through, on the op with an attention behind it."""
    from test_gpu_fd import R, fd_case
    g = R(ref, 77)
    fd_case(gpu, ref, [g(T, Hq * hd), g(T, Hkv * hd), g(T, Hkv * hd), 1 + 0.3 * g(hd), 1 + 0.3 * g(hd)],
            lambda ag, q, k, v, wq, wk: ag.attention(*ag.qk_norm_rope(q, k, wq, wk, T, Hq, Hkv, hd, EPS, 1e4, 2), v, T, Hq, Hkv, hd), "qk_norm_rope")


@pytest.mark.gpu
def test_frozen_leaves_an_unused_output_and_positions(gpu):
    full = graph(gpu, True, 37, 2, 4, 2, 64, 21)
    for frozen in (("wq",), ("wk", "wq"), ("q",), ("k", "wk"), ("q", "k")):        # what is left out changes no bit of the rest
        some = graph(gpu, True, 37, 2, 4, 2, 64, 21, frozen=frozen)
        assert set(some) == set(full) - {"d" + m for m in frozen}
        assert all(np.array_equal(some[n], full[n]) for n in some), frozen
    a, b = (graph(gpu, f, 8, 2, 2, 1, 16, 22, attend=False) for f in (True, False))      # nothing reads k's output
    assert not np.any(a["dk"]) and not np.any(a["dwk"])
    for n in ("out", "dq", "dwq"):
        assert np.linalg.norm(a[n].astype(np.float64) - b[n]) <= 1e-6 * np.linalg.norm(b[n]), n
    # positions that spell out (row mod T) + 3
    c = graph(gpu, True, 8, 2, 2, 1, 16, 22, attend=False, positions=[r % 8 + 3 for r in range(16)])
    assert all(np.array_equal(a[n], c[n]) for n in a)


@pytest.mark.gpu
def test_two_consumers_keep_the_rotated_gradient(gpu):
    """A rotated q that something besides the attention reads takes its gradient rotated, whichever consumer writes first."""
    ag = mod("autograd")
    T, Hq, Hkv, hd = 128, 2, 1, 64
    got = []
    for fused in (True, False):
        rs = np.random.RandomState(23)
        n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
        q, k, v, wq, wk = n(T, Hq * hd), n(T, Hkv * hd), n(T, Hkv * hd), n(hd), n(hd)
        gpu.install()
        try:
            if fused:
                qo, ko = ag.qk_norm_rope(q, k, wq, wk, T, Hq, Hkv, hd, EPS, 1e4)
            else:
                qo = ag.rope(ag.rms_norm_heads(q, wq, T, Hq, hd, EPS), T, Hq, hd, 1e4)
                ko = ag.rope(ag.rms_norm_heads(k, wk, T, Hkv, hd, EPS), T, Hkv, hd, 1e4)
            out = ag.add(ag.attention(qo, ko, v, T, Hq, Hkv, hd), ag.scale(qo, 0.25))
            backward_from(gpu, ag, out, rs.standard_normal(out.size))
            gpu.sync([])
        finally:
            gpu.uninstall()
        got.append([t.grad.copy() for t in (q, k, v, wq, wk)])
    for a, b in zip(*got):
        assert np.linalg.norm(a.astype(np.float64) - b) <= 1e-6 * np.linalg.norm(b)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [128, 40])
def test_two_backwards_over_one_graph(gpu, T):
    """Gradients of intermediates accumulate over backward passes, as the four calls' do: with the rotation undone by the attention (T = 128)
    and by the op itself."""
    ag = mod("autograd")
    Hq, Hkv, hd = 2, 1, 64
    got = []
    for fused in (True, False):
        rs = np.random.RandomState(24)
        n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
        q, k, v, wq, wk = n(T, Hq * hd), n(T, Hkv * hd), n(T, Hkv * hd), n(hd), n(hd)
        up = rs.standard_normal(T * Hq * hd)
        gpu.install()
        try:
            if fused:
                qo, ko = ag.qk_norm_rope(q, k, wq, wk, T, Hq, Hkv, hd, EPS, 1e4)
            else:
                qn, kn = ag.rms_norm_heads(q, wq, T, Hq, hd, EPS), ag.rms_norm_heads(k, wk, T, Hkv, hd, EPS)
                # scaled by one: a consumer between the rotation and the attention keeps its backward a launch of its own
                qo, ko = ag.scale(ag.rope(qn, T, Hq, hd, 1e4), 1.0), ag.scale(ag.rope(kn, T, Hkv, hd, 1e4), 1.0)
            out = ag.attention(qo, ko, v, T, Hq, Hkv, hd)
            backward_from(gpu, ag, out, up)
            first = [gpu.read_state_buffer(gpu.buffers_for(t)["grad"], t.size).copy() for t in (q, k, wq, wk)]
            gpu.sync([])
        finally:
            gpu.uninstall()
        got.append(first + [t.grad.copy() for t in (q, k, v, wq, wk)])
    for a, b in zip(*got):
        assert np.linalg.norm(a.astype(np.float64) - b) <= 1e-6 * np.linalg.norm(b)
    # the same graph differentiated twice: every leaf's gradient is its first one three times over, intermediates having added up,
    # but v's, which only the attention itself writes, twice
    rs = np.random.RandomState(24)
    n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
    q, k, v, wq, wk = n(T, Hq * hd), n(T, Hkv * hd), n(T, Hkv * hd), n(hd), n(hd)
    up = rs.standard_normal(T * Hq * hd)
    gpu.install()
    try:
        qo, ko = ag.qk_norm_rope(q, k, wq, wk, T, Hq, Hkv, hd, EPS, 1e4)
        out = ag.attention(qo, ko, v, T, Hq, Hkv, hd)
        for _ in range(2):
            backward_from(gpu, ag, out, up)
        gpu.sync([])
    finally:
        gpu.uninstall()
    for t, once, times in ((q, got[0][4], 3), (k, got[0][5], 3), (v, got[0][6], 2), (wq, got[0][7], 3), (wk, got[0][8], 3)):
        assert np.linalg.norm(t.grad.astype(np.float64) - times * once.astype(np.float64)) <= 1e-6 * times * np.linalg.norm(once)


@pytest.mark.gpu
@pytest.mark.parametrize("name,T", [("qwen3", 21), ("gemma3", 21), ("gemma3-window", 128), ("qwen3-hd128", 128)])
@pytest.mark.parametrize("recompute", [False, True])
def test_models_call_it(gpu, ref, name, T, recompute):
    """With fuse_qk_norm_rope the model graphs with QK-norm launch the op once per layer each way (once more forward where layers are
    recomputed) and no separate head norm or rotation; stacked and one sequence at a time on four streams; loss and gradients
    are the oracle's to the suite's parity bound."""
    from test_gpu_model import REAL, SMALL, batches, build_pair, compare, hip_step, ref_step
    kw = SMALL[name] if name in SMALL else dict(REAL[name], layers=2)
    rmodel, model = build_pair(ref, kw, seed=3, std=0.05)
    seqs = batches(ref, kw["vocab"], T, 3, seed=4, mask_every=7)
    ref.set_threads(min(16, ref.max_threads()))
    try:
        lr, gr = ref_step(ref, rmodel, seqs)
    finally:
        ref.set_threads(1)
    gpu.fuse_qk_norm_rope = True
    try:
        for stacked in (True, False):
            gpu.start_profile()
            loss, grads = hip_step(gpu, model, seqs, stacked, T, recompute=recompute)
            prof = gpu.stop_profile()
            n = kw["layers"] * (1 if stacked else 3)
            assert prof["qknorm.rope"][1] == n * (2 if recompute else 1) and prof["qknorm.rope.bwd"][1] == n
            assert not any(label.startswith("rope") for label in prof), sorted(prof)
            compare(loss, grads, lr, gr, f"{name}, fused QK-norm, stacked {stacked}")
    finally:
        gpu.fuse_qk_norm_rope = False
