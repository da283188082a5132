"""QK-norm with rotation where the numbers or the arguments reach their limits: rows whose squares overflow, rows too small for the cube of their
reciprocal root, calls that the library has to refuse or to take. The bounds are those derived in test_gpu_qk_norm_rope.py."""
import numpy as np
import pytest

from gpu_common import mod
from test_gpu_qk_norm_rope import EPS, U, angles, bufs, inputs, ref_bwd, ref_fwd, wide  # noqa: F401

# heads of every lane count of the vector kernels, and what takes the generic ones: an odd number of chunks, too long, misaligned
HEADS = [(16, 0), (64, 0), (128, 0), (256, 0), (512, 0), (6, 0), (514, 0), (64, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,shift", HEADS, ids=str)
def test_rows_whose_squares_overflow(gpu, bufs, hd, shift):  # noqa: F811
    """A mean square past FP32 has the reciprocal root zero: a head of zeros and no gradient, as from the norm by itself, and every
    other head as without it. One head has squares that overflow by themselves, another only their sum."""
    L = mod("lib")
    rows, Hq, Hkv = 5, 2, 3
    q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, 61)
    big = 1e20 * np.sign(q[1, 0])
    lots = np.full(hd, 1.7e19, np.float32)
    q[1, 0], k[3, 2], q[4, 1] = big, -big, lots
    bad = dict(q=[(1, 0), (4, 1)], k=[(3, 2)])
    put = lambda a: bufs.put(a, shift)  # noqa: E731
    bq, bk, bwq, bwk, bgq, bgk = (put(a) for a in (q, k, wq, wk, gq, gk))
    oq, ok, dq, dk, dwq, dwk = (put(np.full_like(a, 7.0)) for a in (q, k, q, k, wq, wk))
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, rows, rows, Hq, Hkv, hd, EPS, 1e4, 0, 0, bq, Hq * hd, bwq, oq, Hq * hd, bk, Hkv * hd, bwk, ok, Hkv * hd), "fwd")
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, rows, rows, Hq, Hkv, hd, EPS, 1e4, 0, 0, bq, Hq * hd, bwq, bgq, Hq * hd, 1, dq, 0, dwq, 0,
                                               bk, Hkv * hd, bwk, bgk, Hkv * hd, 1, dk, 0, dwk, 0), "bwd")
    # the norm alone, on the same rows
    nq, rinv = bufs.raw(q.nbytes), bufs.raw(rows * Hq * 4)
    L.check(gpu.ctx, L.lib.gt_rmsnorm_fwd(gpu.ctx, rows * Hq, hd, EPS, bq, bwq, nq, rinv), "norm")
    alone = gpu.read_state_buffer(nq, q.size).reshape(q.shape)
    cs = angles(rows, rows, hd, 1e4, 0)
    for name, x, w, g, o, d, dw in (("q", q, wq, gq, oq, dq, dwq), ("k", k, wk, gk, ok, dk, dwk)):
        fine = np.ones(x.shape[:2], bool)
        for i in bad[name]:
            fine[i] = False
        got, gd, gw = (gpu.read_state_buffer(b, n.size).reshape(n.shape) for b, n in ((o, x), (d, x), (dw, w)))
        assert not np.any(got[~fine]) and not np.any(gd[~fine]), name
        x0 = np.where(fine[:, :, None], x, 0)                       # a head of zeros adds nothing to the gain's sums either
        want, size = ref_fwd(x0, w, cs)
        dx, sums, odx, osum = ref_bwd(x0, w, g, cs, True)
        assert np.all((np.abs(got - want) <= 24 * U * size)[fine]) and np.all((np.abs(gd - dx) <= odx)[fine]), name
        assert np.all(np.abs(gw - sums) <= osum + 2 * U * np.abs(sums)), name
    assert all(not np.any(alone[i]) for i in bad["q"])


@pytest.mark.gpu
@pytest.mark.parametrize("acc", [0, 1])
@pytest.mark.parametrize("hd,shift", HEADS, ids=str)
def test_backward_of_rows_too_small_for_the_cube_of_their_root(gpu, bufs, hd, shift, acc):  # noqa: F811
    """Without an eps, rows whose root mean square is 1e-20 and 3e-20: r is up to 1e20 and its cube past FP32, the gradient is not. Each square is off by
    at most 2^-150, and they are above 1e-41 on the average, so r is off by less than d = 4e-5 of itself, w g r by d more than the bound on its
    roundings and x r^3 S by three times that, the gain's terms by d."""
    L = mod("lib")
    rows, d = 4, 4e-5
    q, k, wq, wk, gq, gk = inputs(rows, 2, 1, hd, 62)
    q, k = (1e-20 * q / np.sqrt((q * q).mean(axis=2, keepdims=True))).astype(np.float32), (3e-20 * k / np.sqrt((k * k).mean(axis=2, keepdims=True))).astype(np.float32)
    put = lambda a: bufs.put(a, shift)  # noqa: E731
    old = [np.full(a.shape, 1e18, np.float32) for a in (q, k)]
    dq, dk, dwq, dwk = put(old[0]), put(old[1]), put(np.zeros(hd, np.float32)), put(np.zeros(hd, np.float32))
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, rows, rows, 2, 1, hd, 0.0, 1e4, 0, 0, put(q), 2 * hd, put(wq), put(gq), 2 * hd, 1, dq, acc, dwq, 0,
                                               put(k), hd, put(wk), put(gk), hd, 1, dk, acc, dwk, 0), "bwd")
    cs = angles(rows, rows, hd, 1e4, 0)
    for x, w, g, o, b, bw in ((q, wq, gq, old[0], dq, dwq), (k, wk, gk, old[1], dk, dwk)):
        dx, dw, off, offw = ref_bwd(x, w, g, cs, True, 0.0)
        x64 = x.astype(np.float64)
        r = 1 / np.sqrt((x64 * x64).mean(axis=2, keepdims=True))
        h = hd // 2
        size = np.tile(np.abs(g[..., :h].astype(np.float64)) + np.abs(g[..., h:]), 2)
        off = off + d * np.abs(w) * size * r + 3.01 * d * np.abs(x64) * r ** 3 * (size * np.abs(w * x64)).sum(axis=2, keepdims=True) / hd
        want = dx + (o if acc else 0)
        got = gpu.read_state_buffer(b, x.size).reshape(x.shape)
        assert np.all(np.isfinite(got)) and np.all(np.abs(got - want) <= off + 2 * U * (np.abs(want) + acc * np.abs(o)))
        got = gpu.read_state_buffer(bw, hd)
        assert np.all(np.abs(got - dw) <= offw + d * (size * np.abs(x64) * r).sum(axis=(0, 1)) + 2 * U * np.abs(dw))


# ---- which buffers may share memory -----------------------------------------------------------------------------------


def forward_args(rows, Hq, Hkv, hd, **kw):
    a = dict(rows=rows, T=rows, Hq=Hq, Hkv=Hkv, hd=hd, eps=EPS, base=1e4, pos=0, places=0, q=0, ldq=Hq * hd, wq=0, qo=0, ldqo=Hq * hd, k=0, ldk=Hkv * hd, wk=0, ko=0,
             ldko=Hkv * hd)
    return {**a, **kw}


def backward_args(rows, Hq, Hkv, hd, **kw):
    a = dict(rows=rows, T=rows, Hq=Hq, Hkv=Hkv, hd=hd, eps=EPS, base=1e4, pos=0, places=0, q=0, ldq=Hq * hd, wq=0, gq=0, ldgq=Hq * hd, rot_q=1, dq=0, acc_q=0, dwq=0,
             acc_wq=0, k=0, ldk=Hkv * hd, wk=0, gk=0, ldgk=Hkv * hd, rot_k=1, dk=0, acc_k=0, dwk=0, acc_wk=0)
    return {**a, **kw}


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 6])
def test_overlapping_buffers_are_refused(gpu, bufs, hd):  # noqa: F811
    """What would let one workgroup write what another has still to read. Nothing is launched."""
    L = mod("lib")
    rows, Hq, Hkv = 40, 4, 2
    nq, nk = rows * Hq * hd * 4, rows * Hkv * hd * 4
    fill = lambda n: bufs.put(np.ones(n // 4, np.float32))  # noqa: E731
    b = {m: fill(n) for m, n in dict(q=nq, k=nk, gq=nq, gk=nk, qo=nq, ko=nk, dq=nq, dk=nk).items()}
    b.update({m: fill(4 * hd) for m in ("wq", "wk", "dwq", "dwk")})
    at = bufs.put(np.zeros(rows, np.int32))
    parts = [bufs.raw(1 << 22) for _ in range(2)]
    pick = lambda *names: {m: b[m] for m in names}  # noqa: E731
    okf = forward_args(rows, Hq, Hkv, hd, places=at, **pick("q", "k", "wq", "wk", "qo", "ko"))
    okb = backward_args(rows, Hq, Hkv, hd, places=at, **pick("q", "k", "wq", "wk", "gq", "gk", "dq", "dk", "dwq", "dwk"))
    fwd = lambda **kw: L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, *{**okf, **kw}.values()), "fwd")  # noqa: E731
    bwd = lambda **kw: L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, *{**okb, **kw}.values()), "bwd")  # noqa: E731

    def leave(pq, pk, **kw):
        a = {n: v for n, v in {**okb, **kw}.items() if n not in ("dwq", "acc_wq", "dwk", "acc_wk")}
        names = list(a)
        i = names.index("acc_q") + 1
        L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd_parts(gpu.ctx, *[a[n] for n in names[:i]], pq, *[a[n] for n in names[i:]], pk), "parts")
    fwd()
    bwd()
    leave(*parts)
    gpu.sync([])
    before = {m: gpu.read_state_buffer(x, hd) for m, x in b.items()}
    row, head = Hkv * hd * 4, hd * 4
    for kw in (dict(qo=b["k"]), dict(ko=b["q"]), dict(ko=b["q"] + nq - 4), dict(qo=b["q"] + 4), dict(qo=b["q"] + head), dict(ko=b["k"] + row), dict(qo=b["ko"] + nk - 4),
               dict(ko=b["qo"] + 4 * Hq * hd), dict(qo=b["wq"]), dict(ko=b["wq"] - nk + 4), dict(qo=b["wk"]), dict(qo=at), dict(ko=at + 4 * rows - 4),
               dict(ko=b["k"], q=b["k"], ldq=Hq * hd)):
        with pytest.raises(L.HipError, match="overlap"):
            fwd(**kw)
    for kw in (dict(dq=b["gk"]), dict(dk=b["gq"]), dict(dq=b["k"]), dict(dk=b["q"]), dict(dq=b["q"] + 4), dict(dq=b["gq"] + head), dict(dk=b["dq"] + 4),
               dict(dq=b["dk"] + nk - 4), dict(dk=b["wk"]), dict(dk=b["wq"]), dict(dq=b["wk"] - nq + 4), dict(dq=at), dict(dwq=b["dq"]), dict(dwk=b["dq"] + 8),
               dict(dwq=b["dk"] + nk - 4), dict(dwk=b["dwq"] + 4), dict(dq=b["gq"], gk=b["gq"]), dict(dq=b["q"], k=b["q"])):
        with pytest.raises(L.HipError, match="overlap"):
            bwd(**kw)
    for a in ((parts[0], parts[0]), (parts[0], parts[0] + 16), (b["q"], 0), (b["k"], 0), (0, b["gq"]), (b["gk"], 0), (0, b["dq"]), (b["dk"], 0), (b["wq"], 0), (0, b["wk"]), (at, 0)):
        if all(x % 16 == 0 for x in a):
            with pytest.raises(L.HipError, match="overlap"):
                leave(*a)
    # rows that interleave at different strides
    with pytest.raises(L.HipError, match="overlap"):
        fwd(rows=8, T=8, places=0, qo=b["q"] + 4 * Hq * hd, ldqo=3 * Hq * hd, ldq=2 * Hq * hd)
    gpu.sync([])
    assert all(np.array_equal(gpu.read_state_buffer(x, hd), before[m]) for m, x in b.items())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 6])
def test_slices_of_one_product_and_rows_in_place(gpu, bufs, hd):  # noqa: F811
    """q and k, their rotated rows, gradients and results each as slices of one wider row; over their inputs; one row, whose stride is of no account."""
    L = mod("lib")
    for rows, Hq, Hkv in ((13, 4, 2), (1, 4, 2)):
        q, k, wq, wk, gq, gk = inputs(rows, Hq, Hkv, hd, 63)
        ld, step = (Hq + Hkv) * hd + 4, 4 * Hq * hd
        pair = lambda a, b_: np.concatenate([a.reshape(rows, -1), b_.reshape(rows, -1), np.full((rows, 4), 7.0, np.float32)], axis=1).astype(np.float32)  # noqa: E731
        x, g, o, d = (bufs.put(a) for a in (pair(q, k), pair(gq, gk), pair(0 * q, 0 * k), pair(0 * q, 0 * k)))
        bwq, bwk, dwq, dwk = (bufs.put(a) for a in (wq, wk, wq, wk))
        cs = angles(rows, rows, hd, 1e4, 0)
        wants = [ref_fwd(a, w, cs) for a, w in ((q, wq), (k, wk))]
        grads = [ref_bwd(a, w, h, cs, True) for a, w, h in ((q, wq, gq), (k, wk, gk))]

        def read(buf):
            a = gpu.read_state_buffer(buf, rows * ld).reshape(rows, ld)
            assert np.all(a[:, -4:] == 7.0)
            return a[:, :Hq * hd].reshape(q.shape), a[:, Hq * hd:-4].reshape(k.shape)

        def check_fwd(buf):
            for got, (want, size) in zip(read(buf), wants):
                assert np.all(np.abs(got - want) <= 24 * U * size)

        def check_bwd(buf):
            for got, (dx, dw, off, offw), b_ in zip(read(buf), grads, (dwq, dwk)):
                assert np.all(np.abs(got - dx) <= off + 2 * U * np.abs(dx))
                assert np.all(np.abs(gpu.read_state_buffer(b_, hd) - dw) <= offw + 2 * U * np.abs(dw))

        def fwd(out):
            a = forward_args(rows, Hq, Hkv, hd, q=x, ldq=ld, wq=bwq, qo=out, ldqo=ld, k=x + step, ldk=ld, wk=bwk, ko=out + step, ldko=ld)
            L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, *a.values()), "fwd")

        def bwd(out, up):
            a = backward_args(rows, Hq, Hkv, hd, q=x, ldq=ld, wq=bwq, gq=up, ldgq=ld, dq=out, dwq=dwq, k=x + step, ldk=ld, wk=bwk, gk=up + step, ldgk=ld, dk=out + step, dwk=dwk)
            L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, *a.values()), "bwd")
        fwd(o)
        check_fwd(o)
        bwd(d, g)
        check_bwd(d)
        over = bufs.put(pair(gq, gk))
        bwd(over, over)                                  # over the gradients
        check_bwd(over)
        bwd(x, g)                                        # over the rows themselves
        check_bwd(x)
        gpu.write_state_buffer(x, pair(q, k))
        fwd(x)
        check_fwd(x)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0, -3])
def test_with_positions_the_sequence_length_is_not_read(gpu, bufs, T):  # noqa: F811
    L = mod("lib")
    rows, hd = 5, 64
    q, k, wq, wk, gq, gk = inputs(rows, 2, 1, hd, 64)
    at = [3, 0, 70000, 3, 12]
    b = dict(q=bufs.put(q), k=bufs.put(k), wq=bufs.put(wq), wk=bufs.put(wk), places=bufs.put(np.array(at, np.int32)))
    o, d = [bufs.raw(a.nbytes) for a in (q, k)], [bufs.raw(a.nbytes) for a in (q, k, wq, wk)]
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_fwd(gpu.ctx, *forward_args(rows, 2, 1, hd, **{**b, "T": T}, qo=o[0], ko=o[1]).values()), "fwd")
    L.check(gpu.ctx, L.lib.gt_qk_norm_rope_bwd(gpu.ctx, *backward_args(rows, 2, 1, hd, **{**b, "T": T}, gq=bufs.put(gq), gk=bufs.put(gk), dq=d[0], dk=d[1], dwq=d[2], dwk=d[3]).values()), "bwd")
    cs = angles(rows, 1, hd, 1e4, 0, at)
    for x, w, g, out, dx_, dw_ in ((q, wq, gq, o[0], d[0], d[2]), (k, wk, gk, o[1], d[1], d[3])):
        want, size = ref_fwd(x, w, cs)
        dx, dw, off, offw = ref_bwd(x, w, g, cs, True)
        assert np.all(np.abs(gpu.read_state_buffer(out, x.size).reshape(x.shape) - want) <= 24 * U * size)
        assert np.all(np.abs(gpu.read_state_buffer(dx_, x.size).reshape(x.shape) - dx) <= off + 2 * U * np.abs(dx))
        assert np.all(np.abs(gpu.read_state_buffer(dw_, hd) - dw) <= offw + 2 * U * np.abs(dw))
