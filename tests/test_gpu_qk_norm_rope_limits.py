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
