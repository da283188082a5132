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
