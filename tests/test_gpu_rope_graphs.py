"""Graphs around a rotation whose backward the attention takes over (fuse_rope_bwd), differentiated more than once: every leaf's gradient is what
the rotation's own launch gives. Gradients of intermediates add up over backward passes until a sync, on both sides alike; the sides differ by six
roundings an element: 1e-6 relative is sixteen half-steps on every element's root mean square."""
import numpy as np
import pytest

from gpu_common import backward_from, mod

BASE = 1e4
T, HD, H = 128, 64, 2


def both(gpu, body, seed):
    """body(ag, random state, leaves, rotated q, rotated k) with and without fuse_rope_bwd; the leaves' gradients are compared."""
    ag = mod("autograd")
    got = []
    for fuse in (True, False):
        rs = np.random.RandomState(seed)
        n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
        t = dict(x=n(T, 32), Wq=n(H * HD, 32), Wk=n(H * HD, 32), v=n(T, H * HD))
        gpu.install()
        gpu.fuse_rope_bwd = fuse
        try:
            q, k = ag.linear(t["x"], t["Wq"]), ag.linear(t["x"], t["Wk"])
            body(ag, rs, t, ag.rope(q, T, H, HD, BASE), ag.rope(k, T, H, HD, BASE), q, k)
            gpu.sync([])
        finally:
            gpu.fuse_rope_bwd = True
            gpu.uninstall()
        got.append({m: x.grad.astype(np.float64) for m, x in t.items()})
    for m in got[0]:
        off, norm = np.linalg.norm(got[0][m] - got[1][m]), np.linalg.norm(got[1][m])
        assert off <= 1e-6 * norm, (m, off / norm)


LATER = {
    "attention": lambda ag, q, k, v: ag.attention(q, k, v, T, H, H, HD),
    "scales": lambda ag, q, k, v: ag.add(ag.scale(q, 0.25), ag.scale(k, 0.5)),
    "product": lambda ag, q, k, v: ag.mul(q, k),
    "one": lambda ag, q, k, v: ag.scale(q, 0.25),
}


@pytest.mark.gpu
@pytest.mark.parametrize("later", list(LATER))
def test_a_consumer_recorded_after_a_backward(gpu, later):
    def body(ag, rs, t, q, k, *_):
        backward_from(gpu, ag, ag.attention(q, k, t["v"], T, H, H, HD), rs.standard_normal(T * H * HD))
        out = LATER[later](ag, q, k, t["v"])
        for _ in range(2):
            backward_from(gpu, ag, out, rs.standard_normal(out.size))
    both(gpu, body, 51)


@pytest.mark.gpu
def test_one_graph_three_times(gpu):
    def body(ag, rs, t, q, k, *_):
        out = ag.attention(q, k, t["v"], T, H, H, HD)
        for _ in range(3):
            backward_from(gpu, ag, out, rs.standard_normal(T * H * HD))
    both(gpu, body, 52)


@pytest.mark.gpu
def test_a_seed_after_a_backward(gpu):
    """A backward that starts at the rotation's output, from a gradient written by the host."""
    def body(ag, rs, t, q, k, *_):
        backward_from(gpu, ag, ag.attention(q, k, t["v"], T, H, H, HD), rs.standard_normal(T * H * HD))
        for x in (q, k):
            backward_from(gpu, ag, x, rs.standard_normal(T * H * HD))
    both(gpu, body, 53)


@pytest.mark.gpu
@pytest.mark.parametrize("when", ["before", "after"])
def test_another_reader_of_the_rows_before_the_rotation(gpu, when):
    """Their gradient is then more than what the attention gave it."""
    def body(ag, rs, t, q, k, q0, k0):
        other = lambda: ag.add(ag.scale(q0, 0.25), ag.scale(k0, 0.5))  # noqa: E731
        early = other() if when == "before" else None
        backward_from(gpu, ag, ag.attention(q, k, t["v"], T, H, H, HD), rs.standard_normal(T * H * HD))
        for _ in range(2):
            out = ag.add(ag.mul(q, k), early or other())
            backward_from(gpu, ag, out, rs.standard_normal(out.size))
    both(gpu, body, 54)


@pytest.mark.gpu
def test_leaves_as_rows_before_the_rotation(gpu):
    """q and k are leaves, whose gradients outlive the graph."""
    ag = mod("autograd")
    got = []
    for fuse in (True, False):
        rs = np.random.RandomState(55)
        n = lambda: ag.Tensor(rs.standard_normal((T, H * HD)).astype(np.float32), [T, H * HD], True)  # noqa: E731
        q, k, v = n(), n(), n()
        gpu.install()
        gpu.fuse_rope_bwd = fuse
        try:
            a, b = ag.rope(q, T, H, HD, BASE), ag.rope(k, T, H, HD, BASE)
            backward_from(gpu, ag, ag.attention(a, b, v, T, H, H, HD), rs.standard_normal(T * H * HD))
            backward_from(gpu, ag, ag.mul(a, b), rs.standard_normal(T * H * HD))
            gpu.sync([])
        finally:
            gpu.fuse_rope_bwd = True
            gpu.uninstall()
        got.append([x.grad.astype(np.float64) for x in (q, k, v)])
    for a, b in zip(*got):
        assert np.linalg.norm(a - b) <= 1e-6 * np.linalg.norm(b)


@pytest.mark.gpu
def test_an_output_that_is_gone_needs_no_gradient(gpu):
    """The rows before the rotation are kept over a reclaim, the rotation's output is not; what adds to their gradient afterwards adds to
    what the attention left there."""
    def body(ag, rs, t, q, k, q0, k0):
        backward_from(gpu, ag, ag.attention(q, k, t["v"], T, H, H, HD), rs.standard_normal(T * H * HD))
        gpu.reclaim_step_transients([q0, k0])
        out = ag.add(ag.scale(q0, 0.25), ag.scale(k0, 0.5))
        backward_from(gpu, ag, out, rs.standard_normal(out.size))
    both(gpu, body, 56)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["both", "q", "twice"])
def test_a_sum_recorded_after_a_backward(gpu, which):
    """An add hands its upstream gradient on by address where nobody has written one yet."""
    def body(ag, rs, t, q, k, *_):
        backward_from(gpu, ag, ag.attention(q, k, t["v"], T, H, H, HD), rs.standard_normal(T * H * HD))
        out = ag.add(q, {"both": k, "q": t["v"], "twice": q}[which])
        backward_from(gpu, ag, ag.scale(out, 0.5), rs.standard_normal(out.size))
    both(gpu, body, 57)
