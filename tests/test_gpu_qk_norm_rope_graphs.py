"""Graphs around QK-norm with rotation that are differentiated more than once or in parts. Whether the attention's backward undoes the rotation
in its write-backs (fuse_rope_bwd) or the op does it itself changes no gradient but by rounding.

Gradients of intermediates add up over backward passes until a sync, so a second pass hands on the first one's share again: that is the same on both
sides. The sides differ by the rotation of a gradient, undone in one place or another and at most turned back once between, six roundings an element:
1e-6 relative is sixteen half-steps on every element's root mean square."""
import numpy as np
import pytest

from gpu_common import backward_from, mod

EPS, BASE = 1e-6, 1e4
T, HD = 128, 64                                     # the attention keeps its scores and undoes the rotation itself


def leaves(seed, Hq, Hkv):
    ag = mod("autograd")
    rs = np.random.RandomState(seed)
    n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
    return rs, dict(q=n(T, Hq * HD), k=n(T, Hkv * HD), v=n(T, Hkv * HD), wq=n(HD), wk=n(HD))


def rotated(ag, t, Hq, Hkv):
    return ag.qk_norm_rope(t["q"], t["k"], t["wq"], t["wk"], T, Hq, Hkv, HD, EPS, BASE)


def both(gpu, body, seed, Hq=2, Hkv=2):
    """body(ag, random state, leaves, qo, ko) with the rotation undone by the attention and by the op; the leaves' gradients are compared."""
    ag = mod("autograd")
    got = []
    for fused in (True, False):
        rs, t = leaves(seed, Hq, Hkv)
        gpu.install()
        gpu.fuse_rope_bwd = fused
        try:
            body(ag, rs, t, *rotated(ag, t, Hq, Hkv))
            gpu.sync([])
        finally:
            gpu.fuse_rope_bwd = True
            gpu.uninstall()
        got.append({m: x.grad.astype(np.float64) for m, x in t.items()})
    for m in got[0]:
        norm = np.linalg.norm(got[1][m])
        assert np.linalg.norm(got[0][m] - got[1][m]) <= 1e-6 * norm, (m, np.linalg.norm(got[0][m] - got[1][m]) / norm)


LATER = {
    "attention": lambda ag, qo, ko, v: ag.attention(qo, ko, v, T, 2, 2, HD),
    "scales": lambda ag, qo, ko, v: ag.add(ag.scale(qo, 0.25), ag.scale(ko, 0.5)),
    "add": lambda ag, qo, ko, v: ag.add(qo, ko),
    "product": lambda ag, qo, ko, v: ag.mul(qo, ko),
}


@pytest.mark.gpu
@pytest.mark.parametrize("later", list(LATER))
def test_a_consumer_recorded_after_a_backward(gpu, later):
    """The first backward leaves the gradients of the rows before the rotation; what is recorded afterwards adds those of the rotated rows."""
    def body(ag, rs, t, qo, ko):
        backward_from(gpu, ag, ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD))
        out = LATER[later](ag, qo, ko, t["v"])
        for _ in range(2):
            backward_from(gpu, ag, out, rs.standard_normal(out.size))
    both(gpu, body, 31)


@pytest.mark.gpu
def test_the_switch_turned_between_two_backwards(gpu):
    def body(ag, rs, t, qo, ko):
        out, up = ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD)
        backward_from(gpu, ag, out, up)
        gpu.fuse_rope_bwd = False
        backward_from(gpu, ag, out, up)
    both(gpu, body, 32)


@pytest.mark.gpu
def test_a_seed_replaces_what_a_backward_left(gpu):
    """A gradient written from the host is of the rotated rows."""
    def body(ag, rs, t, qo, ko):
        backward_from(gpu, ag, ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD))
        up = [rs.standard_normal(x.size) for x in (qo, ko)]
        out = ag.add(ag.scale(qo, 0.5), ag.scale(ko, 0.5))
        for x, u in zip((qo, ko), up):
            x.grad[:] = u.astype(np.float32)
            gpu.seed_grad_from_host(x)
        backward_from(gpu, ag, out, rs.standard_normal(out.size))
    both(gpu, body, 33)


@pytest.mark.gpu
def test_a_recomputed_block_that_ends_in_the_rotation(gpu):
    """checkpoint hands its output's gradient to the block's replay, whose own rotation is still to be undone."""
    def body(ag, rs, t, *_):
        ag.set_checkpointing(True)
        try:
            ins = [t[m] for m in ("q", "k", "wq", "wk")]
            qo, ko = (ag.checkpoint(ins, lambda i=i: rotated(ag, t, 2, 2)[i]) for i in (0, 1))
            backward_from(gpu, ag, ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD))
        finally:
            ag.set_checkpointing(False)
    both(gpu, body, 34)


@pytest.mark.gpu
def test_the_gradient_buffer_of_an_output_is_of_the_rotated_rows(gpu):
    ag = mod("autograd")
    got = []
    for fused in (True, False):
        rs, t = leaves(35, 2, 2)
        gpu.install()
        gpu.fuse_rope_bwd = fused
        try:
            qo, ko = rotated(ag, t, 2, 2)
            backward_from(gpu, ag, ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD))
            got.append([gpu.read_state_buffer(gpu.buffers_for(x)["grad"], x.size).astype(np.float64) for x in (qo, ko)])
            gpu.sync([])
        finally:
            gpu.fuse_rope_bwd = True
            gpu.uninstall()
    for a, b in zip(*got):
        assert np.linalg.norm(a - b) <= 1e-6 * np.linalg.norm(b)


# ---- backwards that come through one of the two outputs ------------------------------------------------------------------


def chain(ag, rs, Hq, Hkv):
    """q and k as products, so that what lies above them shows who was called again."""
    n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
    t = dict(x=n(T, 32), Wq=n(Hq * HD, 32), Wk=n(Hkv * HD, 32), wq=n(HD), wk=n(HD))
    qo, ko = ag.qk_norm_rope(ag.linear(t["x"], t["Wq"]), ag.linear(t["x"], t["Wk"]), t["wq"], t["wk"], T, Hq, Hkv, HD, EPS, BASE)
    return t, qo, ko


def through(gpu, seed, walks, Hq=2, Hkv=1):
    """Gradients of the leaves after backwards through the named outputs ("q", "k"), each with an upstream gradient of its own."""
    ag = mod("autograd")
    rs = np.random.RandomState(seed)
    ups = dict(q=rs.standard_normal(T * Hq * HD), k=rs.standard_normal(T * Hkv * HD))
    gpu.install()
    try:
        t, qo, ko = chain(ag, rs, Hq, Hkv)
        out = dict(q=ag.scale(qo, 1.0), k=ag.scale(ko, 1.0))
        for w in walks:
            backward_from(gpu, ag, out[w], ups[w])
        gpu.sync([])
    finally:
        gpu.uninstall()
    return {m: x.grad.astype(np.float64) for m, x in t.items()}


@pytest.mark.gpu
def test_a_backward_through_one_output_leaves_the_other_side_alone(gpu):
    """Each side is what it is by itself, bit for bit where one product makes it up; x, which both sides add to, is the sum of the two."""
    q, k, qk, kq = (through(gpu, 41, w) for w in ("q", "k", "qk", "kq"))
    for m in ("Wq", "wq"):
        assert np.any(q[m]) and not np.any(k[m]) and np.array_equal(qk[m], q[m]) and np.array_equal(kq[m], q[m]), m
    for m in ("Wk", "wk"):
        assert np.any(k[m]) and not np.any(q[m]) and np.array_equal(qk[m], k[m]) and np.array_equal(kq[m], k[m]), m
    for g in (qk, kq):
        assert np.linalg.norm(g["x"] - (q["x"] + k["x"])) <= 1e-6 * np.linalg.norm(g["x"])


@pytest.mark.gpu
def test_a_backward_through_one_output_after_one_through_both(gpu):
    """The attention's gradients lie in both outputs; the second backward reaches q's alone, and k's side keeps what the first one gave it."""
    ag = mod("autograd")
    rs, t = leaves(42, 2, 2)
    gpu.install()
    try:
        qo, ko = rotated(ag, t, 2, 2)
        backward_from(gpu, ag, ag.attention(qo, ko, t["v"], T, 2, 2, HD), rs.standard_normal(T * 2 * HD))
        first = {m: gpu.read_state_buffer(gpu.buffers_for(t[m])["grad"], t[m].size) for m in ("k", "wk", "v", "q")}
        backward_from(gpu, ag, ag.scale(qo, 0.25), rs.standard_normal(T * 2 * HD))
        gpu.sync([])
    finally:
        gpu.uninstall()
    for m in ("k", "wk", "v"):
        assert np.array_equal(t[m].grad, first[m]), m
    assert not np.array_equal(t["q"].grad, first["q"])


def test_the_order_of_a_walk_with_an_op_of_two_outputs():
    """On the host: inputs of outputs that the root does not depend on are left out, also where leaving them out leaves out others."""
    ag = mod("autograd")
    t = lambda *prev: (lambda x: setattr(x, "_prev", list(prev)) or x)(ag.Tensor(None, [1]))  # noqa: E731

    def pair(a, b):
        op = t(a, b)
        outs = t(op), t(op)
        op._outs = [(outs[0], [a]), (outs[1], [b])]
        return op, *outs
    x = t()
    op1, a1, b1 = pair(t(x), t(x))
    op2, a2, b2 = pair(t(a1), t(b1))
    for root, there, absent in ((t(a2, b2), (op1, op2, a1, b1, a2, b2, x), ()), (t(a2), (op1, op2, a1, a2, x), (b1, b2)), (t(b2), (op1, op2, b1, b2, x), (a1, a2)),
                                (t(t(b2), b2, a1), (op1, op2, a1, b1, b2, x), (a2,))):
        topo = ag._topo(root, set())
        at = {id(y): i for i, y in enumerate(topo)}
        assert len(at) == len(topo) and topo[-1] is root
        assert all(id(y) in at for y in there) and not any(id(y) in at for y in absent)
        for y in topo:
            for p in y._prev:
                assert id(p) not in at or at[id(p)] < at[id(y)]
        for o, p in ((a2, op2._prev[0]), (b2, op2._prev[1])):
            assert (id(p) in at) == (id(o) in at)
        # tensors that a caller counts as seen stay out, and are still counted
        seen = {id(x)}
        assert id(x) not in {id(y) for y in ag._topo(root, seen)} and id(x) in seen
