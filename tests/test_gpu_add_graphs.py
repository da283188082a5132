"""Sums in graphs that are differentiated more than once: an add hands its upstream gradient on by address (alias_add_grads), which changes no gradient.
Both sides add the same numbers, a copy more or less between them: 1e-6 relative is sixteen half-steps on every element's root mean square."""
import numpy as np
import pytest

from gpu_common import backward_from, mod


def graph(ag, t, which):
    a, b = ag.scale(t["a"], 2.0), ag.scale(t["b"], 3.0)
    if which == "root":
        return ag.add(a, b)
    if which == "below":
        return ag.scale(ag.add(a, b), 0.5)
    if which == "chain":                                             # the handed-on gradient is handed on again
        return ag.scale(ag.add(ag.add(a, b), ag.scale(a, 0.25)), 0.5)
    return ag.linear(ag.rms_norm(ag.add(a, ag.scale(ag.add(a, b), 0.5)), t["w"], 1e-6), t["W"])


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["root", "below", "chain", "residual"])
def test_one_graph_three_times(gpu, which):
    ag = mod("autograd")
    got = []
    for alias in (True, False):
        rs = np.random.RandomState(81)
        n = lambda *s: ag.Tensor(rs.standard_normal(s).astype(np.float32), list(s), True)  # noqa: E731
        t = dict(a=n(24, 64), b=n(24, 64), w=n(64), W=n(48, 64))
        gpu.install()
        gpu.alias_add_grads = alias
        try:
            out = graph(ag, t, which)
            for _ in range(3):
                backward_from(gpu, ag, out, rs.standard_normal(out.size))
            gpu.sync([])
        finally:
            gpu.alias_add_grads = True
            gpu.uninstall()
        got.append({m: x.grad.astype(np.float64) for m, x in t.items()})
    for m in got[0]:
        assert np.linalg.norm(got[0][m] - got[1][m]) <= 1e-6 * np.linalg.norm(got[1][m]), m
