"""Two operators of a training step beside its matrix products, as cases that can be timed and checked.

qk_norm_rope   the normalisation of every head of q and k and the position rotation of the result, one pass each way:
               q_out = R(p) (q * rinv * w_q), rinv = 1 / sqrt(mean(q^2) + eps) per head, k alike; the backward gives dq, dk and
               the gradients of the two gains.
adamw8         an AdamW step over a whole parameter group whose moments are held in 8 bits: m and r = sqrt(v) as OCP e4m3
               values times a power of two for each block of 256 elements, rounded up or down at random in proportion. The states
               come back as the e4m3 values, in units of their block's power of two, and the exponents beside them.

`own` False: the operators in elementary torch operations. `own` True: the library's entry points on the same buffers.
"""
import ctypes
import importlib
import math

import torch

own = False

BLOCK = 256                    # elements that share the exponents of their two moments
EPS, BASE = 1e-6, 1000000.0
BETA1, BETA2, ADAM_EPS, DECAY, LR = 0.9, 0.95, 1e-8, 0.1, 3e-4


def listed():
    return [
        # ---- forward
        # one new token of one sequence: latency is all there is
        dict(name="fwd one token", op="fwd", seqs=1, T=1, hq=16, hkv=8, hd=128, pos=2047, spread=0, pad=0),
        # a decoding batch: every row at its own place in its own sequence, far ones among them
        dict(name="fwd 64 decoding rows", op="fwd", seqs=64, T=1, hq=10, hkv=2, hd=64, pos=0, spread=131072, pad=0),
        # odd lengths and a head size that is no power of two, q and k as slices of wider rows (one product made q, k and v)
        dict(name="fwd 3x683 hd96 strided", op="fwd", seqs=3, T=683, hq=9, hkv=3, hd=96, pos=0, spread=0, pad=96),
        # the micro-batches of a training step, stacked
        dict(name="fwd 8x2048 hd128", op="fwd", seqs=8, T=2048, hq=16, hkv=8, hd=128, pos=0, spread=0, pad=0),
        # ---- backward
        # one short odd sequence
        dict(name="bwd 1x127 hd64", op="bwd", seqs=1, T=127, hq=10, hkv=2, hd=64, pos=0, spread=0, pad=0, rot=1),
        # a training step's micro-batches at head size 64
        dict(name="bwd 8x2048 hd64", op="bwd", seqs=8, T=2048, hq=10, hkv=2, hd=64, pos=0, spread=0, pad=0, rot=1),
        # the same at head size 128 where the attention's backward has undone the rotation already
        dict(name="bwd 8x2048 hd128 norms", op="bwd", seqs=8, T=2048, hq=16, hkv=8, hd=128, pos=0, spread=0, pad=0, rot=0),
        # one long sequence
        dict(name="bwd 1x32768 hd128", op="bwd", seqs=1, T=32768, hq=16, hkv=8, hd=128, pos=0, spread=0, pad=0, rot=1),
        # ---- optimizer
        # the gains of a 30-layer model, an auxiliary group of its own: 61 tensors of 576
        dict(name="adamw8 gains", op="adamw8", layers=30, hidden=576, kv=0, ffn=0, vocab=0, rank=0, clip=1.0, t=100),
        # low-rank adapters of every projection of such a model: 420 small tensors
        dict(name="adamw8 adapters r16", op="adamw8", layers=30, hidden=576, kv=192, ffn=1536, vocab=0, rank=16, clip=1.0, t=10),
        # all of a 135M-parameter model, with the global clip
        dict(name="adamw8 135M", op="adamw8", layers=30, hidden=576, kv=192, ffn=1536, vocab=49152, rank=0, clip=1.0, t=1000),
        # the largest, without a clip
        dict(name="adamw8 640M no clip", op="adamw8", layers=12, hidden=2048, kv=512, ffn=5632, vocab=49152, rank=0, clip=0.0, t=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fwd", "bwd", "adamw8"])
    if op == "adamw8":
        hidden = _log(rng, 64, 1500)
        rank = rng.choice([0, 0, 4, 16, 33])
        case = dict(op=op, layers=rng.randint(1, 14), hidden=hidden, kv=max(1, hidden // rng.choice([2, 3, 4])), ffn=_log(rng, hidden, 4 * hidden),
                    vocab=0 if rank else _log(rng, 300, 60000), rank=rank, clip=rng.choice([0.0, 0.5, 1.0]), t=_log(rng, 1, 20000))
        return case
    hd = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, 160, 256])
    hkv = rng.randint(1, 8)
    hq = hkv * rng.randint(1, 4)
    most = (32768 * 24 * 128) // ((hq + hkv) * hd)                  # rows of the largest listed case's cost
    T = _log(rng, 1, min(16384, most))
    most = min(8, most // T)
    case = dict(op=op, seqs=rng.randint(1, most) if T > 1 else _log(rng, 1, 256), T=T, hq=hq, hkv=hkv, hd=hd, pos=rng.choice([0, 0, 1, rng.randint(2, 100000)]),
                spread=rng.choice([0, 0, 0, 1000000]), pad=rng.choice([0, 0, 4 * rng.randint(1, 64)]))
    if op == "bwd":
        case["rot"] = rng.choice([1, 1, 0])
    return case


def _sizes(c):
    """Element counts of the group's tensors."""
    h, kv, f, n = c["hidden"], c["kv"], c["ffn"], c["layers"]
    if not f:
        return [h] * (2 * n + 1)
    mats = [(h, h), (kv, h), (kv, h), (h, h), (f, h), (f, h), (h, f)]
    if c["rank"]:
        return [s for _ in range(n) for o, i in mats for s in (c["rank"] * i, o * c["rank"])]
    return [c["vocab"] * h, h] + [s for _ in range(n) for s in (h, *[o * i for o, i in mats], h)]


def work(case):
    if case["op"] == "adamw8":
        n = sum(_sizes(case))
        return {"bytes": 16.0 * n + 4.0 * sum(-(-s // BLOCK) for s in _sizes(case)), "flops": 20.0 * n}
    n = case["seqs"] * case["T"] * (case["hq"] + case["hkv"]) * case["hd"]
    gains = 8.0 * case["hd"]
    places = 4.0 * case["seqs"] * case["T"] if case["spread"] else 0.0
    if case["op"] == "fwd":
        return {"bytes": 8.0 * n + gains + places, "flops": 7.0 * n}
    return {"bytes": 12.0 * n + 2 * gains + places, "flops": 15.0 * n}


# ---- what a program has in hand before the call ------------------------------------------------------------------

_ctx = None


def _lib():
    """The library's binding and one context on the first GPU, kept as a training program keeps its backend."""
    global _ctx
    lib = importlib.import_module("gguf-trainer_amd.lib")
    if _ctx is None:
        c = ctypes.c_void_p()
        if lib.lib.gt_ctx_create(0, ctypes.byref(c)) != 0:
            raise RuntimeError((lib.lib.gt_last_error(None) or b"").decode())
        _ctx = c
    return lib


class _Group:
    """An 8-bit AdamW group of the library over the tensors that lie in flat buffers."""

    def __init__(self, sizes, starts, w, g, m, v, e, clip):
        lib = _lib()
        n = len(sizes)
        at = lambda t, scale, by: (lib.buf * n)(*[t.data_ptr() + scale * s // by for s in starts])  # noqa: E731
        self.handle = ctypes.c_void_p()
        lib.check(_ctx, lib.lib.gt_adamw8_create(_ctx, n, at(w, 4, 1), at(g, 4, 1), at(m, 1, 1), at(v, 1, 1), at(e, 2, BLOCK), (ctypes.c_int64 * n)(*sizes),
                                                 BETA1, BETA2, ADAM_EPS, DECAY, clip, ctypes.byref(self.handle)), "gt_adamw8_create")

    def __del__(self):
        lib = _lib()
        lib.lib.gt_adamw_destroy(_ctx, self.handle)


def _flat(sizes):
    """(start of each tensor, total): every tensor starts at a whole block, as allocators place them."""
    starts, at = [], 0
    for s in sizes:
        starts.append(at)
        at += -(-s // BLOCK) * BLOCK
    return starts, at


def _adam_inputs(case, seed):
    sizes = _sizes(case)
    starts, total = _flat(sizes)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda k: torch.randn(k, device="cuda", generator=gen)  # noqa: E731
    live = torch.ones(total, device="cuda", dtype=torch.bool)      # False in the gap between a tensor's end and the next block
    gaps = [(a + s, a + -(-s // BLOCK) * BLOCK) for a, s in zip(starts, sizes) if s % BLOCK]
    if gaps:
        idx = torch.cat([torch.arange(a, b) for a, b in gaps]).cuda()
        live[idx] = False
    # gradients of very different size from block to block and, within one, from element to element; some exactly zero
    # (an embedding row that no token of the batch named)
    blocks = total // BLOCK
    scale = torch.exp(1.5 * new(blocks) - 7.0)
    scale[torch.rand(blocks, device="cuda", generator=gen) < 0.05] = 0.0
    spread = torch.exp(0.7 * new(total)).view(blocks, BLOCK) * scale[:, None]
    w = 0.05 * new(total) * live
    g = (spread * new(total).view(blocks, BLOCK)).view(-1) * live
    m = (0.3 * spread * new(total).view(blocks, BLOCK)).view(-1) * live
    r = (spread * (0.2 + torch.rand(total, device="cuda", generator=gen).view(blocks, BLOCK))).view(-1) * live
    half = torch.full((total,), 32768, device="cuda", dtype=torch.int32)
    mc, me = _encode(m, half)
    rc, re = _encode(r, half)
    return sizes, starts, w, g, mc, rc, torch.stack([me, re], dim=1).contiguous()


def _qk_inputs(case, seed):
    rows, hd = case["seqs"] * case["T"], case["hd"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *k: torch.randn(*k, device="cuda", generator=gen)  # noqa: E731
    s = {}
    for name, heads in (("q", case["hq"]), ("k", case["hkv"])):
        wide = new(rows, heads * hd + case["pad"]) * torch.exp(0.5 * new(rows, 1))
        s[name] = wide[:, :heads * hd]
        s["w" + name] = 1 + 0.3 * new(hd)
        if case["op"] == "bwd":
            s["g" + name] = 0.01 * new(rows, heads * hd)
    s["places"] = None
    if case["spread"]:
        s["places"] = torch.randint(0, case["spread"], (rows,), device="cuda", generator=gen, dtype=torch.int32)
    return s


def prepare(case, seed):
    if case["op"] == "adamw8":
        sizes, starts, w, g, m, v, e = _adam_inputs(case, seed)
        state = dict(case=case, sizes=sizes, w=w, g=g, m=m, v=v, e=e, t=case["t"])
        if own:
            state["group"] = _Group(sizes, starts, w, g, m, v, e, case["clip"])
        return state
    state = dict(case=case, **_qk_inputs(case, seed))
    for name in ("q", "k"):
        x = state[name]
        if case["op"] == "fwd":
            state["out_" + name] = torch.empty(x.shape, device="cuda")
        else:
            state["d" + name] = torch.empty_strided(x.shape, x.stride(), device="cuda")
            state["dw" + name] = torch.empty(case["hd"], device="cuda")
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_adam(state) if op == "adamw8" else _own_forward(state) if op == "fwd" else _own_backward(state)
    return _plain_adam(state) if op == "adamw8" else _plain_forward(state) if op == "fwd" else _plain_backward(state)


def _address(t):
    return 0 if t is None else t.data_ptr()


def _own_forward(s):
    c, lib = s["case"], _lib()
    q, k, qo, ko = s["q"], s["k"], s["out_q"], s["out_k"]
    lib.check(_ctx, lib.lib.gt_qk_norm_rope_fwd(
        _ctx, q.shape[0], c["T"], c["hq"], c["hkv"], c["hd"], EPS, BASE, c["pos"], _address(s["places"]),
        q.data_ptr(), q.stride(0), s["wq"].data_ptr(), qo.data_ptr(), qo.stride(0),
        k.data_ptr(), k.stride(0), s["wk"].data_ptr(), ko.data_ptr(), ko.stride(0)), "gt_qk_norm_rope_fwd")
    return {"q": qo, "k": ko}


def _own_backward(s):
    c, lib = s["case"], _lib()
    q, k, gq, gk = s["q"], s["k"], s["gq"], s["gk"]
    lib.check(_ctx, lib.lib.gt_qk_norm_rope_bwd(
        _ctx, q.shape[0], c["T"], c["hq"], c["hkv"], c["hd"], EPS, BASE, c["pos"], _address(s["places"]),
        q.data_ptr(), q.stride(0), s["wq"].data_ptr(), gq.data_ptr(), gq.stride(0), c["rot"], s["dq"].data_ptr(), 0, s["dwq"].data_ptr(), 0,
        k.data_ptr(), k.stride(0), s["wk"].data_ptr(), gk.data_ptr(), gk.stride(0), c["rot"], s["dk"].data_ptr(), 0, s["dwk"].data_ptr(), 0),
        "gt_qk_norm_rope_bwd")
    return {"dq": s["dq"], "dk": s["dk"], "dwq": s["dwq"], "dwk": s["dwk"]}


def _own_adam(s):
    lib, t = _lib(), s["t"]
    lib.check(_ctx, lib.lib.gt_adamw8_step(_ctx, s["group"].handle, LR, 1 - BETA1 ** t, 1 - BETA2 ** t, t), "gt_adamw8_step")
    s["t"] = t + 1
    return {"w": s["w"], "m": s["m"].view(torch.float8_e4m3fn), "r": s["v"].view(torch.float8_e4m3fn), "exponents": s["e"]}


def _angles(s):
    """cos and sin [rows, hd / 2] of the rotation of each row's pairs (j, j + hd / 2), formed in 64 bits."""
    c = s["case"]
    half = c["hd"] // 2
    p = s["places"]
    if p is None:
        p = torch.arange(c["T"], device="cuda").repeat(c["seqs"]) + c["pos"]
    freq = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 * math.log(BASE) / c["hd"]))
    a = p.double()[:, None] * freq
    return torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]


def _plain_forward(s):
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        x = s[name].unflatten(1, (-1, s["case"]["hd"]))
        y = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + EPS) * s["w" + name]
        lo, hi = y.chunk(2, dim=2)
        out[name] = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], dim=2).flatten(1)
    return out


def _plain_backward(s):
    c = s["case"]
    out = {}
    if c["rot"]:
        cos, sin = _angles(s)
    for name in ("q", "k"):
        x, g, w = s[name].unflatten(1, (-1, c["hd"])), s["g" + name].unflatten(1, (-1, c["hd"])), s["w" + name]
        if c["rot"]:
            lo, hi = g.chunk(2, dim=2)
            g = torch.cat([lo * cos + hi * sin, hi * cos - lo * sin], dim=2)
        r = torch.rsqrt((x * x).mean(dim=2, keepdim=True) + EPS)
        n = x * r
        gw = g * w
        out["d" + name] = (r * (gw - n * (gw * n).mean(dim=2, keepdim=True))).flatten(1)
        out["dw" + name] = (g * n).double().sum(dim=(0, 1)).float()
    return out


def _mix(x):
    """One multiply-xorshift round over 32-bit words held in 64."""
    x = x ^ (x >> 16)
    x = (x * 0x21F0AAAD) & 0xFFFFFFFF
    return x ^ (x >> 15)


def _word(x):
    """The full mixer: two rounds."""
    x = _mix(x)
    x = (x * 0x735A2D97) & 0xFFFFFFFF
    return x ^ (x >> 15)


def _random_words(seed, total):
    """The 32 random bits of every element: a function of the step's seed, the number of the block in the group and the place
    in the block. The low 16 round m, the high 16 round r."""
    lo, hi = seed & 0xFFFFFFFF, seed >> 32
    key = _word(lo ^ _word((hi + 0x9E3779B9) & 0xFFFFFFFF))
    block = torch.arange(total // BLOCK, device="cuda")
    inside = torch.arange(BLOCK, device="cuda") * 0x9E3779B9
    return _mix((_word(block ^ key)[:, None] + inside) & 0xFFFFFFFF).view(-1)


def _power(e):
    """2^e for whole e in [-126, 126], as its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _encode(x, r16):
    """(codes, exponents): |x| <= 448 * 2^e over each block of 256 with the smallest such e, and x / 2^e as an e4m3 value: the
    lower neighbour, or the upper one where what is left over, plus r16 / 65536 of a step, makes a whole step."""
    blocks = x.view(-1, BLOCK)
    top = blocks.abs().amax(dim=1)
    f, k = torch.frexp(top)
    e = torch.where(top > 0, torch.where(f <= 0.875, k - 9, k - 8), -126).clamp(min=-126).to(torch.int32)
    y = (blocks.abs() * _power(-e)[:, None]).view(-1)
    r16 = r16.to(torch.int32)
    normal = ((y.view(torch.int32) + (r16 << 4)) >> 20) - (120 << 3)
    small = torch.floor(y * 512 + r16.float() / 65536).to(torch.int32)
    code = torch.where(y >= 2.0 ** -6, normal, small)
    return (code | ((x < 0).to(torch.int32) << 7)).to(torch.uint8), e.to(torch.int8)


def _decode(code, e):
    return (code.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * _power(e.int())[:, None]).view(-1)


def _plain_adam(s):
    c, t, w, g = s["case"], s["t"], s["w"], s["g"]
    if c["clip"] > 0:
        norm = g.double().square().sum().sqrt()
        g = g * torch.where(norm > c["clip"], c["clip"] / (norm + 1e-12), 1.0).float()
    m = _decode(s["m"], s["e"][:, 0]) * BETA1 + g * (1 - BETA1)
    r = _decode(s["v"], s["e"][:, 1])
    v = (r * r) * BETA2 + (g * (1 - BETA2)) * g
    bits = _random_words(t, w.numel())
    s["m"], em = _encode(m, bits & 0xFFFF)
    code, er = _encode(v.sqrt(), bits >> 16)
    s["v"] = torch.where(v > 0, code.clamp(min=1), code)        # a moment that is there never becomes one that is not
    s["e"] = torch.stack([em, er], dim=1)
    step = (m * (1 / (1 - BETA1 ** t))) / ((v * (1 / (1 - BETA2 ** t))).sqrt() + ADAM_EPS) + DECAY * w
    s["w"] = w - LR * step
    s["t"] = t + 1
    return {"w": s["w"], "m": s["m"].view(torch.float8_e4m3fn), "r": s["v"].view(torch.float8_e4m3fn), "exponents": s["e"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "adamw8":
        return _exact_adam(case, seed)
    s = _qk_inputs(case, seed)
    rows, hd = case["seqs"] * case["T"], case["hd"]
    if s["places"] is not None:
        place = s["places"].double()
    else:
        place = (torch.arange(rows, device="cuda") % case["T"]).double() + case["pos"]
    turn = torch.view_as_complex(torch.stack([torch.zeros(rows, hd // 2, device="cuda", dtype=torch.float64),
                                              place[:, None] * BASE ** (-2.0 / hd * torch.arange(hd // 2, device="cuda").double())], dim=2)).exp()[:, None]
    out = {}
    for name in ("q", "k"):
        x, w = s[name].double().reshape(rows, -1, hd), s["w" + name].double()
        rms = ((x ** 2).sum(-1, keepdim=True) / hd + EPS) ** 0.5
        if case["op"] == "fwd":
            y = x / rms * w
            z = torch.complex(y[..., :hd // 2], y[..., hd // 2:]) * turn
            out[name] = torch.cat([z.real, z.imag], dim=-1).reshape(rows, -1)
            continue
        g = s["g" + name].double().reshape(rows, -1, hd)
        if case["rot"]:
            z = torch.complex(g[..., :hd // 2], g[..., hd // 2:]) * turn.conj()
            g = torch.cat([z.real, z.imag], dim=-1)
        out["dw" + name] = torch.sum(g * x / rms, dim=(0, 1))
        # d/dx of (x / rms) . (g w): the part along x drops out
        h = g * w
        out["d" + name] = ((h * rms ** 2 - x * (h * x).sum(-1, keepdim=True) / hd) / rms ** 3).reshape(rows, -1)
    return out


def _exact_adam(case, seed):
    sizes, _, w, g, mc, rc, e = _adam_inputs(case, seed)
    t, total = case["t"], w.numel()
    two = torch.tensor(2.0, device="cuda", dtype=torch.float64)
    value = lambda code, x: (code.view(torch.float8_e4m3fn).double().view(-1, BLOCK) * two ** x[:, None].double()).view(-1)  # noqa: E731
    g = g.double()
    if case["clip"] > 0:
        norm = torch.linalg.vector_norm(g)
        if norm > case["clip"]:
            g *= case["clip"] / (norm + 1e-12)
    m = BETA1 * value(mc, e[:, 0]) + (1 - BETA1) * g
    v = BETA2 * value(rc, e[:, 1]) ** 2 + (1 - BETA2) * g ** 2
    del g
    word = _random_words(t, total)
    out = {"w": w.double() - LR * (m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)) ** 0.5 + ADAM_EPS) + DECAY * w.double())}
    new = []
    for name, x, bits in (("m", m, word % 65536), ("r", v ** 0.5, word // 65536)):
        b = x.abs().view(-1, BLOCK)
        top = b.amax(dim=1)
        ex = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), -126.0).clamp(min=-126)
        ex = torch.where(top > 448 * two ** ex, ex + 1, torch.where((top <= 448 * two ** (ex - 1)) & (ex > -126), ex - 1, ex))     # log2's last bit
        y = (b / two ** ex[:, None]).view(-1)
        grain = two ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
        y = grain * torch.floor(y / grain + bits.double() / 65536)
        if name == "r":
            y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
        out[name] = torch.where(x < 0, -y, y)
        new.append(ex)
    out["exponents"] = None
    return out
