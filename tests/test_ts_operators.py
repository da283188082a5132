"""What hip.ts does before and around its library calls, run: bodies of the binding are taken out of the file, their type annotations dropped, and
executed by node against a stand-in for the library that records the calls. (Deno is not needed for that, and not here.)"""
import json
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = open(os.path.join(ROOT, "gguf-trainer_amd", "ts", "hip.ts")).read()
needs_node = pytest.mark.skipif(shutil.which("node") is None, reason="no node")


def block(src, at):
    """The text from the first brace at or after `at` to the one that closes it."""
    i = src.index("{", at)
    depth, j = 0, i
    while True:
        depth += {"{": 1, "}": -1}.get(src[j], 0)
        j += 1
        if not depth:
            return src[i:j]


def plain(body):
    """Without the annotations that occur in these bodies."""
    body = re.sub(r"\bas (\[[^\]]*\]|\w+)(\[\])?", "", body)
    body = re.sub(r"(\w+): \[Tensor, Tensor, number, string\]\[\] =", r"\1 =", body)
    body = re.sub(r"(\w+): (Float32Array|DevBuf|number|string)(\[\])? =", r"\1 =", body)
    body = re.sub(r"([\w.]+) \?\? (\w+)", r"(\1 != null ? \1 : \2)", body)       # younger than the node this may meet
    return re.sub(r"(?<=[\w\])])!(?=[.;,)\[])", "", body)


def method(cls, name):
    """(parameter names, plain body) of a method."""
    at = SRC.index(f"export class {cls}")
    m = re.compile(rf"^  (?:async |private )*{name}\(([^)]*)\)[^{{;]*?(?:: [^{{]*(?:\{{[^}}]*\}}[^{{]*)?)? \{{$", re.M).search(SRC, at)
    params = [p.split(":")[0].strip(" ?") for p in m.group(1).split(",") if p.strip()]
    return params, plain(block(SRC, m.end() - 1))


def run(js):
    out = subprocess.run(["node", "-e", js], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr[-2000:]
    return json.loads(out.stdout)


QK = """
const prod = (s) => s.reduce((a, b) => a * b, 1);
function backend() {
  const log = [];
  const be = {
    log, ctx: "ctx", next: 100n,
    sym: new Proxy({}, { get: (_, name) => (...a) => { log.push([name, a.slice(1).map(String)]); return 0; } }),
    check(rc, what) { if (rc !== 0) throw new Error(what); },
    dataOf(t) { return t.d || (t.d = be.next++); },
    makeOut(shape, prev, alloc = true) { const t = { shape, _prev: prev, _backward() {} }, e = { data: alloc ? be.next++ : 0n, gradInit: false }; t.e = e; return { t, e }; },
    gradOf(t) { t.e.gradInit = true; return t.g || (t.g = be.next++); },
    gradDst(t) { const acc = t.acc || 0; t.acc = 1; return [t.gr || (t.gr = be.next++), acc]; },
  };
  be.qkNormRope = function (%s) %s;
  return be;
}
const T = (...shape) => ({ shape, requiresGrad: true, _prev: [] });
// the reference's walk: each tensor after everything below it, then backwards
function walk(root) {
  const seen = new Set(), topo = [];
  (function go(t) { if (seen.has(t)) return; seen.add(t); t._prev.forEach(go); topo.push(t); })(root);
  root.e.gradInit = true;
  topo.reverse().forEach((t) => t._backward && t._backward());
}
"""


def qk(js):
    params, body = method("HipBackend", "qkNormRope")
    return run(QK % (", ".join(params), body) + js)


def tried(call):
    return "(() => { const be = backend(); let err = ''; try { " + call + " } catch (e) { err = e.message; } return [err, be.log.map((x) => x[0])]; })()"


@needs_node
def test_qk_norm_rope_checks_its_shapes_before_it_calls():
    """The library takes addresses: a row count or a width that is not what the tensors have would be read past their ends."""
    cases = ["be.qkNormRope(T(6, 32), T(6, 16), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "be.qkNormRope(T(6, 32), T(5, 16), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "be.qkNormRope(T(6, 24), T(6, 16), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "be.qkNormRope(T(6, 32), T(6, 16), T(8), T(7), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "be.qkNormRope(T(6, 32), T(6, 8), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "be.qkNormRope(T(6, 32), T(96), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0)",
             "const q = T(6, 16); be.qkNormRope(q, q, T(8), T(8), 3, 2, 2, 8, 1e-6, 1e4, 0)"]
    got = qk("console.log(JSON.stringify([" + ", ".join(tried(c) for c in cases) + "]))")
    assert got[0] == ["", ["gt_qk_norm_rope_fwd"]]
    for (err, calls), match in zip(got[1:], ("6 rows and k 5", "q is [6, 24]", "gain of 7", "k is [6, 8]", "k is [96]", "distinct")):
        assert match in err and calls == [], (err, match, calls)


@needs_node
def test_qk_norm_rope_and_backwards_that_reach_one_output():
    """Both outputs in one walk are one call; a walk through one output alone has zeros for the other; but where an earlier walk came through the other,
    its old gradient would be handed on again: that is refused before anything is launched."""
    js = """
    const out = {};
    for (const [name, walks] of Object.entries({ both: ["qk"], twice: ["qk", "qk"], q: ["q"], k: ["k"], qq: ["q", "q"], bothThenQ: ["qk", "q"], bothThenK: ["qk", "k"], kThenQ: ["k", "q"], qThenBoth: ["q", "qk"] })) {
      const be = backend();
      const [qo, ko] = be.qkNormRope(T(6, 32), T(6, 16), T(8), T(8), 3, 4, 2, 8, 1e-6, 1e4, 0);
      let err = "";
      try {
        for (const w of walks) walk({ shape: [1], _prev: w === "qk" ? [qo, ko] : w === "q" ? [qo] : [ko], e: {} });
      } catch (e) { err = e.message; }
      out[name] = [err, be.log.filter((x) => x[0] === "gt_qk_norm_rope_bwd").length];
    }
    console.log(JSON.stringify(out));
    """
    got = qk(js)
    for name, n in dict(both=1, twice=2, q=1, k=1, qq=2, qThenBoth=2).items():
        assert got[name] == ["", n], (name, got[name])
    for name in ("bothThenQ", "bothThenK", "kThenQ"):
        assert "sync()" in got[name][0] and got[name][1] == 1, (name, got[name])


# ---- AdamWHip -----------------------------------------------------------------------------------------------------------

ADAM = """
class Buffers {
  // a backend that counts state buffers and fails at the n-th call of an entry point
  constructor(fail, at) {
    this.live = new Set(); this.n = 0; this.calls = []; this.context = null; this.isDestroyed = false;
    let k = 0;
    this.symbols = new Proxy({}, { get: (_, name) => (...a) => { this.calls.push(name); return name === fail && ++k === at ? 1 : 0; } });
  }
  check(rc, what) { if (rc !== 0) throw new Error(what); }
  createStateBuffer(bytes) { const b = BigInt(++this.n); this.live.add(b); return b; }
  freeStateBuffer(b) { this.live.delete(b); }
  writeStateBuffer() { if (--this.writes === 0) throw new Error("write"); }
  async readStateBuffer(b, n) { if (--this.reads === 0) throw new Error("read"); return new Float32Array(n); }
  buffersFor() { return { data: 1n, grad: 2n }; }
  keepGradOnDevice() {}
}
const Deno = { UnsafePointer: { create: (x) => x } }, u64s = (v) => v;
class AdamWHip {
  %s
}
const P = (n) => ({ size: n });
const S = (...n) => n.map((k) => new Float32Array(k));
async function main() { const out = []; %s; console.log(JSON.stringify(out)); }
main().catch((e) => { console.error(e); process.exit(1); });
"""


def adam(js):
    names = ("constructor", "momentPair", "exportState", "importState", "destroy")
    body = []
    for n in names:
        at = SRC.index("export class AdamWHip")
        m = re.compile(rf"^  ((?:async |private )*){n}\((.*)\)(?:: .*)? \{{$", re.M).search(SRC, at)
        params = [re.sub(r"\W", "", p.split(":")[0]) for p in re.split(r",(?![^{]*\})", m.group(2)) if p.strip()]
        fields = "this.mBufs = []; this.vBufs = []; this.eBufs = []; this.t = 0; this.handle = null;" if n == "constructor" else ""
        text = plain(block(SRC, m.end() - 1))
        body.append(f"{'async ' if 'async' in m.group(1) else ''}{n}({', '.join(params)}) {{ {fields}" + text[1:])
    return run(ADAM % ("\n".join(body), js))


@needs_node
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_gives_its_moment_buffers_back_when_a_call_throws(bits):
    """However far exportState and importState come, the state buffers afterwards are those of the group."""
    js = """
    for (const [what, fail, at] of [["", "", 0], ["export", "gt_adamw8_read", 2], ["exportRead", "", 3], ["import", "gt_adamw8_write", 2], ["importWrite", "", 3]]) {
      const gpu = new Buffers(fail, at), opt = new AdamWHip(gpu, [P(300), P(5)], { lr: 1, stateBits: %d });
      const own = gpu.live.size;
      gpu.reads = what === "exportRead" ? at : -1;
      gpu.writes = what === "importWrite" ? at : -1;
      let err = "";
      try { const s = await opt.exportState(); opt.importState({ m: S(300, 5), v: S(300, 5), t: 3 }); } catch (e) { err = e.message; }
      out.push([what, err, own, gpu.live.size]);
      opt.destroy();
      out.push(gpu.live.size);
    }""" % bits
    got = adam(js)
    for done, rest in zip(got[::2], got[1::2]):
        assert done[2] == done[3] == (6 if bits == 8 else 4) and rest == 0, done
        assert bool(done[1]) == (done[0] != "" and (bits == 8 or done[0] in ("exportRead", "importWrite"))), done


@needs_node
def test_adamw_refuses_other_state_sizes():
    js = """
    for (const bits of [16, 0, "8", 8, 32, undefined]) {
      const gpu = new Buffers("", 1);
      let err = "";
      try { new AdamWHip(gpu, [P(300)], { lr: 1, stateBits: bits }); } catch (e) { err = e.message; }
      out.push([err, gpu.live.size, gpu.calls]);
    }"""
    got = adam(js)
    for err, live, calls in got[:3]:
        assert "stateBits must be 8 or 32" in err and live == 0 and calls == []
    for (err, live, calls), (n, name) in zip(got[3:], ((3, "gt_adamw8_create"), (2, "gt_adamw_create"), (2, "gt_adamw_create"))):
        assert err == "" and live == n and calls == [name]


@needs_node
def test_a_refused_adamw_group_keeps_no_memory():
    js = """
    for (const [bits, fail] of [[8, "gt_adamw8_create"], [32, "gt_adamw_create"]]) {
      const gpu = new Buffers(fail, 1);
      let err = "";
      try { new AdamWHip(gpu, [P(300), P(5)], { lr: 1, stateBits: bits }); } catch (e) { err = e.message; }
      out.push([err, gpu.n, gpu.live.size]);
    }"""
    assert adam(js) == [["gt_adamw8_create", 6, 0], ["gt_adamw_create", 4, 0]]
