"""The training operators around the linear layer, as cases that can be timed and compared.

Three operators, forward and backward: the linear layer with bias, activation, dropout and residual in its epilogue
(mmh_linear), dropout whose mask comes from a counter and is never stored (mmh_dropout), and the cross entropy of a head
over a vocabulary whose logits are never whole in memory (mmh_linear_cross_entropy). With own = True a pass is the call of
the C ABI that a program makes; otherwise it is the same mathematics in elementary torch operations. All values are f32, as
the framework's are; activations ~ N(0, 1), weights ~ N(0, 0.02), as its seeded init draws them, targets uniform over the
vocabulary and on the host, where the framework takes them.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

STD = 0.02
FORMS = {"nn": 0, "nt": 1}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
IGNORE = -1


def listed():
    return [
        # one projection of the smallest preset, 2 x 32 tokens: a call that is all latency
        dict(name="linear_smoke", kind="linear", form="nn", rows=64, k=64, n=176, act="silu", p=0.0, residual=False, pre=False),
        # the wide half of an MLP in training at the large preset's widths, 4 x 1024 tokens: the preactivation is kept
        dict(name="linear_up", kind="linear", form="nt", rows=4096, k=2048, n=5632, act="gelu_tanh", p=0.0, residual=False, pre=True),
        # its narrow half: dropout and the residual stream in the epilogue
        dict(name="linear_down", kind="linear", form="nn", rows=4096, k=5632, n=2048, act="none", p=0.1, residual=True, pre=False),
        # gradients for a batch whose token count and widths are no multiple of anything
        dict(name="linear_bwd_ragged", kind="linear_bwd", form="nn", rows=1003, k=770, n=1517, act="relu", p=0.25),
        # the wide half's gradients at the medium preset's widths, 4 x 1024 tokens
        dict(name="linear_bwd", kind="linear_bwd", form="nt", rows=4096, k=1024, n=2816, act="gelu", p=0.1),
        # the dropout of one micro batch of the smallest preset: latency
        dict(name="dropout_smoke", kind="dropout", n=64 * 64, p=0.1, residual=False),
        # the dropout and residual add of the large preset's stream at 16 x 1024 tokens
        dict(name="dropout_add", kind="dropout", n=16384 * 2048, p=0.1, residual=True),
        # its gradient over an odd number of values
        dict(name="dropout_bwd", kind="dropout_bwd", n=5003 * 1021, p=0.5),
        # evaluation with the large preset's tied head, 4 x 1024 tokens
        dict(name="ce_large", kind="ce", form="nt", n=4096, d=2048, vocab=32000, ignored=0.0),
        # the tiny preset's training batch, 8 x 256 tokens
        dict(name="ce_bwd_tiny", kind="ce_bwd", form="nt", n=2048, d=128, vocab=4096, ignored=0.0),
        # the large preset's training batch, 4 x 1024 tokens
        dict(name="ce_bwd_large", kind="ce_bwd", form="nt", n=4096, d=2048, vocab=32000, ignored=0.0),
        # a vocabulary of four times that, untied head, a ragged batch with padding that is left out of the loss
        dict(name="ce_bwd_wide", kind="ce_bwd", form="nn", n=1021, d=1024, vocab=131071, ignored=0.2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size in [lo, hi], spread over its logarithm: half of them multiples of 64 where there is room, the others as they fall."""
    v = _log(rng, lo, hi)
    return max(64, v // 64 * 64) if v >= 128 and rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_bwd", "linear_bwd", "dropout", "dropout_bwd", "ce", "ce_bwd", "ce_bwd"])
    p = rng.choice([0.0, 0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    if kind in ("dropout", "dropout_bwd"):
        c = dict(kind=kind, n=_log(rng, 1, 16384 * 2048), p=p or 0.1)
        return dict(c, residual=rng.random() < 0.5) if kind == "dropout" else c
    form = rng.choice(["nn", "nt"])
    if kind in ("linear", "linear_bwd"):
        while True:
            rows, k, n = _size(rng, 1, 8192), _size(rng, 8, 8192), _size(rng, 8, 8192)
            if rows * k * n <= 4096 * 2048 * 11264:
                break
        act = rng.choice(list(ACTIVATIONS))
        c = dict(kind=kind, form=form, rows=rows, k=k, n=n, act=act, p=p)
        return dict(c, residual=rng.random() < 0.5, pre=rng.random() < 0.5) if kind == "linear" else c
    while True:
        n, d, vocab = _size(rng, 1, 8192), _size(rng, 16, 4096), _size(rng, 64, 262144)
        if n * vocab <= 4096 * 32000 and d * vocab <= 2048 * 131072 and n * d * vocab <= 4096 * 2048 * 32000:
            break
    return dict(kind=kind, form=form, n=n, d=d, vocab=vocab, ignored=rng.choice([0.0, 0.0, 0.1, 0.5]))


# ---- inputs --------------------------------------------------------------------

_context = None


def _mh():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "midman-ai_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import midman_hip
    return midman_hip


def _ctx():
    """The program's one context."""
    global _context
    if _context is None:
        _context = _mh().Context(0)
    return _context


class _Cuda:
    """A DeviceArray's memory, for torch."""

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = dict(shape=array.shape, typestr="<f4", data=(array.ptr, False), version=2)


def _inputs(c):
    """{name: (shape, std)} of a case's random arrays."""
    kind = c["kind"]
    if kind == "dropout":
        s = {"x": ((c["n"],), 1.0)}
        if c["residual"]:
            s["residual"] = ((c["n"],), 1.0)
        return s
    if kind == "dropout_bwd":
        return {"dout": ((c["n"],), 1.0)}
    if kind in ("ce", "ce_bwd"):
        return {"x": ((c["n"], c["d"]), 1.0), "w": ((c["d"], c["vocab"]) if c["form"] == "nn" else (c["vocab"], c["d"]), STD)}
    r, k, n = c["rows"], c["k"], c["n"]
    s = {"x": ((r, k), 1.0), "w": ((k, n) if c["form"] == "nn" else (n, k), STD)}
    if kind == "linear":
        s["bias"] = ((n,), 0.1)
        if c["residual"]:
            s["residual"] = ((r, n), 1.0)
    else:
        s["pre"] = ((r, n), STD * math.sqrt(k))
        s["dout"] = ((r, n), 1.0)
    return s


def _outputs(c):
    """{name: shape} of the buffers that a program hands to the call."""
    kind = c["kind"]
    if kind == "dropout":
        return {"out": (c["n"],)}
    if kind == "dropout_bwd":
        return {"dx": (c["n"],)}
    if kind == "ce":
        return {}
    s = {n: v for n, (v, _) in _inputs(c).items()}
    if kind == "ce_bwd":
        return {"dx": s["x"], "dw": s["w"]}
    if kind == "linear":
        out = {"out": (c["rows"], c["n"])}
        if c["pre"]:
            out["pre"] = out["out"]
        return out
    return {"dx": s["x"], "dw": s["w"], "dbias": (c["n"],)}


def _drawn(c, seed):
    """The arrays, the targets and the generator's key and first counter of a case, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = {n: torch.randn(s, generator=g, device="cuda") * std for n, (s, std) in _inputs(c).items()}
    r = np.random.default_rng(seed)
    key, offset = int(r.integers(1 << 63)) * 2 + 1, int(r.integers(1 << 40))
    targets = None
    if c["kind"] in ("ce", "ce_bwd"):
        targets = r.integers(0, c["vocab"], c["n"]).astype(np.int32)
        targets[r.random(c["n"]) < c["ignored"]] = IGNORE
    return t, targets, key, offset


def prepare(case, seed):
    c = case
    t, targets, key, offset = _drawn(c, seed)
    s = dict(case=c, key=key, offset=offset, targets=targets)
    if own:
        ctx = _ctx()
        for name, v in t.items():
            s[name] = ctx.empty(tuple(v.shape))
            torch.as_tensor(_Cuda(s[name]), device="cuda").copy_(v)
        outs = _outputs(c)
        for name, shape in outs.items():
            s[name] = ctx.empty(shape)
        s["outs"] = {name: torch.as_tensor(_Cuda(s[name]), device="cuda") for name in outs}
        torch.cuda.synchronize()  # the inputs are there before the context's own stream reads them
    else:
        s.update(t)
    return s


# ---- one pass ------------------------------------------------------------------

def _call(name, *args):
    """One entry point of the C ABI, with DeviceArrays and numpy arrays for its pointers."""
    mh = _mh()
    mh.check(getattr(mh.lib(), name)(_ctx().handle, *[a.ptr if isinstance(a, mh.DeviceArray) else a for a in args]))


def _run_own(s):
    import ctypes
    c = s["case"]
    kind = c["kind"]
    if kind == "dropout":
        _call("mmh_dropout", s["x"], s.get("residual"), c["n"], c["p"], s["key"], s["offset"], s["out"])
    elif kind == "dropout_bwd":
        _call("mmh_dropout_backward", s["dout"], c["n"], c["p"], s["key"], s["offset"], s["dx"])
    elif kind in ("ce", "ce_bwd"):
        loss = ctypes.c_float()
        targets = s["targets"].ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
        grads = [s["dx"], s["dw"]] if kind == "ce_bwd" else []
        _call("mmh_linear_cross_entropy" + ("_backward" if grads else ""), FORMS[c["form"]], s["x"], s["w"], targets,
              c["n"], c["d"], c["vocab"], IGNORE, *grads, ctypes.byref(loss))
        return dict(s["outs"], loss=loss.value)
    elif kind == "linear":
        _call("mmh_linear", FORMS[c["form"]], s["x"], s["w"], s["bias"], s.get("residual"), c["rows"], c["k"], c["n"],
              ACTIVATIONS[c["act"]], c["p"], s["key"], s["offset"], s.get("pre"), s["out"])
    else:
        _call("mmh_linear_backward", FORMS[c["form"]], s["x"], s["w"], s["pre"], s["dout"], c["rows"], c["k"], c["n"],
              ACTIVATIONS[c["act"]], c["p"], s["key"], s["offset"], s["dx"], s["dw"], s["dbias"])
    return s["outs"]


def _threshold(p):
    """Words below it are dropped: p as the f32 that the call takes, times 2^32."""
    return int(float(np.float32(p)) * 4294967296.0)


def _mul32(a, b):
    """High and low 32 bits of a constant times 32-bit values held in int64."""
    t = (b & 0xFFFF) * a
    u = (b >> 16) * a + (t >> 16)
    return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)


def _kept(n, p, key, offset):
    """Which of n values stay: Philox4x32-10, word i % 4 of block offset + i / 4."""
    j = torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda") + offset
    c = [j & 0xFFFFFFFF, (j >> 32) & 0xFFFFFFFF, torch.zeros_like(j), torch.zeros_like(j)]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        h0, l0 = _mul32(0xD2511F53, c[0])
        h1, l1 = _mul32(0xCD9E8D57, c[2])
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack(c, 1).reshape(-1)[:n] >= _threshold(p)


def _drop(x, p, key, offset):
    if p == 0.0:
        return x
    kept = _kept(x.numel(), p, key, offset).view(x.shape)
    return torch.where(kept, x * (1.0 / (1.0 - float(np.float32(p)))), torch.zeros_like(x))


R2 = math.sqrt(0.5)
C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def _act(a, z):
    if a == "relu":
        return torch.clamp(z, min=0.0)
    if a == "gelu":
        return z * 0.5 * (1.0 + torch.erf(z * R2))
    if a == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(C0 * (z + C1 * z * z * z)))
    if a == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(a, z):
    """d act / dz."""
    if a == "relu":
        return (z > 0).to(z.dtype)
    if a == "gelu":
        return 0.5 * (1.0 + torch.erf(z * R2)) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if a == "gelu_tanh":
        t = torch.tanh(C0 * (z + C1 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * C0 * (1.0 + 3.0 * C1 * z * z)
    if a == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    return torch.ones_like(z)


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s)
    kind = c["kind"]
    if kind in ("dropout", "dropout_bwd"):
        y = _drop(s["x" if kind == "dropout" else "dout"], c["p"], s["key"], s["offset"])
        return {"dx": y} if kind == "dropout_bwd" else {"out": y + s["residual"] if c["residual"] else y}
    x, w = s["x"], s["w"] if c["form"] == "nn" else s["w"].T  # [d, vocab] or [k, n]
    if kind == "linear":
        pre = x @ w + s["bias"]
        y = _drop(_act(c["act"], pre), c["p"], s["key"], s["offset"])
        out = {"out": y + s["residual"] if c["residual"] else y}
        return dict(out, pre=pre) if c["pre"] else out
    if kind == "linear_bwd":
        dpre = _drop(s["dout"], c["p"], s["key"], s["offset"]) * _act_grad(c["act"], s["pre"])
        dw = x.T @ dpre if c["form"] == "nn" else dpre.T @ x
        return {"dx": dpre @ w.T, "dw": dw, "dbias": dpre.sum(0, dtype=torch.float64).float()}
    targets = torch.from_numpy(s["targets"]).to("cuda").long()
    kept = targets != IGNORE
    count = kept.sum().clamp(min=1)
    at = targets.clamp(min=0)[:, None]
    z = x @ w
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    rows = (top + torch.log(total) - z.gather(1, at))[:, 0]
    loss = (torch.where(kept, rows, torch.zeros_like(rows)).double().sum() / count).float()
    if kind == "ce":
        return {"loss": loss}
    scale = (kept.float() / count)[:, None]
    dz = e / total * scale
    dz.scatter_add_(1, at, -scale)
    return {"loss": loss, "dx": dz @ w.T, "dw": x.T @ dz if c["form"] == "nn" else dz.T @ x}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    c = case
    kind = c["kind"]
    if kind in ("dropout", "dropout_bwd"):
        return {"bytes": 4.0 * c["n"] * (3 if c.get("residual") else 2), "flops": 2.0 * c["n"]}
    if kind in ("ce", "ce_bwd"):
        n, d, v = c["n"] * (1.0 - c["ignored"]), c["d"], c["vocab"]
        if kind == "ce":
            return {"bytes": 4.0 * (n * d + d * v), "flops": 2.0 * n * d * v}
        return {"bytes": 4.0 * (2 * n * d + 2 * d * v), "flops": 6.0 * n * d * v}
    r, k, n = c["rows"], c["k"], c["n"]
    if kind == "linear":
        return {"bytes": 4.0 * (r * k + k * n + n + r * n * (1 + c["residual"] + c["pre"])), "flops": 2.0 * r * k * n}
    return {"bytes": 4.0 * (2 * r * k + 2 * k * n + 2 * r * n + n), "flops": 4.0 * r * k * n}


# ---- the same in 64 bits -----------------------------------------------------------

def _mask64(n, p, key, offset):
    """The kept values of the generator in unsigned 64-bit products, on the host."""
    out = np.empty((n + 3) // 4 * 4, dtype=bool)
    low, drop = np.uint64(0xFFFFFFFF), np.uint64(math.floor(float(np.float32(p)) * 2.0 ** 32))
    half = np.uint64(32)
    for at in range(0, len(out) // 4, 1 << 18):
        j = np.arange(at, min(at + (1 << 18), len(out) // 4), dtype=np.uint64) + np.uint64(offset)
        x0, x1, x2, x3 = j & low, j >> half, np.zeros_like(j), np.zeros_like(j)
        for i in range(10):
            ka = np.uint64((key % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32)
            kb = np.uint64((key // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32)
            a, b = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
            x0, x1, x2, x3 = (b >> half) ^ x1 ^ ka, b & low, (a >> half) ^ x3 ^ kb, a & low
        for word, x in enumerate((x0, x1, x2, x3)):
            out[4 * at + word:4 * (at + len(j)):4] = x >= drop
    return torch.from_numpy(out[:n]).cuda()


def exact(case, seed):
    c = case
    kind = c["kind"]
    t, targets, key, offset = _drawn(c, seed)
    t = {n: v.double() for n, v in t.items()}

    def dropped(y):
        if c["p"] == 0.0:
            return y
        return y * _mask64(y.numel(), c["p"], key, offset).view(y.shape) / (1.0 - float(np.float32(c["p"])))

    if kind == "dropout":
        return {"out": dropped(t["x"]) + t.get("residual", 0.0)}
    if kind == "dropout_bwd":
        return {"dx": dropped(t["dout"])}
    x, w = t["x"].requires_grad_(), t["w"].requires_grad_()
    head = w if c["form"] == "nn" else w.T
    if kind in ("ce", "ce_bwd"):
        kept = np.flatnonzero(targets != IGNORE)
        if not len(kept):
            return {"loss": 0.0} if kind == "ce" else {"loss": 0.0, "dx": torch.zeros_like(x), "dw": torch.zeros_like(w)}
        total, dx, dw = 0.0, torch.zeros_like(x), torch.zeros_like(w)
        for at in range(0, len(kept), 512):  # some rows of logits at a time
            i = torch.from_numpy(kept[at:at + 512]).cuda()
            y = torch.from_numpy(targets[kept[at:at + 512]]).cuda().long()
            part = torch.nn.functional.cross_entropy(x[i] @ head, y, reduction="sum") / len(kept)
            total += float(part)
            if kind == "ce_bwd":
                gx, gw = torch.autograd.grad(part, (x, w))
                dx += gx
                dw += gw
        return {"loss": total} if kind == "ce" else {"loss": total, "dx": dx, "dw": dw}
    f = torch.nn.functional
    act = {"none": lambda z: z, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda z: f.gelu(z, approximate="tanh"), "silu": f.silu}[c["act"]]
    if kind == "linear":
        with torch.no_grad():
            pre = x @ head + t["bias"]
            out = {"out": dropped(act(pre)) + t.get("residual", 0.0)}
            return dict(out, pre=pre) if c["pre"] else out
    pre = t["pre"].requires_grad_()
    (dpre,) = torch.autograd.grad(dropped(act(pre)), pre, t["dout"])
    with torch.no_grad():
        dw = x.T @ dpre if c["form"] == "nn" else dpre.T @ x
        return {"dx": dpre @ head.T, "dw": dw, "dbias": dpre.sum(0)}
