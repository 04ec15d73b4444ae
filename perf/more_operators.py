"""Scoring tokens, learning from a teacher, and rotary positions, as cases that can be timed and compared.

Three operators: the log probabilities of given tokens with the entropy and the top alternatives of each row of logits
(mmh_token_logprobs and its backward), the distillation loss against a teacher's top logits (mmh_distillation and its
backward), and rotary positions in both layouts, over a part of the head, at given positions, from tables scaled for
long contexts (mmh_rotary_tables, mmh_rotary and its backward). With own = True a pass is the call of the C ABI that a
program makes; otherwise it is the same mathematics in elementary torch operations. All values are f32, as the
framework's are; token ids, positions and targets are on the host, where the framework takes them, and a teacher's ids
on the device, where mmh_token_logprobs leaves them. Logits are spread as a trained model's are: N(0, 2) and a few
tokens of each row well above the rest.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

IGNORE = -1
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def listed():
    return [
        # scoring one micro batch of the smallest preset, 2 x 32 tokens: a call that is all latency
        dict(name="logprobs_smoke", kind="logprobs", n=64, vocab=256, k=5, targets=True, ignored=0.0),
        # what four sequences answer with at one step, over a wide vocabulary: few rows, long ones
        dict(name="logprobs_step", kind="logprobs", n=4, vocab=131071, k=20, targets=False, ignored=0.0),
        # a teacher's top alternatives for the large preset's batch, 4 x 1024 tokens
        dict(name="logprobs_large", kind="logprobs", n=4096, vocab=32000, k=64, targets=True, ignored=0.0),
        # a policy's gradient with an entropy bonus over the same batch, prompts left out
        dict(name="logprobs_bwd", kind="logprobs_bwd", n=4096, vocab=32000, ignored=0.25),
        # the distillation loss of the tiny preset's evaluation batch, 8 x 256 tokens
        dict(name="distill_tiny", kind="distill", n=2048, vocab=4096, k=16, temperature=1.0, alpha=1.0, ignored=0.0, empty=0.0),
        # its gradient for one micro batch of the smallest preset: latency
        dict(name="distill_bwd_smoke", kind="distill_bwd", n=64, vocab=256, k=8, temperature=2.0, alpha=0.5, ignored=0.0, empty=0.0),
        # the large preset's training batch, 4 x 1024 tokens, both terms, softened
        dict(name="distill_bwd_large", kind="distill_bwd", n=4096, vocab=32000, k=64, temperature=2.0, alpha=0.5, ignored=0.0, empty=0.0),
        # a vocabulary of four times that, a ragged batch with padding, rows with fewer alternatives than slots
        dict(name="distill_bwd_wide", kind="distill_bwd", n=1021, vocab=131071, k=50, temperature=1.0, alpha=0.9, ignored=0.2, empty=0.3),
        # one token of each of eight sequences, each at its own far position: latency
        dict(name="rotary_step", kind="rotary", layout="half", b=8, t=1, h=16, hkv=8, hd=128, width=128, table=131072, positions=True),
        # the large preset's queries and keys, 4 x 1024 tokens
        dict(name="rotary_large", kind="rotary", layout="half", b=4, t=1024, h=16, hkv=8, hd=128, width=128, table=1024, positions=False),
        # gradients of packed documents: neighbouring pairs, half of an odd-sized head, odd lengths
        dict(name="rotary_bwd_ragged", kind="rotary_bwd", layout="interleaved", b=3, t=1021, h=12, hkv=4, hd=84, width=42, table=4096, positions=True),
        # tables for a context of 131072 tokens, each frequency scaled by its own part
        dict(name="rotary_tables_long", kind="rotary_tables", width=128, table=131072, scaling="parts", factor=8.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size in [lo, hi], spread over its logarithm: half of them multiples of 64 where there is room, the others as they fall."""
    v = _log(rng, lo, hi)
    return max(64, v // 64 * 64) if v >= 128 and rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "logprobs_bwd", "distill", "distill_bwd", "distill_bwd", "rotary", "rotary_bwd", "rotary_tables"])
    if kind == "rotary_tables":
        return dict(kind=kind, width=2 * rng.randint(1, 64), table=_log(rng, 1, 131072), scaling=rng.choice(list(SCALINGS)),
                    factor=rng.choice([1.0, 2.0, 8.0, round(rng.uniform(1.0, 32.0), 3)]))
    if kind in ("rotary", "rotary_bwd"):
        while True:
            b, t, hkv, hd = _log(rng, 1, 64), _log(rng, 1, 16384), _log(rng, 1, 16), rng.randint(2, 128)
            h = hkv * rng.choice([1, 2, 4, 8])
            if b * t * (h + hkv) * hd <= 4 * 4096 * 24 * 128:
                break
        width = hd // 2 * 2 if rng.random() < 0.5 else 2 * rng.randint(1, hd // 2)
        positions = rng.random() < 0.5
        return dict(kind=kind, layout=rng.choice(list(LAYOUTS)), b=b, t=t, h=h, hkv=hkv, hd=hd, width=width,
                    table=_log(rng, t, 131072), positions=positions)
    while True:
        n, vocab = _size(rng, 1, 8192), _size(rng, 64, 262144)
        if n * vocab <= 4096 * 32000:
            break
    ignored = rng.choice([0.0, 0.0, 0.1, 0.5])
    if kind == "logprobs":
        return dict(kind=kind, n=n, vocab=vocab, k=min(vocab, rng.choice([0, _log(rng, 1, 256)])), targets=rng.random() < 0.75, ignored=ignored)
    if kind == "logprobs_bwd":
        return dict(kind=kind, n=n, vocab=vocab, ignored=ignored)
    return dict(kind=kind, n=n, vocab=vocab, k=min(vocab, _log(rng, 1, 256)), temperature=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 5.0), 2)]),
                alpha=rng.choice([1.0, 0.5, round(rng.random(), 3)]), ignored=ignored, empty=rng.choice([0.0, 0.3]))


# ---- inputs --------------------------------------------------------------------

THETA = 10000.0  # (tables are built for bases from there to 100 times that)
TRAINED, LOW, HIGH = 8192, 1.0, 32.0  # rotary scaling by parts: the trained length, the turns between which it blends

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
        self.__cuda_array_interface__ = dict(shape=array.shape, typestr=array.dtype.str, data=(array.ptr, False), version=2)


def _amplitude(c):
    return 1.0 + 0.1 * math.log(c["factor"]) if c["scaling"] == "parts" else 1.0


def _frequencies(width, theta=THETA, scaling="none", factor=1.0):
    """w_i of the pairs, in 64 bits."""
    i = torch.arange(width // 2, dtype=torch.float64, device="cuda")
    base = theta * factor ** (width / (width - 2)) if scaling == "base" and width > 2 else theta
    w = torch.exp(i * (-2.0 / width * math.log(base)))
    if scaling == "linear":
        return w / factor
    if scaling == "parts":
        kept = torch.clamp((TRAINED / (2.0 * math.pi) * w - LOW) / (HIGH - LOW), 0.0, 1.0)
        return w * (kept + (1.0 - kept) / factor)
    return w


def _drawn(c, seed):
    """The inputs of a case, from the seed alone: torch tensors on the GPU, numpy arrays and numbers for what is on the host."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = np.random.default_rng(seed)
    kind = c["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if kind == "rotary_tables":
        return {"theta": float(np.float32(THETA * 100.0 ** r.random()))}
    if kind in ("rotary", "rotary_bwd"):
        b, t, hd = c["b"], c["t"], c["hd"]
        s = dict(q=normal(b, c["h"], t, hd), k=normal(b, c["hkv"], t, hd))
        angle = torch.arange(c["table"], dtype=torch.float64, device="cuda")[:, None] * _frequencies(c["width"])
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        if c["positions"]:  # documents that start anywhere in the context, one per sequence
            first = r.integers(0, c["table"] - t + 1, (b, 1))
            s["positions"] = (first + np.arange(t)).astype(np.int32)
        return s
    n, vocab = c["n"], c["vocab"]
    z = normal(n, vocab).mul_(2.0)
    ahead = min(8, vocab)
    at = torch.randint(vocab, (n, ahead), generator=g, device="cuda")
    z.scatter_add_(1, at, 4.0 + 3.0 * torch.rand(n, ahead, generator=g, device="cuda"))
    s = dict(logits=z)
    if c.get("targets", True):
        y = r.integers(0, vocab, n).astype(np.int32)
        top = at[:, 0].cpu().numpy()
        y = np.where(r.random(n) < 0.5, top, y).astype(np.int32)  # half of them tokens that the row holds likely
        y[r.random(n) < c["ignored"]] = IGNORE
        s["targets"] = y
    if kind == "logprobs_bwd":
        s["dlogprobs"], s["dentropy"] = normal(n), 0.01 * normal(n)
    if kind in ("distill", "distill_bwd"):
        k = c["k"]
        values, ids = torch.empty(n, k, device="cuda"), torch.empty(n, k, dtype=torch.int32, device="cuda")
        for i in range(0, n, 512):  # the teacher agrees with the student up to some noise
            v, j = torch.topk(z[i:i + 512] + normal(min(512, n - i), vocab), k)
            values[i:i + 512], ids[i:i + 512] = v, j.int()
        if c["empty"] > 0.0:  # rows whose last slots are not filled
            count = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
            some = torch.rand(n, 1, generator=g, device="cuda") < c["empty"]
            ids[some & (torch.arange(k, device="cuda")[None] >= count)] = -1
        s["teacher_ids"], s["teacher_logits"] = ids, values
    return s


def _outputs(c):
    """{name: (shape, type)} of the buffers that a program hands to the call."""
    kind = c["kind"]
    f, i = np.float32, np.int32
    if kind == "rotary_tables":
        return {n: ((c["table"], c["width"] // 2), f) for n in ("cos_out", "sin_out")}
    if kind in ("rotary", "rotary_bwd"):
        return {"q_out": ((c["b"], c["h"], c["t"], c["hd"]), f), "k_out": ((c["b"], c["hkv"], c["t"], c["hd"]), f)}
    if kind == "logprobs":
        out = {"entropy": ((c["n"],), f)}
        if c["targets"]:
            out["logprobs"] = ((c["n"],), f)
        if c["k"]:
            out["top_ids"], out["top_logprobs"] = ((c["n"], c["k"]), i), ((c["n"], c["k"]), f)
        return out
    return {} if kind == "distill" else {"dlogits": ((c["n"], c["vocab"]), f)}


def prepare(case, seed):
    c = case
    t = _drawn(c, seed)
    s = dict(case=c)
    if not own:
        s.update(t)
        return s
    ctx = _ctx()
    for name, v in t.items():
        if not isinstance(v, torch.Tensor):
            s[name] = v
            continue
        s[name] = ctx.empty(tuple(v.shape), np.int32 if v.dtype == torch.int32 else np.float32)
        torch.as_tensor(_Cuda(s[name]), device="cuda").copy_(v)
    outs = _outputs(c)
    for name, (shape, dtype) in outs.items():
        s[name] = ctx.empty(shape, dtype)
    s["outs"] = {name: torch.as_tensor(_Cuda(s[name]), device="cuda") for name in outs}
    torch.cuda.synchronize()  # the inputs are there before the context's own stream reads them
    return s


# ---- one pass ------------------------------------------------------------------

def _call(name, *args):
    """One entry point of the C ABI, with DeviceArrays and numpy arrays for its pointers."""
    import ctypes
    mh = _mh()

    def arg(a):
        if isinstance(a, mh.DeviceArray):
            return a.ptr
        return a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)) if isinstance(a, np.ndarray) else a

    mh.check(getattr(mh.lib(), name)(_ctx().handle, *[arg(a) for a in args]))


def _run_own(s):
    import ctypes
    c = s["case"]
    kind = c["kind"]
    if kind == "rotary_tables":
        _call("mmh_rotary_tables", c["width"], c["table"], s["theta"], SCALINGS[c["scaling"]], c["factor"], TRAINED, LOW, HIGH, _amplitude(c),
              s["cos_out"], s["sin_out"])
    elif kind in ("rotary", "rotary_bwd"):
        _call("mmh_rotary" if kind == "rotary" else "mmh_rotary_backward", LAYOUTS[c["layout"]], s["q"], s["k"], s.get("positions"),
              c["b"], c["h"], c["hkv"], c["t"], c["hd"], c["width"], c["table"], s["cos"], s["sin"], s["q_out"], s["k_out"])
    elif kind == "logprobs":
        _call("mmh_token_logprobs", s["logits"], s.get("targets"), c["n"], c["vocab"], IGNORE, c["k"], s.get("logprobs"), s["entropy"],
              s.get("top_ids"), s.get("top_logprobs"))
    elif kind == "logprobs_bwd":
        _call("mmh_token_logprobs_backward", s["logits"], s["targets"], c["n"], c["vocab"], IGNORE, s["dlogprobs"], s["dentropy"],
              s["dlogits"])
    else:
        loss = ctypes.c_float()
        grads = [s["dlogits"]] if kind == "distill_bwd" else []
        _call("mmh_distillation" + ("_backward" if grads else ""), s["logits"], s["targets"], c["n"], c["vocab"], IGNORE,
              s["teacher_ids"], s["teacher_logits"], c["k"], c["temperature"], c["alpha"], *grads, ctypes.byref(loss))
        return dict(s["outs"], loss=loss.value)
    return s["outs"]


def _rotate(x, cos, sin, layout, width):
    """x [b, h, t, hd] with its first `width` columns rotated by cos, sin [b or 1, 1, t, width / 2]."""
    out = x.clone()
    if layout == "half":
        a, b = x[..., :width // 2], x[..., width // 2:width]
        out[..., :width // 2] = a * cos - b * sin
        out[..., width // 2:width] = b * cos + a * sin
    else:
        a, b = x[..., 0:width:2], x[..., 1:width:2]
        out[..., 0:width:2] = a * cos - b * sin
        out[..., 1:width:2] = b * cos + a * sin
    return out


def _top(z, k):
    """The k largest of each row, the lowest ids first among equals: keys whose order is (value, -id)."""
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    last = z.shape[1] - 1
    key = order * (1 << 20) + (last - torch.arange(z.shape[1], device=z.device))
    best = torch.topk(key, k, dim=1).values
    return last - (best & ((1 << 20) - 1))


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s)
    kind = c["kind"]
    if kind == "rotary_tables":
        at = torch.arange(c["table"], dtype=torch.float64, device="cuda")
        angle = at[:, None] * _frequencies(c["width"], s["theta"], c["scaling"], float(np.float32(c["factor"])))
        a = float(np.float32(_amplitude(c)))
        return {"cos_out": (torch.cos(angle) * a).float(), "sin_out": (torch.sin(angle) * a).float()}
    if kind in ("rotary", "rotary_bwd"):
        if c["positions"]:
            at = torch.from_numpy(s["positions"]).to("cuda").long()
        else:
            at = torch.arange(c["t"], device="cuda")[None]
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        if kind == "rotary_bwd":
            sin = -sin
        return {"q_out": _rotate(s["q"], cos, sin, c["layout"], c["width"]), "k_out": _rotate(s["k"], cos, sin, c["layout"], c["width"])}
    z = s["logits"]
    n = c["n"]
    kept = torch.ones(n, dtype=torch.bool, device="cuda")
    if "targets" in s:
        y = torch.from_numpy(s["targets"]).to("cuda").long()
        kept = y != IGNORE
        y = y.clamp(min=0)[:, None]
    d = z - z.max(1, keepdim=True).values
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    if kind in ("logprobs", "logprobs_bwd"):
        entropy = (log_total - (e * d).sum(1, keepdim=True) / total)
        if kind == "logprobs_bwd":
            dl, dh = (torch.where(kept, s[v], torch.zeros_like(s[v]))[:, None] for v in ("dlogprobs", "dentropy"))
            dz = e / total * (-dl - dh * (d - log_total + entropy))
            dz.scatter_add_(1, y, dl)
            return {"dlogits": dz}
        zero = torch.zeros(n, device="cuda")
        out = {"entropy": torch.where(kept, entropy[:, 0], zero)}
        if c["targets"]:
            out["logprobs"] = torch.where(kept, (d.gather(1, y) - log_total)[:, 0], zero)
        if c["k"]:
            ids = _top(z, c["k"])
            values = d.gather(1, ids) - log_total
            out["top_ids"] = torch.where(kept[:, None], ids, torch.full_like(ids, -1)).int()
            out["top_logprobs"] = torch.where(kept[:, None], values, torch.full_like(values, -math.inf))
        return out
    tau, alpha = float(np.float32(c["temperature"])), float(np.float32(c["alpha"]))
    count = kept.sum().clamp(min=1)
    ids = s["teacher_ids"].long()
    filled = ids >= 0
    ids = ids.clamp(min=0)
    u = torch.where(filled, s["teacher_logits"] / tau, torch.full_like(s["teacher_logits"], -math.inf))
    u = u - u.max(1, keepdim=True).values
    q = torch.exp(u)
    q_total = q.sum(1, keepdim=True)
    q = q / q_total
    e_soft = torch.exp(d / tau)
    soft_total = e_soft.sum(1, keepdim=True)
    log_p = d.gather(1, ids) / tau - torch.log(soft_total)
    terms = torch.where(q > 0, q * (u - torch.log(q_total) - log_p), torch.zeros_like(q))
    rows = alpha * tau * tau * terms.sum(1) + (1.0 - alpha) * (log_total - d.gather(1, y))[:, 0]
    loss = (torch.where(kept, rows, torch.zeros_like(rows)).double().sum() / count).float()
    if kind == "distill":
        return {"loss": loss}
    weight = (kept.float() / count)[:, None]
    soft, hard = alpha * tau * weight, (1.0 - alpha) * weight
    dz = e_soft * (soft / soft_total) + e * (hard / total)
    dz.scatter_add_(1, ids, torch.where(filled, -soft * q, torch.zeros_like(q)))
    dz.scatter_add_(1, y, -hard)
    return {"loss": loss, "dlogits": dz}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    c = case
    kind = c["kind"]
    if kind == "rotary_tables":
        values = float(c["table"]) * c["width"]
        return {"bytes": 4.0 * values, "flops": 2.0 * values}
    if kind in ("rotary", "rotary_bwd"):
        heads = c["b"] * c["t"] * (c["h"] + c["hkv"])
        places = min(c["table"], c["b"] * c["t"]) if c["positions"] else c["t"]
        return {"bytes": 4.0 * (2.0 * heads * c["hd"] + places * c["width"]), "flops": 3.0 * heads * c["width"]}
    n, vocab = float(c["n"]), c["vocab"]
    rows = n * (1.0 - c["ignored"]) if c.get("targets", True) else n
    if kind == "logprobs":
        return {"bytes": 4.0 * (rows * vocab + 2 * n + 2 * n * c["k"]), "flops": 6.0 * rows * vocab}
    if kind == "logprobs_bwd":
        return {"bytes": 4.0 * (rows * vocab + n * vocab + 2 * n), "flops": 10.0 * rows * vocab}
    exps = 2 if c["temperature"] != 1.0 and 0.0 < c["alpha"] < 1.0 else 1
    if kind == "distill":
        return {"bytes": 4.0 * (rows * vocab + 2 * rows * c["k"]), "flops": 3.0 * exps * rows * vocab}
    return {"bytes": 4.0 * (rows * vocab + 2 * rows * c["k"] + n * vocab), "flops": 6.0 * exps * rows * vocab}


# ---- the same in 64 bits -----------------------------------------------------------

def _pairs64(x, turn, layout, width):
    """Pairs as complex numbers times turn [b or 1, 1, t, width / 2]."""
    x = x.double()
    head, rest = x[..., :width], x[..., width:]
    if layout == "half":
        z = torch.complex(*(v.contiguous() for v in head.split(width // 2, dim=-1))) * turn
        return torch.cat([z.real, z.imag, rest], dim=-1)
    z = torch.view_as_complex(head.contiguous().unflatten(-1, (width // 2, 2))) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), rest], dim=-1)


def exact(case, seed):
    c = case
    kind = c["kind"]
    if kind == "rotary_tables":
        m, width, factor = c["table"], c["width"], float(np.float32(c["factor"]))
        theta = _drawn(c, seed)["theta"]
        if c["scaling"] == "base" and width > 2:
            theta *= math.pow(factor, width / (width - 2.0))
        w = [math.pow(theta, -2.0 * i / width) for i in range(width // 2)]
        if c["scaling"] == "linear":
            w = [v / factor for v in w]
        if c["scaling"] == "parts":
            for i, v in enumerate(w):
                turns = TRAINED * v / (2.0 * math.pi)
                share = 1.0 if turns >= HIGH else 0.0 if turns <= LOW else (turns - LOW) / (HIGH - LOW)
                w[i] = share * v + (1.0 - share) * v / factor
        turn = torch.polar(torch.full((m, width // 2), float(np.float32(_amplitude(c))), dtype=torch.float64, device="cuda"),
                           torch.outer(torch.arange(m, dtype=torch.float64, device="cuda"), torch.tensor(w, dtype=torch.float64, device="cuda")))
        return {"cos_out": turn.real.contiguous(), "sin_out": turn.imag.contiguous()}
    t = _drawn(c, seed)
    if kind in ("rotary", "rotary_bwd"):
        turn = torch.complex(t["cos"].double(), t["sin"].double())
        if kind == "rotary_bwd":
            turn = turn.conj()
        turn = turn[torch.from_numpy(t["positions"]).long().cuda()] if c["positions"] else turn[None, :c["t"]]
        return {n + "_out": _pairs64(t[n], turn[:, None], c["layout"], c["width"]) for n in ("q", "k")}
    n = c["n"]
    y = torch.from_numpy(t["targets"]).long().cuda() if "targets" in t else None
    kept = y != IGNORE if y is not None else torch.ones(n, dtype=torch.bool, device="cuda")
    parts, loss = [], 0.0
    step = max(1, (1 << 24) // c["vocab"])
    tau, alpha = (float(np.float32(c[v])) if v in c else 1.0 for v in ("temperature", "alpha"))
    for i in range(0, n, step):  # some rows at a time
        at = slice(i, min(n, i + step))
        z = t["logits"][at].double().requires_grad_(kind.endswith("_bwd"))
        keep = kept[at]
        log_p = torch.log_softmax(z, 1)
        own_y = y[at].clamp(min=0) if y is not None else None
        if kind in ("logprobs", "logprobs_bwd"):
            entropy = -(log_p.exp() * log_p).sum(1) * keep
            given = log_p[torch.arange(len(z), device="cuda"), own_y] * keep if y is not None else None
            if kind == "logprobs_bwd":
                s = (given * t["dlogprobs"][at].double() + entropy * t["dentropy"][at].double()).sum()
                parts.append({"dlogits": torch.autograd.grad(s, z)[0]})
                continue
            out = {"entropy": entropy}
            if given is not None:
                out["logprobs"] = given
            if c["k"]:
                ids = torch.sort(t["logits"][at], dim=1, descending=True, stable=True).indices[:, :c["k"]]
                out["top_ids"] = torch.where(keep[:, None], ids, -1).int()
                out["top_logprobs"] = log_p.gather(1, ids).masked_fill(~keep[:, None], -math.inf)
            parts.append(out)
            continue
        ids = t["teacher_ids"][at].long()
        u = (t["teacher_logits"][at].double() / tau).masked_fill(ids < 0, -math.inf)
        log_q = torch.log_softmax(u, 1)
        q = log_q.exp()
        log_soft = torch.log_softmax(z / tau, 1).gather(1, ids.clamp(min=0))
        gap = (log_q.masked_fill(ids < 0, 0.0) - log_soft) * q
        row = alpha * tau ** 2 * gap.sum(1) - (1.0 - alpha) * log_p[torch.arange(len(z), device="cuda"), own_y]
        part = (row * keep).sum() / max(1, int(kept.sum()))
        loss += float(part)
        if kind == "distill_bwd":
            parts.append({"dlogits": torch.autograd.grad(part, z)[0]})
    out = {name: torch.cat([p[name] for p in parts]) for name in (parts[0] if parts else ())}
    return dict(out, loss=loss) if kind.startswith("distill") else out
