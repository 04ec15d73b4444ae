"""GPU checks of rotary positions in their several forms (rotary.hip), and a run of them together with the scoring and
distillation operators, as a student learns from a teacher."""
import numpy as np
import pytest

import midman_hip as mh
import scoring_oracle as R
from test_gpu_scoring import Box, empty, near, ptr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", ["none", "linear", "base", "parts"])
@pytest.mark.parametrize("width,positions,theta", [(2, 1, 1e4), (8, 33, 1e4), (42, 4097, 5e5), (128, 131072, 1e6), (250, 7, 1e4)])
def test_tables(ctx, width, positions, theta, scaling):
    print(f"\n[rotary_tables] {width} x {positions} {scaling}", flush=True)
    t = mh.ScaledRotaryTables(ctx, width, positions, theta, scaling, 8.0, 4096, 1.0, 32.0, 1.2)
    angle = np.outer(np.arange(positions), R.frequencies(width, theta, scaling, 8.0, 4096, 1.0, 32.0))
    a = float(np.float32(1.2))
    # half a step of f32, and the angle's own f64 roundings (a few 2^-53 of up to 2^17)
    for got, want in ((t.cos, np.cos(angle) * a), (t.sin, np.sin(angle) * a)):
        near(got.numpy(), want, R.U * np.abs(want) + 16 * 2.0 ** -53 * (1 + angle), "table")


def test_plain_tables_are_the_ropes(ctx):
    for width, positions in ((16, 64), (128, 2048)):
        a, b = mh.RotaryTables(ctx, width, positions), mh.ScaledRotaryTables(ctx, width, positions)
        for x, y in ((a.cos, b.cos), (a.sin, b.sin)):
            x, y = x.numpy(), y.numpy()
            assert np.abs(x - y).max() <= 2 * R.U and (x == y).mean() > 0.999


# (b, h, hkv, t, hd, width): single tokens, odd heads and lengths, parts of heads, whole ones
SHAPES = [(1, 1, 1, 1, 2, 2), (8, 16, 8, 1, 128, 128), (2, 4, 2, 33, 64, 64), (3, 6, 3, 21, 84, 42), (2, 3, 1, 17, 7, 6), (1, 2, 2, 130, 96, 10),
          (2, 5, 5, 9, 33, 2), (2, 8, 2, 513, 80, 80), (1, 1, 1, 1000, 130, 128), (40, 2, 1, 1, 20, 12), (2, 2, 2, 3, 1000, 1000), (1, 3, 1, 5, 72, 36)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_rotary(ctx, i, layout):
    b, h, hkv, t, hd, width = SHAPES[i]
    r = np.random.default_rng(i)
    table = t + 50
    tables = mh.ScaledRotaryTables(ctx, width, table, 1e4, "linear", 2.0)
    cos, sin = tables.cos.numpy(), tables.sin.numpy()
    q, k = (r.standard_normal((b, x, t, hd)).astype(np.float32) for x in (h, hkv))
    for positions in (None, r.integers(0, table, (b, t)).astype(np.int32)):
        at = np.broadcast_to(np.arange(t), (b, t)) if positions is None else positions
        c, s = cos[at][:, None], sin[at][:, None]
        for back in (False, True):
            name = "mmh_rotary" + ("_backward" if back else "")
            want = [R.rotate(x, c, s, layout, width, back) for x in (q, k)]
            for shift in (0, 1, 2, 3):
                print(f"\n[rotary] {SHAPES[i]} {layout} back={back} positions={positions is not None} shift={shift}", flush=True)
                Q, K, C, S = (Box(ctx, x, shift) for x in (q, k, cos, sin))
                inplace = (shift + back) % 2 == 1
                QO, KO = (Q, K) if inplace else (empty(ctx, q.shape, shift), empty(ctx, k.shape, (shift + 1) % 4))
                mh.check(getattr(mh.lib(), name)(ctx.handle, mh.ROTARY_LAYOUTS[layout], Q.ptr, K.ptr, ptr(positions), b, h, hkv, t, hd, width,
                                                 table, C.ptr, S.ptr, QO.ptr, KO.ptr))
                assert np.array_equal(QO.numpy(), want[0]) and np.array_equal(KO.numpy(), want[1])
                if not inplace:
                    assert np.array_equal(Q.numpy(), q) and np.array_equal(K.numpy(), k)
    # one of them alone
    tables_args = (tables, layout, positions)
    q_out, none = mh.rotary(ctx, ctx.to_device(q), None, *tables_args)
    assert none is None and np.array_equal(q_out.numpy(), R.rotate(q, c, s, layout, width))
    none, k_out = mh.rotary_backward(ctx, None, ctx.to_device(k), *tables_args)
    assert none is None and np.array_equal(k_out.numpy(), R.rotate(k, c, s, layout, width, True))


def test_half_layout_has_the_bits_of_apply_rope(ctx):
    x = np.random.default_rng(0).standard_normal((3, 4, 65, 64)).astype(np.float32)
    tables = mh.RotaryTables(ctx, 64, 80)
    X = ctx.to_device(x)
    q, _ = mh.rotary(ctx, X, None, tables)
    assert np.array_equal(q.numpy(), mh.apply_rope(ctx, X, tables).numpy())
    dq, _ = mh.rotary_backward(ctx, X, None, tables)
    assert np.array_equal(dq.numpy(), mh.apply_rope_backward(ctx, X, tables).numpy())


def test_values_that_are_not_finite_stay_in_their_pairs(ctx):
    x = np.ones((1, 1, 4, 10), np.float32)
    x[0, 0, 1, 2], x[0, 0, 2, 9] = np.nan, np.inf
    tables = mh.ScaledRotaryTables(ctx, 8, 4)
    for layout, pair in (("half", [2, 6]), ("interleaved", [2, 3])):
        out = mh.rotary(ctx, ctx.to_device(x), None, tables, layout)[0].numpy()
        assert np.argwhere(np.isnan(out[0, 0])).tolist() == [[1, j] for j in pair]
        assert out[0, 0, 2, 9] == np.inf and np.isfinite(np.delete(out[0, 0, 2], 9)).all()


def test_positions_of_queued_calls_are_each_calls_own(ctx):
    r = np.random.default_rng(2)
    x = r.standard_normal((16, 2, 100, 32)).astype(np.float32)
    X, tables = ctx.to_device(x), mh.ScaledRotaryTables(ctx, 32, 500)
    cos, sin = tables.cos.numpy(), tables.sin.numpy()
    got, want = [], []
    for _ in range(10):
        at = r.integers(0, 500, (16, 100)).astype(np.int32)
        want.append(R.rotate(x, cos[at][:, None], sin[at][:, None], "half", 32))
        got.append(mh.rotary(ctx, X, None, tables, positions=at)[0])
        at[:] = 0
    for g, w in zip(got, want):
        assert np.array_equal(g.numpy(), w)


def test_a_student_learns_from_a_teacher(ctx):
    """One attention layer and a head, twice: the teacher's with neighbouring pairs, a part of the head and scaled
    frequencies, its top alternatives, and the student's loss and gradients through its head, attention and rotary
    positions, against the same program in 64 bits under autograd."""
    import torch
    b, t, h, hkv, hd, vocab, k = 2, 48, 4, 2, 32, 2000, 40
    d, kv, n = h * hd, hkv * hd, b * t
    r = np.random.default_rng(7)

    def weights():
        w = {m: (r.standard_normal((d, c)) / np.sqrt(d)).astype(np.float32) for m, c in (("q", d), ("k", kv), ("v", kv))}
        w["head"] = (r.standard_normal((d, vocab)) * (4.0 / np.sqrt(d))).astype(np.float32)
        return w

    x = r.standard_normal((n, d)).astype(np.float32)
    y = r.integers(0, vocab, n).astype(np.int32)
    y[5:9] = -1
    start = r.integers(0, 400, (b, 1))
    positions = (start + np.arange(t)).astype(np.int32)
    tw, sw = weights(), weights()
    X = ctx.to_device(x)

    def heads(a, m):  # [n, m hd] -> [b, m, t, hd]
        return np.ascontiguousarray(a.reshape(b, t, m, hd).transpose(0, 2, 1, 3))

    def forward(w, tables, layout):
        W = {m: ctx.to_device(a) for m, a in w.items()}
        q, key, v = (ctx.to_device(heads(mh.matmul(ctx, X, W[m]).numpy(), c)) for m, c in (("q", h), ("k", hkv), ("v", hkv)))
        q, key = mh.rotary(ctx, q, key, tables, layout, positions)
        o = mh.causal_attention(ctx, q, key, v).numpy()
        o = ctx.to_device(np.ascontiguousarray(o.transpose(0, 2, 1, 3)).reshape(n, d))
        return W, q, key, v, o, mh.matmul(ctx, o, W["head"])

    teacher_tables = mh.ScaledRotaryTables(ctx, 16, 512, 1e4, "parts", 4.0, 128, 1.0, 8.0, 1.1)
    top = mh.token_logprobs(ctx, forward(tw, teacher_tables, "interleaved")[-1], y, k=k)
    tables = mh.ScaledRotaryTables(ctx, 32, 512, 1e4)
    W, q, key, v, o, logits = forward(sw, tables, "half")
    loss, dz = mh.distillation_backward(ctx, logits, top.top_ids, top.top_logprobs, y, 2.0, 0.7)
    do, dhead = _matmul_backward(ctx, o, W["head"], dz)
    dO = ctx.to_device(heads(do, h))
    dq, dk, dv = mh.causal_attention_backward(ctx, q, key, v, dO)
    dq, dk = mh.rotary_backward(ctx, dq, dk, tables, "half", positions)
    got = {"head": dhead}
    for m, g in (("q", dq), ("k", dk), ("v", dv)):
        flat = np.ascontiguousarray(g.numpy().transpose(0, 2, 1, 3)).reshape(n, -1)
        got[m] = _matmul_backward(ctx, X, W[m], ctx.to_device(flat))[1]

    p = {m: torch.tensor(a, dtype=torch.float64, requires_grad=True) for m, a in sw.items()}
    xx = torch.tensor(x, dtype=torch.float64)
    at = torch.tensor(positions).long()
    angle = at[:, None, :, None] * torch.tensor(R.frequencies(32, 1e4))
    cos, sin = torch.cos(angle), torch.sin(angle)

    def split(a, m):
        return a.reshape(b, t, m, hd).transpose(1, 2)

    def rope(a):
        u, w = a[..., :16], a[..., 16:]
        return torch.cat([u * cos - w * sin, w * cos + u * sin], -1)

    qq, kk, vv = rope(split(xx @ p["q"], h)), rope(split(xx @ p["k"], hkv)), split(xx @ p["v"], hkv)
    kk, vv = (a.repeat_interleave(h // hkv, 1) for a in (kk, vv))
    sc = (qq @ kk.transpose(-1, -2).contiguous()) / np.sqrt(hd)
    sc = sc.masked_fill(torch.ones(t, t, dtype=torch.bool).triu(1), -np.inf)
    zz = ((torch.softmax(sc, -1) @ vv).transpose(1, 2).reshape(n, d)) @ p["head"]
    keep = torch.tensor(y != -1)
    u = torch.tensor(np.where(np.isfinite(top.top_logprobs.numpy()), top.top_logprobs.numpy(), 0.0), dtype=torch.float64)
    qt = torch.softmax(u / 2.0, -1)
    ids = torch.tensor(top.top_ids.numpy()).long().clamp(min=0)
    kl = (qt * (torch.log(qt) - torch.log_softmax(zz / 2.0, -1).gather(1, ids))).sum(-1)
    ce = -torch.log_softmax(zz, -1).gather(1, torch.tensor(y).long().clamp(min=0)[:, None])[:, 0]
    alpha = float(np.float32(0.7))
    want = ((alpha * 4.0 * kl + (1 - alpha) * ce) * keep).sum() / keep.sum()
    want.backward()
    assert abs(loss - want.item()) <= 1e-4 * abs(want.item())
    for m in got:  # the model's own tolerance for gradients: 2e-3 of each parameter's largest
        g = p[m].grad.numpy()
        assert np.abs(got[m] - g).max() <= 2e-3 * np.abs(g).max(), m


def _matmul_backward(ctx, a, w, dc):
    """(da, dw) of a w as host arrays."""
    rows, k = a.shape
    da, dw = ctx.empty(a.shape), ctx.empty(w.shape)
    mh.check(mh.lib().mmh_matmul_backward(ctx.handle, a.ptr, w.ptr, dc.ptr, da.ptr, dw.ptr, rows, k, w.shape[1]))
    return da.numpy(), dw.numpy()
