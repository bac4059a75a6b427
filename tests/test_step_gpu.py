"""The decode operators on the GPU against their formulas in 64 bits (written out in numpy), at the sizes,
slots, pages and masks where they can go wrong; and a run of them together behind a prefill.

A rounding to bf16 is off by at most half a step, 2^-8 of the value, one to float32 by 2^-24; the
tolerances below count those."""
import ctypes as C

import numpy as np
import pytest

import oracle as O
from helpers import bf, f32, ulp_diff
from system1_omni_b200 import lib as L

pytestmark = pytest.mark.gpu

D = 128
HALF = 2.0 ** -8        # half a bf16 step, relative
EPS = 2.0 ** -24
NAN = np.uint16(0x7fc0)


def up(a, st):
    return L.to_device(np.ascontiguousarray(a), st)


def ints(a, st):
    return None if a is None else up(np.asarray(a, np.int32), st)


def at(buf):
    return None if buf is None else buf.at()


def down(buf, shape, st, dtype=np.uint16):
    return L.from_device(buf, shape, dtype, st)


def status():
    return L.device_status()


@pytest.fixture(autouse=True)
def clean_status(cs1, stream):
    status()
    yield
    assert status() == (0, 0, 0)        # a test that provokes a code reads it itself


# ---- delta rule ----

def delta_inputs(rows, H, HK, slots, seed):
    rng = np.random.default_rng(seed)
    n = rng.standard_normal
    return dict(q=bf(n((rows, HK, D))), k=bf(n((rows, HK, D))), v=bf(n((rows, H, D))), g=-np.exp(n((rows, H)) - 1).astype(np.float32),
                beta=bf(1 / (1 + np.exp(-n((rows, H))))), states=(n((slots, H, D, D)) * 0.3).astype(np.float32))


def delta_formula(x, start, si, so, H, HK, scale):
    """Outputs, states and per-element error bounds."""
    q, k, v, beta = (f32(x[m]).astype(np.float64) for m in ("q", "k", "v", "beta"))
    g, states = x["g"].astype(np.float64), x["states"].astype(np.float64)
    new, o, tol_o, tol_s = states.copy(), np.full(v.shape, np.nan), np.zeros(v.shape), np.zeros(states.shape)
    head = np.arange(H) // (H // HK)
    for i in range(len(so)):
        if so[i] < 0:
            continue
        S = states[si[i]].copy() if si[i] >= 0 else np.zeros((H, D, D))
        err = np.zeros((H, D))       # of a column of S, in the 2-norm
        for r in range(start[i], start[i + 1]):
            kk = k[r, head] / np.sqrt((k[r, head] ** 2).sum(-1, keepdims=True) + 1e-6)
            qq = q[r, head] / np.sqrt((q[r, head] ** 2).sum(-1, keepdims=True) + 1e-6) * scale
            S = S * np.exp(g[r])[:, None, None]
            d = beta[r][:, None] * (v[r] - np.einsum("hi,hij->hj", kk, S))
            # |k| <= 1, so a product over the keys is at most the column's norm; its 128 terms go through 35
            # sums, and the norm, exp and scaling before them through some 13 more roundings: 48 in all, the
            # same again for the update. I - beta k k^T and the decay enlarge no error that came in.
            size = np.sqrt((S ** 2).sum(1)) + np.abs(v[r]) + np.abs(d)
            err = err + 96 * EPS * size
            S = S + kk[:, :, None] * d[:, None, :]
            o[r] = np.einsum("hi,hij->hj", qq, S)
            tol_o[r] = HALF * np.abs(o[r]) + scale * (err + 48 * EPS * size) * 1.01
        new[so[i]], tol_s[so[i]] = S, err[:, None, :] + EPS * np.abs(S)
    return o, new, tol_o, tol_s


def run_delta(cs1, st, x, start, si, so, H, HK, scale, stride=None, rows=None, fill=0x4242):
    n_slots, nseq = len(x["states"]), len(so)
    stride = stride or H * D * D
    rows = len(x["v"]) if rows is None else rows
    pool = np.full((n_slots, stride), 7.0, np.float32)
    pool[:, :H * D * D] = x["states"].reshape(n_slots, -1)
    d = {m: up(x[m], st) for m in ("q", "k", "v", "g", "beta")}
    o = up(np.full(x["v"].shape, fill, np.uint16), st)
    pd = up(pool, st)
    s, a, b = ints(start, st), ints(si, st), ints(so, st)
    L.check(cs1.s1_gdn_step(d["q"].at(), d["k"].at(), d["v"].at(), d["g"].at(), d["beta"].at(), o.at(), rows, H, HK, scale, pd.at(), n_slots,
                            stride, at(s), a.at(), b.at(), nseq, st.handle), "step")
    got = down(pd, pool.shape, st, np.float32)
    assert (got[:, H * D * D:] == 7.0).all()
    return down(o, x["v"].shape, st), got[:, :H * D * D].reshape(x["states"].shape)


@pytest.mark.parametrize("lens,H,HK,case", [
    ([1], 1, 1, "own"), ([1], 32, 16, "own"), ([1] * 5, 6, 2, "own"), ([1] * 40, 3, 1, "own"), ([3, 0, 1, 17, 2], 4, 2, "own"),
    ([2, 5, 1], 48, 16, "shared"), ([1, 1, 1], 4, 4, "zeros"), ([2, 1, 4, 1], 6, 3, "mixed"), ([1] * 300, 2, 1, "own"),
    ([130], 2, 2, "own"), ([0, 0], 4, 2, "shared"), ([1] * 3, 5, 5, "stride")])
def test_delta_rule_step_matches_the_formula(cs1, stream, lens, H, HK, case):
    nseq, rows = len(lens), sum(lens)
    rng = np.random.default_rng(H * 1000 + nseq)
    slots = rng.permutation(nseq + 4)
    so = slots[:nseq].copy()
    si = {"own": so, "shared": np.full(nseq, slots[nseq]), "zeros": np.full(nseq, -1), "stride": so}.get(case, so).copy()
    if case == "mixed":
        si = np.array([slots[nseq], -1, so[2], slots[nseq]])
        so[3] = -1                      # sits out
    start = None if all(n == 1 for n in lens) else np.concatenate([[0], np.cumsum(lens)])
    bounds = np.arange(nseq + 1) if start is None else start
    x = delta_inputs(rows, H, HK, nseq + 4, 5)
    scale = D ** -0.5 if case != "zeros" else 0.37
    want, states, tol_o, tol_s = delta_formula(x, bounds, si, so, H, HK, scale)
    got, new = run_delta(cs1, stream, x, start, si, so, H, HK, scale, stride=H * D * D + 12 if case == "stride" else None)
    skipped = np.isnan(want)
    assert (got[skipped] == 0x4242).all()
    err = np.abs(f32(got).astype(np.float64) - want)[~skipped]
    assert (err <= tol_o[~skipped]).all(), err.max()
    err = np.abs(new.astype(np.float64) - states)
    assert (err <= tol_s).all(), (err - tol_s).max()      # the slots that nobody writes keep their bits: tolerance 0
    again = run_delta(cs1, stream, x, start, si, so, H, HK, scale, stride=H * D * D + 12 if case == "stride" else None)
    assert (again[0] == got).all() and (again[1] == new).all()


def test_delta_rule_step_agrees_with_the_oracle_and_the_prefill(cs1, stream):
    """Token by token from zeros is the oracle's recurrence, and a prefill of 64 tokens followed by steps is a longer prefill."""
    t, n, H, HK = 64, 9, 6, 2
    q, k, v, g, beta = (a.reshape(t + n, -1) for a in __import__("helpers").gdn_inputs(t + n, H, HK, 0.3, 1.0))
    want, s_want = O.gdn_recurrent_f64(q, k, v, g, beta, t + n, H, HK, want_state=True)
    dv = {m: up(a, stream) for m, a in dict(q=q, k=k, v=v, g=g, beta=beta).items()}
    o = L.DeviceBuffer((t + n) * H * D * 2)
    ws = L.DeviceBuffer(cs1.cs1_gdn_workspace_floats(t, H) * 4)
    pool = L.DeviceBuffer(2 * H * D * D * 4)
    L.check(cs1.cs1_gdn_prefill_x(dv["q"].at(), dv["k"].at(), dv["v"].at(), dv["g"].at(), dv["beta"].at(), o.at(), ws.at(), t, H, HK, D ** -0.5,
                                  None, pool.at(), stream.handle), "prefill")
    start, si, so = ints([t, t + n, t + n], stream), ints([0, -1], stream), ints([0, 1], stream)
    L.check(cs1.s1_gdn_step(dv["q"].at(), dv["k"].at(), dv["v"].at(), dv["g"].at(), dv["beta"].at(), o.at(), t + n, H, HK, D ** -0.5, pool.at(), 2,
                            H * D * D, start.at(), si.at(), so.at(), 2, stream.handle), "step")
    got = f32(down(o, (t + n, H, D), stream))
    # the prefill's own gate: 2e-2 of the largest value (its operands go through bf16)
    assert np.abs(got - want).max() <= 2e-2 * np.abs(want).max()
    states = down(pool, (2, H, D, D), stream, np.float32)
    assert np.abs(states[0] - s_want).max() <= 2e-2 * np.abs(s_want).max()
    assert (states[1] == 0).all()       # an empty sequence from zeros leaves zeros
    # all of it by steps, from zeros, against the oracle: float32 against 64 bits
    x = dict(q=q, k=k, v=v.reshape(t + n, H, D), g=g, beta=beta, states=np.ones((1, H, D, D), np.float32))
    f, s, tol_o, tol_s = delta_formula(dict(x, q=q.reshape(-1, HK, D), k=k.reshape(-1, HK, D)), [0, t + n], [-1], [0], H, HK, D ** -0.5)
    assert np.abs(f - want).max() < 1e-12 * np.abs(want).max() + 1e-12
    got, new = run_delta(cs1, stream, x, [0, t + n], [-1], [0], H, HK, D ** -0.5)
    assert (np.abs(f32(got) - want) <= tol_o).all()
    assert (np.abs(new[0] - s_want) <= tol_s[0]).all()


@pytest.mark.parametrize("start,si,so,code,live", [
    (None, [0, 9, 2], [0, 1, 2], 61, [0, 2]),                   # a slot behind the pool, read
    (None, [0, 1, 2], [0, 1, 6], 61, [0, 1]),                   # and written
    (None, [0, 1, 1], [0, 1, 2], 62, [0]),                      # 1 writes what 2 begins with
    (None, [0, 1, 2], [4, 4, 2], 62, [2]),                      # one slot twice
    ([0, 1, 4, 5], [0, 1, 2], [0, 1, 2], 60, [0]),              # rows behind the operands
    ([0, 2, 1, 1], [0, 1, 2], [0, 1, 2], 60, [0, 2]),           # rows that run backwards
    ([-1, 1, 2, 3], [0, 1, 2], [0, 1, 2], 60, [1, 2])])
def test_delta_rule_step_refuses_sequences_on_the_device(cs1, stream, start, si, so, code, live):
    H, HK = 4, 2
    x = delta_inputs(3, H, HK, 5, 8)
    got, new = run_delta(cs1, stream, x, start, si, so, H, HK, 1.0)
    assert status() == (0, 0, code)
    bounds = np.arange(4) if start is None else np.array(start)
    keep = [so[i] if i in live else -1 for i in range(3)]
    want, states, tol_o, tol_s = delta_formula(x, bounds, si, keep, H, HK, 1.0)
    skipped = np.isnan(want)
    assert (got[skipped] == 0x4242).all()
    assert (np.abs(f32(got) - want)[~skipped] <= tol_o[~skipped]).all()
    assert (np.abs(new - states) <= tol_s).all()


def test_delta_rule_step_offsets_pass_32_bits(cs1, stream):
    H, HK = 2, 1
    stride = (1 << 30) + 4          # floats: the third slot begins behind 2^31 elements
    x = delta_inputs(2, H, HK, 3, 3)
    pool = L.DeviceBuffer((2 * stride + H * D * D) * 4)
    for i in range(3):
        L.check(cs1.cs1_upload(pool.at(i * stride * 4), x["states"][i].ctypes.data, x["states"][i].nbytes, stream.handle), "upload")
    d = {m: up(x[m], stream) for m in ("q", "k", "v", "g", "beta")}
    o = L.DeviceBuffer(2 * H * D * 2)
    si, so = ints([0, 1], stream), ints([2, 1], stream)
    L.check(cs1.s1_gdn_step(d["q"].at(), d["k"].at(), d["v"].at(), d["g"].at(), d["beta"].at(), o.at(), 2, H, HK, 1.0, pool.at(), 3, stride, None,
                            si.at(), so.at(), 2, stream.handle), "step")
    want, states, tol_o, tol_s = delta_formula(x, [0, 1, 2], [0, 1], [2, 1], H, HK, 1.0)
    assert (np.abs(f32(down(o, (2, H, D), stream)) - want) <= tol_o).all()
    for i in range(3):
        got = L.from_device(pool, (H, D, D), np.float32, stream, offset_bytes=i * stride * 4)
        assert (np.abs(got - states[i]) <= tol_s[i]).all()


# ---- convolution and gates ----

def conv_case(rows, kd, vd, H, slots, pad, seed):
    rng = np.random.default_rng(seed)
    ch = 2 * kd + vd
    ld = (ch + 2 * H + 7) // 8 * 8 + pad
    n = rng.standard_normal
    return dict(x=bf(n((rows, ld))), ld=ld, w=bf(n((ch, 4)) * 0.4), al=bf(rng.uniform(0, 2.7, H)), dt=bf(n(H) * 0.2),
                tails=bf(n((slots, 3, ch))), kd=kd, vd=vd, H=H, ch=ch)


def run_conv(cs1, st, c, start, si, so, stride=None, rows=None):
    rows = len(c["x"]) if rows is None else rows
    n, ch, H, slots = len(c["x"]), c["ch"], c["H"], len(c["tails"])
    stride = stride or 3 * ch
    pool = np.full((slots, stride), 0x1234, np.uint16)
    pool[:, :3 * ch] = c["tails"].reshape(slots, -1)
    x, w, al, dt, pd = (up(a, st) for a in (c["x"], c["w"], c["al"], c["dt"], pool))
    outs = {m: up(np.full((n, width), 0x4242, np.uint16), st) for m, width in (("q", c["kd"]), ("k", c["kd"]), ("v", c["vd"]), ("beta", H))}
    g = up(np.full((n, H), 99.0, np.float32), st)
    s, a, b = ints(start, st), ints(si, st), ints(so, st)
    L.check(cs1.s1_gdn_conv_gates_step(x.at(), c["ld"], w.at(), outs["q"].at(), outs["k"].at(), outs["v"].at(), rows, c["kd"], c["vd"],
                                       x.at(2 * ch), x.at(2 * (ch + H)), al.at(), dt.at(), outs["beta"].at(), g.at(), H, pd.at(), slots,
                                       stride, at(s), a.at(), b.at(), len(so), st.handle), "conv step")
    got = down(pd, pool.shape, st)
    assert (got[:, 3 * ch:] == 0x1234).all()
    res = {m: down(o, (n, o.nbytes // 2 // max(n, 1)), st) for m, o in outs.items()}
    return res, down(g, (n, H), st, np.float32), got[:, :3 * ch].reshape(c["tails"].shape)


def conv_formula(c, start, si, so):
    x, w = f32(c["x"]).astype(np.float64), f32(c["w"]).astype(np.float64)
    n, ch, H = len(x), c["ch"], c["H"]
    y, bound, tails = np.full((n, ch), np.nan), np.zeros((n, ch)), c["tails"].copy()
    for i in range(len(so)):
        if so[i] < 0:
            continue
        raw = np.concatenate([c["tails"][si[i]] if si[i] >= 0 else np.zeros((3, ch), np.uint16), c["x"][start[i]:start[i + 1], :ch]])
        line = f32(raw).astype(np.float64)
        for t in range(start[i], start[i + 1]):
            win = line[t - start[i]: t - start[i] + 4]
            y[t] = (win * w.T).sum(0)
            bound[t] = np.abs(win * w.T).sum(0)
        tails[so[i]] = raw[-3:]
    out = y / (1 + np.exp(-y))
    # 4 products and sums in float32; SiLU's slope is below 1.1, its exp and division are good to a few 2^-21
    tol = HALF * np.abs(out) + 1.1 * 8 * EPS * bound + 2.0 ** -19 * np.abs(out)
    live = ~np.isnan(y[:, 0])
    b, a = x[:, ch:ch + H], x[:, ch + H:ch + 2 * H] + f32(c["dt"]).astype(np.float64)
    beta = 1 / (1 + np.exp(-b))
    g = -np.exp(f32(c["al"]).astype(np.float64)) * np.logaddexp(a, 0)
    return out, tol, live, beta, g, tails, y


@pytest.mark.parametrize("lens,kd,vd,H,case,pad", [
    ([1], 2048, 4096, 32, "own", 4096), ([1] * 7, 128, 384, 3, "own", 0), ([2, 0, 5, 1, 3, 4], 256, 512, 4, "own", 8),
    ([1, 2, 3], 128, 128, 1, "shared", 0), ([1, 2, 3, 4], 8, 16, 2, "zeros", 0), ([3, 1, 1], 1024, 1032, 5, "mixed", 16),
    ([1] * 260, 16, 24, 3, "own", 0), ([40, 1], 128, 256, 2, "stride", 0)])
def test_convolution_step_matches_the_formula(cs1, stream, lens, kd, vd, H, case, pad):
    nseq, rows = len(lens), sum(lens)
    rng = np.random.default_rng(rows)
    slots = rng.permutation(nseq + 3)
    so = slots[:nseq].copy()
    si = {"shared": np.full(nseq, slots[nseq]), "zeros": np.full(nseq, -1)}.get(case, so).copy()
    if case == "mixed":
        si[0], so[2] = slots[nseq], -1
    start = None if all(n == 1 for n in lens) else np.concatenate([[0], np.cumsum(lens)])
    bounds = np.arange(nseq + 1) if start is None else start
    c = conv_case(rows, kd, vd, H, nseq + 3, pad, 3)
    got, g, tails = run_conv(cs1, stream, c, start, si, so, stride=3 * c["ch"] + 8 if case == "stride" else None)
    want, tol, live, beta, gw, tw, _ = conv_formula(c, bounds, si, so)
    all_got = np.concatenate([got["q"], got["k"], got["v"]], 1)
    assert (all_got[~live] == 0x4242).all() and (got["beta"][~live] == 0x4242).all() and (g[~live] == 99.0).all()
    err = np.abs(f32(all_got).astype(np.float64) - want)[live]
    assert (err <= tol[live]).all(), (err - tol[live]).max()
    # sigmoid of a bf16 in float32: expf, sum and quotient good to 2^-21, then bf16
    assert (np.abs(f32(got["beta"]) - beta)[live] <= (HALF + 2.0 ** -20) * beta[live]).all()
    # the sum a + dt is rounded by 2^-24 of |a| + |dt|, softplus has slope <= 1 and, where small, is as steep
    # as it is large; exp, log1p and two products: 2^-20
    h = np.abs(f32(c["x"])[:, c["ch"] + H:c["ch"] + 2 * H]) + np.abs(f32(c["dt"]))
    assert (np.abs(g - gw)[live] <= (np.abs(gw) * (2.0 ** -20 + EPS * h))[live] + 1e-30).all()
    assert (tails == tw).all()


def test_convolution_step_continues_the_prefill(cs1, stream):
    """The rows of the one-launch prefill operator, within its rounding of the convolution before the SiLU."""
    t, n, kd, vd, H = 20, 6, 256, 512, 4
    c = conv_case(t + n, kd, vd, H, 1, 0, 9)
    x, w, al, dt = (up(a, stream) for a in (c["x"], c["w"], c["al"], c["dt"]))
    out = {m: L.DeviceBuffer((t + n) * width * 2) for m, width in (("q", kd), ("k", kd), ("v", vd), ("beta", H))}
    g = L.DeviceBuffer((t + n) * H * 4)
    L.check(cs1.s1_gdn_conv_gates(x.at(), c["ld"], w.at(), out["q"].at(), out["k"].at(), out["v"].at(), t + n, kd, vd, x.at(2 * c["ch"]),
                                  x.at(2 * (c["ch"] + H)), al.at(), dt.at(), out["beta"].at(), g.at(), H, stream.handle), "prefill conv")
    tail = dict(c, x=c["x"][t:], tails=c["x"][t - 3:t, :c["ch"]][None].copy())
    got, gs, tails = run_conv(cs1, stream, tail, [0, n], [0], [0])
    out64, _, _, _, _, _, y = conv_formula(tail, [0, n], [0], [0])
    theirs = np.concatenate([f32(down(out[m], (t + n, got[m].shape[1]), stream)[t:]) for m in ("q", "k", "v")], 1)
    ours = f32(np.concatenate([got[m] for m in ("q", "k", "v")], 1))
    # SiLU's slope is below 1.1; the last rounding on both sides, and the float32 parts
    assert (np.abs(ours - theirs) <= HALF * (1.1 * np.abs(y) + 2.02 * np.abs(out64)) + 2.0 ** -18).all()
    assert (got["beta"] == down(out["beta"], (t + n, H), stream)[t:]).all()
    assert (gs == down(g, (t + n, H), stream, np.float32)[t:]).all()
    assert (tails[0] == c["x"][-3:, :c["ch"]]).all()


def test_convolution_step_refuses_sequences_on_the_device(cs1, stream):
    for start, si, so, code, live in [(None, [0, 9, 2], [0, 1, 2], 61, [0, 2]), (None, [0, 1, 1], [0, 1, 2], 62, [0]),
                                      (None, [0, 3, 3], [4, 4, 2], 62, [2]), ([0, 1, 4, 5], [0, 1, 2], [0, 1, 2], 60, [0])]:
        c = conv_case(3, 128, 256, 2, 5, 0, 1)
        got, g, tails = run_conv(cs1, stream, c, start, si, so)
        assert status() == (0, 0, code)
        keep = [so[i] if i in live else -1 for i in range(3)]
        want, tol, rows, beta, gw, tw, _ = conv_formula(c, np.arange(4) if start is None else start, si, keep)
        y = np.concatenate([got["q"], got["k"], got["v"]], 1)
        assert (y[~rows] == 0x4242).all() and (np.abs(f32(y) - want)[rows] <= tol[rows]).all()
        assert (g[~rows] == 99.0).all() and (tails == tw).all()


# ---- paged cache ----

def many_sequences(nseq, spare, hurt, seed):
    """Windows of 0 to 3 rows; slots to begin with: the own one, none, or one of `spare` that nobody writes; who is refused."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 4, nseq)
    start = np.concatenate([[0], np.cumsum(lens)])
    so = rng.permutation(nseq)
    si = np.where(rng.random(nseq) < 0.3, -1, np.where(rng.random(nseq) < 0.5, so, nseq + rng.integers(0, spare, nseq)))
    so[rng.permutation(nseq)[:nseq // 20]] = -1                     # sit out
    refused = np.zeros(nseq, bool)
    if hurt:
        some = rng.permutation(nseq)[:80]
        so[some[:20]] = so[some[20:40]]                              # two write one slot
        si[some[40:50]] = np.abs(so[some[50:60]])                    # one begins with what another writes
        so[some[60:70]] = nseq + spare + rng.integers(0, 9, 10)      # no such slot
        si[some[70:80]] = 2 ** 31 - 1
        refused = (so >= nseq + spare) | (si >= nseq + spare)
    outs = so[so >= 0]
    writes, reads = (dict(zip(*np.unique(a, return_counts=True))) for a in (outs, si[(so >= 0) & (si >= 0)]))
    for i in np.flatnonzero(so >= 0):
        own = si[i] == so[i]
        refused[i] |= writes[so[i]] > 1 or reads.get(so[i], 0) > own or (si[i] >= 0 and writes.get(si[i], 0) > own)
    return lens, start, si, so, refused & (so >= 0)


@pytest.mark.parametrize("nseq", [4095, 4096, 5003, 20003])
@pytest.mark.parametrize("hurt", [False, True])
def test_convolution_step_of_many_sequences(cs1, stream, nseq, hurt):
    lens, start, si, so, refused = many_sequences(nseq, 50, hurt, nseq)
    assert refused.any() == hurt
    c = conv_case(start[-1], 8, 16, 2, nseq + 50, 0, nseq)
    out, g, tails = run_conv(cs1, stream, c, start, si, so)
    assert status()[2] in ((61, 62) if hurt else (0,))
    y, tol, live, beta, g64, want, _ = conv_formula(c, start, si, np.where(refused, -1, so))
    got = np.concatenate([out[m] for m in "qkv"], 1)
    assert (got[~live] == 0x4242).all() and (out["beta"][~live] == 0x4242).all() and (g[~live] == 99.0).all()
    assert (np.abs(f32(got) - y)[live] <= tol[live]).all()
    assert (np.abs(f32(out["beta"]) - beta)[live] <= (HALF + 2.0 ** -20) * beta[live]).all()
    h = np.abs(f32(c["x"])[:, c["ch"] + 2:c["ch"] + 4]) + np.abs(f32(c["dt"]))
    assert (np.abs(g - g64)[live] <= (np.abs(g64) * (2.0 ** -20 + EPS * h))[live] + 1e-30).all()
    assert (tails == want).all()


@pytest.mark.parametrize("nseq", [2561, 9001])
@pytest.mark.parametrize("hurt", [False, True])
def test_delta_rule_step_of_many_sequences(cs1, stream, nseq, hurt):
    H, HK, spare, scale = 4, 2, 8, D ** -0.5
    lens, start, si, so, refused = many_sequences(nseq, spare, hurt, nseq)
    x = delta_inputs(start[-1], H, HK, spare, nseq)
    one = H * D * D
    pool = L.DeviceBuffer((nseq + spare) * one * 4)                  # zeros, and the spare states at its end
    L.check(cs1.s1_memset_async(pool.at(), 0, nseq * one * 4, stream.handle), "memset")
    L.check(cs1.cs1_upload(pool.at(nseq * one * 4), x["states"].ctypes.data_as(C.c_void_p), x["states"].nbytes, stream.handle), "upload")
    d = {m: up(x[m], stream) for m in ("q", "k", "v", "g", "beta")}
    o = up(np.full(x["v"].shape, 0x4242, np.uint16), stream)
    s, a, b = ints(start, stream), ints(si, stream), ints(so, stream)
    L.check(cs1.s1_gdn_step(d["q"].at(), d["k"].at(), d["v"].at(), d["g"].at(), d["beta"].at(), o.at(), start[-1], H, HK, scale, pool.at(), nseq + spare,
                            one, s.at(), a.at(), b.at(), nseq, stream.handle), "step")
    got = down(o, x["v"].shape, stream)
    assert status()[2] in ((61, 62) if hurt else (0,))
    rows_of = np.repeat(np.arange(nseq), lens)
    done = (so >= 0) & ~refused
    assert (got[~done[rows_of]] == 0x4242).all() and (f32(got[done[rows_of]]) < 1e4).all()
    # what no sequence leaves stays as it was
    state = np.empty((H, D, D), np.float32)

    def slot(i):
        L.check(cs1.cs1_download(state.ctypes.data_as(C.c_void_p), pool.at(int(i) * one * 4), state.nbytes, stream.handle), "download")
        stream.sync()
        return state

    written = set(so[done])
    for i in [j for j in range(nseq) if j not in written][::max(1, nseq // 400)] + list(np.unique(so[refused & (so < nseq)])[:20]):
        if i not in written:
            assert (slot(i) == 0).all()
    pick = np.flatnonzero(done)[::max(1, nseq // 50)]
    rows = np.concatenate([np.arange(start[i], start[i + 1]) for i in pick])
    part = {m: x[m][rows] for m in ("q", "k", "v", "g", "beta")}
    part["states"] = np.concatenate([x["states"], np.zeros((len(pick), H, D, D), np.float32)])
    at0 = np.concatenate([[0], np.cumsum(lens[pick])])
    w, new, tol, tol_s = delta_formula(part, at0, np.where(si[pick] >= nseq, si[pick] - nseq, -1), spare + np.arange(len(pick)), H, HK, scale)
    assert (np.abs(f32(got[rows]) - w) <= tol).all()
    for n, i in enumerate(pick):
        assert (np.abs(slot(so[i]) - new[spare + n]) <= tol_s[spare + n]).all()


def make_table(need, n_pages, wide, seed):
    """Shuffled pages for sequences that need so many; -1 behind them."""
    order = np.random.default_rng(seed).permutation(n_pages)
    table, used = np.full((len(need), wide), -1, np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[used:used + n]
        used += n
    assert used <= n_pages
    return table


def prep_inputs(rows, Hq, Hk, Dh, half, angles, n_pages, page, pad, seed):
    rng = np.random.default_rng(seed)
    n = rng.standard_normal
    ld = 2 * Hq * Dh + 2 * Hk * Dh + pad
    turn = rng.uniform(0, 6.28, (angles, half))
    return dict(x=bf(n((rows, ld)) * 2), ld=ld, qw=bf(n(Dh) * 0.2), kw=bf(n(Dh) * 0.2), cos=bf(np.cos(turn)), sin=bf(np.sin(turn)),
                kp=bf(n((n_pages, page, Hk, Dh))), vp=bf(n((n_pages, page, Hk, Dh))), Hq=Hq, Hk=Hk, Dh=Dh, half=half)


def run_prep(cs1, st, c, table, seq, pos, angle=None):
    rows, Hq, Hk, Dh = len(c["x"]), c["Hq"], c["Hk"], c["Dh"]
    n_pages, page = c["kp"].shape[:2]
    d = {m: up(c[m], st) for m in ("x", "qw", "kw", "cos", "sin", "kp", "vp")}
    q, gate = (up(np.full((rows, Hq, Dh), 0x4242, np.uint16), st) for _ in range(2))
    t, s, p, a = ints(table, st), ints(seq, st), ints(pos, st), ints(angle, st)
    kr = 2 * Hq * Dh * 2
    L.check(cs1.s1_attn_prep_paged(d["x"].at(), d["x"].at(kr), d["x"].at(kr + 2 * Hk * Dh), c["ld"], d["qw"].at(), d["kw"].at(), d["cos"].at(),
                                   d["sin"].at(), len(c["cos"]), at(a), q.at(), gate.at(), d["kp"].at(), d["vp"].at(), n_pages, page, t.at(),
                                   table.shape[1], len(table), at(s), p.at(), rows, Hq, Hk, Dh, c["half"], 1e-6, st.handle), "prep")
    return (down(q, (rows, Hq, Dh), st), down(gate, (rows, Hq, Dh), st), down(d["kp"], c["kp"].shape, st), down(d["vp"], c["vp"].shape, st))


def prep_formula(c, turn):
    rows, Hq, Hk, Dh, half = len(c["x"]), c["Hq"], c["Hk"], c["Dh"], c["half"]
    cos, sin = (f32(c[m]).astype(np.float64)[turn][:, None] for m in ("cos", "sin"))

    def one(x, w):
        y = f32(x).astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * (1 + f32(w).astype(np.float64))
        a, b = y[..., :half], y[..., half:2 * half]
        out = np.concatenate([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1)
        big = np.concatenate([np.abs(a) + np.abs(b)] * 2 + [np.abs(y[..., 2 * half:])], -1)
        # the mean over Dh squares, rsqrt, three products and two rotary products with their sum: under 64 roundings
        return out, HALF * np.abs(out) + 64 * EPS * big

    h = c["x"][:, :2 * Hq * Dh].reshape(rows, Hq, 2, Dh)
    kv = c["x"][:, 2 * Hq * Dh:2 * (Hq + Hk) * Dh].reshape(rows, 2, Hk, Dh)
    return one(h[:, :, 0], c["qw"]), h[:, :, 1], one(kv[:, 0], c["kw"]), kv[:, 1]


@pytest.mark.parametrize("Dh,Hq,Hk,half,page,pad", [(128, 4, 2, 16, 16, 0), (128, 24, 4, 32, 64, 8), (256, 16, 4, 32, 48, 0), (256, 2, 2, 128, 5, 16),
                                                    (128, 1, 1, 64, 1, 0), (128, 7, 7, 8, 33, 0), (256, 40, 1, 64, 16, 0)])
@pytest.mark.parametrize("angles", ["positions", "own"])
def test_prep_matches_the_formula_and_fills_the_cache(cs1, stream, Dh, Hq, Hk, half, page, pad, angles):
    seq = np.array([2, 0, 0, 1, 3, 0, 2])
    pos = np.array([0, page - 1, page, 2 * page + page // 2, -1, 3 * page - 1 if page > 1 else 2, 1])
    rows = len(seq)
    n_angles = 4 * page + 4 if angles == "positions" else rows + 2
    c = prep_inputs(rows, Hq, Hk, Dh, half, n_angles, 14, page, pad, Dh + Hq)
    table = make_table([3, 3, 2, 0], 14, 4, 1)
    angle = None if angles == "positions" else np.arange(rows)[::-1].copy() + 1
    q, gate, kp, vp = run_prep(cs1, stream, c, table, seq, pos, angle)
    (wq, tq), wg, (wk, tk), wv = prep_formula(c, np.maximum(pos, 0) if angle is None else angle)
    live = pos >= 0
    assert (q[~live] == 0x4242).all() and (gate[~live] == 0x4242).all()
    assert (np.abs(f32(q) - wq)[live] <= tq[live]).all()
    assert (gate[live] == wg[live]).all()
    touched = np.zeros(c["kp"].shape[:2], bool)
    for r in np.flatnonzero(live):
        place = table[seq[r], pos[r] // page], pos[r] % page
        assert not touched[place]
        touched[place] = True
        assert (np.abs(f32(kp[place]) - wk[r]) <= tk[r]).all()
        assert (vp[place] == wv[r]).all()
    assert (kp[~touched] == c["kp"][~touched]).all() and (vp[~touched] == c["vp"][~touched]).all()


def test_prep_refuses_rows_on_the_device(cs1, stream):
    page, rows = 16, 4
    c = prep_inputs(rows, 4, 2, 128, 16, 40, 8, page, 0, 2)
    table = make_table([2, 2, 2], 8, 2, 4)
    shared = table.copy()
    shared[1] = shared[0]
    bad_page, low_page = table.copy(), table.copy()
    bad_page[1, 0], low_page[1, 0] = 8, -2
    cases = [(table, [0, 3, 1, 2], [0, 0, 0, 0], None, 31, [1], []), (table, [0, -1, 1, 2], [0, 0, 0, 0], None, 31, [1], []),
             (table, [0, 1, 1, 2], [0, 32, 0, 0], None, 31, [1], []), (bad_page, [0, 1, 2, 2], [0, 0, 3, 0], None, 32, [1], []),
             (low_page, [0, 1, 2, 2], [0, 0, 3, 0], None, 32, [1], []), (table, [0, 1, 2, 2], [0, 0, 3, 0], [0, 40, 1, 1], 33, [1], []),
             (table, [0, 1, 2, 2], [0, 0, 3, 0], [0, -1, 1, 1], 33, [1], []), (table, [0, 1, 2, 1], [0, 5, 3, 5], None, 34, [], [1, 3]),
             (shared, [0, 1, 2, 0], [17, 17, 17, 0], None, 34, [], [0, 1])]
    for t, seq, pos, angle, code, out, uncached in cases:
        q, gate, kp, vp = run_prep(cs1, stream, c, t, np.array(seq), np.array(pos), angle)
        assert status() == (0, code, 0)
        (wq, tq), wg, (wk, tk), wv = prep_formula(c, np.clip(pos if angle is None else angle, 0, 39))
        touched = np.zeros(c["kp"].shape[:2], bool)
        for r in range(rows):
            if r in out:
                assert (q[r] == 0x4242).all() and (gate[r] == 0x4242).all()
                continue
            assert (np.abs(f32(q[r]) - wq[r]) <= tq[r]).all() and (gate[r] == wg[r]).all()
            if r in uncached:
                continue
            place = t[seq[r], pos[r] // page], pos[r] % page
            touched[place] = True
            assert (np.abs(f32(kp[place]) - wk[r]) <= tk[r]).all() and (vp[place] == wv[r]).all()
        assert (kp[~touched] == c["kp"][~touched]).all() and (vp[~touched] == c["vp"][~touched]).all()


@pytest.mark.parametrize("rows,Dh,Hq,Hk,page", [(512, 128, 4, 2, 16), (513, 128, 4, 2, 16), (513, 256, 12, 2, 7), (700, 128, 20, 4, 64), (2100, 128, 1, 1, 1),
                                                (3001, 256, 2, 1, 300), (9000, 128, 2, 1, 1024), (40001, 128, 1, 1, 48)])
@pytest.mark.parametrize("hurt", [False, True])
def test_prep_of_many_rows(cs1, stream, rows, Dh, Hq, Hk, page, hurt):
    """A chunk of a prompt and more into the cache, whole; and with rows that sit out, are refused, or share a place."""
    rng = np.random.default_rng(rows + hurt)
    nseq, half, angles = 5, 16, 64
    need = [-(-rows // nseq // page) + 1] * nseq
    n_pages = sum(need) + 1
    c = prep_inputs(rows, Hq, Hk, Dh, half, angles, n_pages, page, 0, rows)
    table = make_table(need, n_pages, max(need) + 1, 3)
    places = rng.permutation(nseq * need[0] * page)[:rows]           # no place twice
    if not hurt:
        places.sort()
    seq, pos, angle = places // (need[0] * page), places % (need[0] * page), rng.integers(0, angles, rows)
    lost = np.zeros(rows, bool)                                      # rows that leave nothing at all
    if hurt:
        table[4, 0] = table[3, 0]                                    # two sequences name one page
        some = rng.permutation(rows)[:50].reshape(5, 10)
        pos[some[0]], lost[some[0]] = -1 - rng.integers(0, 9, 10), True
        seq[some[1]], lost[some[1]] = np.where(rng.random(10) < 0.5, -1, nseq), True
        pos[some[2]], lost[some[2]] = np.array([max(need) * page, (max(need) + 1) * page, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1] * 2), True
        angle[some[3]], lost[some[3]] = np.where(rng.random(10) < 0.5, -1, angles), True
        other = rng.integers(0, rows, 10)
        seq[some[4]], pos[some[4]] = seq[other], pos[other]          # twice at one place, or lost with the row copied
        lost[some[4]] |= (pos[some[4]] < 0) | (seq[some[4]] < 0) | (seq[some[4]] >= nseq) | (pos[some[4]] >= max(need) * page)
    q, gate, kp, vp = run_prep(cs1, stream, c, table, seq, pos, angle)
    code = status()[1]
    assert code in ((31, 32, 33, 34) if hurt else (0,))
    (wq, tq), wg, (wk, tk), wv = prep_formula(c, np.clip(angle, 0, angles - 1))
    assert (q[lost] == 0x4242).all() and (gate[lost] == 0x4242).all()
    assert (np.abs(f32(q) - wq)[~lost] <= tq[~lost]).all() and (gate[~lost] == wg[~lost]).all()
    # every row with a place in the table counts for it, one with a bad angle too
    named = (pos >= 0) & (pos < table.shape[1] * page) & (seq >= 0) & (seq < nseq)
    at = np.where(named, table[np.where(named, seq, 0), np.where(named, pos, 0) // page].astype(np.int64) * page + pos % page, -1)
    held, count = np.unique(at[named], return_counts=True)
    alone = np.isin(at, held[count == 1]) & ~lost
    assert (count > 1).any() == hurt
    kp2, vp2 = kp.reshape(-1, Hk, Dh), vp.reshape(-1, Hk, Dh)
    assert (np.abs(f32(kp2[at[alone]]) - wk[alone]) <= tk[alone]).all() and (vp2[at[alone]] == wv[alone]).all()
    rest = np.ones(len(kp2), bool)
    rest[at[alone]] = False
    assert (kp2[rest] == c["kp"].reshape(kp2.shape)[rest]).all() and (vp2[rest] == c["vp"].reshape(vp2.shape)[rest]).all()


def test_prep_agrees_with_the_prefill_operator(cs1, stream):
    """The rows of cs1_attn_prep, within the bf16 steps of its roundings in between."""
    T, Hq, Hk, Dh, half, page = 37, 8, 2, 128, 32, 16
    c = prep_inputs(T, Hq, Hk, Dh, half, T, 4, page, 0, 6)
    d = {m: up(c[m], stream) for m in ("x", "qw", "kw", "cos", "sin")}
    q, gate, k = (L.DeviceBuffer(T * h * Dh * 2) for h in (Hq, Hq, Hk))
    L.check(cs1.cs1_attn_prep(d["x"].at(), d["x"].at(4 * Hq * Dh), c["ld"], d["qw"].at(), d["kw"].at(), d["cos"].at(), d["sin"].at(), q.at(), gate.at(),
                              k.at(), T, Hq, Hk, Dh, half, 1e-6, stream.handle), "prep")
    table = make_table([3], 4, 3, 0)
    q2, gate2, kp, vp = run_prep(cs1, stream, c, table, np.zeros(T, int), np.arange(T))
    assert (gate2 == down(gate, gate2.shape, stream)).all()
    keys = kp[table[0]].reshape(-1, Hk, Dh)[:T]
    for got, want in ((q2, down(q, q2.shape, stream)), (keys, down(k, keys.shape, stream))):
        a, b = f32(got), f32(want)
        # theirs rounds the normed pair and both products before the sum: each adds half a step of a pair's
        # length, at most sqrt(2) of the largest value, and both round the result
        assert np.abs(a - b).max() <= (2 * 2 ** 0.5 + 2) * 1.01 * HALF * np.abs(b).max()
        assert (got[..., 2 * half:] == want[..., 2 * half:]).all()     # without rotary: one rounding on both sides


# ---- attention ----

def attn_case(lens, Hq, Hk, Dh, page, seed, amp=1.0, seq=None, spare=2, extra_width=1):
    rng = np.random.default_rng(seed)
    nseq = len(lens) if seq is None else max(seq) + 1
    need = np.zeros(nseq, int)
    for r, n in enumerate(lens):
        i = r if seq is None else seq[r]
        need[i] = max(need[i], -(-max(n, 0) // page))
    n_pages = int(need.sum()) + spare
    table = make_table(need, n_pages, int(need.max()) + extra_width, seed)
    n = rng.standard_normal
    kp, vp = bf(n((n_pages, page, Hk, Dh)) * amp), bf(n((n_pages, page, Hk, Dh)))
    # what no row sees is NaN: the rest of the last pages and the spare ones
    seen = np.zeros((n_pages, page), bool)
    for r, m in enumerate(lens):
        i = r if seq is None else seq[r]
        for t in range(0, max(m, 0), page):
            seen[table[i, t // page], :min(page, m - t)] = True
    kp[~seen], vp[~seen] = NAN, NAN
    return dict(q=bf(n((len(lens), Hq, Dh)) * amp), gate=bf(n((len(lens), Hq, Dh)) * 2), kp=kp, vp=vp, table=table, lens=lens, seq=seq,
                Hq=Hq, Hk=Hk, Dh=Dh, page=page)


def run_attn(cs1, st, c, gated, scale, stream=None, ws_fill=0xff):
    rows, Hq, Hk, Dh = len(c["lens"]), c["Hq"], c["Hk"], c["Dh"]
    d = {m: up(c[m], st) for m in ("q", "gate", "kp", "vp", "table")}
    out = up(np.full((rows, Hq, Dh), 0x4242, np.uint16), st)
    floats = cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)
    ws = L.DeviceBuffer(floats * 4)
    L.check(cs1.s1_memset_async(ws.at(), ws_fill, floats * 4, st.handle), "memset")       # all NaN: nothing may be read before it is written
    seq, n = ints(c["seq"], st), ints(c["lens"], st)
    L.check(cs1.s1_attention_paged(d["q"].at(), d["gate"].at() if gated else None, out.at(), d["kp"].at(), d["vp"].at(), len(c["kp"]), c["page"],
                                   d["table"].at(), c["table"].shape[1], len(c["table"]), at(seq), n.at(), rows, Hq, Hk, Dh, scale, ws.at(),
                                   floats, st.handle), "attention")
    return down(out, (rows, Hq, Dh), st)


def attn_formula(c, r, gated, scale):
    i, n = r if c["seq"] is None else c["seq"][r], c["lens"][r]
    Hq, Hk, Dh, page = c["Hq"], c["Hk"], c["Dh"], c["page"]
    pages = c["table"][i, :-(-n // page)]
    k, v = (f32(c[m][pages]).astype(np.float64).reshape(-1, Hk, Dh)[:n] for m in ("kp", "vp"))
    q = f32(c["q"][r]).astype(np.float64).reshape(Hk, -1, Dh)
    s = np.einsum("hgd,thd->hgt", q, k) * scale
    # a score is a float32 sum of Dh products: off by Dh * 2^-24 of the sum of their sizes
    ds = Dh * EPS * (np.einsum("hgd,thd->hgt", np.abs(q), np.abs(k)) * abs(scale)).max(-1, keepdims=True)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    o = np.einsum("hgt,thd->hgd", p, v)
    size = np.einsum("hgt,thd->hgd", p, np.abs(v))
    # probabilities: bf16 for the product (2^-8), the score's error twice (its own and the maximum's), exp2 and sums 2^-18
    tol = (HALF + 2 * ds + 2.0 ** -18) * size
    o, tol = o.reshape(Hq, Dh), tol.reshape(Hq, Dh)
    if gated:
        w = 1 / (1 + np.exp(-f32(c["gate"][r]).astype(np.float64)))
        o, tol = o * w, tol * w * (1 + 2.0 ** -19)
    return o, tol + HALF * np.abs(o) + 2.0 ** -19 * np.abs(o)


def check_attn(c, got, gated, scale, rows=None):
    for r in range(len(c["lens"])) if rows is None else rows:
        n = c["lens"][r]
        if n < 0:
            assert (got[r] == 0x4242).all()
        elif n == 0:
            assert (got[r] == 0).all()
        else:
            want, tol = attn_formula(c, r, gated, scale)
            err = np.abs(f32(got[r]).astype(np.float64) - want)
            assert (err <= tol).all(), (r, n, (err / tol).max())


@pytest.mark.parametrize("Dh", [128, 256])
@pytest.mark.parametrize("Hq,Hk,page,gated", [(24, 4, 64, True), (16, 4, 16, True), (4, 4, 48, False), (8, 1, 32, True), (32, 1, 16, False),
                                              (20, 1, 64, True), (40, 2, 128, False), (17, 1, 16, True)])
def test_paged_attention_matches_the_formula(cs1, stream, Dh, Hq, Hk, page, gated):
    lens = [1, 2, 0, 15, 16, 17, 63, -1, 64, 65, 127, 128, 129, 300, 0, 777]
    c = attn_case(lens, Hq, Hk, Dh, page, Hq + page)
    got = run_attn(cs1, stream, c, gated, Dh ** -0.5)
    check_attn(c, got, gated, Dh ** -0.5)
    assert (run_attn(cs1, stream, c, gated, Dh ** -0.5, ws_fill=0) == got).all()


@pytest.mark.parametrize("Dh,Hq,Hk,page,lens", [
    (128, 24, 4, 64, [20001]), (256, 16, 4, 16, [9001]), (128, 4, 1, 16, [40000, 3, 5000]), (256, 8, 8, 80, [1, 6000, 64]),
    (128, 16, 4, 32, [1]), (128, 16, 4, 32, [0]), (128, 16, 4, 32, [-1, -1]), (128, 6, 2, 16, [64] * 200), (256, 6, 1, 256, [513] * 75),
    (128, 24, 4, 64, [500 + 37 * i for i in range(60)]), (128, 9, 3, 1024, [5000, 1024, 1025]), (256, 64, 1, 16, [700, 33]),
    (256, 12, 6, 4096, [4096, 1, 9000])])
def test_paged_attention_cut_over_many_blocks(cs1, stream, Dh, Hq, Hk, page, lens):
    """Rows cut in the middle, at their ends, into one tile each; many rows per block; nothing at all."""
    c = attn_case(lens, Hq, Hk, Dh, page, len(lens) + Dh)
    got = run_attn(cs1, stream, c, True, Dh ** -0.5)
    rows = range(len(lens)) if len(lens) < 20 else range(0, len(lens), 7)
    check_attn(c, got, True, Dh ** -0.5, rows)


@pytest.mark.parametrize("Hq,Hk,tile,tiles", [(Hq, Hk, tile, tiles) for Hq, Hk, tile in ((8, 4, 16), (6, 2, 32), (3, 1, 64))
                                              for tiles in (63, 64, 65, 95, 97, 191, 511, 512, 513, 769, 2367, 2369) if tiles * tile < 80000])
def test_paged_attention_where_runs_grow(cs1, stream, Hq, Hk, tile, tiles):
    """One row at the tile counts where its runs go from one tile to eight, and from there to one per block."""
    for n in (tiles * tile, tiles * tile - tile + 1):
        c = attn_case([n], Hq, Hk, 128, 64, tiles + tile)
        check_attn(c, run_attn(cs1, stream, c, True, 128 ** -0.5), True, 128 ** -0.5)


def test_paged_attention_of_very_many_rows(cs1, stream):
    """More rows than a block has threads, most of them next to nothing: lengths 0, 1, 17, 40 and rows that sit out."""
    lens = [(0, 1, -1, 17, 1, 40, 0)[(i * i) % 7] for i in range(20011)]
    seq = [i % 50 for i in range(len(lens))]
    c = attn_case(lens, 2, 1, 128, 16, 9, seq=seq)
    got = run_attn(cs1, stream, c, True, 128 ** -0.5)
    check_attn(c, got, True, 128 ** -0.5, list(range(0, len(lens), 97)) + list(range(len(lens) - 20, len(lens))))


def test_paged_attention_rows_of_one_sequence_are_a_causal_window(cs1, stream):
    seq = [0, 0, 0, 1, 2, 2]
    c = attn_case([198, 199, 200, 64, 1, 2], 8, 2, 128, 16, 3, seq=seq)
    check_attn(c, run_attn(cs1, stream, c, True, 128 ** -0.5), True, 128 ** -0.5)
    # the last row alone gives the same bits: a row does not depend on the others but for the cut
    one = dict(c, q=c["q"][4:5], gate=c["gate"][4:5], lens=[1], seq=[2])
    assert (run_attn(cs1, stream, one, True, 128 ** -0.5) == run_attn(cs1, stream, c, True, 128 ** -0.5)[4:5]).all()


def windows_of(spec):
    """Rows of (sequence, first length, rows, growth) windows."""
    lens = [n + i * grow for _, n, rows, grow in spec for i in range(rows)]
    return lens, [q for q, _, rows, _ in spec for _ in range(rows)]


def wide(c):
    """The case with a table that could hold 70 MB: rows of one sequence share tiles in such caches."""
    n, w = c["table"].shape
    more = max(0, int(70e6 / (n * c["page"] * c["Hk"] * c["Dh"] * 4)) + 1 - w)
    return dict(c, table=np.concatenate([c["table"], np.full((n, more), -1, c["table"].dtype)], 1))


@pytest.mark.parametrize("Dh", [128, 256])
@pytest.mark.parametrize("Hq,Hk", [(24, 4), (16, 4), (16, 2), (8, 8), (5, 1), (12, 1), (40, 2), (6, 2), (9, 3)])
@pytest.mark.parametrize("spec", [
    [(0, 1, 3, 1), (1, 14, 5, 1), (2, 100, 1, 1), (3, 60, 17, 1)],                     # from the first token on; over a tile's end
    [(0, 500, 3, 1), (0, 503, 2, 1), (1, 503, 3, 1), (1, 400, 3, 1), (2, 2000, 9, 1)],  # two windows of one sequence, a shorter one behind
    [(0, 300, 4, 0), (1, 64, 4, 16), (2, 64, 4, 17), (3, 129, 2, 1), (3, -1, 2, 0), (3, 131, 2, 1), (4, 0, 3, 0), (4, 1, 2, 0)],
    [(0, 40, 70, 1), (1, 700, 49, 1), (2, 9, 1, 1)]])                                  # longer than rows look back
def test_paged_attention_windows_share_tiles(cs1, stream, Dh, Hq, Hk, spec):
    """Rows of one sequence, as many at once as fit a product: each over its own length, those that sit out left alone."""
    lens, seq = windows_of(spec)
    c = wide(attn_case(lens, Hq, Hk, Dh, 32, Hq + Dh, seq=seq))
    got = run_attn(cs1, stream, c, True, Dh ** -0.5)
    check_attn(c, got, True, Dh ** -0.5)
    assert (run_attn(cs1, stream, c, True, Dh ** -0.5, ws_fill=0) == got).all()


@pytest.mark.parametrize("Dh,Hq,Hk", [(128, 16, 4), (128, 8, 8), (256, 12, 2), (128, 5, 1)])
def test_paged_attention_windows_cut_over_many_blocks(cs1, stream, Dh, Hq, Hk):
    lens, seq = windows_of([(0, 9000, 5, 1), (1, 3, 2, 1), (2, 4000, 3, 5), (3, 2500, 16, 1)])
    c = wide(attn_case(lens, Hq, Hk, Dh, 64, Hq, seq=seq))
    check_attn(c, run_attn(cs1, stream, c, False, Dh ** -0.5), False, Dh ** -0.5)


@pytest.mark.parametrize("Dh,Hq,Hk", [(128, 16, 4), (128, 8, 8), (256, 16, 4), (128, 4, 1), (256, 6, 2)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_paged_attention_a_window_keeps_later_tokens_from_earlier_rows(cs1, stream, Dh, Hq, Hk, bad):
    """What only the later rows of a window may see is infinite or NaN: the earlier ones do not change."""
    lens, seq = windows_of([(0, 190, 8, 1), (1, 30, 4, 5), (2, 47, 4, 1)])
    c = wide(attn_case(lens, Hq, Hk, Dh, 16, 7, seq=seq))
    clean = run_attn(cs1, stream, c, True, Dh ** -0.5)
    hurt = dict(c, kp=c["kp"].copy(), vp=c["vp"].copy())
    first = {0: 194, 1: 36, 2: 48}   # the first token that is hurt
    for s, t0 in first.items():
        for t in range(t0, max(n for n, q in zip(lens, seq) if q == s)):
            for m in ("kp", "vp"):
                hurt[m][c["table"][s, t // 16], t % 16] = bf(np.full((Hk, Dh), bad))
    got = run_attn(cs1, stream, hurt, True, Dh ** -0.5)
    early = [r for r in range(len(lens)) if lens[r] <= first[seq[r]]]
    assert 6 < len(early) < len(lens)
    assert (got[early] == clean[early]).all()
    if np.isnan(bad):
        assert np.isnan(f32(got[[r for r in range(len(lens)) if r not in early]])).all()


@pytest.mark.parametrize("rows", [513, 2999, 8191, 8192, 8193])
def test_paged_attention_windows_of_many_rows(cs1, stream, rows):
    """More rows than a block has threads, in windows of 1 to 40 rows: up to 8192 they share tiles, above they do not."""
    spec, left, i = [], rows, 0
    while left:
        n = min(left, (3, 1, 7, 40, 2, 4, 16)[i * i % 7])
        spec.append((i, 1 + (i * 37) % 90, n, 1))
        left, i = left - n, i + 1
    lens, seq = windows_of(spec)
    c = wide(attn_case(lens, 8, 2, 128, 16, rows, seq=seq))
    got = run_attn(cs1, stream, c, True, 128 ** -0.5)
    check_attn(c, got, True, 128 ** -0.5, list(range(0, rows, 41)) + list(range(rows - 45, rows)))


def test_paged_attention_windows_refuse_rows_on_the_device(cs1, stream):
    """Rows without a sequence, or past their table, between rows that share tiles; more rows than sequences and no list of them."""
    lens, seq = windows_of([(0, 190, 3, 1), (1, 30, 4, 1), (2, 47, 4, 1)])
    c = wide(attn_case(lens, 16, 4, 128, 16, 7, seq=seq))
    longest = c["table"].shape[1] * 16
    for r, (s, n) in {1: (-1, 191), 4: (3, 31), 5: (1, longest + 1), 8: (2 ** 31 - 1, 48)}.items():
        hurt = dict(c, seq=list(c["seq"]), lens=list(c["lens"]))
        hurt["seq"][r], hurt["lens"][r] = s, n
        got = run_attn(cs1, stream, hurt, True, 128 ** -0.5)
        assert status() == (0, 31, 0)
        assert (got[r] == 0x4242).all()
        rest = [i for i in range(len(lens)) if i != r]
        check_attn(c, got, True, 128 ** -0.5, rest)
    got = run_attn(cs1, stream, dict(c, seq=None, lens=[190, 30, 47] + [5] * 8), True, 128 ** -0.5)
    assert status() == (0, 31, 0) and (got[3:] == 0x4242).all() and (got[:3] != 0x4242).any()


@pytest.mark.parametrize("climb", [0.0, 0.4, -0.4, 30.0])
def test_paged_attention_with_scores_that_climb(cs1, stream, climb):
    """Scores that grow or fall along the cache by up to several hundred: the running maximum moves in every tile, or never."""
    n, Hq, Hk, Dh, page = 700, 8, 2, 128, 16
    c = attn_case([n], Hq, Hk, Dh, page, 11, amp=0.5)
    q = f32(c["q"])
    q[..., 0] = 8.0
    c["q"] = bf(q)
    kp = f32(c["kp"])
    for t in range(n):
        kp[c["table"][0, t // page], t % page, :, 0] = climb * t / 8
    c["kp"] = np.where(np.isnan(kp), c["kp"], bf(np.nan_to_num(kp)))
    check_attn(c, run_attn(cs1, stream, c, False, 1.0), False, 1.0)


def test_paged_attention_with_infinities(cs1, stream):
    """-inf scores are masks, wherever they lie; a row of nothing else is zeros; NaN in a seen key shows."""
    n, Hq, Hk, Dh, page = 400, 4, 2, 128, 16
    c = attn_case([n, n, n, n], Hq, Hk, Dh, page, 12)
    q = np.abs(f32(c["q"])) * 0
    q[..., 0] = 1.0
    q[..., 1:9] = f32(c["q"])[..., 1:9]
    c["q"] = bf(q)
    keep = np.ones((4, n), bool)
    keep[0, :130] = False            # whole tiles at the start, so whole parts
    keep[1, 200:] = False
    keep[2, :] = False               # nothing is left
    for r in range(4):
        for t in np.flatnonzero(~keep[r]):
            c["kp"][c["table"][r, t // page], t % page, :, 0] = 0xff80      # -inf
    c["kp"][c["table"][3, 5], 7, 1, 0] = NAN
    got = f32(run_attn(cs1, stream, c, False, 1.0))
    for r in range(2):
        pages = c["table"][r, :-(-n // page)]
        k, v = (f32(c[m][pages]).astype(np.float64).reshape(-1, Hk, Dh)[:n][keep[r]] for m in ("kp", "vp"))
        s = np.einsum("hgd,thd->hgt", q[r].astype(np.float64).reshape(Hk, -1, Dh), k)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want, size = (np.einsum("hgt,thd->hgd", p, x).reshape(Hq, Dh) for x in (v, np.abs(v)))
        assert (np.abs(got[r] - want) <= (HALF + 2.0 ** -16) * size + HALF * np.abs(want)).all()
    assert (got[2] == 0).all()
    assert np.isnan(got[3][2:]).all() and np.isfinite(got[3][:2]).all()     # the heads of the key-value head that has it


def test_paged_attention_refuses_rows_on_the_device(cs1, stream):
    c = attn_case([40, 50, 60, 70], 8, 2, 128, 16, 5)
    wide = c["table"].shape[1]
    for change, code, bad, kept in [(dict(seq=[0, 4, 2, 3]), 31, 1, True), (dict(seq=[0, -1, 2, 3]), 31, 1, True),
                                    (dict(lens=[40, wide * 16 + 1, 60, 70]), 31, 1, True), ("low", 32, 1, False), ("high", 32, 1, False)]:
        if isinstance(change, str):
            table = c["table"].copy()
            table[1, 2] = -1 if change == "low" else len(c["kp"])
            change = dict(table=table)
        x = dict(c, **change)
        got = run_attn(cs1, stream, x, True, 128 ** -0.5)
        assert status() == (0, code, 0)
        check_attn(c, got, True, 128 ** -0.5, [r for r in range(4) if r != bad])
        if kept:
            assert (got[bad] == 0x4242).all()


def test_paged_attention_offsets_pass_32_bits(cs1, stream):
    Hq, Hk, Dh, page = 8, 8, 256, 16
    token = Hk * Dh * 2
    n_pages = (1 << 32) // (token * page) + 40           # a pool of more than 2^32 bytes and 2^31 elements
    n = 100
    c = attn_case([n], Hq, Hk, Dh, page, 4, spare=0)
    pools = []
    table = np.arange(n_pages - 7, n_pages, dtype=np.int32)[::-1].copy()[None]
    for m in ("kp", "vp"):
        pool = L.DeviceBuffer(n_pages * page * token)
        for i in range(7):
            a = np.ascontiguousarray(c[m][c["table"][0, i]])
            L.check(cs1.cs1_upload(pool.at(int(table[0, i]) * page * token), a.ctypes.data, a.nbytes, stream.handle), "upload")
        pools.append(pool)
    q, t, ln = up(c["q"], stream), up(table, stream), ints([n], stream)
    out = L.DeviceBuffer(Hq * Dh * 2)
    floats = cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)
    ws = L.DeviceBuffer(floats * 4)
    L.check(cs1.s1_attention_paged(q.at(), None, out.at(), pools[0].at(), pools[1].at(), n_pages, page, t.at(), 7, 1, None, ln.at(), 1, Hq, Hk, Dh,
                                   Dh ** -0.5, ws.at(), floats, stream.handle), "attention")
    check_attn(c, down(out, (1, Hq, Dh), stream), False, Dh ** -0.5)
    # and the writer of such a pool
    p = prep_inputs(1, Hq, Hk, Dh, 32, 200, 1, page, 0, 3)
    d = {m: up(p[m], stream) for m in ("x", "qw", "kw", "cos", "sin")}
    pos = ints([n], stream)
    q2, gate = L.DeviceBuffer(Hq * Dh * 2), L.DeviceBuffer(Hq * Dh * 2)
    kr = 4 * Hq * Dh
    L.check(cs1.s1_attn_prep_paged(d["x"].at(), d["x"].at(kr), d["x"].at(kr + 2 * Hk * Dh), p["ld"], d["qw"].at(), d["kw"].at(), d["cos"].at(),
                                   d["sin"].at(), 200, None, q2.at(), gate.at(), pools[0].at(), pools[1].at(), n_pages, page, t.at(), 7, 1, None,
                                   pos.at(), 1, Hq, Hk, Dh, 32, 1e-6, stream.handle), "prep")
    where = (int(table[0, 6]) * page + n % page) * token
    (_, _), _, (wk, tk), wv = prep_formula(p, np.array([n]))
    assert (np.abs(f32(L.from_device(pools[0], (Hk, Dh), np.uint16, stream, where)) - wk[0]) <= tk[0]).all()
    assert (L.from_device(pools[1], (Hk, Dh), np.uint16, stream, where) == wv[0]).all()


def test_paged_attention_agrees_with_the_prefill_operator(cs1, stream):
    T, Hq, Hk, Dh, page = 333, 8, 2, 256, 16
    c = attn_case([T], Hq, Hk, Dh, page, 21)
    k, v = (c[m][c["table"][0, :21]].reshape(-1, Hk, Dh)[:T] for m in ("kp", "vp"))
    q = np.zeros((T, Hq, Dh), np.uint16)
    q[-1] = c["q"][0]
    dq, dk, dv = up(q, stream), up(k, stream), up(v, stream)
    o = L.DeviceBuffer(T * Hq * Dh * 2)
    L.check(cs1.cs1_attention(dq.at(), dk.at(), dv.at(), Hk * Dh, o.at(), T, Hq, Hk, Dh, Dh ** -0.5, stream.handle), "attention")
    want, tol = attn_formula(c, 0, False, Dh ** -0.5)
    theirs = f32(down(o, (T, Hq, Dh), stream)[-1])
    ours = f32(run_attn(cs1, stream, c, False, Dh ** -0.5)[0])
    assert (np.abs(ours - want) <= tol).all()
    assert np.abs(ours - theirs).max() < 1.6e-2 * np.abs(want).max()     # the prefill's own gate


# ---- pages ----

@pytest.mark.parametrize("page_bytes,n_pools,n_pages,pairs,fan", [(16, 1, 4, 1, 1), (48, 3, 9, 4, 2), (65536, 2, 20, 7, 7), (16400, 5, 30, 11, 3),
                                                                  (32, 70, 1000, 490, 1), (16384, 65, 12, 5, 2), (1 << 20, 1, 6, 3, 1)])
def test_page_copies(cs1, stream, page_bytes, n_pools, n_pages, pairs, fan):
    rng = np.random.default_rng(pairs)
    pools = [rng.integers(0, 256, (n_pages, page_bytes), dtype=np.uint8) for _ in range(n_pools)]
    order = rng.permutation(n_pages).astype(np.int32)
    src, dst = order[:pairs][np.arange(pairs) // fan].copy(), order[n_pages - pairs:].copy()
    bufs = [up(p, stream) for p in pools]
    ptrs = (C.c_void_p * n_pools)(*[b.ptr.value for b in bufs])
    L.check(cs1.s1_pages_copy(ptrs, n_pools, n_pages, page_bytes, src.ctypes.data, dst.ctypes.data, pairs, stream.handle), "copy")
    src[:], dst[:] = 0, 0              # the lists are the caller's again
    for i in range(n_pools):
        ptrs[i] = None
    for p, b in zip(pools, bufs):
        want = p.copy()
        want[order[n_pages - pairs:]] = p[order[:pairs][np.arange(pairs) // fan]]
        assert (down(b, p.shape, stream, np.uint8) == want).all()


def test_recorded_page_copies_keep_their_lists(cs1, stream):
    st = L.Stream()
    pool = np.arange(6 * 16, dtype=np.uint8).reshape(6, 16)
    buf = up(pool, st)
    ptrs = (C.c_void_p * 1)(buf.ptr.value)
    src, dst = np.array([0, 0, 1], np.int32), np.array([3, 4, 5], np.int32)
    exec_ = C.c_void_p()
    L.check(cs1.cs1_graph_begin(st.handle), "begin")
    L.check(cs1.s1_pages_copy(ptrs, 1, 6, 16, src.ctypes.data, dst.ctypes.data, 3, st.handle), "copy")
    L.check(cs1.cs1_graph_end(st.handle, C.byref(exec_)), "end")
    src[:], dst[:], ptrs[0] = 2, 2, None
    for k in range(2):
        pool[:2] += 7
        L.check(cs1.cs1_upload(buf.at(), pool.ctypes.data, pool.nbytes, st.handle), "upload")
        L.check(cs1.cs1_graph_launch(exec_, st.handle), "launch")
        pool[[3, 4, 5]] = pool[[0, 0, 1]]
        assert (down(buf, pool.shape, st, np.uint8) == pool).all()
    cs1.cs1_graph_destroy(exec_)


# ---- together ----

def test_recorded_step_replays_with_new_contents(cs1, stream):
    """One step of both kinds recorded into a graph and replayed with other rows, slots, tables, positions and lengths."""
    st = L.Stream()
    H, HK, Hq, Hk, Dh, page, half, rows = 4, 2, 8, 2, 128, 16, 16, 3
    rng = np.random.default_rng(0)
    xs = [delta_inputs(rows, H, HK, 6, s) for s in (1, 2)]
    ps = [prep_inputs(rows, Hq, Hk, Dh, half, 64, 12, page, 0, s) for s in (3, 4)]
    slots = [([0, 1, 2], [0, 1, 2]), ([5, -1, 5], [4, 0, 3])]
    tables = [make_table([2, 2, 2], 12, 3, s) for s in (5, 6)]
    poss = [[16, 3, 31], [0, 20, -1]]
    lens = [[17, 4, 32], [1, 21, -1]]
    d = {m: up(xs[0][m], st) for m in ("q", "k", "v", "g", "beta", "states")}
    e = {m: up(ps[0][m], st) for m in ("x", "qw", "kw", "cos", "sin", "kp", "vp")}
    si, so, table, pos, ln = ints(slots[0][0], st), ints(slots[0][1], st), up(tables[0], st), ints(poss[0], st), ints(lens[0], st)
    o, q, gate, out = (L.DeviceBuffer(rows * h * w * 2) for h, w in ((H, D), (Hq, Dh), (Hq, Dh), (Hq, Dh)))
    floats = cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)
    ws = L.DeviceBuffer(floats * 4)
    kr = 4 * Hq * Dh

    def queue():
        L.check(cs1.s1_gdn_step(d["q"].at(), d["k"].at(), d["v"].at(), d["g"].at(), d["beta"].at(), o.at(), rows, H, HK, 1.0, d["states"].at(), 6,
                                H * D * D, None, si.at(), so.at(), rows, st.handle), "step")
        L.check(cs1.s1_attn_prep_paged(e["x"].at(), e["x"].at(kr), e["x"].at(kr + 2 * Hk * Dh), ps[0]["ld"], e["qw"].at(), e["kw"].at(), e["cos"].at(),
                                       e["sin"].at(), 64, None, q.at(), gate.at(), e["kp"].at(), e["vp"].at(), 12, page, table.at(), 3, 3, None,
                                       pos.at(), rows, Hq, Hk, Dh, half, 1e-6, st.handle), "prep")
        L.check(cs1.s1_attention_paged(q.at(), gate.at(), out.at(), e["kp"].at(), e["vp"].at(), 12, page, table.at(), 3, 3, None, ln.at(), rows, Hq,
                                       Hk, Dh, Dh ** -0.5, ws.at(), floats, st.handle), "attention")

    def put(buf, a):
        a = np.ascontiguousarray(a)
        L.check(cs1.cs1_upload(buf.at(), a.ctypes.data, a.nbytes, st.handle), "upload")

    def fill(i):
        for m in d:
            put(d[m], xs[i][m])
        for m in e:
            put(e[m], ps[i][m])
        for buf, a in ((si, slots[i][0]), (so, slots[i][1]), (pos, poss[i]), (ln, lens[i])):
            put(buf, np.asarray(a, np.int32))
        put(table, tables[i])
        for b in (o, q, gate, out):
            L.check(cs1.s1_memset_async(b.at(), 0x42, b.nbytes, st.handle), "memset")

    def read():
        return [down(b, (b.nbytes // 2,), st) for b in (o, q, gate, out, d["states"], e["kp"], e["vp"])]

    want = []
    for i in range(2):
        fill(i)
        queue()
        want.append(read())
    exec_ = C.c_void_p()
    L.check(cs1.cs1_graph_begin(st.handle), "begin")
    queue()
    L.check(cs1.cs1_graph_end(st.handle, C.byref(exec_)), "end")
    for i in (0, 1, 1, 0):
        fill(i)
        L.check(cs1.cs1_graph_launch(exec_, st.handle), "launch")
        for a, b in zip(read(), want[i]):
            assert (a == b).all()
    cs1.cs1_graph_destroy(exec_)


@pytest.mark.parametrize("mode", [1, 2])
def test_steps_as_dependent_launches_give_the_same_bits(cs1, stream, mode):
    """A chain of steps in place, queued without a wait, with and without programmatic dependent launch."""
    H, HK, nseq = 32, 16, 4
    x = delta_inputs(nseq, H, HK, nseq, 5)
    c = conv_case(nseq, HK * D, H * D, H, nseq, 0, 6)
    ids = np.arange(nseq)
    res = []
    for m in (0, mode):
        before = cs1.s1_set_dependent_launch(m)
        d = {k: up(x[k], stream) for k in ("g", "beta", "states")}
        cd = {k: up(c[k], stream) for k in ("x", "w", "al", "dt", "tails")}
        q, k, v, o = (L.DeviceBuffer(nseq * w * D * 2) for w in (HK, HK, H, H))
        s = ints(ids, stream)
        for _ in range(12):
            L.check(cs1.s1_gdn_conv_gates_step(cd["x"].at(), c["ld"], cd["w"].at(), q.at(), k.at(), v.at(), nseq, HK * D, H * D, cd["x"].at(2 * c["ch"]),
                                               cd["x"].at(2 * (c["ch"] + H)), cd["al"].at(), cd["dt"].at(), d["beta"].at(), d["g"].at(), H,
                                               cd["tails"].at(), nseq, 3 * c["ch"], None, s.at(), s.at(), nseq, stream.handle), "conv")
            L.check(cs1.s1_gdn_step(q.at(), k.at(), v.at(), d["g"].at(), d["beta"].at(), o.at(), nseq, H, HK, D ** -0.5, d["states"].at(), nseq,
                                    H * D * D, None, s.at(), s.at(), nseq, stream.handle), "step")
        cs1.s1_set_dependent_launch(before)
        res.append((down(o, (nseq, H, D), stream), down(d["states"], x["states"].shape, stream, np.float32)))
    assert (res[0][0] == res[1][0]).all() and (res[0][1] == res[1][1]).all()


def test_two_attentions_at_once_on_their_own_workspaces(cs1, stream):
    a, b = (attn_case([3000 + 100 * i for i in range(6)], 24, 4, 128, 16, s) for s in (1, 2))
    want = [run_attn(cs1, stream, c, True, 128 ** -0.5) for c in (a, b)]
    sts = [L.Stream(), L.Stream()]
    state = []
    for c, st in zip((a, b), sts):
        d = {m: up(c[m], st) for m in ("q", "gate", "kp", "vp", "table")}
        floats = cs1.s1_attention_paged_workspace_floats(24, 4, 128)
        state.append((d, ints(c["lens"], st), L.DeviceBuffer(floats * 4), L.DeviceBuffer(6 * 24 * 128 * 2), floats))
    for _ in range(20):
        for c, st, (d, ln, ws, out, floats) in zip((a, b), sts, state):
            L.check(cs1.s1_attention_paged(d["q"].at(), d["gate"].at(), out.at(), d["kp"].at(), d["vp"].at(), len(c["kp"]), 16, d["table"].at(),
                                           c["table"].shape[1], 6, None, ln.at(), 6, 24, 4, 128, 128 ** -0.5, ws.at(), floats, st.handle), "attention")
    for st, w, s in zip(sts, want, state):
        assert (down(s[3], w.shape, st) == w).all()


def test_layer_steps_continue_its_prefill(cs1, stream):
    """One Gated DeltaNet layer: prompts of several lengths, then tokens one at a time and a window of them, from their
    slots and from a shared one, against the oracle's layer on the whole sequences."""
    from system1_omni_b200.gdn_layer import GdnLayer
    from test_gdn_layer_gpu import make_case, oracle_layer, rel_l2
    hidden, hk, hv = 1024, 4, 8
    prompts, more = [70, 2, 64, 1], 5
    total = [n + more for n in prompts]
    layer = GdnLayer(hidden, hk, hv, max_tokens=128, stream=stream, slots=7)
    try:
        xs = [make_case(n, hidden, hk, hv, seed=i)[0] for i, n in enumerate(total)]
        w = make_case(1, hidden, hk, hv)[1]
        layer.set_weights(**w)
        for slot, (n, x) in enumerate(zip(prompts, xs)):
            x_dev = up(x[:n], stream)
            layer.forward(x_dev.at(), n, slot=slot)
            stream.sync()
        got = [np.zeros((more, hidden), np.float32) for _ in prompts]
        slots = ints([0, 1, 2, 3], stream)
        for t in range(more - 3):
            x_dev = up(np.stack([x[n + t] for n, x in zip(prompts, xs)]), stream)
            y = f32(down(layer.step(x_dev.at(), 4, slots.at(), slots.at(), 4), (128, hidden), stream))
            for i in range(4):
                got[i][t] = y[i]
        # the last three tokens of each as one window; two more sequences begin where the first one stands
        rows = np.concatenate([x[-3:] for x in xs] + [xs[0][-3:-1], xs[0][-3:-2]])
        start, si, so = ints([0, 3, 6, 9, 12, 14, 15], stream), ints([0, 1, 2, 3, 0, 0], stream), ints([4, 1, 2, 3, 5, 6], stream)
        x_dev = up(rows, stream)
        y = f32(down(layer.step(x_dev.at(), 15, si.at(), so.at(), 6, start.at()), (128, hidden), stream))
        for i in range(4):
            got[i][-3:] = y[3 * i:3 * i + 3]
            want = f32(oracle_layer(xs[i], w, total[i], hidden, hk, hv, float64_core=True))[-more:]
            # bf16 activations with float32 accumulation on both sides: the gate of the layer's prefill
            assert rel_l2(got[i], want) < 2e-2, i
            assert np.abs(got[i] - want).max() < 5e-2 * np.abs(want).max()
        # the candidates' rows are those of the first sequence, up to the row counts' summation order in the projections
        assert rel_l2(y[12:14], y[0:2]) < 1e-2 and rel_l2(y[14:15], y[0:1]) < 1e-2
        with pytest.raises(ValueError):
            layer.forward(x_dev.at(), 3, slot=7)
    finally:
        layer.close()


@pytest.mark.parametrize("Dh,page", [(128, 16), (256, 32)])
def test_candidates_of_a_prefix_in_a_paged_cache(cs1, stream, Dh, page):
    """A prompt written to pages, forked for three candidates whose tokens follow one at a time, a page copied when a
    shared one is written, the pool compacted in between: each row against the prefill's attention over the same rows."""
    from system1_omni_b200.pages import Pages, copy
    Hq, Hk, half, eps, T, more = 8, 4, 32, 1e-6, 75, 20
    n_pages, wide = 40, 8
    angles = T + more
    common = prep_inputs(T, Hq, Hk, Dh, half, angles, n_pages, page, 0, 1)
    tails = [prep_inputs(more, Hq, Hk, Dh, half, angles, 1, page, 0, 10 + i) for i in range(3)]
    d = {m: up(common[m], stream) for m in ("qw", "kw", "cos", "sin", "kp", "vp")}
    ld, kr, page_bytes = common["ld"], 4 * Hq * Dh, page * Hk * Dh * 2
    floats = cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)
    ws = L.DeviceBuffer(floats * 4)
    p = Pages(n_pages, page, 4, wide)
    try:
        def step(x, seq, pos):
            """New rows x at places (seq, pos): written to the cache and attended over it."""
            rows = len(x)
            table, _ = p.table()
            x, table = up(x, stream), up(table, stream)
            s, q_pos, n = ints(seq, stream), ints(pos, stream), ints([t + 1 for t in pos], stream)
            q, gate, out = (L.DeviceBuffer(rows * Hq * Dh * 2) for _ in range(3))
            L.check(cs1.s1_attn_prep_paged(x.at(), x.at(kr), x.at(kr + 2 * Hk * Dh), ld, d["qw"].at(), d["kw"].at(), d["cos"].at(), d["sin"].at(),
                                           angles, None, q.at(), gate.at(), d["kp"].at(), d["vp"].at(), n_pages, page, table.at(), wide, 4,
                                           s.at(), q_pos.at(), rows, Hq, Hk, Dh, half, eps, stream.handle), "prep")
            L.check(cs1.s1_attention_paged(q.at(), gate.at(), out.at(), d["kp"].at(), d["vp"].at(), n_pages, page, table.at(), wide, 4, s.at(),
                                           n.at(), rows, Hq, Hk, Dh, Dh ** -0.5, ws.at(), floats, stream.handle), "attention")
            return down(out, (rows, Hq, Dh), stream)

        assert p.append(0, T) == []
        got = [step(common["x"], [0] * T, list(range(T)))] + [np.zeros((more, Hq, Dh), np.uint16) for _ in range(3)]
        for i in range(3):
            p.fork(0, 1 + i)
        copies = 0
        for t in range(more):
            pairs = sum((p.append(1 + i, 1) for i in range(3)), [])
            copies += len(pairs)
            copy([d["kp"].at(), d["vp"].at()], n_pages, page_bytes, pairs, stream)
            y = step(np.stack([x["x"][t] for x in tails]), [1, 2, 3], [T + t] * 3)
            for i in range(3):
                got[1 + i][t] = y[i]
            if t == 4:
                p.truncate(0)                   # the prompt alone is not needed any more
                copy([d["kp"].at(), d["vp"].at()], n_pages, page_bytes, p.compact(), stream)
        assert copies == 3                      # the half-filled page of the prompt, once per candidate
        used = n_pages - p.free_pages()
        assert used == T // page + 3 * -(-(T % page + more) // page) and p.table(1)[0].max() < used + 3
        for i in range(3):
            x = np.concatenate([common["x"], tails[i]["x"]])
            n = T + more
            dx = up(x, stream)
            q, gate, k, out = (L.DeviceBuffer(n * h * Dh * 2) for h in (Hq, Hq, Hk, Hq))
            L.check(cs1.cs1_attn_prep(dx.at(), dx.at(kr), ld, d["qw"].at(), d["kw"].at(), d["cos"].at(), d["sin"].at(), q.at(), gate.at(), k.at(), n, Hq,
                                      Hk, Dh, half, eps, stream.handle), "prefill prep")
            L.check(cs1.cs1_attention_gated(q.at(), k.at(), dx.at(kr + 2 * Hk * Dh), ld, gate.at(), out.at(), n, Hq, Hk, Dh, Dh ** -0.5,
                                            stream.handle), "prefill attention")
            want = f32(down(out, (n, Hq, Dh), stream)).astype(np.float64)
            mine = f32(np.concatenate([got[0], got[1 + i]])).astype(np.float64)
            # the prefill's own gate for its attention against float64, twice: both sides have such an error
            assert np.abs(mine - want).max() < 2 * 1.6e-2 * np.abs(want).max()
            assert np.linalg.norm(mine - want) < 2 * 1.6e-2 * np.linalg.norm(want)
    finally:
        p.close()


def test_cache_writes_reach_the_attention_launched_as_its_dependent(cs1, stream):
    """Prep, then attention over what it just wrote, as programmatic dependents and without: the same bits."""
    Hq, Hk, Dh, page, rows = 8, 4, 128, 16, 48
    c = prep_inputs(rows, Hq, Hk, Dh, 16, 64, 30, page, 0, 5)
    table = make_table([3] * 8, 30, 4, 2)
    seq, pos = np.arange(rows) % 8, np.arange(rows) // 8
    kr, floats = 4 * Hq * Dh, cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)
    want = None
    for mode in (0, 1, 1, 1):
        d = {m: up(c[m], stream) for m in ("x", "qw", "kw", "cos", "sin", "kp", "vp")}
        t, s, p, n = ints(table, stream), ints(seq, stream), ints(pos, stream), ints(pos + 1, stream)
        q, gate, out = (L.DeviceBuffer(rows * Hq * Dh * 2) for _ in range(3))
        ws = L.DeviceBuffer(floats * 4)
        stream.sync()
        before = cs1.s1_set_dependent_launch(mode)
        for _ in range(8):
            L.check(cs1.s1_attn_prep_paged(d["x"].at(), d["x"].at(kr), d["x"].at(kr + 2 * Hk * Dh), c["ld"], d["qw"].at(), d["kw"].at(), d["cos"].at(),
                                           d["sin"].at(), 64, None, q.at(), gate.at(), d["kp"].at(), d["vp"].at(), 30, page, t.at(), 4, 8, s.at(),
                                           p.at(), rows, Hq, Hk, Dh, 16, 1e-6, stream.handle), "prep")
            L.check(cs1.s1_attention_paged(q.at(), gate.at(), out.at(), d["kp"].at(), d["vp"].at(), 30, page, t.at(), 4, 8, s.at(), n.at(), rows, Hq,
                                           Hk, Dh, Dh ** -0.5, ws.at(), floats, stream.handle), "attention")
        cs1.s1_set_dependent_launch(before)
        got = down(out, (rows, Hq, Dh), stream)
        if want is None:
            want = got
        assert (got == want).all()


@pytest.mark.parametrize("mode", [0, 1])
def test_lengths_written_by_the_kernel_before(cs1, stream, mode):
    """Attentions queued without a wait, each behind a kernel that changes the lengths it is cut by: each as alone."""
    Hq, Hk, Dh, page = 8, 4, 128, 16
    sets = [[3000, 1, 700, 0], [1, 4000, 16, 2500], [0, 33, 0, 1], [2048, 2048, 2048, 2048]]
    c = attn_case([max(s[i] for s in sets) for i in range(4)], Hq, Hk, Dh, page, 11)
    want = [run_attn(cs1, stream, dict(c, lens=s), True, Dh ** -0.5) for s in sets]
    d = {m: up(c[m], stream) for m in ("q", "gate", "kp", "vp", "table")}
    lens, floats = ints([sets[0]] + sets, stream), cs1.s1_attention_paged_workspace_floats(Hq, Hk, Dh)     # page 0: the live ones
    ws, pool = L.DeviceBuffer(floats * 4), (C.c_void_p * 1)(lens.ptr.value)
    order = [1, 0, 3, 2, 0, 2, 1, 3] * 4
    outs = [L.DeviceBuffer(4 * Hq * Dh * 2) for _ in order]
    stream.sync()
    before = cs1.s1_set_dependent_launch(mode)
    for k, out in zip(order, outs):
        src, dst = np.array([k + 1], np.int32), np.array([0], np.int32)
        L.check(cs1.s1_pages_copy(pool, 1, 5, 16, src.ctypes.data, dst.ctypes.data, 1, stream.handle), "lengths")
        L.check(cs1.s1_attention_paged(d["q"].at(), d["gate"].at(), out.at(), d["kp"].at(), d["vp"].at(), len(c["kp"]), page, d["table"].at(),
                                       c["table"].shape[1], 4, None, lens.at(), 4, Hq, Hk, Dh, Dh ** -0.5, ws.at(), floats, stream.handle), "attention")
    cs1.s1_set_dependent_launch(before)
    for k, out in zip(order, outs):
        assert (down(out, (4, Hq, Dh), stream) == want[k]).all()
