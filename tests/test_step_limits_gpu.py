"""The decode operators on the GPU where their promises are tightest: the probabilities' precision, infinite values,
codes next to a prefill, grouped calls at their limits."""
import numpy as np
import pytest

import test_step_gpu as S
from helpers import bf, f32
from system1_omni_b200 import lib as L
from test_step_gpu import up

pytestmark = pytest.mark.gpu

HALF, EPS, NAN = S.HALF, S.EPS, S.NAN


@pytest.fixture(autouse=True)
def clean_status(cs1, stream):
    S.status()
    yield
    assert S.status() == (0, 0, 0)


# ---- attention: the precision of the probabilities ----

def exact_scores(c, seed):
    """The case with queries and keys whose scores float32 holds exactly: four dims of quarters up to 2."""
    rng = np.random.default_rng(seed)
    quarters = lambda shape: bf(rng.integers(-8, 9, shape) * 0.25 * (np.arange(shape[-1]) < 4))
    return dict(c, q=quarters(c["q"].shape), kp=np.where(c["kp"] == NAN, NAN, quarters(c["kp"].shape)))


def tight_formula(c, r, gated):
    """Result and bound with exact scores s, |s| <= 16, scale 1 and up to 64 tokens. Of p: 2^-15 from its two bf16 terms;
    s log2(e) up to 24 and rounded twice (constant and product), as the maximum is, then their difference rounded:
    ln 2 * (4 * 24 + 48) * 2^-24 < 2^-17; exp2f 2^-22. Sums of p over at most 4 slices of 16 tokens, 2^-24 an addition:
    24 additions, 2^-19. The product: 8 MMAs of 16 terms and what came before, 17 * 2^-24 each, 2^-16.9. Rescaling
    and the division, 2^-21. Together below 2^-14."""
    want, _ = S.attn_formula(c, r, False, 1.0)
    n = c["lens"][r]
    _, size = np.abs(want), S.attn_formula(dict(c, vp=c["vp"] & np.uint16(0x7fff)), r, False, 1.0)[0]   # sum of p |v|
    assert n <= 64
    if gated:
        w = 1 / (1 + np.exp(-f32(c["gate"][r]).astype(np.float64)))
        want, size = want * w, size * w
    # the gate: __expf 2^-21 relative to its argument's size and __fdividef 2^-22, together below 2^-18
    return want, (2.0 ** -14 + (2.0 ** -18 if gated else 0)) * size + HALF * np.abs(want) * (1 + 2.0 ** -13)


@pytest.mark.parametrize("Dh", [128, 256])
@pytest.mark.parametrize("Hq,Hk,page", [(24, 4, 64), (8, 8, 16), (6, 2, 16), (16, 2, 32), (5, 1, 16), (32, 1, 16)])
@pytest.mark.parametrize("gated", [False, True])
def test_probabilities_enter_the_product_as_float32(cs1, stream, Dh, Hq, Hk, page, gated):
    c = exact_scores(S.attn_case([2, 64, 17, 33, 48, 3, 63, 1, 9, 40], Hq, Hk, Dh, page, Hq + Dh), 5)
    got = S.run_attn(cs1, stream, c, gated, 1.0)
    for r in range(len(c["lens"])):
        want, tol = tight_formula(c, r, gated)
        err = np.abs(f32(got[r]).astype(np.float64) - want)
        assert (err <= tol).all(), (r, (err / tol).max())


@pytest.mark.parametrize("Dh,Hq,Hk", [(128, 16, 4), (128, 24, 4), (128, 8, 8), (256, 6, 2), (256, 16, 4), (128, 5, 1)])
def test_probabilities_of_a_window_enter_the_product_as_float32(cs1, stream, Dh, Hq, Hk):
    lens, seq = S.windows_of([(0, 30, 3, 1), (1, 60, 5, 1), (2, 9, 4, 5)])     # over the ends of slices and within them
    c = S.wide(exact_scores(S.attn_case(lens, Hq, Hk, Dh, 16, Hq + Dh, seq=seq), 6))
    got = S.run_attn(cs1, stream, c, False, 1.0)
    for r in range(len(lens)):
        want, tol = tight_formula(c, r, False)
        err = np.abs(f32(got[r]).astype(np.float64) - want)
        assert (err <= tol).all(), (r, (err / tol).max())


@pytest.mark.parametrize("Dh,Hq,Hk", [(128, 8, 4), (256, 8, 2), (128, 5, 1)])
@pytest.mark.parametrize("equal", [True, False])
@pytest.mark.parametrize("window", [True, False])
def test_infinite_values_keep_their_sign(cs1, stream, Dh, Hq, Hk, equal, window):
    """An infinite value of a token that a row sees makes that dim infinite, whichever weight the token has, and no other dim."""
    lens, seq = S.windows_of([(0, 40, 4, 1), (1, 1, 1, 0), (2, 100, 3, 1)])
    c = S.attn_case(lens, Hq, Hk, Dh, 16, 8, seq=seq)
    if equal:
        c["q"] = c["q"] * np.uint16(0)
    if window:
        c = S.wide(c)
    finite = [S.attn_formula(c, r, False, Dh ** -0.5) for r in range(len(lens))]
    for s, t, d, bits in [(0, 0, 3, 0x7f80), (0, 39, 70, 0xff80), (1, 0, 9, 0x7f80), (2, 57, 127, 0xff80)]:
        c["vp"][c["table"][s, t // 16], t % 16, :, d] = bits
    got = f32(S.run_attn(cs1, stream, c, False, Dh ** -0.5))
    for r, s in enumerate(seq):
        hit = {0: {3: np.inf, 70: -np.inf}, 1: {9: np.inf}, 2: {127: -np.inf}}[s]
        for d, x in hit.items():
            assert (got[r, :, d] == x).all(), (r, d)
        rest = [d for d in range(Dh) if d not in hit]
        want, tol = finite[r]
        assert (np.abs(got[r][:, rest] - want[:, rest]) <= tol[:, rest]).all()


# ---- codes next to a prefill ----

@pytest.fixture(scope="module")
def model(cs1):
    from helpers import random_weights, tiny_config
    from system1_omni_b200 import model as M
    L.set_device(0)
    cfg = tiny_config()
    m = M.Model(cfg, device=0)
    m.set_tensors(random_weights(cfg, seed=4))
    yield m
    m.close()


@pytest.mark.parametrize("family", ["delta rule", "convolution", "prep", "attention"])
def test_a_refused_index_fails_no_prefill(cs1, stream, model, family):
    """A step operator's refusal is its caller's: a pass of the executor behind it gives its rows, and the code is still there."""
    prompts = [list(range(1, 50)), list(range(7, 300))]
    before = model.forward_batch(prompts)
    if family == "delta rule":
        x = S.delta_inputs(2, 2, 1, 3, 1)
        S.run_delta(cs1, stream, x, None, np.array([0, 9]), np.array([0, 1]), 2, 1, 1.0)
        want = (0, 0, 61)
    elif family == "convolution":
        S.run_conv(cs1, stream, S.conv_case(2, 128, 128, 1, 3, 0, 1), None, np.array([0, 1]), np.array([1, 1]))
        want = (0, 0, 62)
    elif family == "prep":
        p = S.prep_inputs(2, 2, 1, 128, 32, 50, 4, 16, 0, 1)
        S.run_prep(cs1, stream, p, np.array([[0, 1], [2, 9]], np.int32), [0, 1], [3, 20])
        want = (0, 32, 0)
    else:
        c = S.attn_case([20, 30], 2, 1, 128, 16, 1)
        S.run_attn(cs1, stream, dict(c, seq=[0, 5]), False, 1.0)
        want = (0, 31, 0)
    stream.sync()
    assert (model.forward_batch(prompts) == before).all()
    assert (model.forward_batch(prompts) == before).all()
    assert S.status() == want


@pytest.mark.parametrize("read,want", [("attn_status", 31), ("gdn_status", 61)])
def test_the_families_status_calls_report_the_steps_codes(cs1, stream, read, want):
    c = S.attn_case([20, 30], 2, 1, 128, 16, 1)
    S.run_attn(cs1, stream, dict(c, seq=[0, 5]), False, 1.0)
    S.run_delta(cs1, stream, S.delta_inputs(2, 2, 1, 3, 1), None, np.array([0, 9]), np.array([0, 1]), 2, 1, 1.0)
    assert getattr(L, read)() == want
    assert getattr(L, read)() == 0
    assert S.status() == ((0, 0, 61) if read == "attn_status" else (0, 31, 0))     # the other family's stays until it is read


# ---- large calls ----

def device_us(call, st, n=8):
    """The quickest of n calls between events."""
    a, b, us = L.Event(), L.Event(), []
    for i in range(n + 2):
        a.record(st)
        call()
        b.record(st)
        st.sync()
        us.append(a.elapsed_ms(b) * 1e3)
    return min(us[2:])


@pytest.mark.parametrize("nseq", [16384, 65535])
def test_a_shared_slot_costs_a_large_call_no_more_than_own_ones(cs1, stream, nseq):
    """The candidates of one prefix: sequences that all begin with one slot, against ones that continue in their own."""
    kd, vd, H = 8, 16, 1
    ch = 2 * kd + vd
    ld = ch + 8
    x, w, tails = up(bf(np.ones((nseq, ld))), stream), up(bf(np.ones((ch, 4))), stream), up(np.zeros((nseq + 1, 3, ch), np.uint16), stream)
    al = up(bf(np.ones(8)), stream)
    q, k, v, beta, g = (L.DeviceBuffer(nseq * 4 * n) for n in (kd, kd, vd, 8, 8))
    own, one = S.ints(np.arange(nseq), stream), S.ints(np.full(nseq, nseq), stream)
    times = [device_us(lambda: L.check(cs1.s1_gdn_conv_gates_step(
        x.at(), ld, w.at(), q.at(), k.at(), v.at(), nseq, kd, vd, x.at(2 * ch), x.at(2 * ch + 2), al.at(), al.at(), beta.at(), g.at(), H, tails.at(),
        nseq + 1, 3 * ch, None, begin.at(), own.at(), nseq, stream.handle), "step"), stream) for begin in (own, one)]
    print(nseq, times)
    assert times[1] < 2 * times[0]


# ---- the layer ----

def test_layer_rows_that_are_not_run_are_zeros(cs1, stream):
    """A sequence that sits out, one that is refused and rows that nobody owns show nothing of an earlier call."""
    from system1_omni_b200.gdn_layer import GdnLayer
    from test_gdn_layer_gpu import make_case
    hidden, hk, hv = 256, 1, 4
    layer = GdnLayer(hidden, hk, hv, max_tokens=64, stream=stream, slots=6)
    try:
        x, w = make_case(5, hidden, hk, hv)
        layer.set_weights(**w)
        x_dev = up(x, stream)
        for i in range(5):
            layer.forward(x_dev.at(i * hidden * 2), 1, slot=i)
        si = S.ints([0, 1, 2, 3, 4], stream)
        keep = {n: L.from_device(getattr(layer, n), getattr(layer, n).nbytes, np.uint8, stream) for n in ("states", "tails")}
        first = S.down(layer.step(x_dev.at(), 5, si.at(), si.at(), 5), (5, hidden), stream)
        assert (first != 0).any(1).all()
        for n, a in keep.items():       # the same step again, from the same slots
            L.check(cs1.cs1_upload(getattr(layer, n).at(), a.ctypes.data, a.nbytes, stream.handle), "upload")
        so = S.ints([0, -1, 9, 3, 3], stream)                 # goes on, sits out, no such slot, two that write one
        start = S.ints([0, 1, 2, 3, 4, 5], stream)
        y = S.down(layer.step(x_dev.at(), 5, si.at(), so.at(), 4, start.at()), (5, hidden), stream)
        assert S.status()[2] == 61
        assert (y[0] == first[0]).all() and (y[3] == first[3]).all()
        assert (y[[1, 2, 4]] == 0).all()
        y = S.down(layer.step(x_dev.at(), 5, si.at(), so.at(), 5, start.at()), (5, hidden), stream)
        assert S.status()[2] in (61, 62)
        assert (y[1:] == 0).all() and (y[0] != 0).any()
        assert (L.from_device(layer.states, layer.states.nbytes // 6, np.uint8, stream, layer.states.nbytes // 6 * 4) != 0).any()
        layer.forward(x_dev.at(), 0, slot=4)                  # no tokens: the slot of a sequence that has not begun
        for buf in (layer.states, layer.tails):
            assert (L.from_device(buf, buf.nbytes // 6, np.uint8, stream, buf.nbytes // 6 * 4) == 0).all()
    finally:
        layer.close()


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 2), (3, 3), (2, 6), (5, 5)])
def test_layer_steps_with_any_number_of_heads(cs1, stream, hk, hv):
    """Heads whose gates leave a projected row at no multiple of 8: the step takes them as the prefill does."""
    from system1_omni_b200.gdn_layer import GdnLayer
    from test_gdn_layer_gpu import make_case, oracle_layer, rel_l2
    hidden, n, more = 256, 11, 3
    layer = GdnLayer(hidden, hk, hv, max_tokens=32, stream=stream, slots=1)
    try:
        x, w = make_case(n + more, hidden, hk, hv, seed=hv)
        layer.set_weights(**w)
        x_dev, slot = up(x, stream), S.ints([0], stream)
        y = f32(S.down(layer.forward(x_dev.at(), n, slot=0), (32, hidden), stream))[:n]
        for t in range(more):
            y = np.concatenate([y, f32(S.down(layer.step(x_dev.at((n + t) * hidden * 2), 1, slot.at(), slot.at(), 1), (1, hidden), stream))])
        want = f32(oracle_layer(x, w, n + more, hidden, hk, hv, float64_core=True))
        assert rel_l2(y, want) < 2e-2                          # the gate of the layer's prefill
        assert np.abs(y - want).max() < 5e-2 * np.abs(want).max()
    finally:
        layer.close()


# ---- groups at their limits ----

@pytest.mark.parametrize("hurt", [False, True])
def test_convolution_of_the_most_sequences(cs1, stream, hurt):
    """65535 sequences, 127 to a block, the last block short."""
    S.test_convolution_step_of_many_sequences(cs1, stream, 65535, hurt)


@pytest.mark.parametrize("hurt", [False, True])
def test_prep_of_the_most_rows(cs1, stream, hurt):
    """65536 rows, 128 to a block."""
    S.test_prep_of_many_rows(cs1, stream, 65536, 128, 2, 1, 48, hurt)


@pytest.mark.parametrize("nseq,H,HK,per", [(65535, 9, 3, 128), (43000, 16, 8, 128), (3000, 6, 6, 4)])
@pytest.mark.parametrize("hurt", [False, True])
def test_delta_rule_with_the_most_sequences_to_a_block(cs1, stream, nseq, H, HK, per, hurt):
    """Sequences that sit out, but for some: scattered, and every one of a block; all rows against the formula."""
    assert min(128, nseq * H // 4096) == per
    rng = np.random.default_rng(nseq + hurt)
    block = per * (nseq // per // 2)
    live = np.unique(np.concatenate([rng.permutation(nseq)[:60], block + np.arange(per), [0, per - 1, per, nseq - 1]]))
    lens = np.zeros(nseq, int)
    lens[live] = rng.integers(0, 4, len(live))
    lens[rng.permutation(nseq)[:50]] = 1                          # rows of sequences that sit out
    start = np.concatenate([[0], np.cumsum(lens)])
    so, si = np.full(nseq, -1), rng.integers(-1, 300, nseq)       # what begins a sequence that sits out is nobody's matter
    n = len(live)
    slots = n + 2
    so[live] = rng.permutation(n)
    si[live] = np.where(rng.random(n) < 0.4, n, np.where(rng.random(n) < 0.5, so[live], -1))
    refused = np.zeros(nseq, bool)
    if hurt:
        a, b, c, d, e = live[rng.permutation(n)[:5]]
        so[a] = so[b]                                             # two write one slot
        si[c], si[d] = so[d], -1                                  # one begins with what another writes
        so[e] = slots                                             # no such slot
        for i in live:
            others = [j for j in live if j != i]
            refused[i] = so[i] >= slots or any(so[i] in (so[j], si[j]) or (si[i] >= 0 and si[i] == so[j]) for j in others)
        assert refused[[a, b, c, d, e]].all() and refused.sum() < 12
    x = S.delta_inputs(start[-1], H, HK, slots, nseq)
    w, states, tol, tol_s = S.delta_formula(x, start, si, np.where(refused, -1, so), H, HK, S.D ** -0.5)
    got, new = S.run_delta(cs1, stream, x, start, si, so, H, HK, S.D ** -0.5, fill=int(NAN))
    assert (S.status()[2] in (61, 62)) == hurt
    rest = np.isnan(w)
    assert (got[rest] == NAN).all() and np.isfinite(f32(got[~rest])).all()
    assert (np.abs(f32(got).astype(np.float64) - w)[~rest] <= tol[~rest]).all()
    assert (np.abs(new.astype(np.float64) - states) <= tol_s).all()


@pytest.mark.parametrize("nseq", [2561, 9001])
def test_delta_rule_of_many_sequences_writes_every_row(cs1, stream, nseq):
    H, HK, scale = 4, 2, S.D ** -0.5
    x = S.delta_inputs(nseq, H, HK, 1, nseq)
    pool = L.DeviceBuffer(nseq * H * S.D * S.D * 4)
    d = {m: up(x[m], stream) for m in ("q", "k", "v", "g", "beta")}
    o = up(np.full(x["v"].shape, NAN, np.uint16), stream)
    so, si = S.ints(np.random.default_rng(1).permutation(nseq), stream), S.ints(np.full(nseq, -1), stream)
    L.check(cs1.s1_gdn_step(d["q"].at(), d["k"].at(), d["v"].at(), d["g"].at(), d["beta"].at(), o.at(), nseq, H, HK, scale, pool.at(), nseq,
                            H * S.D * S.D, None, si.at(), so.at(), nseq, stream.handle), "step")
    got = f32(S.down(o, x["v"].shape, stream)).astype(np.float64)
    # from zeros: S = k (beta v)^T, o = (q.k) beta v
    q, k, v, beta = (f32(x[m]).astype(np.float64) for m in ("q", "k", "v", "beta"))
    q, k = (a / np.sqrt((a ** 2).sum(-1, keepdims=True) + 1e-6) for a in (q, k))
    head = np.arange(H) // (H // HK)
    want = ((q * k).sum(-1) * scale)[:, head, None] * beta[..., None] * v
    # q.k is a sum of 128 products of unit vectors (48 roundings as in delta_formula), the rest a few more
    tol = HALF * np.abs(want) + 96 * EPS * scale * beta[..., None] * np.abs(v)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("nseq,H,HK,tokens", [(40, 16, 8, 2), (4100, 4, 2, 1)])
def test_dependent_launches_of_wide_and_grouped_steps_give_the_same_bits(cs1, stream, nseq, H, HK, tokens):
    """Convolution and delta rule in a chain, in place, with four warps to a block and with several sequences to one."""
    rows = nseq * tokens
    kd, vd = HK * S.D, H * S.D
    c = S.conv_case(rows, kd, vd, H, nseq, 0, 6)
    start = None if tokens == 1 else S.ints(np.arange(nseq + 1) * tokens, stream)
    res = []
    for mode in (0, 1, 2):
        before = cs1.s1_set_dependent_launch(mode)
        cd = {k: up(c[k], stream) for k in ("x", "w", "al", "dt", "tails")}
        q, k, v, o = (L.DeviceBuffer(rows * w * 2) for w in (kd, kd, vd, vd))
        beta, g, states = L.DeviceBuffer(rows * H * 2), L.DeviceBuffer(rows * H * 4), L.DeviceBuffer(nseq * H * S.D * S.D * 4)
        L.check(cs1.s1_memset_async(states.at(), 0, states.nbytes, stream.handle), "memset")
        s = S.ints(np.arange(nseq), stream)
        for _ in range(6):
            L.check(cs1.s1_gdn_conv_gates_step(cd["x"].at(), c["ld"], cd["w"].at(), q.at(), k.at(), v.at(), rows, kd, vd, cd["x"].at(2 * c["ch"]),
                                               cd["x"].at(2 * (c["ch"] + H)), cd["al"].at(), cd["dt"].at(), beta.at(), g.at(), H, cd["tails"].at(),
                                               nseq, 3 * c["ch"], S.at(start), s.at(), s.at(), nseq, stream.handle), "conv")
            L.check(cs1.s1_gdn_step(q.at(), k.at(), v.at(), g.at(), beta.at(), o.at(), rows, H, HK, S.D ** -0.5, states.at(), nseq, H * S.D * S.D,
                                    S.at(start), s.at(), s.at(), nseq, stream.handle), "step")
        cs1.s1_set_dependent_launch(before)
        res.append((S.down(o, (rows, vd), stream), S.down(states, (nseq * H * S.D * S.D,), stream, np.float32)))
    assert np.isfinite(f32(res[0][0])).all() and np.abs(res[0][1]).max() > 0
    for other in res[1:]:
        assert (other[0] == res[0][0]).all() and (other[1] == res[0][1]).all()
