"""The decode operators without a GPU: the owner of the pages (append, copy on write, fork, truncate,
compact) against a plain model of it, and the calls that the operators refuse before they touch the device."""
import ctypes as C
import random

import numpy as np
import pytest

from system1_omni_b200 import lib as L

ARGUMENT, PAGES, INVALID = 3000, 3009, 1


class Pool:
    """A handle, with the copies it asks for carried out on host pages of token labels."""

    def __init__(self, so, n_pages, page_tokens, seqs, seq_pages):
        self.so, self.page, self.wide = so, page_tokens, seq_pages
        self.h = C.c_void_p()
        assert so.s1_pages_create(n_pages, page_tokens, seqs, seq_pages, C.byref(self.h)) == 0
        self.mem = np.full((n_pages, page_tokens), -1, np.int64)
        self.text = [[] for _ in range(seqs)]       # what each sequence should read

    def close(self):
        self.so.s1_pages_destroy(self.h)

    def copies(self, call, cap=64):
        src, dst, n = np.full(cap, -7, np.int32), np.full(cap, -7, np.int32), C.c_int(-1)
        rc = call(src.ctypes.data, dst.ctypes.data, cap, C.byref(n))
        if rc == 0:
            assert 0 <= n.value <= cap and (src[n.value:] == -7).all()
            assert len(set(dst[:n.value])) == n.value and not set(dst[:n.value]) & set(src[:n.value])
            self.mem[dst[:n.value]] = self.mem[src[:n.value]]
        return rc

    def row(self, s):
        table, n = np.empty((1, self.wide), np.int32), np.empty(1, np.int32)
        assert self.so.s1_pages_table(self.h, s, 1, table.ctypes.data, self.wide, n.ctypes.data) == 0
        return table[0], int(n[0])

    def append(self, s, labels, cap=1):
        rc = self.copies(lambda a, b, c, n: self.so.s1_pages_append(self.h, s, len(labels), a, b, c, n), cap)
        if rc == 0:
            table, _ = self.row(s)
            for x in labels:
                at = len(self.text[s])
                self.mem[table[at // self.page], at % self.page] = x
                self.text[s].append(x)
        return rc

    def fork(self, a, b):
        rc = self.so.s1_pages_fork(self.h, a, b)
        if rc == 0:
            self.text[b] = list(self.text[a])
        return rc

    def truncate(self, s, n):
        rc = self.so.s1_pages_truncate(self.h, s, n)
        if rc == 0:
            del self.text[s][n:]
        return rc

    def compact(self, cap=64):
        return self.copies(lambda a, b, c, n: self.so.s1_pages_compact(self.h, a, b, c, n), cap)

    def check(self):
        used = set()
        for s, want in enumerate(self.text):
            table, n = self.row(s)
            assert n == len(want)
            pages = -(-n // self.page)
            assert (table[:pages] >= 0).all() and (table[pages:] == -1).all()
            assert len(set(table[:pages])) == pages
            used |= set(table[:pages].tolist())
            assert [self.mem[table[t // self.page], t % self.page] for t in range(n)] == want
        assert self.so.s1_pages_free_count(self.h) == len(self.mem) - len(used)
        return used


@pytest.mark.parametrize("page,seed", [(1, 0), (4, 1), (7, 2), (16, 3)])
def test_pages_keep_what_every_sequence_wrote(cs1, page, seed):
    rng = random.Random(seed)
    p = Pool(cs1, 40, page, 6, 12)
    label = 0
    failed = 0
    try:
        for _ in range(600):
            s = rng.randrange(6)
            what = rng.choice(["append", "append", "append", "fork", "cut", "free", "compact"])
            if what == "append":
                n = rng.choice([0, 1, 1, page, rng.randrange(1, 3 * page + 1)])
                rc = p.append(s, range(label, label + n))
                label += n
            elif what == "fork":
                rc = p.fork(s, rng.randrange(6))
            elif what == "cut":
                rc = p.truncate(s, rng.randrange(len(p.text[s]) + 1))
            elif what == "free":
                rc = p.truncate(s, 0)
            else:
                rc = p.compact()
                assert rc == 0
                used = p.check()
                assert used == set(range(len(used)))
            assert rc in (0, ARGUMENT, PAGES)
            failed += rc != 0
            p.check()
        assert failed > 0        # the walk met a full pool and forks onto used numbers
    finally:
        p.close()


def test_pages_share_until_one_writes(cs1):
    p = Pool(cs1, 8, 4, 3, 4)
    try:
        assert p.append(0, range(6)) == 0
        assert p.fork(0, 1) == 0 and p.fork(0, 2) == 0
        assert cs1.s1_pages_free_count(p.h) == 6
        before = p.row(0)[0].copy()
        assert p.append(1, [100], cap=0) == PAGES       # the copy has nowhere to be listed
        assert p.append(1, [100]) == 0                  # copies the half-filled page
        a, b = p.row(0)[0], p.row(1)[0]
        assert a[0] == b[0] and a[1] != b[1] and (a == before).all()
        assert p.append(2, [200]) == 0
        assert p.append(0, [6], cap=0) == 0             # alone on its page now: no copy
        assert p.row(0)[0][1] == before[1]
        # a full last page is shared on: nothing of it is written
        assert p.truncate(1, 4) == 0 and p.truncate(2, 4) == 0
        assert p.append(1, [9], cap=0) == 0
        p.check()
    finally:
        p.close()


def test_pages_refuse_and_change_nothing(cs1):
    p = Pool(cs1, 4, 4, 3, 3)
    h = p.h
    n = C.c_int()
    try:
        assert p.append(0, range(9)) == 0
        assert p.append(0, range(4)) == PAGES           # a fourth page does not fit its table row
        assert p.append(1, range(5)) == PAGES           # one page is free
        assert p.append(1, range(4)) == 0
        for rc in (cs1.s1_pages_append(h, 3, 1, None, None, 0, C.byref(n)), cs1.s1_pages_append(h, -1, 1, None, None, 0, C.byref(n)),
                   cs1.s1_pages_append(h, 0, -1, None, None, 0, C.byref(n)), cs1.s1_pages_append(h, 0, 1, None, None, 1, C.byref(n)),
                   cs1.s1_pages_append(h, 0, 1, None, None, 0, None), cs1.s1_pages_append(None, 0, 1, None, None, 0, C.byref(n)),
                   cs1.s1_pages_fork(h, 0, 0), cs1.s1_pages_fork(h, 0, 1), cs1.s1_pages_fork(h, 0, 3), cs1.s1_pages_fork(h, -1, 2),
                   cs1.s1_pages_truncate(h, 0, 10), cs1.s1_pages_truncate(h, 0, -1), cs1.s1_pages_truncate(h, 5, 0),
                   cs1.s1_pages_table(h, 0, 1, np.empty(2, np.int32).ctypes.data, 2, None),
                   cs1.s1_pages_table(h, 2, 2, None, 0, None), cs1.s1_pages_table(h, -1, 1, None, 0, None),
                   cs1.s1_pages_compact(h, None, None, 0, None)):
            assert rc == ARGUMENT
        p.check()
        assert cs1.s1_pages_fork(h, 0, 2) == 0
        p.text[2] = list(p.text[0])
        assert p.append(2, [1]) == PAGES                # its copy finds no free page
        assert cs1.s1_pages_append(h, 2, 0, None, None, 0, C.byref(n)) == 0 and n.value == 0
        assert p.truncate(0, 0) == 0
        assert p.append(2, [1], cap=0) == 0
        p.check()
        for args in ((0, 4, 1, 1), (4, 0, 1, 1), (4, 4, 0, 1), (4, 4, 1, 0), (4, 1 << 20, 1, 1 << 20)):
            out = C.c_void_p()
            assert cs1.s1_pages_create(*args, C.byref(out)) == ARGUMENT and not out.value
        assert cs1.s1_pages_create(4, 4, 1, 1, None) == ARGUMENT
        assert b"pages" in cs1.cs1_error_string(PAGES)
        cs1.s1_pages_destroy(None)
        assert cs1.s1_pages_free_count(None) == 0
    finally:
        p.close()


def test_pages_compaction_needs_room_for_its_list(cs1):
    p = Pool(cs1, 8, 2, 3, 8)
    try:
        for s in range(3):
            assert p.append(s, range(10 * s, 10 * s + 4)) == 0
        assert p.truncate(0, 0) == 0
        before = [p.row(s)[0].tolist() for s in range(3)]
        assert p.compact(cap=1) == PAGES
        assert [p.row(s)[0].tolist() for s in range(3)] == before
        assert p.compact(cap=2) == 0
        assert p.check() == {0, 1, 2, 3}
        assert p.compact(cap=0) == 0                    # nothing left to move
    finally:
        p.close()


A = 1 << 20      # a plausible, aligned address; nothing below reaches the device


def step(cs1, **kw):
    a = dict(q=A, k=A, v=A, g=A, beta=A, o=A, rows=4, H=4, HK=2, scale=1.0, states=A, n_slots=4, stride=4 * 16384, start=None, si=A,
             so=A, nseq=4)
    a.update(kw)
    return cs1.s1_gdn_step(a["q"], a["k"], a["v"], a["g"], a["beta"], a["o"], a["rows"], a["H"], a["HK"], a["scale"], a["states"],
                           a["n_slots"], a["stride"], a["start"], a["si"], a["so"], a["nseq"], None)


@pytest.mark.parametrize("bad", [dict(H=0), dict(HK=0), dict(HK=3), dict(rows=-1), dict(nseq=-1), dict(n_slots=-1), dict(stride=4 * 16384 - 4),
                                 dict(stride=4 * 16384 + 2), dict(si=None), dict(so=None), dict(states=None), dict(states=A + 4),
                                 dict(q=None), dict(k=A + 8), dict(v=A + 2), dict(o=None), dict(g=None), dict(beta=None),
                                 dict(nseq=65536), dict(nseq=65535, H=1 << 15, HK=1, stride=(1 << 15) * 16384)])
def test_delta_rule_step_refuses(cs1, bad):
    assert step(cs1, **bad) == INVALID


def test_steps_without_sequences_do_nothing(cs1):
    assert step(cs1, nseq=0, q=None, states=None, si=None, so=None) == 0
    assert conv(cs1, nseq=0, x=None, tails=None, si=None, so=None) == 0
    assert prep(cs1, rows=0, qg=None, table=None, pos=None) == 0
    assert attention(cs1, rows=0, q=None, table=None, len=None) == 0
    assert copy(cs1, n=0, src=None, dst=None) == 0 and copy(cs1, pools=[]) == 0


def conv(cs1, **kw):
    a = dict(x=A, ld=64, w=A, q=A, k=A, v=A, rows=4, kd=16, vd=16, b=A, a=A, al=A, dt=A, beta=A, g=A, H=2, tails=A, n_slots=4, stride=144,
             start=None, si=A, so=A, nseq=4)
    a.update(kw)
    return cs1.s1_gdn_conv_gates_step(a["x"], a["ld"], a["w"], a["q"], a["k"], a["v"], a["rows"], a["kd"], a["vd"], a["b"], a["a"], a["al"],
                                      a["dt"], a["beta"], a["g"], a["H"], a["tails"], a["n_slots"], a["stride"], a["start"], a["si"],
                                      a["so"], a["nseq"], None)


@pytest.mark.parametrize("bad", [dict(ld=40), dict(ld=60), dict(kd=12), dict(vd=4), dict(kd=0), dict(H=0), dict(rows=-1), dict(nseq=-1),
                                 dict(nseq=65536), dict(n_slots=-2), dict(stride=136), dict(stride=148), dict(si=None), dict(so=None),
                                 dict(tails=None), dict(tails=A + 2), dict(w=None), dict(w=A + 8), dict(x=None), dict(x=A + 2), dict(q=A + 8),
                                 dict(k=None), dict(v=A + 4), dict(b=None), dict(a=None), dict(al=None), dict(dt=None), dict(beta=None),
                                 dict(g=None), dict(kd=1 << 30, vd=1 << 30, ld=2147483640)])
def test_convolution_step_refuses(cs1, bad):
    assert conv(cs1, **bad) == INVALID


def prep(cs1, **kw):
    a = dict(qg=A, kr=A, vr=A, ld=2048, qw=A, kw=A, cos=A, sin=A, angles=64, angle=None, q=A, gate=A, kp=A, vp=A, n_pages=4, page=16, table=A,
             wide=4, seqs=4, seq=None, pos=A, rows=4, Hq=4, Hk=2, Dh=128, half=16)
    a.update(kw)
    return cs1.s1_attn_prep_paged(a["qg"], a["kr"], a["vr"], a["ld"], a["qw"], a["kw"], a["cos"], a["sin"], a["angles"], a["angle"], a["q"],
                                  a["gate"], a["kp"], a["vp"], a["n_pages"], a["page"], a["table"], a["wide"], a["seqs"], a["seq"], a["pos"],
                                  a["rows"], a["Hq"], a["Hk"], a["Dh"], a["half"], 1e-6, None)


@pytest.mark.parametrize("bad", [dict(Dh=64), dict(Hq=0), dict(Hk=0), dict(ld=2047), dict(ld=1016), dict(rows=-1), dict(rows=65537), dict(half=0), dict(half=12),
                                 dict(half=24), dict(half=128), dict(angles=-1), dict(n_pages=0), dict(page=0), dict(table=None),
                                 dict(wide=0), dict(seqs=0), dict(pos=None), dict(n_pages=1 << 28), dict(wide=1 << 27), dict(qg=None),
                                 dict(kr=A + 2), dict(vr=None), dict(qw=A + 8), dict(kw=None), dict(cos=None), dict(sin=A + 4),
                                 dict(q=None), dict(gate=A + 2), dict(kp=None), dict(vp=A + 8)])
def test_prep_refuses(cs1, bad):
    assert prep(cs1, **bad) == INVALID


def attention(cs1, **kw):
    a = dict(q=A, gate=None, out=A, kp=A, vp=A, n_pages=4, page=16, table=A, wide=4, seqs=4, seq=None, len=A, rows=4, Hq=4, Hk=2, Dh=128,
             ws=A, floats=None)
    a.update(kw)
    if a["floats"] is None:
        a["floats"] = cs1.s1_attention_paged_workspace_floats(4, 2, 128)
    return cs1.s1_attention_paged(a["q"], a["gate"], a["out"], a["kp"], a["vp"], a["n_pages"], a["page"], a["table"], a["wide"], a["seqs"],
                                  a["seq"], a["len"], a["rows"], a["Hq"], a["Hk"], a["Dh"], 1.0, a["ws"], a["floats"], None)


@pytest.mark.parametrize("bad", [dict(Dh=64), dict(Hk=3), dict(Hk=0), dict(Hq=0), dict(rows=-1), dict(rows=(1 << 20) + 1), dict(page=8),
                                 dict(page=24), dict(page=0), dict(n_pages=0), dict(n_pages=1 << 27), dict(wide=0), dict(wide=1 << 27),
                                 dict(seqs=0), dict(table=None), dict(len=None), dict(q=None), dict(q=A + 8), dict(out=None),
                                 dict(out=A + 4), dict(gate=A + 2), dict(kp=None), dict(kp=A + 8), dict(vp=A + 2), dict(ws=None),
                                 dict(ws=A + 4), dict(floats=100)])
def test_paged_attention_refuses(cs1, bad):
    assert attention(cs1, **bad) == INVALID


def test_paged_attention_workspace(cs1):
    f = cs1.s1_attention_paged_workspace_floats
    assert 0 < f(24, 4, 128) < f(16, 4, 128) and f(24, 4, 256) < f(16, 4, 256)      # rows of a product: 2 * 6 and 4 * 4
    assert max(f(q, k, d) for q in range(1, 65) for k in range(1, q + 1) for d in (128, 256)) < 5 << 20
    assert f(16, 1, 256) == f(32, 1, 256)          # more than 16 heads of one key-value head go in parts
    assert f(4, 3, 128) == f(0, 1, 128) == f(4, 0, 128) == f(4, 4, 64) == 0


def copy(cs1, pools=(A, 2 * A), n_pages=8, page_bytes=32, src=(0, 1), dst=(4, 5), n=2):
    arr = (C.c_void_p * max(1, len(pools)))(*pools)
    ints = [None if x is None else np.array(x, np.int32) for x in (src, dst)]
    return cs1.s1_pages_copy(arr, len(pools), n_pages, page_bytes, *(x if x is None else x.ctypes.data for x in ints), n, None)


@pytest.mark.parametrize("bad", [dict(page_bytes=0), dict(page_bytes=24), dict(page_bytes=1 << 35), dict(n_pages=-1), dict(n=-1), dict(src=None),
                                 dict(dst=None), dict(pools=(A, 0)), dict(pools=(A + 8,)), dict(src=(0, 8)), dict(src=(-1, 0)),
                                 dict(dst=(8, 1)), dict(dst=(4, -4)), dict(dst=(4, 4)), dict(dst=(4, 0)), dict(src=(0, 4)),
                                 dict(src=(3, 1), dst=(3, 2))])
def test_page_copies_refuse(cs1, bad):
    assert copy(cs1, **bad) == INVALID


def test_direct_calls_answer_as_ctypes_does(cs1):
    """Plain numbers go straight to the library, everything else through ctypes: the same answers and errors."""
    from system1_omni_b200 import _fastcall
    assert set(_fastcall.NAMES) == {"s1_gdn_step", "s1_gdn_conv_gates_step", "s1_attn_prep_paged", "s1_attention_paged", "s1_pages_copy"}
    for name in _fastcall.NAMES:
        assert type(getattr(cs1, name)).__name__ == "Bound"
    f = cs1.s1_gdn_step
    plain = [A, A, A, A, A, A, 4, 4, 2, 1.0, A, 4, 4 * 16384, None, A, A, 0, None]
    assert f(*plain) == 0                                               # no sequences
    for i in (0, 9, 10, 13, 17):                                        # another kind of argument at one place
        a = list(plain)
        a[i] = C.c_void_p(a[i]) if i != 9 else 1
        assert f(*a) == 0
    bad = list(plain)
    bad[7] = 0                                                          # H
    assert f(*bad) == INVALID
    bad[0] = C.c_void_p(A)
    assert f(*bad) == INVALID
    for args in ([], plain[:-1], [object()] + plain[1:], plain[:6] + ["4"] + plain[7:]):
        with pytest.raises((TypeError, C.ArgumentError)):
            f(*args)
    wide = list(plain)
    wide[16] = 1 << 32                                                  # ctypes keeps the low 32 bits of an int: nseq 0
    assert f(*wide) == 0
    assert f(*plain[:6], True, *plain[7:]) == 0


def test_an_error_code_names_one_thing():
    """s1_device_status reports a family's waits and its step operators' refusals in one place: no code stands for both."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "system1_omni_b200", "csrc")
    read = lambda name: open(os.path.join(csrc, name)).read()
    for waits, steps, enum in (("attention_tc5.cu", "paged.cu", r"PAGED_\w+ = (\d+)"), ("gdn.cu", "step.h", r"STEP_[A-Z_]+ = (\d+)")):
        of_waits = set(re.findall(r"fail\((\d+)\)", read(waits))) | set(re.findall(r"atomicCAS\(&\w+, 0, (\d+)\)", read(waits)))
        of_steps = set(re.findall(enum, read(steps)))
        assert of_waits and len(of_steps) >= 3
        assert not of_waits & of_steps
