"""The decode operators of libqwen3_5_cuda.so as measured cases: the tokens after a prefill.

s1_gdn_step             the gated delta rule token by token on float32 states kept in slots
s1_gdn_conv_gates_step  the causal convolution and the gates of new tokens, the last three rows kept in slots
s1_attn_prep_paged      norm, rotary and gate split of new tokens, keys and values appended to a paged cache
s1_attention_paged      attention of one new token per row over the paged cache
s1_pages_copy           copies of pages (fork, copy on write, compaction) over all layers' pools

`run` computes a case in its plain form with torch, or with `own` through the library. All
sizes of a case follow from its own values; the seed fills the tensors and shuffles slots and pages.
"""
import functools
import math

import torch

own = False

KEY = 128           # head dim of the delta rule
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def spread(n, lo, hi):
    """n whole numbers between lo and hi, spread evenly over their logarithm, the first one hi."""
    return [hi if i == 0 else int(round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def windows(case):
    """New tokens of each sequence."""
    return [1 + (i * 5 + 2) % case["tokens"] for i in range(case["nseq"])]


def listed():
    return [
        # the next token of one request on the 4B-shaped decoder: all latency
        dict(name="delta rule, 1 sequence", op="delta", nseq=1, H=32, HK=16, tokens=1, share=False),
        # a serving batch on the 27B-shaped decoder, one token each, states updated in place
        dict(name="delta rule, 193 sequences", op="delta", nseq=193, H=48, HK=16, tokens=1, share=False),
        # short candidates of one captured prefix: every sequence starts from the prefix's state
        dict(name="delta rule, 37 candidates", op="delta", nseq=37, H=32, HK=16, tokens=9, share=True),
        # the convolution and gates before the first and the second of these
        dict(name="convolution, 1 sequence", op="conv", nseq=1, H=32, HK=16, tokens=1, share=False),
        dict(name="convolution, 193 sequences", op="conv", nseq=193, H=48, HK=16, tokens=1, share=False),
        # keys, values and queries of the next token: one request, and a batch at head dim 256
        dict(name="prep, 1 row", op="prep", rows=1, Hq=24, Hk=4, Dh=128, half=32, page=64, longest=1500),
        dict(name="prep, 251 rows", op="prep", rows=251, Hq=16, Hk=4, Dh=256, half=32, page=16, longest=9000),
        # attention of one request behind a prompt of ordinary length
        dict(name="attention, 1 x 1500", op="attention", rows=1, Hq=24, Hk=4, Dh=128, page=64, shortest=1500, longest=1500, gated=True, per_seq=1),
        # a serving batch whose lengths differ by a factor of thirty
        dict(name="attention, 65 ragged", op="attention", rows=65, Hq=24, Hk=4, Dh=128, page=64, shortest=500, longest=16000, gated=True, per_seq=1),
        # one request at the longest positions of the configuration
        dict(name="attention, 1 x 250001", op="attention", rows=1, Hq=16, Hk=4, Dh=256, page=16, shortest=250001, longest=250001, gated=True, per_seq=1),
        # a fork's copies: the partly filled last page of a prefix for three candidates, in the 16 attention layers' two pools each
        dict(name="pages, fork by 3", op="pages", pools=32, pages=40, page_bytes=65536, pairs=3, fan=3),
        # a compaction: a third of the pool moves down
        dict(name="pages, 337 moved", op="pages", pools=32, pages=1024, page_bytes=65536, pairs=337, fan=1),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["delta", "delta", "conv", "prep", "attention", "attention", "attention", "pages"])
    if op in ("delta", "conv"):
        HK, H = rng.choice([(16, 16), (16, 32), (16, 48), (8, 24), (2, 6), (4, 4)])
        share = rng.random() < 0.3
        tokens = 1 if rng.random() < 0.6 else log(2, 17)
        return dict(op=op, nseq=log(1, 193 if tokens == 1 else 48), H=H, HK=HK, tokens=tokens, share=share)
    Hq, Hk = rng.choice([(24, 4), (16, 4), (16, 2), (8, 8), (12, 1), (32, 1), (40, 2)])
    Dh = rng.choice([128, 256])
    page = rng.choice([16, 32, 48, 64, 80, 128, 256])
    if op == "prep":
        return dict(op=op, rows=log(1, 400), Hq=Hq, Hk=Hk, Dh=Dh, half=rng.choice([16, 32, 64]), page=page, longest=log(2, 20000))
    if op == "attention":
        rows = log(1, 200)
        longest = log(1, max(2, min(200000, 200000 * 1024 // (rows * Hk * Dh))))
        return dict(op=op, rows=rows, Hq=Hq, Hk=Hk, Dh=Dh, page=page, shortest=max(1, longest // rng.choice([1, 5, 40])), longest=longest,
                    gated=rng.random() < 0.7, per_seq=rng.choice([1, 1, 3]))
    fan = rng.choice([1, 1, 2, 5])
    pairs = log(1, 300)
    return dict(op=op, pools=log(1, 32), pages=pairs + -(-pairs // fan) + log(1, 300), page_bytes=rng.choice([2048, 16384, 49152, 65536]), pairs=pairs, fan=fan)


def lengths(case):
    """Cache tokens that each row of an attention or prep case sees, its own one among them."""
    if case["op"] == "prep":
        return spread(case["rows"], 1, case["longest"])
    n = -(-case["rows"] // case["per_seq"])
    base = spread(n, case["shortest"], case["longest"])
    return [max(1, base[r // case["per_seq"]] - (case["per_seq"] - 1 - r % case["per_seq"])) for r in range(case["rows"])]


def work(case):
    op = case["op"]
    if op in ("delta", "conv"):
        n, H, HK = sum(windows(case)), case["H"], case["HK"]
        kd, vd = HK * KEY, H * KEY
        if op == "delta":
            state = H * KEY * KEY * 4
            return dict(bytes=(state if case["share"] else case["nseq"] * state) + case["nseq"] * state + n * (2 * kd + 2 * vd + H) * 2 + n * H * 4,
                        flops=n * H * KEY * KEY * 7)
        ch = 2 * kd + vd
        tail = 3 * ch * 2
        return dict(bytes=(tail if case["share"] else case["nseq"] * tail) + case["nseq"] * tail + 2 * n * ch * 2 + ch * 8 + n * H * (4 + 2 + 4) + 4 * H,
                    flops=n * ch * 12)
    if op == "prep":
        qw, kw = case["Hq"] * case["Dh"], case["Hk"] * case["Dh"]
        return dict(bytes=case["rows"] * (2 * (2 * qw + 2 * kw) * 2 + 2 * case["half"] * 2) + case["Dh"] * 4, flops=case["rows"] * (qw + kw) * 8)
    if op == "attention":
        # rows of one sequence read one cache: its longest row's part of it
        seen = {}
        for r, t in enumerate(lengths(case)):
            seen[r // case["per_seq"]] = max(seen.get(r // case["per_seq"], 0), t)
        wide = case["Hq"] * case["Dh"]
        return dict(bytes=sum(seen.values()) * case["Hk"] * case["Dh"] * 4 + case["rows"] * wide * (6 if case["gated"] else 4),
                    flops=4 * sum(lengths(case)) * wide)
    sources = -(-case["pairs"] // case["fan"])
    return dict(bytes=case["pools"] * case["page_bytes"] * (sources + case["pairs"]), flops=0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)

    def normal(*shape, std=1.0, dtype=BF):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=F32) * std).to(dtype)

    def shuffled(n):
        return torch.randperm(n, generator=gen, device="cuda")

    def ints(values):
        return torch.tensor(values, dtype=I32, device="cuda")

    op = case["op"]
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if op in ("delta", "conv"):
        nseq, H, HK = case["nseq"], case["H"], case["HK"]
        lens = windows(case)
        n = sum(lens)
        order = shuffled(nseq + 3).to(I32)
        s["rows"], s["slots"] = n, nseq + 3
        s["slot_out"] = order[:nseq].contiguous()
        s["slot_in"] = order[nseq:nseq + 1].repeat(nseq) if case["share"] else s["slot_out"].clone()
        s["start"] = None if case["tokens"] == 1 else ints([sum(lens[:i]) for i in range(nseq + 1)])
        kd, vd = HK * KEY, H * KEY
        a_log = torch.rand(H, generator=gen, device="cuda") * math.log(16.0)
        dt = normal(H, std=0.1)
        if op == "delta":
            act = torch.nn.functional.silu
            s["q"], s["k"] = act(normal(n, HK, KEY, dtype=F32)).to(BF), act(normal(n, HK, KEY, dtype=F32)).to(BF)
            s["v"] = act(normal(n, H, KEY, dtype=F32)).to(BF)
            s["g"] = (-a_log.exp() * torch.nn.functional.softplus(normal(n, H, dtype=F32) + dt.float())).contiguous()
            s["beta"] = torch.sigmoid(normal(n, H, dtype=F32)).to(BF)
            s["o"] = torch.zeros(n, H, KEY, dtype=BF, device="cuda")
            s["states"] = normal(nseq + 3, H, KEY, KEY, std=0.1, dtype=F32)
        else:
            ch = 2 * kd + vd
            s["ld"] = ch + vd + 2 * H
            s["x"] = normal(n, s["ld"])
            s["w"] = normal(ch, 4, std=0.3)
            s["a_log"], s["dt"] = a_log.to(BF), dt
            s["q"], s["k"] = (torch.zeros(n, kd, dtype=BF, device="cuda") for _ in range(2))
            s["v"] = torch.zeros(n, vd, dtype=BF, device="cuda")
            s["beta"], s["g"] = torch.zeros(n, H, dtype=BF, device="cuda"), torch.zeros(n, H, dtype=F32, device="cuda")
            s["tails"] = normal(nseq + 3, 3, ch)
    elif op in ("prep", "attention"):
        rows, Hq, Hk, Dh, page = case["rows"], case["Hq"], case["Hk"], case["Dh"], case["page"]
        lens = lengths(case)
        per = case.get("per_seq", 1)
        nseq = -(-rows // per)
        seq = [r // per for r in range(rows)]
        need = [0] * nseq
        for r in range(rows):
            need[seq[r]] = max(need[seq[r]], -(-lens[r] // page))
        wide = max(need) + 1
        total = sum(need)
        n_pages = total + 5
        ids = shuffled(n_pages)[:total].cpu().tolist()
        table, at = [], 0
        for p in need:
            table.append(ids[at:at + p] + [-1] * (wide - p))
            at += p
        s["table"], s["seq"], s["n_pages"], s["nseq"] = ints(table), ints(seq), n_pages, nseq
        if op == "prep":
            s["pos"] = ints([t - 1 for t in lens])
            s["ld"] = 2 * Hq * Dh + 2 * Hk * Dh
            s["x"] = normal(rows, s["ld"])
            s["qw"], s["kw"] = normal(Dh, std=0.1), normal(Dh, std=0.1)
            inv = 1e7 ** (-torch.arange(case["half"], device="cuda", dtype=F64) / case["half"])
            angle = torch.arange(case["longest"], device="cuda", dtype=F64)[:, None] * inv
            s["cos"], s["sin"] = angle.cos().to(BF), angle.sin().to(BF)
            s["q"], s["gate"] = (torch.zeros(rows, Hq, Dh, dtype=BF, device="cuda") for _ in range(2))
            s["k_pages"], s["v_pages"] = (normal(n_pages, page, Hk, Dh) for _ in range(2))
        else:
            s["len"] = ints(lens)
            s["q"], s["gate"] = normal(rows, Hq, Dh), normal(rows, Hq, Dh)
            s["out"] = torch.zeros(rows, Hq, Dh, dtype=BF, device="cuda")
            s["k_pages"], s["v_pages"] = (normal(n_pages, page, Hk, Dh) for _ in range(2))
            # what lies behind a sequence's end in its last page was never written
            for i, p in enumerate(need):
                end = max(lens[r] for r in range(i * per, min(rows, i * per + per)))
                if end % page:
                    for pool in (s["k_pages"], s["v_pages"]):
                        pool[table[i][p - 1], end % page:] = float("nan")
            s["floats"] = 8 << 20
            s["work"] = torch.empty(s["floats"], dtype=F32, device="cuda")
    else:
        order = shuffled(case["pages"]).tolist()
        src = [order[i // case["fan"]] for i in range(case["pairs"])]
        dst = order[-case["pairs"]:]
        s["src"], s["dst"] = torch.tensor(src, dtype=I32), torch.tensor(dst, dtype=I32)   # host lists: the page tables' owner makes them
        s["src_at"], s["dst_at"] = s["src"].cuda().long(), s["dst"].cuda().long()
        s["pool"] = normal(case["pools"], case["pages"], case["page_bytes"] // 2)
        s["pools"] = torch.tensor([s["pool"][i].data_ptr() for i in range(case["pools"])], dtype=torch.int64)
    # the addresses that a program which owns these buffers passes
    s["at"] = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return s


# ---- plain forms ----

def row_places(s):
    """Sequence of each row and its place in the sequence."""
    case = s["case"]
    n = torch.tensor(windows(case), device="cuda")
    seq = torch.repeat_interleave(torch.arange(case["nseq"], device="cuda"), n)
    return n, seq, torch.arange(s["rows"], device="cuda") - (torch.cumsum(n, 0) - n)[seq]


def plain_delta(s):
    case = s["case"]
    H, HK = case["H"], case["HK"]

    def unit(x):
        x = x.float()
        return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)

    q = unit(s["q"]).repeat_interleave(H // HK, 1) * KEY ** -0.5
    k = unit(s["k"]).repeat_interleave(H // HK, 1)
    v, decay, beta = s["v"].float(), s["g"].exp(), s["beta"].float()
    state = s["states"][s["slot_in"].long()]
    n, seq, place = row_places(s)
    first = torch.cumsum(n, 0) - n
    o = torch.zeros_like(v)
    for t in range(case["tokens"]):
        live = (n > t).nonzero()[:, 0] if case["tokens"] > 1 else slice(None)
        r = first[live] + t
        S = state[live] * decay[r][..., None, None]
        delta = (v[r] - (k[r][..., None] * S).sum(-2)) * beta[r][..., None]
        S = S + k[r][..., None] * delta[..., None, :]
        o[r] = (q[r][..., None] * S).sum(-2)
        state[live] = S
    s["o"].copy_(o)
    s["states"][s["slot_out"].long()] = state
    return {"o": s["o"], "states": s["states"]}


def plain_conv(s):
    case = s["case"]
    H, kd, vd = case["H"], case["HK"] * KEY, case["H"] * KEY
    ch = 2 * kd + vd
    n, seq, place = row_places(s)
    x = s["x"][:, :ch].float()
    tail = s["tails"][s["slot_in"].long()].float()
    # the row `back` rows before each row, out of the kept rows where it lies before the first
    y = torch.zeros_like(x)
    rows = torch.arange(s["rows"], device="cuda")
    for back in range(4):
        old = place < back
        before = torch.where(old[:, None], tail[seq, torch.where(old, 3 + place - back, 0)], x[(rows - back).clamp(min=0)])
        y = y + before * s["w"].float()[:, 3 - back]
    y = y / (1 + (-y).exp())
    s["q"].copy_(y[:, :kd])
    s["k"].copy_(y[:, kd:2 * kd])
    s["v"].copy_(y[:, 2 * kd:])
    b, a = s["x"][:, ch + vd:ch + vd + H].float(), s["x"][:, ch + vd + H:].float() + s["dt"].float()
    s["beta"].copy_(1 / (1 + (-b).exp()))
    s["g"].copy_(-s["a_log"].float().exp() * (a.clamp(min=0) + torch.log1p((-a.abs()).exp())))
    # the last three rows of the kept ones and the new ones
    last = torch.cumsum(n, 0) - 1
    back = torch.arange(2, -1, -1, device="cuda")
    at = n[:, None] - 1 - back
    kept = torch.where((at < 0)[..., None], s["tails"][s["slot_in"].long()[:, None], (3 + at).clamp(0, 2)],
                       s["x"][(last[:, None] - back).clamp(min=0), :ch])
    s["tails"][s["slot_out"].long()] = kept
    return {k: s[k] for k in ("q", "k", "v", "beta", "g", "tails")}


def plain_prep(s):
    case = s["case"]
    rows, Hq, Hk, Dh, half = case["rows"], case["Hq"], case["Hk"], case["Dh"], case["half"]
    pos = s["pos"].long()
    cos, sin = s["cos"][pos].float()[:, None], s["sin"][pos].float()[:, None]

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.float())
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    qg = s["x"][:, :2 * Hq * Dh].view(rows, Hq, 2, Dh)
    kv = s["x"][:, 2 * Hq * Dh:].view(rows, 2, Hk, Dh)
    s["q"].copy_(turned(qg[:, :, 0], s["qw"]))
    s["gate"].copy_(qg[:, :, 1])
    at = s["table"].long()[s["seq"].long(), pos // case["page"]]
    s["k_pages"][at, pos % case["page"]] = turned(kv[:, 0], s["kw"]).to(BF)
    s["v_pages"][at, pos % case["page"]] = kv[:, 1]
    return {k: s[k] for k in ("q", "gate", "k_pages", "v_pages")}


def plain_attention(s):
    case = s["case"]
    rows, Hq, Hk, Dh = case["rows"], case["Hq"], case["Hk"], case["Dh"]
    most = -(-case["longest"] // case["page"])
    pages = s["table"].long()[s["seq"].long(), :most].clamp(min=0)
    T = most * case["page"]
    seen = torch.arange(T, device="cuda") < s["len"][:, None]
    k = torch.where(seen[..., None, None], s["k_pages"][pages].view(rows, T, Hk, Dh), 0).permute(0, 2, 3, 1).float()
    q = s["q"].view(rows, Hk, Hq // Hk, Dh).float() * Dh ** -0.5
    score = (q @ k).masked_fill(~seen[:, None, None], float("-inf"))
    del k
    p = (score - score.amax(-1, keepdim=True)).exp()
    v = torch.where(seen[..., None, None], s["v_pages"][pages].view(rows, T, Hk, Dh), 0).transpose(1, 2).float()
    o = ((p @ v) / p.sum(-1, keepdim=True)).view(rows, Hq, Dh)
    if case["gated"]:
        o = o / (1 + (-s["gate"].float()).exp())
    s["out"].copy_(o)
    return s["out"]


def plain_pages(s):
    s["pool"][:, s["dst_at"]] = s["pool"][:, s["src_at"]]
    return s["pool"]


# ---- the library's entry points ----

@functools.lru_cache(maxsize=1)
def binding():
    from system1_omni_b200 import lib
    return lib, lib.load()


def own_delta(s):
    lib, so = binding()
    c, at = s["case"], s["at"]
    lib.check(so.s1_gdn_step(at["q"], at["k"], at["v"], at["g"], at["beta"], at["o"], s["rows"], c["H"], c["HK"], KEY ** -0.5, at["states"],
                             s["slots"], c["H"] * KEY * KEY, at.get("start"), at["slot_in"], at["slot_out"], c["nseq"], s["stream"]), "delta rule step")
    return {"o": s["o"], "states": s["states"]}


def own_conv(s):
    lib, so = binding()
    c, at = s["case"], s["at"]
    kd, vd = c["HK"] * KEY, c["H"] * KEY
    b = at["x"] + 2 * (2 * kd + 2 * vd)
    lib.check(so.s1_gdn_conv_gates_step(at["x"], s["ld"], at["w"], at["q"], at["k"], at["v"], s["rows"], kd, vd, b, b + 2 * c["H"], at["a_log"], at["dt"],
                                        at["beta"], at["g"], c["H"], at["tails"], s["slots"], 3 * (2 * kd + vd), at.get("start"), at["slot_in"],
                                        at["slot_out"], c["nseq"], s["stream"]), "convolution step")
    return {k: s[k] for k in ("q", "k", "v", "beta", "g", "tails")}


def own_prep(s):
    lib, so = binding()
    c, at = s["case"], s["at"]
    kr = at["x"] + 2 * (2 * c["Hq"] * c["Dh"])
    lib.check(so.s1_attn_prep_paged(at["x"], kr, kr + 2 * c["Hk"] * c["Dh"], s["ld"], at["qw"], at["kw"], at["cos"], at["sin"], c["longest"], None,
                                    at["q"], at["gate"], at["k_pages"], at["v_pages"], s["n_pages"], c["page"], at["table"], s["table"].shape[1],
                                    s["nseq"], at["seq"], at["pos"], c["rows"], c["Hq"], c["Hk"], c["Dh"], c["half"], 1e-6, s["stream"]), "prep")
    return {k: s[k] for k in ("q", "gate", "k_pages", "v_pages")}


def own_attention(s):
    lib, so = binding()
    c, at = s["case"], s["at"]
    lib.check(so.s1_attention_paged(at["q"], at["gate"] if c["gated"] else None, at["out"], at["k_pages"], at["v_pages"], s["n_pages"], c["page"],
                                    at["table"], s["table"].shape[1], s["nseq"], at["seq"], at["len"], c["rows"], c["Hq"], c["Hk"], c["Dh"],
                                    c["Dh"] ** -0.5, at["work"], s["floats"], s["stream"]), "attention")
    return s["out"]


def own_pages(s):
    lib, so = binding()
    c, at = s["case"], s["at"]
    lib.check(so.s1_pages_copy(at["pools"], c["pools"], c["pages"], c["page_bytes"], at["src"], at["dst"], c["pairs"], s["stream"]), "page copies")
    return s["pool"]


PLAIN = dict(delta=plain_delta, conv=plain_conv, prep=plain_prep, attention=plain_attention, pages=plain_pages)
OWN = dict(delta=own_delta, conv=own_conv, prep=own_prep, attention=own_attention, pages=own_pages)


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- 64 bits, sequence by sequence ----

def exact(case, seed):
    s = prepare(case, seed)
    return dict(delta=exact_delta, conv=exact_conv, prep=exact_prep, attention=exact_attention, pages=exact_pages)[case["op"]](s, case)


def exact_delta(s, case):
    H, HK = case["H"], case["HK"]
    states = s["states"].double()
    o = torch.zeros(s["rows"], H, KEY, dtype=F64, device="cuda")
    q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "g", "beta"))
    head = torch.arange(H, device="cuda") // (H // HK)
    row = 0
    before = states.clone()
    for i, n in enumerate(windows(case)):
        S = before[int(s["slot_in"][i])].clone()                      # [H, key, value]
        for _ in range(n):
            kk = k[row, head] / (k[row, head].square().sum(-1, keepdim=True) + 1e-6).sqrt()
            qq = q[row, head] / (q[row, head].square().sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(KEY)
            S = S * torch.exp(g[row])[:, None, None]
            held = torch.einsum("hi,hij->hj", kk, S)
            S = S + torch.einsum("hi,hj->hij", kk, beta[row][:, None] * (v[row] - held))
            o[row] = torch.einsum("hi,hij->hj", qq, S)
            row += 1
        states[int(s["slot_out"][i])] = S
    return {"o": o, "states": states}


def exact_conv(s, case):
    H, kd, vd = case["H"], case["HK"] * KEY, case["H"] * KEY
    ch = 2 * kd + vd
    x, w = s["x"].double(), s["w"].double()
    y = torch.zeros(s["rows"], ch, dtype=F64, device="cuda")
    tails = s["tails"].double()
    before = tails.clone()
    row = 0
    for i, n in enumerate(windows(case)):
        line = torch.cat([before[int(s["slot_in"][i])], x[row:row + n, :ch]])
        y[row:row + n] = torch.einsum("tcj,cj->tc", line.unfold(0, 4, 1), w)
        tails[int(s["slot_out"][i])] = line[-3:]
        row += n
    y = y * torch.sigmoid(y)
    b, a = x[:, ch + vd:ch + vd + H], x[:, ch + vd + H:] + s["dt"].double()
    return {"q": y[:, :kd], "k": y[:, kd:2 * kd], "v": y[:, 2 * kd:], "beta": torch.sigmoid(b),
            "g": -s["a_log"].double().exp() * torch.logaddexp(a, torch.zeros_like(a)), "tails": tails}


def exact_prep(s, case):
    rows, Hq, Hk, Dh, half, page = (case[n] for n in ("rows", "Hq", "Hk", "Dh", "half", "page"))
    x = s["x"].double()
    pos = s["pos"].tolist()
    spin = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()]      # [rows, half]

    def turned(y, w):
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + w.double())
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * spin[:, None]
        return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)

    heads = x[:, :2 * Hq * Dh].reshape(rows, Hq, 2 * Dh)
    keys = turned(x[:, 2 * Hq * Dh:(2 * Hq + Hk) * Dh].reshape(rows, Hk, Dh), s["kw"])
    values = x[:, (2 * Hq + Hk) * Dh:].reshape(rows, Hk, Dh)
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    table = s["table"].tolist()
    for r, i in enumerate(s["seq"].tolist()):
        k_pages[table[i][pos[r] // page], pos[r] % page] = keys[r]
        v_pages[table[i][pos[r] // page], pos[r] % page] = values[r]
    return {"q": turned(heads[..., :Dh], s["qw"]), "gate": heads[..., Dh:], "k_pages": k_pages, "v_pages": v_pages}


def exact_attention(s, case):
    Hq, Hk, Dh, page = case["Hq"], case["Hk"], case["Dh"], case["page"]
    out = torch.zeros(case["rows"], Hq, Dh, dtype=F64, device="cuda")
    for r, (i, n) in enumerate(zip(s["seq"].tolist(), s["len"].tolist())):
        ids = s["table"][i, :-(-n // page)].long()
        k = s["k_pages"][ids].reshape(-1, Hk, Dh)[:n].double()
        v = s["v_pages"][ids].reshape(-1, Hk, Dh)[:n].double()
        p = torch.softmax(torch.einsum("hgd,thd->hgt", s["q"][r].double().view(Hk, -1, Dh), k) / math.sqrt(Dh), -1)
        out[r] = torch.einsum("hgt,thd->hgd", p, v).reshape(Hq, Dh)
    return out * torch.sigmoid(s["gate"].double()) if case["gated"] else out


def exact_pages(s, case):
    pool = s["pool"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        pool[:, b] = s["pool"][:, a]
    return pool.double()
