"""Performance cases of the paged key-value cache's operators: what writes it, reads it and thins it.

Three kinds, each with its own ranges in draw():

  append   the rows of a step into the cache: every head's norm of queries and keys and their rotation in one pass
           (one token a sequence, or the rows of prompts)
  attn     the attention of a step's rows over the pages: single tokens, the few rows of a verify pass, whole prompts,
           with or without a sliding window and first tokens that stay visible; "weights" adds up what every slot got
  evict    sequences thinned to a budget of slots by what their slots got

Sequences of a batch differ in length by a fixed rule of the case (_lens), in an order that the seed sets, so that the
work of a case does not depend on the seed.  Head shapes are the benchmark's models' (packs.cfg_c0, _c2, _c3, _c4) and a
generic one of 32 heads on 8.
"""
import math

import torch

own = False

SHAPES = {"c0": (8, 2, 128), "c2": (24, 4, 256), "c3": (16, 2, 256), "c4": (16, 4, 256), "g8": (32, 8, 128)}   # heads, kv heads, head dimension
ROPE, BASE, EPS = 64, 1.0e7, 1.0e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a chat's next token on the small model: latency and one launch only
        dict(name="append-token", kind="append", shape="c0", el="bf16", el_in="f32", page=16, seqs=1, rows=1, far=900),
        # one token of each of many users, far into long contexts, a batch of no round size
        dict(name="append-batch", kind="append", shape="c2", el="f16", el_in="f32", page=64, seqs=37, rows=1, far=200000),
        # prompts of three users together, rows as a 16-bit projection leaves them
        dict(name="append-prompts", kind="append", shape="c2", el="bf16", el_in="bf16", page=64, seqs=3, rows=4001, far=4100),
        # the same chat's attention: one token, a short context
        dict(name="token", kind="attn", shape="c0", el="bf16", page=16, seqs=1, rows=1, len=701, window=0, sinks=0, weights=False),
        # a serving batch, contexts of all lengths
        dict(name="batch", kind="attn", shape="c4", el="bf16", page=64, seqs=32, rows=1, len=8192, window=0, sinks=0, weights=False),
        # two very long documents
        dict(name="long", kind="attn", shape="c2", el="f16", page=128, seqs=2, rows=1, len=131071, window=0, sinks=0, weights=False),
        # many users whose caches are thinned by weight: what every slot got is added up
        dict(name="batch-weights", kind="attn", shape="g8", el="bf16", page=32, seqs=48, rows=1, len=6000, window=0, sinks=0, weights=True),
        # a verify pass of k = 3 with a sliding window
        dict(name="verify-window", kind="attn", shape="c3", el="f16", page=16, seqs=16, rows=4, len=12000, window=2048, sinks=4, weights=False),
        # the headline's prompt
        dict(name="prompt", kind="attn", shape="c2", el="bf16", page=64, seqs=1, rows=3011, len=3011, window=0, sinks=0, weights=False),
        # pieces of several prompts behind earlier ones, window and first tokens
        dict(name="prompt-window", kind="attn", shape="g8", el="f16", page=32, seqs=4, rows=2000, len=9000, window=1024, sinks=16, weights=False),
        # one user's cache thinned
        dict(name="evict-one", kind="evict", shape="c0", el="bf16", page=16, seqs=1, len=1500, budget=512, sinks=4, recent=64),
        # a batch's, long ones
        dict(name="evict-batch", kind="evict", shape="c4", el="bf16", page=64, seqs=16, len=20000, budget=4096, sinks=4, recent=256),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    shape, el, page = rng.choice(sorted(SHAPES)), rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    kind = rng.choice(["append", "attn", "attn", "attn", "evict"])
    if kind == "append":
        rows = rng.choice([1, 1, _log(rng, 2, 3000)])
        return dict(kind=kind, shape=shape, el=el, el_in=rng.choice(["f32", el]), page=page, seqs=_log(rng, 1, 64) if rows == 1 else rng.randint(1, 3), rows=rows, far=_log(rng, rows, 250000))
    if kind == "evict":
        length = _log(rng, 600, 20000)
        budget = max(64, int(length * rng.uniform(0.1, 0.7)))
        return dict(kind=kind, shape=shape, el=el, page=page, seqs=_log(rng, 1, 12), len=length, budget=budget, sinks=rng.choice([0, 4, 17]), recent=rng.choice([0, 32, budget // 4]))
    form = rng.choice(["token", "token", "few", "prompt"])
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 100, 4000), rng.choice([0, 4, 33]))])
    if form == "prompt":
        rows = _log(rng, 65, 2500)
        return dict(kind=kind, shape=shape, el=el, page=page, seqs=rng.randint(1, 3), rows=rows, len=rows + rng.choice([0, _log(rng, 1, 5000)]), window=window, sinks=sinks, weights=False)
    seqs, rows = _log(rng, 1, 32), 1 if form == "token" else rng.randint(2, 5)
    return dict(kind=kind, shape=shape, el=el, page=page, seqs=seqs, rows=rows, len=_log(rng, 30, 200000 // seqs), window=window, sinks=sinks,
                weights=rng.random() < 0.35)


# ---- a case's sequences ----------------------------------------------------------------------------
def _lens(case):
    """(rows, length) of every sequence: the first is the longest, the others spread over the range below it."""
    out = []
    for b in range(case["seqs"]):
        part = 1.0 - 0.9 * ((b * 0.6180339887) % 1.0)
        n = case.get("rows", 1)
        n = n if n <= 8 else max(1, int(n * part))
        out.append((n, max(n, int(case.get("len", n) * part))))
    return out


def _visible(e, window, sinks):
    """How many slots a row at slot e sees."""
    if not window or e < window:
        return e + 1
    return window + min(sinks, e + 1 - window)


def _pool(case, seqs, slots, kv, hd, gen, fill=True):
    """A pool of pages, a third more than the sequences hold, and their pages in no order; entries of no page are -1."""
    page, dev, dt = case["page"], "cuda", TYPES[case["el"]]
    need = [-(-n // page) for n in slots]
    total = sum(need)
    pages = total + total // 3 + 1
    order = torch.randperm(pages - 1, device=dev, generator=gen)[:total].to(torch.int32)   # (the last page is nobody's)
    table = torch.full((seqs, max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (pages, kv, page, hd)
    if fill:
        return [torch.randn(shape, device=dev, generator=gen, dtype=dt) for _ in range(2)] + [table]
    return [torch.zeros(shape, device=dev, dtype=dt) for _ in range(2)] + [table]


def prepare(case, seed):
    H, KV, hd = SHAPES[case["shape"]]
    dev, dt, B = "cuda", TYPES[case["el"]], case["seqs"]
    gen = torch.Generator(device=dev).manual_seed(seed)
    seqs = _lens(case)
    turn = seed % B
    seqs = seqs[turn:] + seqs[:turn]
    n, lens = [s[0] for s in seqs], [s[1] for s in seqs]
    start = [0]
    for i in n:
        start.append(start[-1] + i)
    R = start[-1]

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=dev)

    s = dict(case=case, H=H, KV=KV, hd=hd, R=R, max_rows=max(n), max_len=max(lens), lens=ints(lens), row_start=ints(start),
             row_seq=ints([b for b, i in enumerate(n) for _ in range(i)], torch.int64), row_in=ints([i for m in n for i in range(m)], torch.int64))
    if case["kind"] == "append":
        s["k"], s["v"], s["table"] = _pool(case, B, lens, KV, hd, gen, fill=False)
        ti = TYPES[case["el_in"]]
        # rows of one projection: queries, keys and values of a row side by side
        s["x"] = torch.randn(R, (H + 2 * KV) * hd, device=dev, generator=gen, dtype=ti) * 1.7
        s["qn"], s["kn"] = (1.0 + 0.2 * torch.randn(hd, device=dev, generator=gen) for _ in range(2))
        s["invfreq"] = BASE ** (-2.0 * torch.arange(ROPE // 2, dtype=torch.float64, device=dev) / ROPE)
        far = case["far"]
        s["pos"] = ints([max(0, far - m - int(far * 0.37 * b / B)) for b, m in enumerate(n)])
        s["q_out"] = torch.zeros(R, H, hd, device=dev, dtype=dt)
    elif case["kind"] == "attn":
        s["k"], s["v"], s["table"] = _pool(case, B, lens, KV, hd, gen)
        s["q"] = torch.randn(R, H, hd, device=dev, generator=gen, dtype=dt) * 1.5
        s["out"] = torch.zeros(R, H, hd, device=dev, dtype=dt)
        if case["weights"]:
            s["w_in"] = torch.rand(B, KV, max(lens), device=dev, generator=gen) * 0.01
            s["w_out"] = torch.zeros(B, KV, max(lens), device=dev)
    else:
        s["k"], s["v"], s["table"] = _pool(case, B, lens, KV, hd, gen)
        kept = [min(i, case["budget"]) for i in lens]
        s["k2"], s["v2"], s["table2"] = _pool(case, B, kept, KV, hd, gen, fill=False)
        s["lens2"] = torch.zeros(B, dtype=torch.int32, device=dev)
        # sums of softmax weights: over many orders of magnitude, a good part of them exactly zero
        w = torch.exp(3.0 * torch.randn(B, KV, max(lens), device=dev, generator=gen) - 6.0)
        s["w"] = torch.where(torch.rand(w.shape, device=dev, generator=gen) < 0.3, torch.zeros_like(w), w)
        s["w2"] = torch.zeros(B, KV, case["budget"], device=dev)
        s["kept"] = torch.full((B, KV, case["budget"]), -1, dtype=torch.int32, device=dev)
    return s


# ---- the operators' plain forms --------------------------------------------------------------------
def _rotated(x, w, pos, invfreq):
    """x [R][heads][hd] normed, weighted and rotated by the position, as f32."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    th = pos.to(torch.float64)[:, None] * invfreq
    c, sn = th.cos().float()[:, None], th.sin().float()[:, None]
    h = invfreq.numel()
    a, b = y[..., :h], y[..., h:2 * h]
    return torch.cat([a * c - b * sn, a * sn + b * c, y[..., 2 * h:]], -1)


def _plain_append(s):
    H, KV, hd, page = s["H"], s["KV"], s["hd"], s["case"]["page"]
    x = s["x"].float().view(s["R"], H + 2 * KV, hd)
    b, i = s["row_seq"], s["row_in"]
    rows = (s["row_start"][1:] - s["row_start"][:-1])[b]
    slot = (s["lens"][b] - rows + i).long()
    pos = s["pos"][b] + i
    at = s["table"][b, slot // page].long()
    s["q_out"].copy_(_rotated(x[:, :H], s["qn"], pos, s["invfreq"]))
    s["k"][at, :, slot % page] = _rotated(x[:, H:H + KV], s["kn"], pos, s["invfreq"]).to(s["k"].dtype)
    s["v"][at, :, slot % page] = x[:, H + KV:].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _slots(pool, table, count):
    """The slots of every sequence side by side: [seqs][kv heads][count][hd]."""
    x = pool[table.clamp(min=0).long()]
    x = x.permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :count]


def _plain_attn(s):
    c, H, KV, hd, n, L = s["case"], s["H"], s["KV"], s["hd"], s["max_rows"], s["max_len"]
    dev, B, G = s["q"].device, c["seqs"], H // KV
    K, V = _slots(s["k"], s["table"], L).float(), _slots(s["v"], s["table"], L).float()
    start, rows = s["row_start"][:-1].long(), (s["row_start"][1:] - s["row_start"][:-1]).long()
    i = torch.arange(n, device=dev)
    r = (start[:, None] + i).clamp(max=s["R"] - 1)
    q = s["q"].float()[r].view(B, n, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, n * G, hd)
    e = (s["lens"].long() - rows)[:, None] + i                                     # the slot of every row
    j = torch.arange(L, device=dev)
    see = (j <= e[..., None]) & (i < rows[:, None])[..., None]
    if c["window"]:
        see = see & ((j > e[..., None] - c["window"]) | (j < c["sinks"]))
    see = see[:, None, :, None].expand(B, 1, n, G, L).reshape(B, 1, n * G, L)
    S = ((q @ K.transpose(-1, -2)) * (1.0 / math.sqrt(hd))).masked_fill(~see, -math.inf)
    m = S.amax(-1, keepdim=True)
    P = torch.exp(S - torch.where(m == -math.inf, torch.zeros_like(m), m))
    P = P / P.sum(-1, keepdim=True).clamp(min=1e-37)
    O = (P @ V).view(B, KV, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B, n, H, hd)
    s["out"].copy_(O[s["row_seq"], s["row_in"]])
    if not c["weights"]:
        return {"out": s["out"]}
    held = (j < s["lens"][:, None])[:, None]
    s["w_out"].copy_(torch.where(held, s["w_in"] + P.sum(2), s["w_out"]))
    return {"out": s["out"], "weights": s["w_out"]}


def _plain_evict(s):
    c, page = s["case"], s["case"]["page"]
    dev, L, B, KV, budget = s["w"].device, s["max_len"], c["seqs"], s["KV"], c["budget"]
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(L, device=dev)
    first = torch.where(((j < c["sinks"]) | (j >= lens - c["recent"])), math.inf, s["w"])
    first = torch.where(j < lens, first, -math.inf)
    kept = torch.sort(first, dim=-1, descending=True, stable=True)[1][..., :budget]
    kept = torch.sort(kept, dim=-1)[0]                                            # (a short sequence's slots come before those behind its end)
    if kept.shape[-1] < budget:
        kept = torch.cat([kept, kept.new_zeros(B, KV, budget - kept.shape[-1])], -1)
    new = lens.clamp(max=budget)
    i = torch.arange(budget, device=dev)
    on = i < new
    s["lens2"].copy_(new[:, 0, 0])
    s["kept"].copy_(torch.where(on, kept, -1))
    s["w2"].copy_(torch.where(on, torch.gather(s["w"], 2, kept), 0.0))
    for a, z in (("k", "k2"), ("v", "v2")):
        rows = torch.gather(_slots(s[a], s["table"], L), 2, kept[..., None].expand(B, KV, budget, s["hd"]))
        P = s["table2"].shape[1]
        rows = torch.nn.functional.pad(torch.where(on[..., None], rows, 0.0), (0, 0, 0, max(0, P * page - budget)))[:, :, :P * page]
        rows = rows.view(B, KV, P, page, s["hd"]).permute(0, 2, 1, 3, 4)
        # entries of no page go to the pool's last page, which is nobody's, as zeros
        s[z][torch.where(s["table2"] < 0, s["spare"], s["table2"]).long()] = rows
    return {"k": s["k2"], "v": s["v2"], "weights": s["w2"], "kept": s["kept"], "lens": s["lens2"]}


# ---- the framework's calls --------------------------------------------------------------------------
def _framework():
    import importlib
    llb = importlib.import_module("eureka-engine_b200").llb
    llb.init(torch.cuda.current_device())
    return llb


def _cache(llb, s, k, v, table, lens):
    pool = s[k]
    return llb.Kv(el=llb.EL[s["case"]["el"]], kv_heads=s["KV"], head_dim=s["hd"], page=s["case"]["page"], n_pages=pool.shape[0], seqs=s["case"]["seqs"],
                  table_stride=s[table].shape[1], k=pool.data_ptr(), v=s[v].data_ptr(), table=s[table].data_ptr(), lens=s[lens].data_ptr())


def _describe(s):
    """The descriptions of cache and call that a program fills in once and keeps, and the call's workspace."""
    llb, c, hd = _framework(), s["case"], s["hd"]
    s["llb"], s["kv"] = llb, _cache(llb, s, "k", "v", "table", "lens")
    if c["kind"] == "append":
        x, H, KV, w = s["x"], s["H"], s["KV"], s["x"].element_size()
        s["call"] = llb.KvAppend(rows=s["R"], heads=H, el_in=llb.EL[c["el_in"]], rope_dim=ROPE, eps=EPS, q=x.data_ptr(), k=x.data_ptr() + H * hd * w,
                                 v=x.data_ptr() + (H + KV) * hd * w, q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0), q_head_stride=hd,
                                 q_norm=s["qn"].data_ptr(), k_norm=s["kn"].data_ptr(), invfreq=s["invfreq"].data_ptr(), row_start=s["row_start"].data_ptr(),
                                 pos=s["pos"].data_ptr(), q_out=s["q_out"].data_ptr(), q_out_stride=s["H"] * hd)
    elif c["kind"] == "attn":
        s["call"] = llb.KvAttn(rows=s["R"], max_rows=s["max_rows"], max_len=s["max_len"], heads=s["H"], window=c["window"], sinks=c["sinks"], scale=0.0,
                               el_out=llb.EL[c["el"]], q=s["q"].data_ptr(), q_stride=s["H"] * hd, out=s["out"].data_ptr(), out_stride=s["H"] * hd,
                               row_start=s["row_start"].data_ptr())
        if c["weights"]:
            s["call"].w_in, s["call"].w_out, s["call"].w_stride = s["w_in"].data_ptr(), s["w_out"].data_ptr(), s["max_len"]
        s["ws"] = torch.empty(max(16, llb.kv_attn_ws(s["kv"], s["call"])), dtype=torch.uint8, device=s["q"].device)
        s["call"].ws, s["call"].ws_bytes = s["ws"].data_ptr(), s["ws"].numel()
    else:
        s["kv2"] = _cache(llb, s, "k2", "v2", "table2", "lens2")
        s["call"] = llb.KvEvict(budget=c["budget"], sinks=c["sinks"], recent=c["recent"], max_len=s["max_len"], w=s["w"].data_ptr(), w_stride=s["max_len"],
                                w_out=s["w2"].data_ptr(), w_out_stride=c["budget"], kept=s["kept"].data_ptr(), kept_stride=c["budget"])
        s["ws"] = torch.empty(max(16, llb.kv_evict_ws(s["kv"], s["call"])), dtype=torch.uint8, device=s["w"].device)
        s["call"].ws, s["call"].ws_bytes = s["ws"].data_ptr(), s["ws"].numel()


def _own(s):
    if "call" not in s:
        _describe(s)
    llb, kind = s["llb"], s["case"]["kind"]
    if kind == "append":
        llb.kv_append(s["kv"], s["call"])
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if kind == "attn":
        llb.kv_attn(s["kv"], s["call"])
        return {"out": s["out"], "weights": s["w_out"]} if s["case"]["weights"] else {"out": s["out"]}
    llb.kv_evict(s["kv"], s["kv2"], s["call"])
    return {"k": s["k2"], "v": s["v2"], "weights": s["w2"], "kept": s["kept"], "lens": s["lens2"]}


def run(state):
    if own:
        return _own(state)
    if state["case"]["kind"] == "evict" and "spare" not in state:
        state["spare"] = torch.tensor(state["k2"].shape[0] - 1, dtype=torch.int32, device="cuda")
    return {"append": _plain_append, "attn": _plain_attn, "evict": _plain_evict}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------
def work(case):
    H, KV, hd = SHAPES[case["shape"]]
    seqs = _lens(case)
    R = sum(n for n, _ in seqs)
    if case["kind"] == "append":
        return {"bytes": R * (H + 2 * KV) * hd * (TYPES[case["el_in"]].itemsize + 2), "flops": R * (H + KV) * (4 * hd + 3 * ROPE)}
    if case["kind"] == "evict":
        kept = sum(min(m, case["budget"]) for _, m in seqs)
        return {"bytes": 4 * KV * sum(m for _, m in seqs) + kept * KV * (2 * 2 * hd * 2 + 4 + 4), "flops": KV * sum(m for _, m in seqs)}
    W, S = case["window"], case["sinks"]
    by = 2 * R * H * hd * 2
    pairs = 0
    for n, m in seqs:
        pairs += sum(_visible(e, W, S) for e in range(m - n, m))
        # the slots that some row sees: those of the first row and the rows behind it, and the first tokens
        lo = max(0, m - n - W + 1) if W else 0
        by += (m - lo + min(S, lo)) * KV * hd * 2 * 2
        if case["weights"]:
            by += 8 * KV * m
    return {"bytes": by, "flops": 4 * hd * H * pairs}


# ---- the definition in 64 bits ----------------------------------------------------------------------
def _exact_rows(s, b):
    """First row, rows, length and the places (page, slot in it) of sequence b's slots."""
    a, z, m = int(s["row_start"][b]), int(s["row_start"][b + 1]), int(s["lens"][b])
    j = torch.arange(m, device="cuda")
    return a, z - a, m, s["table"][b].long()[j // s["case"]["page"]], j % s["case"]["page"]


def exact(case, seed):
    s = prepare(case, seed)
    B, H, KV, hd = case["seqs"], s["H"], s["KV"], s["hd"]
    if case["kind"] == "append":
        out, k, v = s["q_out"].double(), s["k"].double(), s["v"].double()
        h = ROPE // 2
        for b in range(B):
            a, n, m, page, at = _exact_rows(s, b)
            x = s["x"][a:a + n].double().view(n, H + 2 * KV, hd)
            turn = (float(s["pos"][b]) + torch.arange(n, device="cuda").double())[:, None] * s["invfreq"]
            z = torch.exp(1j * turn)[:, None]
            done = []
            for w, y in ((s["qn"], x[:, :H]), (s["kn"], x[:, H:H + KV])):
                y = y * w.double() / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
                t = torch.complex(y[..., :h].contiguous(), y[..., h:2 * h].contiguous()) * z
                done.append(torch.cat([t.real, t.imag, y[..., 2 * h:]], -1))
            out[a:a + n] = done[0]
            k[page[m - n:], :, at[m - n:]] = done[1]
            v[page[m - n:], :, at[m - n:]] = x[:, H + KV:]
        return {"q": out, "k": k, "v": v}
    if case["kind"] == "attn":
        out = torch.zeros(s["R"], H, hd, dtype=torch.float64, device="cuda")
        wt = s["w_out"].double() if case["weights"] else None
        G = H // KV
        for b in range(B):
            a, n, m, page, at = _exact_rows(s, b)
            slot = torch.arange(m, device="cuda")
            for g in range(KV):
                k, v = s["k"][page, g, at].double(), s["v"][page, g, at].double()
                total = torch.zeros(m, dtype=torch.float64, device="cuda")
                for i in range(0, n, 256):
                    e = torch.arange(m - n + i, m - n + min(n, i + 256), device="cuda")
                    hide = slot[None] > e[:, None]
                    if case["window"]:
                        hide |= (slot[None] <= e[:, None] - case["window"]) & (slot[None] >= case["sinks"])
                    q = s["q"][a + i:a + i + len(e), g * G:(g + 1) * G].double()
                    sc = torch.einsum("rgd,jd->rgj", q, k) / hd ** 0.5
                    sc[hide[:, None].expand_as(sc)] = -math.inf
                    p = torch.softmax(sc, -1)
                    out[a + i:a + i + len(e), g * G:(g + 1) * G] = torch.einsum("rgj,jd->rgd", p, v)
                    total += p.sum((0, 1))
                if wt is not None:
                    wt[b, g, :m] = s["w_in"][b, g, :m].double() + total
        return {"out": out} if wt is None else {"out": out, "weights": wt}
    # evict moves values: what comes out are the inputs' own
    page = case["page"]
    k, v, w2, kept, lens = s["k2"].double(), s["v2"].double(), s["w2"].double(), s["kept"], s["lens2"]
    for b in range(B):
        _, _, m, pg, at = _exact_rows(s, b)
        new = min(m, case["budget"])
        i = torch.arange(new, device="cuda")
        lens[b] = new
        for g in range(KV):
            lo, hi = (case["sinks"], m - case["recent"]) if m > new else (m, m)
            mid = s["w"][b, g, lo:hi].cpu().numpy()
            few = (-mid).argsort(kind="stable")[:new - lo - (m - hi)]
            ids = sorted(list(range(lo)) + [lo + int(t) for t in few] + list(range(hi, m)))
            ids = torch.tensor(ids, device="cuda")
            kept[b, g, :new] = ids.int()
            w2[b, g, :new] = s["w"][b, g][ids].double()
            to = s["table2"][b].long()[i // page]
            k[to, g, i % page] = s["k"][pg[ids], g, at[ids]].double()
            v[to, g, i % page] = s["v"][pg[ids], g, at[ids]].double()
    return {"k": k, "v": v, "weights": w2, "kept": kept, "lens": lens}
