"""The paged key-value cache's operators against their definitions in 64 bits.

Every pool starts as NaN: only slots that a row of the call may look at hold numbers, and table entries of other slots
are no page at all.  Bounds on the errors follow from the formats: a rounding to type t is off by at most
finfo(t).eps / 2 of the value, f32 sums of n terms by n 2^-23 of the terms' magnitudes (tensor cores truncate)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}     # half a step of the smallest numbers (f16: below 2^-14)
GARBAGE = (-1, 2 ** 31 - 1, -2 ** 31, 1 << 20)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


class Cache:
    """Sequences of the given lengths on a pool of NaN; `live(b, j)` says which slots hold numbers."""

    def __init__(self, llb, el, KV, hd, page, lens, seed, live=None, spare=3, seqs_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.llb, self.el, self.KV, self.hd, self.page, self.lens_list = llb, el, KV, hd, page, list(lens)
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g).tolist()
        stride = max(need + [1]) + 2
        live = live or (lambda b, j: True)
        self.k = torch.full((self.n_pages, KV, page, hd), math.nan, dtype=DT[el], device="cuda")
        self.v = self.k.clone()
        self.K, self.V, rows, at = [], [], [], 0
        for b, n in enumerate(lens):
            pages = order[at:at + need[b]]
            at += need[b]
            on = torch.tensor([bool(live(b, j)) for j in range(n)], dtype=torch.bool)
            k, v = (torch.randn(n, KV, hd, generator=g).to(DT[el]) for _ in range(2))
            entry = []
            for i, p in enumerate(pages):
                m = slice(i * page, min(n, (i + 1) * page))
                if not bool(on[m].any()):
                    entry.append(GARBAGE[(b + i) % len(GARBAGE)])
                    continue
                entry.append(p)
                w = on[m].cuda()
                idx = w.nonzero()[:, 0]
                self.k[p][:, idx] = k[m].cuda()[idx].transpose(0, 1)
                self.v[p][:, idx] = v[m].cuda()[idx].transpose(0, 1)
            rows.append(entry + [GARBAGE[(b + i) % len(GARBAGE)] for i in range(stride - len(entry))])
            self.K.append(k.double())
            self.V.append(v.double())
        self.table, self.lens = _ints(rows), _ints(self.lens_list)
        self.stride = stride

    def desc(self, **kw):
        a = dict(el=self.llb.EL[self.el], kv_heads=self.KV, head_dim=self.hd, page=self.page, n_pages=self.n_pages, seqs=len(self.lens_list), table_stride=self.stride,
                 k=self.k.data_ptr(), v=self.v.data_ptr(), table=self.table.data_ptr(), lens=self.lens.data_ptr())
        a.update(kw)
        return self.llb.Kv(**a)

    def slots(self, b, n, what="k"):
        """Slots 0 .. n - 1 of sequence b as they lie in the pool: [n][KV][hd]."""
        pool = self.k if what == "k" else self.v
        j = torch.arange(n, device="cuda")
        return pool[self.table[b][j // self.page].long(), :, j % self.page]


def _sees(j, e, window, sinks):
    return j <= e and (not window or j > e - window or j < sinks)


def _clean(llb):
    assert llb.lib().llb_b200_wait_errors() == 0
    assert llb.kv_errors() == 0


def _attn(llb, c, H, rows, window=0, sinks=0, el_out=None, scale=0.0, weights=False, seed=0, pad=0, behind=2, kvkw={}, max_rows=None, max_len=None, q=None):
    """Runs the call; returns what it wrote and what it was given."""
    g = torch.Generator().manual_seed(seed + 1)
    hd, el_out = c.hd, el_out or c.el
    start = np.concatenate([[0], np.cumsum(rows)]).tolist()
    R = start[-1] + behind
    qs, os = H * hd + 8 * pad, H * hd + 16 * pad
    qt = torch.full((R, qs), math.nan, dtype=DT[c.el], device="cuda")
    qt[:, :H * hd] = ((torch.randn(R, H * hd, generator=g) * 1.5) if q is None else q).to(DT[c.el]).cuda()
    out = torch.full((R, os), 7.0, dtype=DT[el_out], device="cuda")
    rs = _ints(start)
    L = max(c.lens_list + [0]) if max_len is None else max_len
    a = llb.KvAttn(rows=R, max_rows=max_rows or max(rows + [1]), max_len=L, heads=H, window=window, sinks=sinks, scale=scale, el_out=llb.EL[el_out],
                   q=qt.data_ptr(), out=out.data_ptr(), q_stride=qs, out_stride=os, row_start=rs.data_ptr())
    w_in = w_out = None
    if weights:
        w_in = torch.rand(len(rows), c.KV, L + 3, generator=g).cuda()
        w_out = torch.full_like(w_in, 7.0)
        a.w_in, a.w_out, a.w_stride = w_in.data_ptr(), w_out.data_ptr(), L + 3
    kv = c.desc(**kvkw)
    ws = torch.full((llb.kv_attn_ws(kv, a),), 255, dtype=torch.uint8, device="cuda")
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    llb.kv_attn(kv, a)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    return dict(q=qt, out=out, start=start, w_in=w_in, w_out=w_out, R=R, H=H, window=window, sinks=sinks, scale=scale or hd ** -0.5, el_out=el_out, rows=rows,
                keep=(rs, ws), call=(kv, a))


def _check_attn(c, r):
    H, KV, hd, W, S = r["H"], c.KV, c.hd, r["window"], r["sinks"]
    G = H // KV
    out = r["out"].double().cpu()
    worst = 0.0
    for b, n in enumerate(r["rows"]):
        m, a0 = c.lens_list[b], r["start"][b]
        total, slack = np.zeros((KV, m)), np.zeros((KV, m))
        j = torch.arange(m)
        for i in range(n):
            e = m - n + i
            see = (j <= e) & ((j > e - W) | (j < S)) if W else j <= e
            idx = see.nonzero()[:, 0]
            got = out[a0 + i, :H * hd].view(H, hd)
            if not len(idx):
                assert torch.all(got == 0), (b, i)
                continue
            q = r["q"][a0 + i, :H * hd].double().cpu().view(KV, G, hd)
            K, V = c.K[b][idx].permute(1, 0, 2), c.V[b][idx].permute(1, 0, 2)           # [KV][seen][hd]
            s = torch.einsum("ghd,gjd->ghj", q, K) * r["scale"]
            mag = torch.einsum("ghd,gjd->ghj", q.abs(), K.abs()) * r["scale"]
            ds = mag * hd * 2.0 ** -23 + s.abs() * 2.0 ** -21 + 2.0 ** -20               # a score's error, and what exp makes of it
            x = torch.exp(s - s.amax(-1, keepdim=True))
            L = x.sum(-1, keepdim=True)
            p = x / L
            want = torch.einsum("ghj,gjd->ghd", p, V).reshape(H, hd)
            # a probability: off by its score's error, rounded to the cache's type; their sum likewise; then sums of as many products
            dp = p * (2 * ds + HALF[c.el] + len(idx) * 2.0 ** -23) + TINY[c.el] / L + p * (p * 2 * ds).sum(-1, keepdim=True)
            bound = torch.einsum("ghj,gjd->ghd", dp, V.abs()).reshape(H, hd)
            bound = bound * 1.001 + (want.abs() + bound) * HALF[r["el_out"]] + TINY[r["el_out"]] + 1e-30
            d = (got - want).abs()
            assert torch.all(d <= bound), (b, i, float((d / bound).max()), float(d.max()))
            worst = max(worst, float((d / bound).max()))
            ii = idx.numpy()
            total[:, ii] += p.sum(1).numpy()
            slack[:, ii] += (p * (2 * ds + 2 * (p * ds).sum(-1, keepdim=True) + (len(idx) + 8) * 2.0 ** -23)).sum(1).numpy()
        if r["w_out"] is not None:
            w = r["w_out"][b].double().cpu().numpy()
            want = r["w_in"][b, :, :m].double().cpu().numpy() + total
            d = np.abs(w[:, :m] - want)
            assert np.all(d <= slack + (want + slack) * 2.0 ** -22 + 1e-30), (b, float((d / (slack + 1e-30)).max()))
            assert np.all(w[:, m:] == 7.0)
    assert torch.all(r["out"][r["start"][-1]:] == 7.0)              # rows behind the last sequence
    assert torch.all(r["out"][:, H * hd:] == 7.0)                   # and what lies between rows
    return worst


def _live_of(rows, lens, window, sinks):
    return lambda b, j: any(_sees(j, lens[b] - rows[b] + i, window, sinks) for i in range(rows[b]))


# ---- attention ---------------------------------------------------------------------------------------
FORMS = [(1, 1, 64), (8, 2, 128), (24, 4, 256), (16, 2, 256), (3, 3, 128), (32, 8, 128), (16, 1, 64), (64, 1, 128)]


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_tokens_of_many_lengths(llb, form, page, el):
    H, KV, hd = form
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 300, 0, 1, 513]
    c = Cache(llb, el, KV, hd, page, lens, seed=1)
    r = _attn(llb, c, H, [1] * len(lens), weights=True, pad=1)
    _check_attn(c, r)
    _clean(llb)


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("form,lens,rows", [
    ((8, 2, 128), [900, 5, 0, 77, 1300], [4, 4, 0, 2, 1]), ((24, 4, 256), [700, 33, 64], [5, 8, 3]), ((16, 2, 256), [300, 301], [8, 7]), ((16, 16, 64), [130, 999], [60, 7]),
    ((6, 1, 128), [200, 17], [10, 10]), ((64, 1, 64), [100, 500], [1, 1])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (64, 70), (7, 16)])
def test_few_rows(llb, form, lens, rows, window, sinks, el):
    """Rows of verify passes: row counts that differ, windows inside and across pages, first tokens that meet the window."""
    H, KV, hd = form
    c = Cache(llb, el, KV, hd, 16, lens, seed=2, live=_live_of(rows, lens, window, sinks))
    r = _attn(llb, c, H, rows, window=window, sinks=sinks, weights=H // KV * max(rows) <= 64, seed=3)
    _check_attn(c, r)
    _clean(llb)


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("form", [(8, 2, 128), (24, 4, 256), (3, 3, 64), (16, 2, 256), (32, 8, 128)])
@pytest.mark.parametrize("rows,lens", [([130], [130]), ([300, 1, 0, 77], [300, 1, 0, 500]), ([65, 129, 128], [1000, 129, 640]), ([257], [290])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5), (33, 0), (200, 130)])
def test_prompts(llb, form, rows, lens, window, sinks, el):
    H, KV, hd = form
    c = Cache(llb, el, KV, hd, 32, lens, seed=4, live=_live_of(rows, lens, window, sinks))
    _check_attn(c, _attn(llb, c, H, rows, window=window, sinks=sinks, seed=5, pad=2))
    _clean(llb)


@pytest.mark.parametrize("page", [16, 64, 128])
def test_prompt_pages_and_f32_out(llb, page):
    c = Cache(llb, "bf16", 2, 128, page, [333, 190], seed=6)
    _check_attn(c, _attn(llb, c, 8, [333, 100], el_out="f32", scale=0.11, seed=7))
    c = Cache(llb, "f16", 2, 256, page, [333, 190], seed=6)
    _check_attn(c, _attn(llb, c, 8, [2, 1], el_out="f32", scale=0.02, seed=7, weights=True))
    _clean(llb)


def test_rows_before_the_first_slot_see_nothing(llb):
    """Lengths smaller than the rows: the first rows are at slots below 0."""
    for rows, lens in (([4, 1], [2, 0]), ([200, 70], [3, 0])):
        c = Cache(llb, "f16", 2, 128, 16, lens, seed=8)
        _check_attn(c, _attn(llb, c, 4, rows, seed=9, max_len=64, weights=max(rows) < 8))
    _clean(llb)


@pytest.mark.parametrize("rows", [[1, 1, 1], [100, 90, 1]])
def test_no_slots_and_no_rows(llb, rows):
    c = Cache(llb, "bf16", 1, 64, 16, [0, 0, 0], seed=10)
    _check_attn(c, _attn(llb, c, 4, rows, seed=9, max_len=0))
    c = Cache(llb, "bf16", 1, 64, 16, [30, 0, 40], seed=10)
    r = _attn(llb, c, 4, [0, 0, 0], seed=9, weights=True)
    for b, m in enumerate([30, 0, 40]):
        assert torch.equal(r["w_out"][b, :, :m], r["w_in"][b, :, :m])
    _check_attn(c, r)
    r = _attn(llb, c, 4, [0, 0, 0], seed=9, behind=0)
    _clean(llb)


@pytest.mark.parametrize("what", ["inf", "nan"])
@pytest.mark.parametrize("rows,H,KV", [([4], 8, 2), ([3], 24, 4), ([150], 8, 2), ([140], 4, 4)])
def test_a_later_rows_infinities_do_not_reach_earlier_rows(llb, rows, H, KV, what):
    """The last row's own K and V are no numbers: rows before it do not see that slot and are right to the last bit of their bounds."""
    n = rows[0]
    c = Cache(llb, "bf16", KV, 128, 16, [n + 40], seed=11)
    bad = math.inf if what == "inf" else math.nan
    j = n + 39
    c.v[int(c.table[0, j // 16]), :, j % 16] = bad
    c.k[int(c.table[0, j // 16]), :, j % 16] = bad
    r = _attn(llb, c, H, rows, seed=12)
    assert not torch.isfinite(r["out"][n - 1, :H * 128].float()).any() or what == "inf"
    r["out"][n - 1] = 7.0
    r["rows"], r["start"] = [n - 1], [0, n - 1]
    c.lens_list, c.K, c.V = [n + 39], [c.K[0][:-1]], [c.V[0][:-1]]
    _check_attn(c, r)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows,window", [(1, 0), (3, 0), (150, 0), (150, 100)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_key_that_is_no_number(llb, hd, rows, window, bad):
    """One component of one key of every kv head, each at another place among eight slots: a row that sees a score of NaN or of plus infinity is
    NaN, minus infinity takes no part, and the rows that do not see the slot are right.

    Bounds: a score is off by |q| |K| hd 2^-23 / sqrt(hd) < 8e-4 at most here, a probability by four times that (its own and the sum's) and its rounding
    to bf16, 2^-8: less than 2^-7 together; then the result's own rounding."""
    n, KV, G = 190, 8, 2
    c = Cache(llb, "bf16", KV, hd, 16, [n], seed=71)
    at = [n - 75 + g for g in range(KV)] if rows > 75 else [n - 75 - g for g in range(KV)]
    for g, j in enumerate(at):
        c.k[int(c.table[0, j // 16]), g, j % 16, 5 * g] = bad
        c.K[0][j, g, 5 * g] = bad
    r = _attn(llb, c, KV * G, [rows], window=window, seed=72)
    _clean(llb)
    out = r["out"][:rows].double().cpu().view(rows, KV, G, hd)
    for i in range(rows):
        e = n - rows + i
        a0 = max(0, e - window + 1) if window else 0
        q = r["q"][i].double().cpu().view(KV, G, hd)
        x = torch.einsum("kgd,jkd->kgj", q, c.K[0][a0:e + 1]) * r["scale"]
        p = torch.softmax(x, -1)
        V = c.V[0][a0:e + 1].permute(1, 0, 2)
        want, size = torch.matmul(p, V), torch.matmul(p, V.abs())
        assert torch.equal(torch.isnan(want), torch.isnan(out[i])), i
        d = (out[i] - want).abs().nan_to_num(0.0)
        assert torch.all(d <= (size * 2.0 ** -7 + want.abs() * 2.0 ** -8).nan_to_num(0.0) * 1.01 + 1e-30), i


@pytest.mark.parametrize("H,KV", [(4, 1), (24, 4)])
def test_weights_of_a_row_that_is_no_number(llb, H, KV):
    """The last row's own key is no number: what its slots get is none either, what only the rows before it see is right, and so are other sequences."""
    c = Cache(llb, "bf16", KV, 128, 16, [60, 70], seed=65)
    c.k[int(c.table[0, 59 // 16]), 0, 59 % 16] = math.nan
    r = _attn(llb, c, H, [1, 1], seed=66, weights=True)
    w = r["w_out"]
    assert torch.isnan(w[0, 0, :60]).all()
    total = (w - r["w_in"]).double()
    assert torch.all((total[1, :, :70].sum(-1) - H // KV).abs() < 1e-4)
    if KV > 1:
        assert torch.all((total[0, 1:, :60].sum(-1) - H // KV).abs() < 1e-4)


def test_scores_of_minus_infinity_and_large_ones(llb):
    """Keys that overflow a score to minus infinity take no part; scores of thousands do not overflow."""
    c = Cache(llb, "bf16", 1, 128, 16, [200, 200], seed=13)
    q = torch.randn(2, 128, generator=torch.Generator().manual_seed(1)).abs()
    for b in range(2):
        for j in range(0, 200, 3):
            c.k[int(c.table[b, j // 16]), 0, j % 16] = -math.inf
            c.K[b][j] = -math.inf
        for j in range(1, 200, 3):
            c.k[int(c.table[b, j // 16]), 0, j % 16] *= 300.0
            c.K[b][j] *= 300.0
            c.K[b][j] = c.k[int(c.table[b, j // 16]), 0, j % 16].double().cpu()
    r = _attn(llb, c, 1, [1, 1], q=q, behind=0)
    for b in range(2):
        keep = torch.isfinite(c.K[b][:, 0]).all(-1).nonzero()[:, 0]
        p = torch.softmax((c.K[b][keep, 0] @ r["q"][b].double().cpu()) / 128 ** 0.5, 0)
        want = p @ c.V[b][keep, 0]
        assert torch.all((r["out"][b].double().cpu() - want).abs() <= 2 ** -7 * (p @ c.V[b][keep, 0].abs()) + 1e-3 * want.abs() + 1e-2 * p.max())


def test_every_score_minus_infinity(llb):
    """No visible slot has a weight then: not a number, as 0 / 0 is, or zeros; no neighbour is touched."""
    c = Cache(llb, "bf16", 1, 64, 16, [20, 20], seed=14)
    c.k[c.table[0, :2].long()] = -math.inf
    r = _attn(llb, c, 1, [1, 1], q=torch.ones(2, 64), behind=0)
    assert not r["out"][0].float().nan_to_num(0.0).any()
    c.lens_list[0], r["rows"] = 0, [0, 1]
    r["start"] = [1, 1, 2]
    c.K[0], c.V[0] = c.K[0][:0], c.V[0][:0]
    _check_attn(c, r)


@pytest.mark.parametrize("bad", [None, -1, -2, -2 ** 31])
@pytest.mark.parametrize("rows", [1, 80])
def test_bad_pages_are_not_seen(llb, rows, bad):
    """An entry of a visible slot that is no page: its slots are left out, and the error word says so."""
    c = Cache(llb, "f16", 2, 64, 16, [150], seed=15)
    c.table[0, 3] = c.n_pages if bad is None else bad
    r = _attn(llb, c, 4, [rows], seed=16, weights=rows == 1)
    assert llb.kv_errors() == 1
    llb.lib().llb_b200_kv_errors_clear()
    keep = torch.tensor([j for j in range(150) if j // 16 != 3])
    for i in range(rows):
        e = 150 - rows + i
        idx = keep[keep <= e]
        q = r["q"][i, :256].double().cpu().view(2, 2, 64)
        p = torch.softmax(torch.einsum("ghd,jgd->ghj", q, c.K[0][idx]) / 8.0, -1)
        want = torch.einsum("ghj,jgd->ghd", p, c.V[0][idx]).reshape(-1)
        mass = torch.einsum("ghj,jgd->ghd", p, c.V[0][idx].abs()).reshape(-1)
        assert torch.all((r["out"][i, :256].double().cpu() - want).abs() <= 2 ** -9 * mass)
    _clean(llb)


def test_lengths_and_rows_that_do_not_fit_are_reported(llb):
    c = Cache(llb, "f16", 1, 64, 16, [40, 40], seed=17)
    c.lens[0] = -5
    c.lens[1] = 1 << 30
    _attn(llb, c, 1, [1, 1], seed=18, max_len=40)
    assert llb.kv_errors() == 2
    llb.lib().llb_b200_kv_errors_clear()
    c.lens.copy_(_ints([40, 40]))
    r = _attn(llb, c, 1, [3, 1], seed=18, max_rows=2)                # one row more than the call was told of
    assert llb.kv_errors() == 4
    assert torch.all(r["out"][2] == 7.0) and torch.all(r["out"][3].float().abs() < 7.0)
    llb.lib().llb_b200_kv_errors_clear()
    for start in ([0, 2, 1], [-1, 1, 2], [0, 1, 1 << 20]):
        r["keep"][0].copy_(_ints(start))
        llb.kv_attn(*r["call"])
        assert llb.kv_errors() == 4, start
        llb.lib().llb_b200_kv_errors_clear()
    _clean(llb)


def test_a_pool_beyond_32_bits_of_bytes(llb):
    """Pages at the end of a pool of six GB, one long sequence."""
    KV, hd, page = 4, 256, 64
    per = KV * page * hd
    n_pages = 6 * (1 << 30) // (per * 2)
    k, v = (torch.empty(n_pages, KV, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = Cache(llb, "bf16", KV, hd, page, [1000], seed=19, spare=0)
    top = _ints(list(range(n_pages - c.n_pages, n_pages)))
    k[top.long()], v[top.long()] = c.k, c.v
    c.k, c.v, c.table, c.n_pages = k, v, torch.where(c.table < c.n_pages, c.table + (n_pages - c.n_pages), c.table), n_pages
    c.table[0, 16:] = -1
    _check_attn(c, _attn(llb, c, 24, [1], seed=20))
    _check_attn(c, _attn(llb, c, 24, [100], seed=20))
    _clean(llb)


@pytest.mark.parametrize("window,sinks", [(0, 0), (3000, 9)])
def test_a_long_sequence_beside_short_ones(llb, window, sinks):
    lens = [40000, 3, 1, 700]
    c = Cache(llb, "bf16", 2, 128, 128, lens, seed=21)
    _check_attn(c, _attn(llb, c, 16, [1, 1, 1, 1], window=window, sinks=sinks, weights=True, seed=22))
    lens = [20000, 90]
    c = Cache(llb, "f16", 2, 128, 64, lens, seed=23)
    _check_attn(c, _attn(llb, c, 2, [70, 80], window=window, sinks=sinks, seed=24))
    _clean(llb)


@pytest.mark.parametrize("form", [(16, 4, 256), (8, 2, 128), (4, 2, 64)])
def test_stretches_that_go_round_the_ring_many_times(llb, form):
    """Sequences enough for blocks that bring a few hundred chunks through their rings, over the ends of units, twice with the same bits."""
    H, KV, hd = form
    lens = [16000, 900, 12345, 16, 9000, 15999, 1, 7000, 11111, 14000]
    c = Cache(llb, "bf16", KV, hd, 64, lens, seed=63)
    one = _attn(llb, c, H, [1] * len(lens), seed=64)
    _check_attn(c, one)
    for _ in range(5):
        assert torch.equal(one["out"], _attn(llb, c, H, [1] * len(lens), seed=64)["out"])
    _clean(llb)


def test_weights_in_place_and_from_nothing(llb):
    c = Cache(llb, "bf16", 2, 128, 16, [400, 90], seed=25)
    r = _attn(llb, c, 8, [2, 1], weights=True, seed=26)
    want = r["w_out"][:, :, :400].clone()
    kv, a = r["call"]
    a.w_in = 0
    llb.kv_attn(kv, a)
    got = r["w_out"][:, :, :400]
    for b, m in enumerate((400, 90)):
        assert torch.all((got[b, :, :m] + r["w_in"][b, :, :m] - want[b, :, :m]).abs() <= 1e-6)
    r["w_out"].copy_(r["w_in"])
    a.w_in = a.w_out
    llb.kv_attn(kv, a)
    for b, m in enumerate((400, 90)):
        assert torch.equal(r["w_out"][b, :, :m], want[b, :, :m])
    _clean(llb)


@pytest.mark.parametrize("rows", [[1, 1], [3, 2], [200, 90]])
def test_the_same_call_gives_the_same_bits(llb, rows):
    c = Cache(llb, "bf16", 4, 128, 32, [3000, 800], seed=27)
    one = _attn(llb, c, 16, rows, seed=28, weights=max(rows) < 8)
    for _ in range(3):
        two = _attn(llb, c, 16, rows, seed=28, weights=max(rows) < 8)
        assert torch.equal(one["out"], two["out"])
        assert one["w_out"] is None or torch.equal(one["w_out"], two["w_out"])


def test_sequences_may_share_pages(llb):
    c = Cache(llb, "bf16", 2, 64, 16, [100, 90], seed=29)
    c.table[1] = c.table[0]
    c.K[1], c.V[1] = c.K[0][:90], c.V[0][:90]
    _check_attn(c, _attn(llb, c, 4, [1, 1], seed=30, weights=True))
    _check_attn(c, _attn(llb, c, 4, [100, 90], seed=30))
    _clean(llb)


# ---- rows in ------------------------------------------------------------------------------------------
def _append(llb, c, H, rows, el_in, rope=64, norm=True, pos=None, gate=False, pad=0, seed=0, q=True, eps=1e-6, behind=2, shift=0):
    g = torch.Generator().manual_seed(seed)
    hd, KV = c.hd, c.KV
    start = np.concatenate([[0], np.cumsum(rows)]).tolist()
    R = start[-1] + behind
    qh = 2 * hd if gate else hd
    qs, ks = H * qh + pad, KV * hd + 3 * pad
    es = torch.finfo(DT[el_in]).bits // 8
    buf = [torch.full((R * s + shift,), math.nan, dtype=DT[el_in], device="cuda") for s in (qs, ks, ks)]
    x = [b[shift:].view(R, -1) for b in buf]
    x[0][:, :H * qh] = (torch.randn(R, H * qh, generator=g) * 1.7).to(DT[el_in]).cuda()
    for t in x[1:]:
        t[:, :KV * hd] = (torch.randn(R, KV * hd, generator=g) * 1.7).to(DT[el_in]).cuda()
    qn, kn = ((1 + 0.2 * torch.randn(hd, generator=g)).cuda() for _ in range(2))
    inv = 1.0e7 ** (-2.0 * torch.arange(max(1, rope // 2), dtype=torch.float64) / max(1, rope))
    invd, rs = inv.cuda(), _ints(start)
    out = torch.full((R, H * hd + pad), 7.0, dtype=DT[c.el], device="cuda")
    ps = None if pos is None else _ints(pos)
    a = llb.KvAppend(rows=R, heads=H, el_in=llb.EL[el_in], rope_dim=rope, eps=eps, q=x[0].data_ptr() if q else 0, k=x[1].data_ptr(), v=x[2].data_ptr(), q_stride=qs,
                     k_stride=ks, v_stride=ks, q_head_stride=qh, q_norm=qn.data_ptr() if norm else 0, k_norm=kn.data_ptr() if norm else 0, invfreq=invd.data_ptr() if rope else 0,
                     row_start=rs.data_ptr(), pos=ps.data_ptr() if ps is not None else 0, q_out=out.data_ptr() if q else 0, q_out_stride=H * hd + pad)
    llb.kv_append(c.desc(), a)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    h = rope // 2
    for b, n in enumerate(rows):
        m = c.lens_list[b]
        for i in range(n):
            r, slot = start[b] + i, m - n + i
            p = slot if pos is None else pos[b] + i
            th = p * inv[:h]
            co, si = th.cos(), th.sin()

            def turned(y, w):
                y = y.double().cpu()
                if norm:
                    y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
                t = y.clone()
                t[:, :h] = y[:, :h] * co - y[:, h:2 * h] * si
                t[:, h:2 * h] = y[:, :h] * si + y[:, h:2 * h] * co
                mag = y.abs()
                mag[:, :2 * h] = (y[:, :h].abs() + y[:, h:2 * h].abs()).repeat(1, 2)
                # sixteen f32 roundings of norm and products, an angle rounded to f32 (2^-22 with sine and cosine), then the type's rounding
                return t, t.abs() * HALF[c.el] + mag * (16 * 2.0 ** -24 + 2.0 ** -22) + TINY[c.el]

            if q:
                want, bound = turned(x[0][r, :H * qh].view(H, qh)[:, :hd], qn)
                d = (out[r, :H * hd].double().cpu().view(H, hd) - want).abs()
                assert torch.all(d <= bound), (b, i, float((d / bound).max()))
            if slot < 0:
                continue
            page, at = int(c.table[b, slot // c.page]), slot % c.page
            want, bound = turned(x[1][r, :KV * hd].view(KV, hd), kn)
            d = (c.k[page, :, at].double().cpu() - want).abs()
            assert torch.all(d <= bound), (b, i, float((d / bound).max()))
            assert torch.equal(c.v[page, :, at], x[2][r, :KV * hd].view(KV, hd).float().to(DT[c.el]))
    if q:
        assert torch.all(out[start[-1]:] == 7.0) and torch.all(out[:, H * hd:] == 7.0)
    assert es
    return a, (x, out, rs, ps, qn, kn, invd)


def _untouched(c, rows):
    """Every slot but the rows' own is still NaN."""
    k = c.k.clone()
    for b, n in enumerate(rows):
        for slot in range(max(0, c.lens_list[b] - n), c.lens_list[b]):
            k[int(c.table[b, slot // c.page]), :, slot % c.page] = math.nan
    assert torch.isnan(k).all()


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("el_in", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("form", [(24, 4, 256), (8, 2, 128), (3, 3, 64), (1, 1, 128)])
def test_append(llb, form, el, el_in):
    H, KV, hd = form
    rows, lens = [1, 0, 5, 20, 1], [1, 7, 5, 50, 333]
    c = Cache(llb, el, KV, hd, 16, lens, seed=31, live=lambda b, j: j >= lens[b] - rows[b])
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    _append(llb, c, H, rows, el_in, pos=[0, 3, 262143, 1000, 77], seed=32)
    _untouched(c, rows)
    _clean(llb)


@pytest.mark.parametrize("kw", [dict(rope=0), dict(rope=128), dict(rope=2), dict(rope=30), dict(norm=False), dict(gate=True), dict(pad=8), dict(pad=1), dict(shift=1), dict(shift=1, pad=3, gate=True),
                                dict(q=False), dict(eps=0.5), dict(pos=None), dict(pos=[2 ** 31 - 10, 0]), dict(pos=[-40, 5])])
def test_append_forms(llb, kw):
    """Strides and addresses of no round numbers, gates between the heads, keys and values alone, the rotation's widths, positions at the ends of their range."""
    kw = {**dict(pos=[9, 100]), **kw}
    c = Cache(llb, "bf16", 2, 128, 32, [40, 33], seed=33)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    _append(llb, c, 6, [3, 33], "bf16" if kw.get("shift") else "f32", seed=34, **kw)
    _untouched(c, [3, 33])
    _clean(llb)


def test_append_of_many_sequences(llb):
    """Sequences enough for several steps of the search for a row's own, many of them without rows."""
    rows = [(b * 7) % 3 if b % 5 else 0 for b in range(2500)]
    c = Cache(llb, "bf16", 1, 64, 16, [max(1, n) for n in rows], seed=35)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    _append(llb, c, 1, rows, "f32", rope=16, seed=36)
    _untouched(c, rows)
    _clean(llb)


def test_append_of_rows_without_a_slot(llb):
    """Lengths smaller than the rows: queries are rotated, nothing is stored below slot 0; bad pages store nothing."""
    c = Cache(llb, "f16", 2, 64, 16, [2, 0], seed=37)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    _append(llb, c, 2, [4, 1], "f32", seed=38, pos=[10, 20])
    _untouched(c, [2, 0])
    _clean(llb)
    c = Cache(llb, "f16", 2, 64, 16, [20], seed=37)
    c.k.fill_(math.nan), c.v.fill_(math.nan)
    keep = int(c.table[0, 1])
    a, more = _append(llb, c, 2, [20], "f32", seed=38)
    c.k.fill_(math.nan)
    c.table[0, 1] = -7
    llb.kv_append(c.desc(), a)
    assert llb.kv_errors() == 1 and torch.isnan(c.k[keep]).all() and not torch.isnan(c.k[int(c.table[0, 0])]).any()
    llb.lib().llb_b200_kv_errors_clear()
    for start in ([-1, 20], [0, 30]):
        more[2].copy_(_ints(start))
        llb.kv_append(c.desc(), a)
        assert llb.kv_errors() & 4
        llb.lib().llb_b200_kv_errors_clear()
    _clean(llb)


# ---- eviction -------------------------------------------------------------------------------------------
def _evict(llb, c, budget, sinks, recent, w, page2=16, kept=True, want_w=True, max_len=None, check=True):
    B, L = len(c.lens_list), max(c.lens_list + [1])
    most = min(budget, max_len or L)
    d = Cache(llb, c.el, c.KV, c.hd, page2, [min(n, budget) for n in c.lens_list], seed=40)
    d.k.fill_(math.nan), d.v.fill_(math.nan)
    if d.stride * page2 < most:
        extra = torch.full((B, -(-most // page2) - d.stride), -1, dtype=torch.int32, device="cuda")
        d.table, d.stride = torch.cat([d.table, extra], 1).contiguous(), -(-most // page2)
    d.lens.fill_(-9)
    ids = torch.full((B, c.KV, most + 2), -5, dtype=torch.int32, device="cuda")
    w2 = torch.full((B, c.KV, most + 1), 7.0, device="cuda")
    e = llb.KvEvict(budget=budget, sinks=sinks, recent=recent, max_len=max_len or L, w=w.data_ptr(), w_stride=w.shape[2], w_out=w2.data_ptr() if want_w else 0, w_out_stride=most + 1,
                    kept=ids.data_ptr() if kept else 0, kept_stride=most + 2)
    src, dst = c.desc(), d.desc()
    ws = torch.full((llb.kv_evict_ws(src, e),), 255, dtype=torch.uint8, device="cuda")
    e.ws, e.ws_bytes = ws.data_ptr(), ws.numel()
    llb.kv_evict(src, dst, e)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    for b, n in enumerate(c.lens_list if check else []):
        now = min(n, budget)
        assert int(d.lens[b]) == now
        for g in range(c.KV):
            if n <= budget:
                want = list(range(n))
            else:
                x = w[b, g, sinks:n - recent].double().cpu().numpy()
                x = np.where(np.isnan(x), -np.inf, x)
                nan = np.isnan(w[b, g, sinks:n - recent].cpu().numpy())
                order = sorted(range(len(x)), key=lambda i: (nan[i], -x[i], i))[:budget - sinks - recent]
                want = list(range(sinks)) + sorted(sinks + i for i in order) + list(range(n - recent, n))
            if kept:
                assert ids[b, g, :now].tolist() == want, (b, g)
                assert torch.all(ids[b, g, now:] == -5)
            idx = torch.tensor(want, dtype=torch.long)
            for what, X in (("k", c.K), ("v", c.V)):
                assert torch.equal(d.slots(b, now, what)[:, g].double().cpu(), X[b][idx][:, g])
            if want_w:
                assert torch.equal(w2[b, g, :now].nan_to_num(-3.0), w[b, g, idx.cuda()].nan_to_num(-3.0)) and torch.all(w2[b, g, now:] == 7.0)
    return d, ids, w2, (src, dst, e, ws)


def _weights(B, KV, L, seed, ties=0.3):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(3 * torch.randn(B, KV, L, generator=g) - 6)
    return torch.where(torch.rand(w.shape, generator=g) < ties, torch.zeros_like(w), w).cuda()


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("form,page", [((2, 128), 16), ((4, 256), 64), ((1, 64), 128)])
@pytest.mark.parametrize("budget,sinks,recent", [(100, 4, 20), (1, 0, 0), (64, 0, 64), (40, 40, 0), (40, 10, 30), (2000, 4, 64), (1023, 0, 1)])
def test_evict(llb, form, page, el, budget, sinks, recent):
    KV, hd = form
    lens = [1500, 3, 0, 100, 101, 64, 1024, 1025]
    c = Cache(llb, el, KV, hd, page, lens, seed=41)
    _evict(llb, c, budget, sinks, recent, _weights(len(lens), KV, 1503, 42), page2=128 if page == 16 else 16)
    _clean(llb)


@pytest.mark.parametrize("kind", ["equal", "zeros", "nan", "negative", "inf", "close"])
def test_evict_ties_and_odd_weights(llb, kind):
    """The lowest slots of equal weights; both zeros alike; NaN below everything; weights that differ in the last bit."""
    lens = [700, 650]
    c = Cache(llb, "bf16", 2, 64, 16, lens, seed=43)
    w = _weights(2, 2, 700, 44)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "zeros":
        w = torch.where(torch.rand(w.shape, device="cuda") < 0.5, torch.zeros_like(w), -torch.zeros_like(w))
    elif kind == "nan":
        w[:, :, ::2] = math.nan
        w[0, 0, 50:600] = math.nan
    elif kind == "negative":
        w = -w
    elif kind == "inf":
        w[:, :, ::3] = math.inf
        w[:, :, 1::3] = -math.inf
    else:
        w = (torch.full_like(w, 1.5).view(torch.int32) + torch.randint(0, 3, w.shape, device="cuda", dtype=torch.int32)).view(torch.float32)
    _evict(llb, c, 300, 4, 30, w)
    _clean(llb)


def test_evict_without_what_is_not_wanted(llb):
    c = Cache(llb, "bf16", 2, 128, 32, [500, 20], seed=45)
    _evict(llb, c, 130, 3, 7, _weights(2, 2, 500, 46), kept=False)
    _evict(llb, c, 130, 3, 7, _weights(2, 2, 500, 46), kept=False, want_w=False)
    _evict(llb, c, 130, 3, 7, _weights(2, 2, 500, 46), want_w=False)
    _clean(llb)


def test_evict_of_a_long_sequence(llb):
    c = Cache(llb, "bf16", 1, 64, 128, [70001, 5000], seed=47)
    _evict(llb, c, 9000, 16, 500, _weights(2, 1, 70001, 48))
    _clean(llb)


@pytest.mark.parametrize("budget,sinks,recent", [(9000, 16, 500), (19999, 19990, 7), (12999, 12997, 1), (1, 0, 0), (20000, 0, 0)])
@pytest.mark.parametrize("kind", ["mixed", "equal", "zeros", "nan", "two"])
def test_evict_of_long_sequences_goes_by_the_order(llb, budget, sinks, recent, kind):
    """Equal weights stay in the order of their slots, also over the parts that several blocks have, of which some may have no slot to choose from."""
    lens = [20001, 13000, 5000, 0, 1]
    w = _weights(len(lens), 2, 20001, 73, ties=0.9 if kind == "mixed" else 0.3)
    if kind == "equal":
        w[:] = 0.25
    elif kind == "zeros":
        w[:, :, 100:] = 0.0
        w[0, 0, 1::2] = -0.0
    elif kind == "nan":
        w[:, :, 7:19000] = math.nan
    elif kind == "two":
        w[:] = torch.where(torch.arange(20001, device="cuda") % 3 == 0, 1.5, 1.25)
    c = Cache(llb, "f16", 2, 64, 64, lens, seed=74)
    _evict(llb, c, budget, sinks, recent, w)
    _clean(llb)


def test_evict_reports_pages_and_lengths(llb):
    c = Cache(llb, "bf16", 2, 64, 16, [300], seed=49)
    w = _weights(1, 2, 300, 50, ties=0.0)
    d, ids, _, call = _evict(llb, c, 100, 0, 10, w)
    full = [d.slots(0, 100, x).clone() for x in ("k", "v")]
    c.table[0, 5] = -1
    d.k.fill_(math.nan)
    llb.kv_evict(*call[:3])
    assert llb.kv_errors() == 1
    llb.lib().llb_b200_kv_errors_clear()
    for g in range(2):
        gone = (ids[0, g, :100] // 16 == 5).cpu()
        now = d.slots(0, 100)[:, g]
        assert torch.isnan(now[gone.cuda()]).all() and torch.equal(now[~gone.cuda()], full[0][~gone.cuda()][:, g])
    d.table[0, 2] = d.n_pages + 5
    llb.kv_evict(*call[:3])
    assert llb.kv_errors() == 1
    llb.lib().llb_b200_kv_errors_clear()
    c.lens[0] = 400                                   # more than max_len: cut to it
    _, _, _, _ = d, ids, w, call
    llb.kv_evict(*call[:3])
    assert llb.kv_errors() & 2 and int(d.lens[0]) == 100
    llb.lib().llb_b200_kv_errors_clear()


# ---- as they are used -------------------------------------------------------------------------------------
def test_a_run_of_them_together(llb, packs):
    """Projections by the GEMM operator, rows into the cache, attention with weights, eviction, and more tokens behind it:
    two sequences through a prompt and eight tokens, one of them thinned on the way, against the same in 64 bits."""
    L = llb.lib()
    H, KV, hd, d, page, rope = 4, 2, 64, 512, 16, 32
    N = (H + 2 * KV) * hd
    g = torch.Generator().manual_seed(51)
    wf = torch.randn(N, d, generator=g) * 0.05
    raw = packs.QUANT["Q8_0"](wf).numpy()
    Wd = packs.dequant("Q8_0", torch.from_numpy(raw), N, d).double()
    w = torch.empty(L.llb_b200_weight_bytes(packs.FMT["Q8_0"], N, d), dtype=torch.uint8, device="cuda")
    llb.check(L.llb_b200_weight_upload(packs.FMT["Q8_0"], N, d, raw.ctypes.data, 0, w.data_ptr()), "upload")
    inv = 1.0e4 ** (-2.0 * torch.arange(rope // 2, dtype=torch.float64) / rope)
    invd = inv.cuda()
    prompts, cap, budget = [70, 33], 128, 48
    pools = [torch.full((40, KV, page, hd), math.nan, dtype=torch.float16, device="cuda") for _ in range(2)]
    free = list(range(40))
    held = [[], []]
    lens, table, starts, pos = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), \
        torch.zeros(2, dtype=torch.int32, device="cuda")
    wt = torch.zeros(2, KV, cap, device="cuda")
    kv = llb.Kv(el=1, kv_heads=KV, head_dim=hd, page=page, n_pages=40, seqs=2, table_stride=8, k=pools[0].data_ptr(), v=pools[1].data_ptr(), table=table.data_ptr(), lens=lens.data_ptr())
    K, V, score = [torch.zeros(0, KV, hd, dtype=torch.float64) for _ in range(2)], [torch.zeros(0, KV, hd, dtype=torch.float64) for _ in range(2)], [torch.zeros(KV, 0, dtype=torch.float64) for _ in range(2)]
    seen, worst = [0, 0], 0.0

    def rot(x, p):
        th = p * inv
        h = rope // 2
        y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        return torch.cat([y[:, :h] * th.cos() - y[:, h:rope] * th.sin(), y[:, :h] * th.sin() + y[:, h:rope] * th.cos(), y[:, rope:]], -1)

    ones = torch.ones(hd, device="cuda")
    for step in range(9):
        rows = prompts if step == 0 else [1, 1]
        R = sum(rows)
        x = torch.randn(R, d, generator=g)
        xd, yd = x.cuda(), torch.zeros(R, N, device="cuda")
        if R <= 8:
            xp = llb.handle(L.llb_b200_xp_new(d, R, 2), "xp")
            llb.check(L.llb_b200_xp_set_f32(xp, xd.data_ptr()), "set")
            llb.gemm(packs.FMT["Q8_0"], [w.data_ptr()], [N], [yd.data_ptr()], d, xp)
        else:
            llb.check(L.llb_b200_pf_gemm(packs.FMT["Q8_0"], w.data_ptr(), N, d, xd.data_ptr(), R, yd.data_ptr(), 0), "pf_gemm")
        now = [len(K[b]) + rows[b] for b in range(2)]
        for b in range(2):
            while len(held[b]) * page < now[b]:
                held[b].append(free.pop(7 % len(free)))
            table[b, :len(held[b])] = _ints(held[b])
        lens.copy_(_ints(now)); starts.copy_(_ints([0, rows[0], R])); pos.copy_(_ints(seen))
        qo, out = torch.zeros(R, H * hd, dtype=torch.float16, device="cuda"), torch.zeros(R, H * hd, dtype=torch.float32, device="cuda")
        llb.kv_append(kv, llb.KvAppend(rows=R, heads=H, el_in=0, rope_dim=rope, eps=1e-6, q=yd.data_ptr(), k=yd.data_ptr() + 4 * H * hd, v=yd.data_ptr() + 4 * (H + KV) * hd, q_stride=N, k_stride=N,
                                       v_stride=N, q_head_stride=hd, q_norm=ones.data_ptr(), k_norm=ones.data_ptr(), invfreq=invd.data_ptr(), row_start=starts.data_ptr(), pos=pos.data_ptr(),
                                       q_out=qo.data_ptr(), q_out_stride=H * hd))
        a = llb.KvAttn(rows=R, max_rows=max(rows), max_len=cap, heads=H, el_out=0, q=qo.data_ptr(), out=out.data_ptr(), q_stride=H * hd, out_stride=H * hd, row_start=starts.data_ptr())
        if step:
            a.w_in = a.w_out = wt.data_ptr()
            a.w_stride = cap
        ws = torch.empty(llb.kv_attn_ws(kv, a), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
        llb.kv_attn(kv, a)
        llb.check(L.llb_b200_sync(), "sync")
        y = x.double() @ Wd.T
        r = 0
        for b in range(2):
            fresh = y[r:r + rows[b]].view(rows[b], H + 2 * KV, hd)
            K[b] = torch.cat([K[b], torch.stack([rot(t[H:H + KV], seen[b] + i) for i, t in enumerate(fresh)])])
            V[b] = torch.cat([V[b], fresh[:, H + KV:]])
            score[b] = torch.cat([score[b], torch.zeros(KV, rows[b], dtype=torch.float64)], 1)
            for i in range(rows[b]):
                q = rot(fresh[i, :H], seen[b] + i).view(KV, H // KV, hd)
                m = now[b] - rows[b] + i + 1
                p = torch.softmax(torch.einsum("ghd,jgd->ghj", q, K[b][:m]) / 8.0, -1)
                want = torch.einsum("ghj,jgd->ghd", p, V[b][:m]).reshape(-1)
                # q, K, V and the probabilities are f16 (2^-11 each): a score is off by 2 * 2^-11 * |q| |k| / 8 <= 2^-10 * 8
                mass = torch.einsum("ghj,jgd->ghd", p, V[b][:m].abs()).reshape(-1)
                dlt = (out[r + i].double().cpu() - want).abs() / (mass * (2 * 8 * 2.0 ** -10 + 2 * 2.0 ** -11) + 1e-4)
                worst = max(worst, float(dlt.max()))
                if step:
                    score[b][:, :m] += p.sum(1)
            seen[b] += rows[b]
            r += rows[b]
        assert worst <= 1.0, (step, worst)
        for b in range(2):
            assert torch.all((wt[b, :, :now[b]].double().cpu() - score[b]).abs() <= 2 * 2 * 8 * 2.0 ** -10 * (score[b] + 1e-3))
        if step == 4:                                 # the longer sequence to 48 slots; the shorter is kept whole
            fresh_pages = [[free.pop(0) for _ in range(3)] for _ in range(2)]
            t2, l2, w2 = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, KV, cap, device="cuda")
            for b in range(2):
                t2[b, :3] = _ints(fresh_pages[b])
            kv2 = llb.Kv(el=1, kv_heads=KV, head_dim=hd, page=page, n_pages=40, seqs=2, table_stride=8, k=pools[0].data_ptr(), v=pools[1].data_ptr(), table=t2.data_ptr(), lens=l2.data_ptr())
            ids = torch.zeros(2, KV, budget, dtype=torch.int32, device="cuda")
            e = llb.KvEvict(budget=budget, sinks=4, recent=8, max_len=cap, w=wt.data_ptr(), w_stride=cap, w_out=w2.data_ptr(), w_out_stride=cap, kept=ids.data_ptr(), kept_stride=budget)
            llb.kv_evict(kv, kv2, e)
            llb.check(L.llb_b200_sync(), "sync")
            for b in range(2):
                n = min(budget, now[b])
                assert int(l2[b]) == n
                idx = ids[b, :, :n].long().cpu()
                K[b] = torch.stack([K[b][idx[h], h] for h in range(KV)], 1)
                V[b] = torch.stack([V[b][idx[h], h] for h in range(KV)], 1)
                score[b] = torch.gather(score[b], 1, idx)
                free += held[b]
                held[b] = fresh_pages[b]
            for pg in free:
                pools[0][pg], pools[1][pg] = math.nan, math.nan
            kv, table, lens, wt = kv2, t2, l2, w2
            kv_keep = (t2, l2)
    assert kv_keep
    _clean(llb)


def test_a_captured_step_runs_again_on_other_contents(llb):
    """A decode step (rows in, attention with weights) captured once and replayed with other rows, lengths and pages."""
    lens = [100, 31]
    c = Cache(llb, "bf16", 2, 128, 16, [140, 60], seed=60)
    c.lens.copy_(_ints(lens))
    a, more = None, None
    x = [torch.randn(2, n * 128, device="cuda") for n in (4, 2, 2)]
    qo, out = torch.zeros(2, 512, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 512, dtype=torch.bfloat16, device="cuda")
    rs, wt = _ints([0, 1, 2]), torch.zeros(2, 2, 160, device="cuda")
    ap = llb.KvAppend(rows=2, heads=4, el_in=0, rope_dim=0, eps=1e-6, q=x[0].data_ptr(), k=x[1].data_ptr(), v=x[2].data_ptr(), q_stride=512, k_stride=256, v_stride=256, q_head_stride=128,
                      row_start=rs.data_ptr(), q_out=qo.data_ptr(), q_out_stride=512)
    at = llb.KvAttn(rows=2, max_rows=1, max_len=140, heads=4, el_out=2, q=qo.data_ptr(), out=out.data_ptr(), q_stride=512, out_stride=512, row_start=rs.data_ptr(), w_out=wt.data_ptr(), w_stride=160)
    ws = torch.empty(llb.kv_attn_ws(c.desc(), at), dtype=torch.uint8, device="cuda")
    at.ws, at.ws_bytes = ws.data_ptr(), ws.numel()

    def step():
        llb.kv_append(c.desc(), ap)
        llb.kv_attn(c.desc(), at)

    stream = torch.cuda.ExternalStream(llb.lib().llb_b200_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for it in range(3):
        for t in x:
            t.normal_()
        c.lens.add_(3)
        if it == 2:
            c.table[0, 8] = c.table[1, 3]             # (pages change hands between steps)
        torch.cuda.synchronize()
        step()
        llb.check(llb.lib().llb_b200_sync(), "sync")
        want = [t.clone() for t in (out, wt, c.k.view(torch.int16))]
        for t in (out, wt):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(wt, want[1]) and torch.equal(c.k.view(torch.int16), want[2])
    del graph
    _clean(llb)


def test_calls_from_another_thread(llb):
    import threading
    c = Cache(llb, "bf16", 2, 128, 16, [500, 90], seed=61)
    want = _attn(llb, c, 8, [1, 1], seed=62)
    got = []

    def work():
        for _ in range(10):
            got.append(_attn(llb, c, 8, [1, 1], seed=62)["out"])

    ts = [threading.Thread(target=work) for _ in range(3)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert len(got) == 30 and all(torch.equal(g, want["out"]) for g in got)
    _clean(llb)
