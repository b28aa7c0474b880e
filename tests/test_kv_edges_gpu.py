"""The paged key-value cache's operators where values, lengths and counts are at the ends of their ranges (bounds as in test_kv_gpu)."""
import math

import pytest
import torch

from test_kv_gpu import Cache, _append, _attn, _check_attn, _clean, _evict, _ints, _weights

pytestmark = pytest.mark.gpu


# ---- rows that see nothing, values that rows do not see ---------------------------------------------------
@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("H,KV", [(4, 2), (1, 1), (6, 1)])
@pytest.mark.parametrize("rows,lens", [([200], [50]), ([300, 140, 5], [64, 139, 3]), ([70], [69])])
def test_rows_without_a_slot_beside_rows_with_many(llb, rows, lens, H, KV, hd, el):
    """Rows at slots below 0 are zeros, to the last bit, also where rows of the same block see slots."""
    c = Cache(llb, el, KV, hd, 16, lens, seed=101)
    _check_attn(c, _attn(llb, c, H, rows, seed=102, max_len=140))
    _check_attn(c, _attn(llb, c, H, rows, seed=102, max_len=140, window=30, sinks=3, el_out="f32"))
    _clean(llb)


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_rows_whose_pages_are_all_bad(llb, page, hd, el):
    """The first 64 slots are on no page: rows that see only those are zeros, and the rows behind them are right."""
    n, H, KV = 150, 4, 2
    c = Cache(llb, el, KV, hd, page, [n], seed=103)
    c.table[0, :64 // page] = -1
    r = _attn(llb, c, H, [n], seed=104)
    assert llb.kv_errors() == 1
    llb.lib().llb_b200_kv_errors_clear()
    out = r["out"][:n].double().cpu().view(n, KV, H // KV, hd)
    assert torch.all(out[:64] == 0)
    c.lens_list, c.K, c.V = [n - 64], [c.K[0][64:]], [c.V[0][64:]]
    r["out"], r["q"], r["rows"], r["start"] = r["out"][64:], r["q"][64:], [n - 64], [0, n - 64]
    _check_attn(c, r)
    _clean(llb)


@pytest.mark.parametrize("el,big", [("bf16", 3.0e38), ("bf16", -2.0 ** 126), ("f16", 65504.0)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,window", [(150, 0), (150, 40), (40, 0), (4, 0)])
def test_a_later_rows_large_values_do_not_reach_earlier_rows(llb, rows, window, hd, el, big):
    """V of the last rows' own slots is as large as the type holds: the rows before them do not see it."""
    KV, G, late = 2, 4, max(1, rows // 8)
    m = rows + 40
    c = Cache(llb, el, KV, hd, 16, [m], seed=105)
    for j in range(m - late, m):
        c.v[int(c.table[0, j // 16]), :, j % 16] = big
    r = _attn(llb, c, KV * G, [rows], window=window, seed=106)
    n = rows - late
    r["out"][n:rows] = 7.0
    r["rows"], r["start"] = [n], [0, n]
    c.lens_list, c.K, c.V = [m - late], [c.K[0][:-late]], [c.V[0][:-late]]
    _check_attn(c, r)
    _clean(llb)


@pytest.mark.parametrize("max_len", [2 ** 31 - 1, 2 ** 31 - 2, 1 << 30])
def test_no_bound_on_the_lengths(llb, max_len):
    """max_len says no more than the table: the same results as with the lengths' own bound."""
    for lens, rows in (([700], [1]), ([700], [3]), ([700], [300])):
        c = Cache(llb, "bf16", 1, 128, 16, lens, seed=114)
        weights = rows[0] < 8
        r = _attn(llb, c, 2, rows, seed=115, weights=weights)
        _check_attn(c, r)
        kv, a = r["call"]
        want = r["out"].clone(), r["w_out"].clone() if weights else None
        r["out"].fill_(7.0)
        a.max_len = max_len
        if weights:
            r["w_out"].fill_(7.0)
            a.w_stride = max_len                       # (one row of one head: the stride is never taken)
        ws = torch.full((llb.kv_attn_ws(kv, a),), 255, dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
        llb.kv_attn(kv, a)
        llb.check(llb.lib().llb_b200_sync(), "sync")
        _check_attn(c, r)
        assert rows[0] > 8 or torch.equal(r["out"], want[0])
        assert not weights or torch.equal(r["w_out"], want[1])
    for n in (700, 13000):
        c = Cache(llb, "bf16", 1, 64, 64, [n], seed=116)
        w = _weights(1, 1, n, 117)
        d, ids, w2, (src, dst, e, _) = _evict(llb, c, 300, 4, 30, w)
        want = ids.clone(), w2.clone(), d.slots(0, 300).clone()
        ids.fill_(-5), w2.fill_(7.0), d.k.fill_(math.nan)
        e.max_len = e.w_stride = max_len
        ws = torch.full((llb.kv_evict_ws(src, e),), 255, dtype=torch.uint8, device="cuda")
        e.ws, e.ws_bytes = ws.data_ptr(), ws.numel()
        llb.kv_evict(src, dst, e)
        llb.check(llb.lib().llb_b200_sync(), "sync")
        assert torch.equal(ids, want[0]) and torch.equal(w2, want[1]) and torch.equal(d.slots(0, 300), want[2])
    _clean(llb)


def test_the_longest_sequence(llb):
    """2^31 - 4096 slots and more, all on one shared page of zeros: a window at the end, and what every slot got."""
    most, hd = 2 ** 31 - 4096, 64
    k = torch.zeros(1, 1, 128, hd, dtype=torch.bfloat16, device="cuda")
    table, rs = torch.zeros(1, 1 << 24, dtype=torch.int32, device="cuda"), _ints([0, 1])
    q, out = torch.ones(1, hd, dtype=torch.bfloat16, device="cuda"), torch.full((1, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    w = torch.full((most + 8,), 7.0, device="cuda")
    w[:most] = 0.5
    for n in (most, most + 300, 2 ** 31 - 1):
        lens = _ints([n])
        kv = llb.Kv(el=2, kv_heads=1, head_dim=hd, page=128, n_pages=1, seqs=1, table_stride=1 << 24, k=k.data_ptr(), v=k.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr())
        a = llb.KvAttn(rows=1, max_rows=1, max_len=2 ** 31 - 1, heads=1, window=100, sinks=3, el_out=2, q=q.data_ptr(), out=out.data_ptr(), q_stride=hd, out_stride=hd,
                       row_start=rs.data_ptr(), w_in=w.data_ptr(), w_out=w.data_ptr(), w_stride=2 ** 31 - 1)
        ws = torch.empty(llb.kv_attn_ws(kv, a), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
        llb.kv_attn(kv, a)
        assert llb.kv_errors() == (2 if n > most else 0)
        llb.lib().llb_b200_kv_errors_clear()
        assert torch.all(out == 0)
    got = w[:most] - 0.5
    seen = torch.cat([got[:3], got[-100:]])
    assert torch.all((seen - 3 / 103).abs() < 1e-6) and not got[3:-100].any() and torch.all(w[most:] == 7.0)
    _clean(llb)
    del w, ws, got, seen
    torch.cuda.empty_cache()


def test_evict_of_more_pieces_than_an_int_counts(llb):
    """2^26 + 1000 slots of 32 pieces each are kept.  All of them lie on one page of ones, and go to one page: what is written there is the same
    from everywhere."""
    n, hd = (1 << 26) + 1000, 256
    stride = n // 128 + 1
    src, dst = (torch.full((1, 1, 128, hd), x, dtype=torch.bfloat16, device="cuda") for x in (1.0, 0.0))
    tables = [torch.zeros(1, stride, dtype=torch.int32, device="cuda") for _ in range(2)]
    lens = [_ints([n]), _ints([-9])]
    w = torch.rand(1, 1, n, device="cuda")
    w2 = torch.full_like(w, 7.0)
    kept = torch.full((1, 1, n), -5, dtype=torch.int32, device="cuda")
    kv = [llb.Kv(el=2, kv_heads=1, head_dim=hd, page=128, n_pages=1, seqs=1, table_stride=stride, k=x.data_ptr(), v=x.data_ptr(), table=t.data_ptr(), lens=m.data_ptr())
          for x, t, m in zip((src, dst), tables, lens)]
    e = llb.KvEvict(budget=n, max_len=n, w=w.data_ptr(), w_stride=n, w_out=w2.data_ptr(), w_out_stride=n, kept=kept.data_ptr(), kept_stride=n)
    llb.kv_evict(kv[0], kv[1], e)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    assert int(lens[1]) == n and torch.equal(w2, w)
    assert torch.equal(kept[0, 0], torch.arange(n, dtype=torch.int32, device="cuda"))
    assert torch.all(dst == 1)
    _clean(llb)


# ---- windows, lengths and counts at the ends of their ranges ----------------------------------------------
@pytest.mark.parametrize("sinks", [2 ** 26, 2 ** 27, 2 ** 28 + 3, 2 ** 31 - 1])
@pytest.mark.parametrize("window", [1, 40, 2 ** 27, 2 ** 30])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_more_first_tokens_than_there_are_slots(llb, hd, window, sinks):
    """... make every slot up to the row's own seen, whatever the window."""
    c = Cache(llb, "bf16", 2, hd, 16, [150, 300, 90], seed=118)
    _check_attn(c, _attn(llb, c, 4, [150, 130, 1], window=window, sinks=sinks, seed=119))
    _check_attn(c, _attn(llb, c, 4, [3, 1, 2], window=window, sinks=sinks, seed=119, weights=True))
    _clean(llb)


@pytest.mark.parametrize("hd", [64, 256])
def test_rows_far_behind_their_first_tokens(llb, hd):
    """Rows at slots from 2^28 on, all slots on shared pages: two for the first tokens, one in between, two for the window."""
    n, rows, window, sinks, page = (1 << 28) + 133, 133, 60, 37, 64
    g = torch.Generator(device="cuda").manual_seed(120)
    k, v = (torch.randn(5, 1, page, hd, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    k[2], v[2] = math.nan, math.nan
    last = -(-n // page)
    table = torch.full((1, last), 2, dtype=torch.int32, device="cuda")
    table[0, 0], table[0, 1] = 0, 1
    table[0, last - 4:] = _ints([3, 4, 3, 4])
    lens, rs = _ints([n]), _ints([0, rows])
    q = torch.randn(rows, hd, device="cuda", dtype=torch.bfloat16, generator=g)
    out = torch.full_like(q, 7.0)
    kv = llb.Kv(el=2, kv_heads=1, head_dim=hd, page=page, n_pages=5, seqs=1, table_stride=last, k=k.data_ptr(), v=v.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr())
    a = llb.KvAttn(rows=rows, max_rows=rows, max_len=n, heads=1, window=window, sinks=sinks, el_out=2, q=q.data_ptr(), out=out.data_ptr(), q_stride=hd, out_stride=hd, row_start=rs.data_ptr())
    ws = torch.full((llb.kv_attn_ws(kv, a),), 255, dtype=torch.uint8, device="cuda")
    a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
    llb.kv_attn(kv, a)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    _clean(llb)
    # the same with the slots in between left out: the first tokens, then the window's slots
    skip = (last - 4) * page - 2 * page
    K, V = (torch.cat([x[0, 0], x[1, 0], x[3, 0], x[4, 0], x[3, 0], x[4, 0]]).double().cpu() for x in (k, v))
    j = torch.arange(len(K))
    for i in range(rows):
        e = n - rows + i - skip
        idx = ((j <= e) & ((j > e - window) | (j < sinks))).nonzero()[:, 0]
        x = (q[i].double().cpu() @ K[idx].T) * hd ** -0.5
        p = torch.softmax(x, 0)
        want, size = p @ V[idx], p @ V[idx].abs()
        # scores below 10 are off by hd 2^-23 of |q| |K| / sqrt(hd) < 40 at most, a probability by four times that and 2^-8; then the result's rounding
        bound = size * (4 * 40 * hd * 2.0 ** -23 + 2.0 ** -8) + want.abs() * 2.0 ** -8
        assert torch.all((out[i].double().cpu() - want).abs() <= bound * 1.01 + 1e-30), i


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30])
@pytest.mark.parametrize("rows,lens", [([200, 130], [50, 130]), ([4, 3], [2, 0]), ([3, 2], [600, 1])])
@pytest.mark.parametrize("sinks", [0, 5])
def test_a_window_larger_than_every_length(llb, rows, lens, sinks, window):
    """... sees all slots up to the row's own, also behind rows at slots below 0."""
    c = Cache(llb, "bf16", 2, 128, 16, lens, seed=107)
    _check_attn(c, _attn(llb, c, 4, rows, window=window, sinks=sinks, seed=108, max_len=640, weights=max(rows) < 8))
    _clean(llb)


@pytest.mark.parametrize("kind", ["mixed", "equal", "nan"])
def test_evict_of_a_sequence_whose_keys_have_no_room(llb, kind):
    """More slots than four blocks' shared memory holds keys of (4 x 49152): the weights are read in every pass."""
    lens = [200001, 196609, 5000]
    w = _weights(3, 1, 200001, 112, ties=0.5)
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "nan":
        w[:, :, 1000:199000:2] = math.nan
    c = Cache(llb, "bf16", 1, 64, 128, lens, seed=113)
    for budget, sinks, recent in ((9000, 16, 500), (150000, 0, 0)):
        _evict(llb, c, budget, sinks, recent, w, page2=128)
    _clean(llb)


def _best(llb, kv, a, times=5):
    stream = torch.cuda.ExternalStream(llb.lib().llb_b200_stream())
    best = math.inf
    for _ in range(times):
        t = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        t[0].record(stream)
        llb.kv_attn(kv, a)
        t[1].record(stream)
        t[1].synchronize()
        best = min(best, t[0].elapsed_time(t[1]))
    return best


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("rows,n,KV", [(1, 100000, 2), (1, 3000, 2), (3, 60000, 1), (700, 2000, 2)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_key_that_is_no_number_costs_no_time(llb, hd, rows, n, KV, bad):
    """Rows that see it are NaN, as before it, in about the time of the same call without it (one slot after the other it is hundreds of times as much)."""
    H = 2 * KV
    c = Cache(llb, "bf16", KV, hd, 128, [n], seed=110)
    r = _attn(llb, c, H, [rows], seed=111, behind=0)
    before = _best(llb, *r["call"])
    c.k[int(c.table[0, 0]), :, 7, 3] = bad
    r["q"].abs_()                                      # (an infinite key's score is plus infinity)
    after = _best(llb, *r["call"])
    assert torch.isnan(r["out"]).all()
    assert after < 4 * before + 0.02, (before, after)
    _clean(llb)


@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("rows,n", [(1, 100000), (1, 3000), (3, 60000)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_an_infinite_value_that_every_row_sees(llb, hd, rows, n, bad):
    """f16, where values beyond its range become infinite: that dimension is infinite, the others are as they were, in about the same time."""
    c = Cache(llb, "f16", 2, hd, 128, [n], seed=121)
    c.k[int(c.table[0, 0]), :, 7] = 0.0                # (scores of 0: probabilities above half a step of f16's smallest numbers)
    r = _attn(llb, c, 4, [rows], seed=122, behind=0, scale=0.1)
    want = r["out"].view(rows, 4, hd).clone()
    before = _best(llb, *r["call"])
    c.v[int(c.table[0, 0]), :, 7, 5] = bad
    after = _best(llb, *r["call"])
    want[:, :, 5] = bad
    assert torch.equal(r["out"].view(rows, 4, hd), want)
    assert after < 4 * before + 0.02, (before, after)
    _clean(llb)


@pytest.mark.parametrize("rows,n", [(1, 60000), (3, 20000), (300, 20000), (80, 3000)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_probabilities_below_the_smallest_f16(llb, hd, rows, n):
    """One slot has nearly all of the weight and V = 0, the others exp(-17.5) = 2^-25.2 of it each and V = 1: what they add up to is the result.

    Bounds.  A score of 17.5 is off by hd 2^-23 of it, its power of two by 2^-21 of itself.  A probability is rounded to f16 after a multiplication by
    2^7 or more: 2^-11 of it, or half a step of 2^-24, which is 2^-32 of the largest.  Sums of n terms by n 2^-23; then the result's rounding."""
    c = Cache(llb, "f16", 1, hd, 64, [n], seed=109)
    c.k.fill_(0.0), c.v.fill_(1.0)
    c.k[..., 0] = -17.5
    p0 = int(c.table[0, 0])
    c.k[p0, 0, 5], c.v[p0, 0, 5] = 0.0, 0.0
    q = torch.zeros(rows, hd)
    q[:, 0] = 1.0
    r = _attn(llb, c, 1, [rows], q=q, scale=1.0, behind=0)
    seen = torch.arange(n - rows + 1, n + 1, dtype=torch.float64) - 1
    tail = seen * math.exp(-17.5)
    want = tail / (1.0 + tail)
    bound = want * (17.5 * hd * 2.0 ** -23 + 2.0 ** -20 + 2 * 2.0 ** -11 + n * 2.0 ** -22) + n * 2.0 ** -32 + 2.0 ** -25
    d = (r["out"].double().cpu() - want[:, None]).abs()
    assert torch.all(d <= bound[:, None]), (float(d.max()), float(want.max()), float(bound.max()))
    _clean(llb)


# ---- outputs over inputs -----------------------------------------------------------------------------------
def _refused(llb, call, word):
    with pytest.raises(llb.LlbError, match=word):
        call()


def _append_call(llb, c, x, out, rs, q=0, k=0, v=0, out_at=0, H=4, es=4, stride=None, out_stride=None):
    stride = stride or x.stride(0)
    w = c.KV * c.hd
    return llb.KvAppend(rows=rs[1], heads=H, el_in=llb.EL["f32"], rope_dim=0, eps=1e-6, q=x.data_ptr() + es * q, k=x.data_ptr() + es * (k or H * c.hd), v=x.data_ptr() + es * (v or H * c.hd + w),
                        q_stride=stride, k_stride=stride, v_stride=stride, q_head_stride=c.hd, row_start=rs[0].data_ptr(), q_out=out.data_ptr() + out_at, q_out_stride=out_stride or out.stride(0))


def test_appended_queries_may_lie_beside_their_rows_and_not_over_them(llb):
    c = Cache(llb, "bf16", 2, 64, 16, [5], seed=123)
    H, R = 4, 5
    rs = (_ints([0, R]), R)
    wide = torch.zeros(R, 800, device="cuda")             # rows of 512 numbers, and 128 more words that 256 queries in 16 bits take
    wide[:, :512] = torch.randn(R, 512, device="cuda")
    apart = torch.zeros(R, 256, dtype=torch.bfloat16, device="cuda")
    llb.kv_append(c.desc(), _append_call(llb, c, wide, apart, rs))
    beside = wide.view(torch.bfloat16)
    llb.kv_append(c.desc(), _append_call(llb, c, wide, beside, rs, out_at=4 * 512))
    llb.check(llb.lib().llb_b200_sync(), "sync")
    assert torch.equal(beside[:, 1024:1280], apart)
    for at in (0, 4 * 255, 4 * 256, 4 * 511, 4 * 700, 4 * 800):      # over q, k, v, and over the next row's q
        _refused(llb, lambda: llb.kv_append(c.desc(), _append_call(llb, c, wide, beside, rs, out_at=at)), "overlaps")
    _refused(llb, lambda: llb.kv_append(c.desc(), _append_call(llb, c, wide, beside, rs, out_at=4 * 512, out_stride=1602)), "overlaps")
    _clean(llb)


def test_attention_over_its_queries_or_weights_is_refused(llb):
    c = Cache(llb, "bf16", 2, 64, 16, [40, 30], seed=124)
    r = _attn(llb, c, 4, [1, 1], seed=125, weights=True)
    _check_attn(c, r)
    kv, a = r["call"]
    want = r["out"].clone(), r["w_out"].clone()
    buf = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    buf[:, :256] = r["q"][:, :256]
    a.q, a.q_stride, a.out_stride = buf.data_ptr(), 512, 512
    for at in (16, 2 * 248, 2 * 264, 2 * 512):
        a.out = buf.data_ptr() + at
        _refused(llb, lambda: llb.kv_attn(kv, a), "out overlaps q")
    a.out = buf.data_ptr() + 2 * 256
    for d in (4, -4, 4 * (r["w_in"].shape[2] - 1)):
        a.w_in = a.w_out + d
        _refused(llb, lambda: llb.kv_attn(kv, a), "w_out overlaps")
    a.w_in = r["w_in"].data_ptr()
    r["w_out"].fill_(7.0)
    llb.kv_attn(kv, a)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    assert torch.equal(buf[:2, 256:], want[0][:2, :256]) and torch.equal(r["w_out"], want[1])
    _clean(llb)


def test_evictions_over_their_inputs_are_refused(llb):
    c = Cache(llb, "bf16", 2, 64, 16, [300, 90], seed=126)
    w = _weights(2, 2, 300, 127)
    d, ids, w2, (src, dst, e, ws) = _evict(llb, c, 100, 4, 20, w)
    want = w2[..., :100].clone()
    for at in (4, 4 * 299, -4 * 50):
        e.w_out = w.data_ptr() + at
        _refused(llb, lambda: llb.kv_evict(src, dst, e), "w_out overlaps w")
    both = torch.zeros(2, 2, 512, device="cuda")           # a head's weights, and the kept slots' behind them
    both[..., :300] = w
    e.w, e.w_stride, e.w_out, e.w_out_stride = both.data_ptr(), 512, both.data_ptr() + 4 * 300, 512
    llb.kv_evict(src, dst, e)
    llb.check(llb.lib().llb_b200_sync(), "sync")
    for b, n in enumerate((100, 90)):
        assert torch.equal(both[b, :, 300:300 + n], want[b, :, :n])
    dst.lens = src.lens + 4
    _refused(llb, lambda: llb.kv_evict(src, dst, e), "lens overlap")
    _clean(llb)


@pytest.mark.parametrize("rows", [[30, 40], [3000, 1]])
def test_positions_that_pass_the_largest_int(llb, rows):
    """A sequence's first row is at a position that an int holds, the rows behind it are where they are."""
    c = Cache(llb, "f16", 1, 64, 64, rows, seed=128)
    _append(llb, c, 1, rows, "f32", seed=129, pos=[2 ** 31 - 10, 2 ** 31 - 1], behind=0)
    _clean(llb)


@pytest.mark.parametrize("el", ["bf16", "f16"])
@pytest.mark.parametrize("rows,n,H,KV,hd", [(4, 60000, 2, 1, 128), (4, 60000, 8, 2, 256), (5, 30000, 4, 4, 64), (100, 60000, 2, 1, 128), (100, 40000, 2, 1, 256), (80, 30000, 2, 2, 64)])
def test_a_row_that_is_no_number_behind_a_long_sequence(llb, rows, n, H, KV, hd, el):
    """K and V of a call's own last row are NaN: the rows before it are what they are without it, and only the part of their slots that holds it is looked at once more."""
    c = Cache(llb, el, KV, hd, 128, [n], seed=130)
    r = _attn(llb, c, H, [rows], seed=131, behind=0)
    want = r["out"].clone()
    before = _best(llb, *r["call"])
    j = n - 1
    for pool in (c.k, c.v):
        pool[int(c.table[0, j // 128]), :, j % 128] = math.nan
    after = _best(llb, *r["call"])
    assert torch.isnan(r["out"][rows - 1]).all()
    r["out"][rows - 1] = 7.0
    r["rows"], r["start"] = [rows - 1], [0, rows - 1]
    c.lens_list, c.K, c.V = [n - 1], [c.K[0][:-1]], [c.V[0][:-1]]
    _check_attn(c, r)
    # a part of 148 of the slots, at most 32 rows of it one after the other, each slot about 0.5 us
    part = -(-n * KV // 148) + 512
    assert after < 4 * before + 1e-3 * part * (1 if rows < 8 else 32), (before, after)
    assert torch.equal(torch.isnan(want), torch.zeros_like(want, dtype=torch.bool))
    _clean(llb)


@pytest.mark.parametrize("el,bad", [("bf16", math.nan), ("f16", math.nan), ("bf16", math.inf), ("f16", -math.inf)])
@pytest.mark.parametrize("rows,lens,H,KV,hd,window", [([1200], [1500], 16, 8, 256, 0), ([1200], [1500], 32, 16, 128, 0), ([700, 300], [1100, 420], 64, 16, 64, 200),
                                                      ([4] * 40, [300 + 7 * b for b in range(40)], 16, 8, 128, 0), ([3] * 40, [500] * 40, 24, 4, 256, 100), ([15, 2] * 60, [90, 300] * 60, 4, 4, 64, 33)])
def test_rows_in_front_of_a_row_that_is_no_number(llb, rows, lens, H, KV, hd, window, el, bad):
    """In the middle of the first sequence's rows K and V are no numbers: what is in front of it is right, and so are all other sequences; in a few times the call's time (one row
    and one slot after the other it is hundreds)."""
    c = Cache(llb, el, KV, hd, 16, lens, seed=132)
    r = _attn(llb, c, H, rows, seed=133, window=window, behind=0)
    before = _best(llb, *r["call"])
    at = rows[0] // 2                                      # (row `at` and those behind it see that slot)
    j = lens[0] - rows[0] + at
    for pool in (c.k, c.v):
        pool[int(c.table[0, j // 16]), :, j % 16] = bad
    after = _best(llb, *r["call"])
    end = rows[0] if not window else min(rows[0], at + window)
    if bad != bad:
        assert torch.isnan(r["out"][at:end]).all()
    r["out"][at:end] = 7.0
    r["start"] = [0] + r["start"][1:]
    # the rows in front, as a sequence that ends before the slot; the others as they are
    keep = c.lens_list, c.K, c.V, r["rows"]
    c.lens_list, c.K, c.V, r["rows"] = [j], [c.K[0][:j]], [c.V[0][:j]], [at]
    full, start = r["out"], r["start"]
    r["out"], r["start"] = full[:at], [0, at]
    _check_attn(c, r)
    c.lens_list, c.K, c.V, r["rows"] = list(keep[0][1:]), keep[1][1:], keep[2][1:], keep[3][1:]
    if r["rows"]:
        r["out"], r["q"], r["start"] = full[rows[0]:], r["q"][rows[0]:], [s - rows[0] for s in start[1:]]
        _check_attn(c, r)
    assert after < 8 * before + 1.5, (before, after)
    _clean(llb)


# ---- captured -------------------------------------------------------------------------------------------------
def test_captured_prompts_and_evictions_run_again_on_other_contents(llb):
    """A prompt over several blocks a row, verify rows with weights and an eviction captured together, replayed with other values, lengths, pages and weights."""
    c = Cache(llb, "bf16", 2, 128, 16, [9000, 700], seed=134)
    prompt, few = _attn(llb, c, 4, [90, 40], seed=135, behind=0, max_len=9000), _attn(llb, c, 4, [3, 2], seed=136, behind=0, weights=True, max_len=9000)
    w = _weights(2, 2, 9000, 137)
    c.K, c.V = [k[:9000] for k in c.K], [v[:9000] for v in c.V]
    d, ids, w2, ev = _evict(llb, c, 500, 4, 60, w)
    held = [prompt["out"], few["out"], few["w_out"], d.k, d.v, d.lens, ids, w2]

    def step():
        llb.kv_attn(*prompt["call"])
        llb.kv_attn(*few["call"])
        llb.kv_evict(*ev[:3])

    stream = torch.cuda.ExternalStream(llb.lib().llb_b200_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for n in ((8000, 650), (3000, 41), (8999, 300)):
        c.lens.copy_(_ints(list(n)))
        w.copy_(_weights(2, 2, 9000, 138 + n[0]))
        prompt["q"].normal_()
        c.table[0, :100] = c.table[0, :100].flip(0)
        torch.cuda.synchronize()
        step()
        llb.check(llb.lib().llb_b200_sync(), "sync")
        want = [t.clone() for t in held]
        for t in held:
            t.fill_(3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in held]
        for t in held:
            t.fill_(3)
        torch.cuda.synchronize()
        step()
        llb.check(llb.lib().llb_b200_sync(), "sync")
        for a, b in zip(again, held):
            assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) if a.is_floating_point() else torch.equal(a, b)
        assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    del graph
    _clean(llb)
