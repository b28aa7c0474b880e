"""The paged key-value cache's calls refuse what they cannot do before anything reaches a GPU: the checks need none."""
import pytest

P = 1 << 20   # an address that nothing looks at


def _kv(llb, **kw):
    a = dict(el=llb.EL["bf16"], kv_heads=4, head_dim=128, page=32, n_pages=64, seqs=3, table_stride=16, k=P, v=P, table=P, lens=P)
    a.update(kw)
    return llb.Kv(**a)


def _append(llb, **kw):
    a = dict(rows=5, heads=8, el_in=llb.EL["f32"], rope_dim=64, eps=1e-6, q=P, k=P, v=P, q_stride=1024, k_stride=512, v_stride=512, q_head_stride=128,
             q_norm=P, k_norm=P, invfreq=P, row_start=P, pos=P, q_out=P, q_out_stride=1024)
    a.update(kw)
    return llb.KvAppend(**a)


def _attn(llb, **kw):
    a = dict(rows=5, max_rows=2, max_len=500, heads=8, window=0, sinks=0, scale=0.0, el_out=llb.EL["bf16"], q=P, out=2 * P, q_stride=1024, out_stride=1024, row_start=P,
             ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return llb.KvAttn(**a)


def _evict(llb, **kw):
    a = dict(budget=100, sinks=4, recent=16, max_len=500, w=P, w_stride=500, w_out=P + 64, w_out_stride=100, kept=P, kept_stride=100, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return llb.KvEvict(**a)


def _refused(llb, call, word):
    with pytest.raises(llb.LlbError, match=word):
        call()


BAD_KV = [(dict(el=0), "el 0"), (dict(el=7), "el 7"), (dict(head_dim=96), "head_dim 96"), (dict(head_dim=0), "head_dim 0"), (dict(kv_heads=0), "0 kv heads"),
          (dict(page=8), "pages of 8"), (dict(page=48), "pages of 48"), (dict(page=256), "pages of 256"), (dict(n_pages=0), "0 pages"), (dict(seqs=0), "0 sequences"),
          (dict(seqs=65536), "65536 sequences"), (dict(table_stride=0), "table_stride 0"), (dict(k=0), "multiples of 16"), (dict(v=P + 8), "multiples of 16"),
          (dict(table=0), "int32"), (dict(lens=P + 2), "int32")]


@pytest.mark.parametrize("bad,word", BAD_KV)
def test_caches_that_are_refused(pkg, bad, word):
    llb = pkg.llb
    kv = _kv(llb, **bad)
    _refused(llb, lambda: llb.kv_append(kv, _append(llb)), word)
    _refused(llb, lambda: llb.kv_attn(kv, _attn(llb)), word)
    _refused(llb, lambda: llb.kv_attn_ws(kv, _attn(llb)), word)
    _refused(llb, lambda: llb.kv_evict(kv, _kv(llb, table=P + 64, lens=P + 64), _evict(llb)), word)
    _refused(llb, lambda: llb.kv_evict(_kv(llb, table=P + 64, lens=P + 64), kv, _evict(llb)), word)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "-1 rows"), (dict(heads=0), "0 heads"), (dict(heads=6), "6 heads on 4"), (dict(heads=4 * 65), "260 heads"), (dict(el_in=3), "el_in 3"),
    (dict(rope_dim=63), "rope_dim 63"), (dict(rope_dim=130), "rope_dim 130"), (dict(rope_dim=-2), "rope_dim -2"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(k=0), "multiples of their elements"), (dict(q=P + 2), "multiples of their elements"), (dict(q_stride=1023), "heads of q"), (dict(q_head_stride=127), "heads of q"),
    (dict(k_stride=511), "k_stride 511"), (dict(v_stride=0), "v_stride 0"), (dict(q_out=0), "q_out"), (dict(q_out_stride=1000), "q_out"), (dict(q_norm=P + 1), "norm weights"),
    (dict(invfreq=0), "invfreq"), (dict(invfreq=P + 4), "invfreq"), (dict(row_start=0), "row_start"), (dict(pos=P + 1), "row_start and pos")])
def test_appends_that_are_refused(pkg, bad, word):
    llb = pkg.llb
    _refused(llb, lambda: llb.kv_append(_kv(llb), _append(llb, **bad)), word)


@pytest.mark.parametrize("bad,word", [
    (dict(rows=-1), "-1 rows"), (dict(heads=6), "6 heads on 4"), (dict(heads=260), "260 heads"), (dict(max_rows=0), "max_rows 0"), (dict(max_len=-1), "max_len -1"),
    (dict(window=-1), "window -1"), (dict(window=8, sinks=-1), "sinks -1"), (dict(sinks=4), "without a window"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(el_out=1), "el_out 1"), (dict(q=0), "multiples of 16"), (dict(out=P), "out is q"), (dict(out=P + 8), "multiples of 16"), (dict(q_stride=1016), "q_stride 1016"),
    (dict(q_stride=1028), "q_stride 1028"), (dict(out_stride=1000), "out_stride 1000"), (dict(row_start=P + 2), "row_start"), (dict(w_in=P), "w_in without w_out"),
    (dict(w_out=P, w_stride=499), "w_stride 499"), (dict(w_out=P + 2, w_stride=500), "weights are f32"), (dict(w_out=P, w_stride=500, max_rows=33), "weights of 33 rows")])
def test_attention_that_is_refused(pkg, bad, word):
    llb = pkg.llb
    _refused(llb, lambda: llb.kv_attn(_kv(llb), _attn(llb, **bad)), word)
    _refused(llb, lambda: llb.kv_attn_ws(_kv(llb), _attn(llb, **bad)), word)


def test_attention_without_its_workspace(pkg):
    llb = pkg.llb
    kv, a = _kv(llb), _attn(llb, w_out=P, w_stride=500)
    need = llb.kv_attn_ws(kv, a)
    assert need >= 5 * 8 * 4
    for bad in (dict(ws=0), dict(ws=P + 8), dict(ws_bytes=need - 1)):
        _refused(llb, lambda: llb.kv_attn(kv, _attn(llb, **{**dict(w_out=P, w_stride=500), **bad})), "workspace")


@pytest.mark.parametrize("bad,word", [
    (dict(budget=0), "budget 0"), (dict(sinks=-1), "-1 first"), (dict(recent=-1), "-1 last"), (dict(sinks=50, recent=51), "50 first and 51"), (dict(max_len=-1), "max_len"),
    (dict(w=0), "weights of"), (dict(w_stride=499), "weights of 499"), (dict(w_out=P), "w_out"), (dict(w_out_stride=99), "w_out"), (dict(kept_stride=99), "kept"),
    (dict(kept=P + 2), "kept"), (dict(budget=600, w_out_stride=500, kept_stride=500, max_len=500, sinks=2 ** 31 - 1, recent=2 ** 31 - 1), "budget 600")])
def test_evictions_that_are_refused(pkg, bad, word):
    llb = pkg.llb
    _refused(llb, lambda: llb.kv_evict(_kv(llb), _kv(llb, table=P + 64, lens=P + 64), _evict(llb, **bad)), word)
    _refused(llb, lambda: llb.kv_evict_ws(_kv(llb), _evict(llb, **bad)), word)


@pytest.mark.parametrize("bad,word", [
    (dict(el=1), "another type"), (dict(kv_heads=2), "another type"), (dict(head_dim=64), "another type"), (dict(seqs=2), "another type"), (dict(table=P), "of its own"),
    (dict(lens=P), "of its own"), (dict(table_stride=3), "96 slots")])
def test_destinations_that_are_refused(pkg, bad, word):
    llb = pkg.llb
    _refused(llb, lambda: llb.kv_evict(_kv(llb), _kv(llb, **{**dict(table=P + 64, lens=P + 64), **bad}), _evict(llb)), word)


def test_eviction_without_its_workspace(pkg):
    llb = pkg.llb
    kv, e = _kv(llb), _evict(llb, kept=0)
    need = llb.kv_evict_ws(kv, e)
    assert need >= 3 * 4 * 100 * 4
    for bad in (dict(ws=0), dict(ws=P + 8), dict(ws_bytes=need - 1)):
        _refused(llb, lambda: llb.kv_evict(kv, _kv(llb, table=P + 64, lens=P + 64), _evict(llb, kept=0, **bad)), "workspace")


def test_calls_that_are_fine_reach_the_library_that_has_no_device(pkg):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    llb = pkg.llb
    for call in (lambda: llb.kv_append(_kv(llb), _append(llb)), lambda: llb.kv_attn(_kv(llb), _attn(llb)),
                 lambda: llb.kv_evict(_kv(llb), _kv(llb, table=P + 64, lens=P + 64), _evict(llb)), lambda: llb.kv_errors()):
        _refused(llb, call, "llb_b200_init")
    assert llb.kv_attn_ws(_kv(llb), _attn(llb)) > 0 and llb.kv_evict_ws(_kv(llb), _evict(llb)) > 0
