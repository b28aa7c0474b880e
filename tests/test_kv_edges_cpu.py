"""The paged key-value cache's barriers, workspaces and refusals at the ends of their ranges, without a GPU."""
import ctypes as C

import pytest

from test_gemm3_barriers_cpu import WAIT, check


def _traces(L, hd, form, n):
    out = []
    while True:
        k = L.llb_b200_pf_trace(3, hd, form, 1, n, len(out), None, 0)
        if k < 0:
            return out
        buf = (C.c_int * max(1, 3 * k))()
        assert L.llb_b200_pf_trace(3, hd, form, 1, n, len(out), buf, 3 * k) == k
        out.append([tuple(buf[3 * i:3 * i + 3]) for i in range(k)])


def _counts(L, hd):
    return [L.llb_b200_pf_bar_count(3, hd, 0, b) for b in range(37)]


@pytest.mark.parametrize("form", range(8))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_no_wait_of_the_prompt_kernel_takes_one_phase_for_another(pkg, hd, form):
    L = pkg.llb.lib()
    for n in range(1, 40):
        t = _traces(L, hd, form, n)
        assert len(t) == (7 if hd == 256 else 12)
        assert check(t, _counts(L, hd)) is None, n


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_last_two_products_phases_could_both_pass(pkg, hd):
    """What the last product's own barrier is for: with the others', a softmax warp that has handed its last probabilities over could meet both phases complete."""
    L = pkg.llb.lib()
    for n in (2, 5, 8):
        t = _traces(L, hd, 0, n)
        for ops in t:
            for k, (kind, b, v) in enumerate(list(ops)):
                if b in (35, 36):
                    ops[k] = (kind, b - 3, n - 1 if kind == WAIT else v)
        assert t[0][-2:] == [(WAIT, 32, n - 2), (WAIT, 32, n - 1)]
        assert "before" in check(t, _counts(L, hd))


def test_what_a_block_that_gave_up_did_not_note_is_not_followed(pkg):
    """The join takes its parts' numbers from the workspace; where a wait ran out those may be anything."""
    parts = pkg.llb.lib().llb_b200_kv_join_parts
    assert [parts(0, 0), parts(3, 3), parts(3, 9), parts(0, 147)] == [1, 1, 7, 148]
    for first, last in ((-1, -1), (-1, 5), (0, 148), (148, 148), (5, 4), (0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, -2 ** 31), (1 << 20, 1 << 20)):
        assert parts(first, last) == 0, (first, last)


def _kv(llb, **kw):
    a = dict(el=llb.EL["bf16"], kv_heads=1, head_dim=128, page=32, n_pages=64, seqs=1, table_stride=16, k=1 << 20, v=1 << 20, table=1 << 20, lens=1 << 20)
    a.update(kw)
    return llb.Kv(**a)


def _attn(llb, max_len, **kw):
    a = dict(rows=1, max_rows=1, max_len=max_len, heads=1, scale=0.0, el_out=llb.EL["bf16"], q=1 << 20, out=2 << 20, q_stride=128, out_stride=128, row_start=1 << 20)
    a.update(kw)
    return llb.KvAttn(**a)


@pytest.mark.parametrize("max_len", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 16, 2 ** 31 - 300, 1 << 30, 513])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("rows", [1, 600])
def test_a_workspace_goes_by_the_slots_that_the_table_holds(pkg, rows, weights, max_len):
    """16 pages of 32 slots: no sequence has more than 512, whatever the call's bound is."""
    llb = pkg.llb
    if weights and rows > 64:
        rows = 64
    kw = dict(rows=rows, max_rows=rows, **(dict(w_out=1 << 20, w_stride=2 ** 31 - 1) if weights else {}))
    want = llb.kv_attn_ws(_kv(llb), _attn(llb, 512, **kw))
    assert not weights or want >= rows * 512 * 4
    assert llb.kv_attn_ws(_kv(llb), _attn(llb, max_len, **kw)) == want


@pytest.mark.parametrize("max_len", [2 ** 31 - 1, 2 ** 31 - 2, 513])
def test_an_evictions_workspace_goes_by_the_slots_that_the_table_holds(pkg, max_len):
    llb = pkg.llb
    e = dict(budget=2 ** 31 - 1, w=1 << 20, w_stride=2 ** 31 - 1)
    want = llb.kv_evict_ws(_kv(llb, seqs=3), llb.KvEvict(max_len=512, **e))
    assert want >= 3 * 512 * 4
    assert llb.kv_evict_ws(_kv(llb, seqs=3), llb.KvEvict(max_len=max_len, **e)) == want


@pytest.mark.parametrize("max_len", [2 ** 31 - 1, 2 ** 31 - 256, 2 ** 31 - 4095])
def test_no_sequence_has_more_slots_than_are_counted(pkg, max_len):
    """Tables of more than 2^31 slots (pages may be shared): lengths end where sums of slots and block sizes still fit 32 bits."""
    llb = pkg.llb
    kw = dict(w_out=1 << 20, w_stride=2 ** 31 - 1)
    kv = _kv(llb, page=128, table_stride=1 << 25)
    want = llb.kv_attn_ws(kv, _attn(llb, 2 ** 31 - 4096, **kw))
    assert want > (2 ** 31 - 4096) * 4
    assert llb.kv_attn_ws(kv, _attn(llb, max_len, **kw)) == want
