"""The paged key-value cache's barriers, workspaces and refusals at the ends of their ranges, without a GPU."""
import ctypes as C

import pytest

from test_gemm3_barriers_cpu import ARRIVE, WAIT, check


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
    return [L.llb_b200_pf_bar_count(3, hd, 0, b) for b in range(35)]


@pytest.mark.parametrize("form", range(8))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_no_wait_of_the_prompt_kernel_takes_one_phase_for_another(pkg, hd, form):
    L = pkg.llb.lib()
    for n in range(1, 40):
        t = _traces(L, hd, form, n)
        assert len(t) == (7 if hd == 256 else 12)
        assert check(t, _counts(L, hd)) is None, n


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_last_products_phase_may_not_pass_before_the_one_before_was_seen(pkg, hd):
    """A softmax warp that hands its last probabilities over before it has seen the product in front of them done could meet both products' phases complete."""
    L = pkg.llb.lib()
    for n in (2, 5, 8):
        t = _traces(L, hd, 0, n)
        for ops in t[:4]:
            i = max(k for k, op in enumerate(ops) if op[0] == ARRIVE)
            assert ops[i - 1] == (WAIT, 32, n - 2)
            ops[i - 1], ops[i] = ops[i], ops[i - 1]
        assert "phase" in check(t, _counts(L, hd))


def test_what_a_block_that_gave_up_did_not_note_is_not_followed(pkg):
    """The join takes its parts' numbers from the workspace; where a wait ran out those may be anything."""
    parts = pkg.llb.lib().llb_b200_kv_join_parts
    assert [parts(0, 0), parts(3, 3), parts(3, 9), parts(0, 147)] == [1, 1, 7, 148]
    for first, last in ((-1, -1), (-1, 5), (0, 148), (148, 148), (5, 4), (0, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, -2 ** 31), (1 << 20, 1 << 20)):
        assert parts(first, last) == 0, (first, last)
