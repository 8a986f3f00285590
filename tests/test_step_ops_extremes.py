"""Steps whose groups share more keys than there are, and the forms of the q/k norm and logits kernels that large calls take."""
import numpy as np
import pytest

from test_shared_prefix import Call, Case
from test_step_ops import (BAD_LENGTH, NO_BLOCKS, LogitCase, QkCase, check_logits, check_qk, run_tables, same, tables_case,
                           tables_oracle)

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("n,extra,carry", [(40, 7, False), (40, 600, False), (300, 7, True), (1500, 3, False), (1500, 5000, True), (4097, 0, False)])
def test_groups_that_share_more_than_a_row_of_the_tables(torch_mod, dev, n, extra, carry):
    """Attention would read past the row, at the last sequence past the array: refused like any bad length. As many as fill the row are taken."""
    case = list(tables_case(50 + n, n, 60, 3, 16, 0, extra=extra, waits=0.1))
    stride = case[5].shape[1]
    case[3] = [(0, 2), (n - 3, 3), (n, 0)]
    case[2][n - 3:] = stride * 16
    same(run_tables(torch_mod, dev, *case, carry=carry), tables_oracle(*case))
    want = {k: v for k, v in tables_oracle(*case[:7], 0).items() if k in ("tables", "row_off", "last_row", "table_off", "groups")}
    for s, keys in ((n - 3, stride * 16 + 1), (n - 1, stride * 16 + 1), (n - 3, 1 << 30), (0, 2 ** 31 - 1)):
        case[2][s] = keys
        got = run_tables(torch_mod, dev, *case, carry=carry)
        same(got, want)
        assert (got["slot"] == -1).all() and (got["meta"][:, 1:] == 0).all() and got["totals"].tolist() == [0, 0, len(case[6]), BAD_LENGTH]
    assert run_tables(torch_mod, dev, *case[:6], case[6][:1], case[7])["totals"][3] == NO_BLOCKS  # what else is wrong comes first


@gpu
@pytest.mark.parametrize("bs", [12, 16, 32])
@pytest.mark.parametrize("members,shared,D", [(3, 500, 64), (2, 300, 16), (9, 640, 64), (20, 640, 128), (3, 2000, 128)])
def test_entries_without_a_block_lead_into_the_pools(torch_mod, dev, members, shared, D, bs):
    """A group's table whose last entries are negative gives what block 0 gives there; members' own tables as well."""
    torch = torch_mod
    case = Case([(members, shared)], [70, 5], 8, 2, D, bs=bs, seed=members + D)
    used = np.array(case.tables)
    held = shared // bs // 2
    ends = [held + 1] + [m[2] + shared // bs for m in case.meta]  # from here on, up to the table's end or a few entries
    stops = [-(-shared // bs)] + [m[2] + -(-m[1] // bs) for m in case.meta]
    for value in (0, -1, -2 ** 31):
        tables = used.copy()
        for lo, hi in zip(ends, stops):
            tables[lo:hi] = value
        case.tables = tables.tolist()
        out = Call(torch, dev, case)().clone()
        torch.cuda.synchronize()
        if value == 0:
            want = out
        assert torch.equal(out, want) and bool(torch.isfinite(out).all())


@gpu
@pytest.mark.parametrize("T,heads,kv_heads,D", [(2101, 9, 3, 64), (1900, 32, 4, 64), (2503, 20, 5, 32), (1777, 32, 8, 128), (1003, 7, 3, 128), (701, 4, 2, 256),
                                               (402, 3, 2, 512), (4999, 5, 2, 16)])
@pytest.mark.parametrize("bias,scale", [(False, False), (True, False), (False, True)])
def test_qk_norm_two_sets_of_heads_a_wave(torch_mod, dev, T, heads, kv_heads, D, bias, scale):
    """One plane of many rows, with a last set of heads that is not whole, and idle rows."""
    assert T * (heads + 2 * kv_heads) * max(4, D // 8) >= 150000
    check_qk(torch_mod, dev, QkCase(T, heads, kv_heads, D, seed=T, bias=bias, scale=scale, idle=(0, 5, T // 2, T - 1)))


@gpu
@pytest.mark.parametrize("out_ld", [9001, 9003, 9004])
@pytest.mark.parametrize("biases", [0, 7])
@pytest.mark.parametrize("rows,history", [(20, 0), (20, 60), (20, 4500), (65, 0), (65, 60), (110, 4500)])
def test_logits_forms(torch_mod, dev, rows, history, biases, out_ld):
    """One and two loads a thread, 256 and 512 threads (histories over 4096), with and without biases, rows that lie alike to 16 bytes or not."""
    case = LogitCase(rows, 9001, history, biases, masks=3, seed=rows + history, ld=9004 if out_ld == 9004 else None)
    check_logits(torch_mod, dev, case, out_ld=out_ld)
    check_logits(torch_mod, dev, case, out_ld=out_ld, shift=1)
    case.mask_of[:] = -1  # (masks that no row uses)
    check_logits(torch_mod, dev, case, out_ld=out_ld, shift=3, next_=False)
