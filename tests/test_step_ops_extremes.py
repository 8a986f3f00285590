"""Steps whose groups share more keys than there are."""
import numpy as np
import pytest

from test_shared_prefix import Call, Case
from test_step_ops import BAD_LENGTH, NO_BLOCKS, run_tables, same, tables_case, tables_oracle

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
