"""The largest sizes that the serving operators take: what their 32-bit counts of positions and steps would not hold is refused
on the host. No GPU needed (the pointers are never followed)."""
import pytest

import nunchi_b200 as nb
from test_serve_ops_cabi import ATTN, call


@pytest.mark.parametrize("bad", [
    # the prompt, a table row, both together
    dict(prefix_len=2 ** 30), dict(width=2 ** 24, table_stride=2 ** 24), dict(width=2 ** 22, table_stride=2 ** 22, page=256),
    dict(prefix_len=2 ** 29, width=2 ** 23, table_stride=2 ** 23),
    # all rows' tables: 4,096 x 2^23 positions are 2^31 steps of 16
    dict(rows=4096, width=2 ** 17, table_stride=2 ** 17), dict(rows=4096, width=2 ** 15, table_stride=2 ** 15, page=256),
    dict(rows=33, width=2 ** 24 - 20, table_stride=2 ** 24)])
def test_prefix_attn_refuses_more_positions_than_it_counts(bad):
    st, msg = call("prefix_attn", nb._PREFIX_ATTN, ATTN, **{**bad, "work_bytes": 1 << 40})
    assert st == 1 and "unsupported shape" in msg
    a = {**ATTN, **bad}
    assert nb.lib().imi_cuda_prefix_attn_work(a["rows"], 32, 8, 64, a["prefix_len"], a["width"], a["page"]) == 0


@pytest.mark.parametrize("rows,prefix,width,page", [(32, 5, 2 ** 24 - 2, 64), (1, 2 ** 30 - 16, 0, 16), (4096, 10 ** 6, 2 ** 16, 64),
                                                    (2047, 2 ** 29, 2 ** 16, 256)])
def test_prefix_attn_takes_sizes_below_the_limits(rows, prefix, width, page):
    a = {**ATTN, "rows": rows, "prefix_len": prefix, "width": width, "table_stride": width, "page": page, "work_bytes": 1 << 50}
    st, msg = call("prefix_attn", nb._PREFIX_ATTN, a)
    assert "unsupported shape" not in msg
    assert nb.lib().imi_cuda_prefix_attn_work(rows, 32, 8, 64, prefix, width, page) > 0


def test_prefix_attn_refuses_a_scale_that_overflows_in_powers_of_two():
    """The kernels work in powers of two: what is finite has to stay so times log2(e) = 1.4427."""
    for scale in (3e38, -2.4e38):
        st, msg = call("prefix_attn", nb._PREFIX_ATTN, ATTN, scale=scale)
        assert st == 1 and "scale" in msg
    for scale in (2.3e38, -2.3e38, 0.0, 1e-45):
        assert "scale" not in call("prefix_attn", nb._PREFIX_ATTN, ATTN, scale=scale)[1]
