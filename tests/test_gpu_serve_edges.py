"""The serving operators on calls at the edge of what the header allows (include/imi_cuda.h), each way of the attention among
them, against their restatement in 64 bits (tests/serve_plain.py)."""
import numpy as np
import pytest

import nunchi_b200 as nb
from test_gpu_serve_ops import FILTERS, I32, attn_case, dev, run_attn, run_sample, scores, torch

pytestmark = pytest.mark.gpu

# rows of 2 kv heads with 4 query heads each: few query rows (registers), one tile of them, several tiles (tensor cores)
ROWS = [3, 9, 40, 130]


def lengths(rows, unused=()):
    return [-1 if i in unused else (7 * i) % 50 for i in range(rows)]


# ------------------------------------------------------------------------------------------------------- the scale
@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.25])
def test_attn_scale_zero_and_negative(rows, dt, d, scale):
    """Scale 0: equal weights, with a ragged end of the prompt, a window and a missing page as well; a negative scale turns the
    scores around."""
    c = attn_case(rows, 2, 4, d, dt, 16, 1400, lengths(rows), seed=rows)
    run_attn(c, scale=scale)
    run_attn(c, scale=scale, window=1000)
    c["prefix"][33] = -1
    run_attn(c, scale=scale, status_want=1)
    run_attn(attn_case(rows, 2, 4, d, dt, 16, 1408, lengths(rows), seed=rows), scale=scale)


# ------------------------------------------------------------------------------------------ NaN and infinite scores
@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("rows", ROWS)
def test_attn_a_visible_key_that_is_not_a_number_shows(rows, dt, d):
    """A NaN in K, or an infinite score, at a position that a row sees makes the row NaN, wherever in a tile it lies; below the
    rows' windows it changes nothing."""
    c = attn_case(rows, 2, 4, d, dt, 16, 1400, [3] * rows, seed=d)
    c["q"].abs_().add_(0.1)                                     # so that an infinite K is an infinite score
    out, lse = torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:2], device="cuda")
    work = nb.prefix_attn_work(c["q"], c["k"], 1400, c["table"])
    for bad in (float("nan"), float("inf")):
        for pos in [*range(128, 160), 0, 1399]:
            page, at = int(c["prefix"][pos // 16]), pos % 16
            was = c["k"][page, :, at].clone()
            c["k"][page, :, at] = bad
            call = lambda window: nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], 1400, c["table"], c["length"], out=out,  # noqa: E731
                                                 lse=lse, work=work, window=window)
            call(0)
            assert out.isnan().all() and lse.isnan().all(), (bad, pos)
            if pos in (134, 153):
                run_attn(c, window=1100)
            c["k"][page, :, at] = was
    run_attn(c)


@pytest.mark.parametrize("rows", ROWS)
def test_attn_a_position_below_a_row_s_window_weighs_nothing(rows):
    """Very large values in V at positions that one row sees and the others' windows have passed."""
    own = [0] + [30] * (rows - 1)
    c = attn_case(rows, 2, 4, 64, "bf16", 16, 1500, own, seed=rows, spread=4.0)
    for pos in range(1302, 1318):                               # row 0 sees from 1300 on, the others from 1330
        c["v"][int(c["prefix"][pos // 16]), :, pos % 16] = 1e37   # row 0's sum of 16 stays finite
    run_attn(c, window=200)


# ---------------------------------------------------------------------------- windows, unused rows, what nobody sees
def poison(c, low):
    """NaN in K and V at the prompt's positions below `low`."""
    for x in (c["k"], c["v"]):
        for p in range(0, low, 16):
            x[int(c["prefix"][p // 16]), :, :min(16, low - p)] = float("nan")


WINDOWS = [(3000, 10), (3000, 130), (3000, 500), (3000, 2990), (2944, 100), (2944, 1024), (140, 60), (3000, 1)]


@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("prefix,window", WINDOWS)
def test_attn_unused_rows_see_nothing(rows, dt, d, prefix, window):
    """Rows that are not in use do not make the others read, under a window, what lies in front of all windows."""
    own = lengths(rows, unused={1, rows - 1})
    c = attn_case(rows, 2, 4, d, dt, 16, prefix, own, seed=window)
    poison(c, (prefix + min(x for x in own if x >= 0) - window) // 128 * 128)
    run_attn(c, window=window)


def test_attn_no_row_in_use():
    for rows in ROWS:
        c = attn_case(rows, 2, 4, 64, "f16", 16, 1500, [5] * rows)
        c["length"].fill_(-1)
        run_attn(c)
        run_attn(c, window=100)


@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("prefix,window", WINDOWS)
def test_attn_what_no_window_includes_may_be_anything(rows, dt, d, prefix, window):
    own = lengths(rows)
    c = attn_case(rows, 2, 4, d, dt, 16, prefix, own, seed=window)
    low = prefix + min(own) - window
    assert low > 0
    poison(c, low)
    run_attn(c, window=window)


@pytest.mark.parametrize("window", [300, 3000, 11990])
def test_attn_windows_on_a_long_prompt_in_many_parts(window):
    """Parts of a prompt that begin below, in and behind the tile in which the lowest window begins, several to a CTA."""
    for rows, kv in ((34, 3), (70, 1), (9, 5)):
        own = lengths(rows, unused={0, 2})
        c = attn_case(rows, kv, 4, 64, "f16", 16, 12000, own, seed=rows)
        poison(c, 12000 + min(x for x in own if x >= 0) - window)
        run_attn(c, window=window)


# -------------------------------------------------------------------------------------------------------- page_map
@pytest.mark.parametrize("n,cap,steps", [(384, 610000, 60), (4096, 40000, 25), (1, 2100, 200)])
def test_page_map_in_place_step_after_step(n, cap, steps):
    """Lengths and the free count in place, over many CTAs, one step behind the other without a wait: every step takes its
    pages from where the one before left the list."""
    rng = np.random.default_rng(n)
    page, n_pages = 16, 16000 if n > 1 else 300
    add = rng.integers(0, 2 if n > 1000 else 9, n)
    width = -(-int(add.max()) * steps // page) + 1
    order = rng.permutation(n_pages)
    held, nf, free, a = dev(np.zeros(n), I32), dev([n_pages], I32), dev(order, I32), dev(add, I32)
    table = torch.full((n, width), -1, dtype=I32, device="cuda")
    start, slots, pos, status = (torch.zeros(k, dtype=I32, device="cuda") for k in (n + 1, cap, cap, 2))
    for _ in range(steps):
        nb.page_map(held, a, table, free, nf, page=page, n_pages=n_pages, start=start, length=held, slots=slots, pos=pos, n_free_out=nf,
                    status=status)
    want, left = np.full((n, width), -1), n_pages
    for k in range(steps):
        for i in range(n):
            for c in range(-(-add[i] * k // page), -(-add[i] * (k + 1) // page)):
                left -= 1
                want[i, c] = order[left]
    assert status.tolist() == [0, 0] and int(nf) == left
    assert np.array_equal(held.cpu().numpy(), add * steps) and np.array_equal(table.cpu().numpy(), want)
    p = np.concatenate([np.arange(x * (steps - 1), x * steps) for x in add])
    i = np.repeat(np.arange(n), add)
    assert np.array_equal(pos.cpu().numpy()[:p.size], p) and (slots.cpu().numpy()[p.size:] == -1).all()
    assert np.array_equal(slots.cpu().numpy()[:p.size], want[i, p // page] * page + p % page)


# ---------------------------------------------------------------------------------------------------------- sample
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 13, 50])
@pytest.mark.parametrize("vocab", [2049, 4097, 8195, 16385, 24000, 50257, 57345, 65537, 100277, 131071])
def test_sample_rows_that_clusters_share_unevenly(vocab, n, dt):
    """Rows just above what a number of CTAs' parts hold, and others that do not divide: the same words at every cluster size; the
    last word of the row, and the words at the CTAs' ends, are drawn too."""
    x = scores(n, vocab, dt, vocab + n)
    rng = np.random.default_rng(vocab)
    for f in (1, 2, 4, 7, 8, 9, 11):
        run_sample(x, rng.random(n), **FILTERS[f])
    y = torch.full((n, vocab), -float("inf"), device="cuda")
    ends = [e for c in (1, 2, 4, 8) for r in range(1, c + 1) for e in (r * -(-vocab // c // 4) * 4, r * -(-vocab // c)) for e in (e - 1, e, e + 1)]
    ends = sorted({e for e in ends + [0, vocab - 1] if 0 <= e < vocab})
    y[:, ends] = torch.linspace(0, 1, len(ends), device="cuda")
    for u in (0.0, 0.37, 0.9999999):
        run_sample(y, u)
        run_sample(y, u, k=max(1, len(ends) - 3), p=0.9)
