"""The serving operators (imi_cuda_page_map / page_write / prefix_attn / sample) against their restatement in 64 bits
(tests/serve_plain.py): sizes and masks where they can go wrong, captured graphs, other streams, and one decode loop of all
of them together."""
import numpy as np
import pytest

import nunchi_b200 as nb
import serve_plain as plain

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
I32 = torch.int32
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}   # a rounding's relative error at most


def dev(x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x)).to("cuda", dtype)


# ---------------------------------------------------------------------------------------------------------- page_map
def map_case(n, page, held_max, add_max, seed, pad=0, spare=3):
    rng = np.random.default_rng(seed)
    held, add = rng.integers(0, held_max + 1, n), rng.integers(0, add_max + 1, n)
    held[rng.random(n) < 0.2] = 0
    if pad:
        held[-pad:] = -1
    width = -(-(held_max + add_max) // page) + 1
    n_pages = n * width + spare
    order = rng.permutation(n_pages)
    table, used = np.full((n, width), -1), 0
    for i in range(n):
        c = -(-max(held[i], 0) // page)
        table[i, :c] = order[used:used + c]
        used += c
    free = np.concatenate((order[used:], np.full(4, -7)))      # the list has room behind its end
    return held, add, table, free, n_pages - used, n_pages


def run_map(held, add, table, free, n_free, page, n_pages, pos0=0, cap=None, in_place=False):
    n = len(held)
    cap = int(np.maximum(add, 0).sum()) + 5 if cap is None else cap
    h, a, t, f, nf = (dev(x, I32) for x in (held, add, table, free, [n_free]))
    mk = lambda k: torch.full((k,), 99, dtype=I32, device="cuda")  # noqa: E731
    start, length, slots, pos, out, status = mk(n + 1), h if in_place else mk(n), mk(cap), mk(cap), nf if in_place else mk(1), mk(2)
    status.zero_()
    nb.page_map(h, a, t, f, nf, page=page, n_pages=n_pages, start=start, length=length, slots=slots, pos=pos, n_free_out=out,
                status=status, pos0=pos0)
    want = plain.page_map(held, add, table, free, n_free, page, n_pages, pos0, cap)
    got = [x.cpu().numpy() for x in (t, start, length, slots, pos, out, status)]
    for g, w, name in zip(got, want, ("table", "start", "length", "slots", "pos", "n_free_out")):
        assert np.array_equal(g, np.atleast_1d(w)), name
    assert got[6][0] == want[6] and got[6][1] == 0
    return got


@pytest.mark.parametrize("n,page,held_max,add_max,pad", [
    (1, 16, 0, 1, 0), (1, 256, 700, 3, 0), (3, 16, 40, 50, 1), (64, 64, 1300, 1, 0), (64, 64, 1300, 1, 7), (511, 32, 100, 9, 2),
    (513, 16, 33, 40, 0), (4096, 16, 64, 2, 100), (40, 128, 300, 2500, 3), (7, 16, 5, 20011, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_map(n, page, held_max, add_max, pad, in_place):
    held, add, table, free, nf, n_pages = map_case(n, page, held_max, add_max, n + page, pad)
    run_map(held, add, table, free, nf, page, n_pages, pos0=17, in_place=in_place)


def test_page_map_nothing_to_add_and_empty_pool():
    held, add, table, free, nf, n_pages = map_case(9, 16, 60, 5, 3)
    run_map(held, add * 0, table, free, nf, 16, n_pages, cap=0)
    run_map(held, add * 0, table, free, 0, 16, n_pages)
    run_map(held, add * 0, table, free[:0], 0, 16, n_pages)


@pytest.mark.parametrize("what", ["pool", "count", "table", "cap", "negative", "huge", "page"])
@pytest.mark.parametrize("cap", [None, 30000])
def test_page_map_device_errors(what, cap):
    held, add, table, free, nf, n_pages = map_case(21, 16, 200, 90, 5, pad=1)
    need = int(sum(-(-(h + a) // 16) - -(-h // 16) for h, a in zip(held, add) if h >= 0))
    if what == "pool":
        nf = need - 1
    if what == "count":
        nf = free.size + 1
    if what == "table":
        add[4] = table.shape[1] * 16 - held[4] + 1
        free, nf, n_pages = np.arange(4000), 4000, 4000
        cap = 30000
    if what == "cap":
        cap = int(add[:-1].sum()) - 1
    if what == "negative":
        add[2] = -1
    if what == "huge":
        held[3] = add[5] = 2 ** 31 - 1
        cap = 30000
    if what == "page":
        free[nf - 2] = n_pages
        table[1, 0] = -3
        held[1], add[1] = 5, 4
    got = run_map(held, add, table, free, nf, 16, n_pages, cap=cap)
    assert got[6][0] == {"pool": 4, "count": 4, "table": 2, "cap": 3, "negative": 5, "huge": got[6][0], "page": 1}[what]
    assert got[6][0] != 0


def test_page_map_steps_never_share_a_page():
    rng = np.random.default_rng(8)
    n, page, width, n_pages = 33, 16, 12, 300
    held, nf = torch.zeros(n, dtype=I32, device="cuda"), dev([n_pages], I32)
    table = torch.full((n, width), -1, dtype=I32, device="cuda")
    free = dev(rng.permutation(n_pages), I32)
    start, slots, pos = (torch.zeros(k, dtype=I32, device="cuda") for k in (n + 1, 700, 700))
    status = torch.zeros(2, dtype=I32, device="cuda")
    seen = set()
    for step in range(9):
        add = dev(rng.integers(0, 21, n), I32)
        nb.page_map(held, add, table, free, nf, page=page, n_pages=n_pages, start=start, length=held, slots=slots, pos=pos,
                    n_free_out=nf, status=status)
        s = slots.cpu().numpy()
        s = s[s >= 0].tolist()
        assert len(s) == int(add.sum()) and len(set(s)) == len(s) and not seen & set(s)
        seen |= set(s)
    assert status.tolist() == [0, 0]
    assert n_pages - int(nf) == int(((held + page - 1) // page).sum())


# -------------------------------------------------------------------------------------------------------- page_write
@pytest.mark.parametrize("rows,kv,d,src,dst,page", [
    (1, 1, 8, "f32", "f16", 16), (5, 3, 64, "f32", "bf16", 32), (130, 8, 64, "f16", "f16", 64), (33, 2, 128, "bf16", "bf16", 16),
    (1000, 5, 72, "f32", "f16", 256), (17, 1, 256, "bf16", "bf16", 128)])
@pytest.mark.parametrize("shift", [0, 1])
def test_page_write(rows, kv, d, src, dst, page, shift):
    rng = np.random.default_rng(rows + d)
    n_pages = rows // page + 3
    big = dev(rng.standard_normal((rows, 2 * kv * d + 24 + shift)) * 3, DT[src])
    if src == "f32":
        big[0, shift] = 1e30                                    # beyond fp16: infinity, as the type's rounding gives
    k, v = (big[:, o + shift:o + shift + kv * d].unflatten(1, (kv, d)) for o in (0, kv * d + 8))
    slots = rng.permutation(n_pages * page)[:rows]
    slots[rng.random(rows) < 0.2] = -1
    slots[rows // 2] = -(2 ** 31)
    pages = [dev(rng.standard_normal((n_pages, kv, page, d)), DT[dst]) for _ in range(2)]
    want = [p.clone() for p in pages]
    for x, w in ((k, want[0]), (v, want[1])):
        for r in np.flatnonzero(slots >= 0):
            w[slots[r] // page, :, slots[r] % page] = x[r].to(DT[dst])
    status = torch.zeros(1, dtype=I32, device="cuda")
    nb.page_write(k, v, dev(slots, I32), *pages, status=status)
    assert torch.equal(pages[0], want[0]) and torch.equal(pages[1], want[1]) and int(status) == 0


def test_page_write_slot_beyond_the_pages_and_no_rows():
    k = torch.randn((4, 2, 64), device="cuda").half()
    pages = [torch.zeros((3, 2, 16, 64), device="cuda", dtype=torch.float16) for _ in range(2)]
    status = torch.zeros(1, dtype=I32, device="cuda")
    nb.page_write(k, k, dev([48, 47, 2 ** 31 - 1, 0], I32), *pages, status=status)
    assert int(status) == 1
    assert torch.equal(pages[0][2, :, 15], k[1]) and torch.equal(pages[1][0, :, 0], k[3])
    assert int((pages[0] != 0).any(-1).sum()) == 4
    nb.page_write(k[:0], k[:0], dev([], I32), *pages)


# ------------------------------------------------------------------------------------------------------- prefix_attn
def attn_case(n, kv, g, d, dt, page, prefix, own, seed=0, spread=1.0, extra=3):
    """own: the rows' lengths. Everything no row sees is NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    pp, width = -(-prefix // page), max(1, -(-max(max(own), 1) // page))
    n_pages = pp + n * width + extra
    order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=I32)
    pages = [torch.full((n_pages, kv, page, d), float("nan"), device="cuda", dtype=DT[dt]) for _ in range(2)]
    pre, table = order[:pp].contiguous(), order[pp:pp + n * width].reshape(n, width).contiguous()
    for x in pages:
        fill = lambda ids, count: [x.index_put_(  # noqa: E731
            (ids[torch.arange(count, device="cuda") // page].long()[:, None], torch.arange(kv, device="cuda")[None],
             (torch.arange(count, device="cuda") % page)[:, None]), r(count, kv, d).to(x.dtype))]
        if prefix:
            fill(pre, prefix)
        for i, L in enumerate(own):
            if L > 0:
                fill(table[i], L)
    return {"q": (r(n, kv * g, d) * spread).to(DT[dt]), "k": pages[0], "v": pages[1], "prefix": pre, "prefix_len": prefix, "table": table,
            "length": dev(own, I32), "dt": dt}


def run_attn(c, window=0, scale=None, out_dtype=None, status_want=0, work=None, stream=None):
    q = c["q"]
    out_name = out_dtype or c["dt"]
    out, lse = torch.full(q.shape, 7.0, device="cuda", dtype=DT[out_name]), torch.full(q.shape[:2], 7.0, device="cuda")
    status = torch.zeros(1, dtype=I32, device="cuda")
    work = nb.prefix_attn_work(q, c["k"], c["prefix_len"], c["table"]) if work is None else work
    work.fill_(0xFF)                                            # NaN everywhere: nothing is expected in it
    nb.prefix_attn(q, c["k"], c["v"], c["prefix"], c["prefix_len"], c["table"], c["length"], out=out, lse=lse, work=work,
                   scale=scale, window=window, status=status, stream=stream)
    torch.cuda.synchronize()
    check_attn(c, out, lse, window, scale, out_name)
    assert int(status) == status_want
    return out, lse


def check_attn(c, out, lse, window, scale, out_name):
    d = c["q"].shape[-1]
    scale = d ** -0.5 if scale is None else scale
    h = lambda t: t.double().cpu().numpy()  # noqa: E731
    want = plain.attn(h(c["q"]), h(c["k"]), h(c["v"]), c["prefix"].cpu().numpy(), c["prefix_len"], c["table"].cpu().numpy(),
                      c["length"].cpu().numpy(), scale, window)
    got, gl = h(out), h(lse)
    e, eo = HALF[c["dt"]], HALF[out_name]
    for i, w in enumerate(want):
        if w is None:
            assert (got[i] == 7.0).all() and (gl[i] == 7.0).all(), i
            continue
        o, z, spread, reach, seen = w
        # a score: d products, exact in 32 bits, summed with an error of 2^-23 of the sum of their sizes each at most, and
        # the scale and the base's change (2^-22 of the score, itself at most scale * reach); a probability then is off by
        # that much, relatively, by the exponential's 2^-22 and by its rounding to the type (below 2^-14 fp16 steps by 2^-24
        # absolutely: 2^-25 of the largest for every position)
        ds = (abs(scale) * reach * (d * 2.0 ** -23 + 2.0 ** -22))[:, None]
        rel = 2 * ds + e + 2.0 ** -21 + seen * 2.0 ** -23
        tol = spread * rel + np.abs(o) * eo + (2.0 ** -25 if out_name == "f16" else 0)
        if c["dt"] == "f16":
            big = np.nanmax(np.abs(np.where(np.isfinite(h(c["v"])), h(c["v"]), 0)))
            tol = tol + seen * 2.0 ** -25 * big
        assert (np.abs(got[i] - o) <= tol).all(), (i, np.max(np.abs(got[i] - o) / tol))
        zt = ds[:, 0] + seen * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22 * np.abs(np.where(np.isfinite(z), z, 0))
        both = np.isneginf(z) & np.isneginf(gl[i])
        assert (both | (np.abs(gl[i] - z) <= zt)).all(), (i, gl[i], z)


@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("prefix,own", [
    (0, [0]), (0, [1]), (1, [0]), (1, [1]), (37, [5, 0, -1, 16]), (16, [15, 17]), (0, [0, 33, -1, 500]), (999, [25, 0, 24]),
    (1000, [40, -1, 0, 700]), (1025, [0, 0, 0]), (2500, [1, 3, 16, 17, 0, -1]), (0, [1500, 2, 0, 1023, 1024])])
def test_attn_lengths(dt, d, prefix, own):
    run_attn(attn_case(len(own), 2, 4, d, dt, 16, prefix, own, seed=prefix + d))


@pytest.mark.parametrize("kv,g", [(1, 1), (3, 2), (2, 3), (1, 5), (2, 7), (1, 8), (2, 9), (1, 16)])
@pytest.mark.parametrize("prefix,own", [(70, [9, 0, 31]), (1300, [100, 7, 0, 257, 64])])
def test_attn_heads(kv, g, prefix, own):
    run_attn(attn_case(len(own), kv, g, 64 if g % 2 else 128, "f16", 32, prefix, own, seed=g))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attn_pages(page):
    run_attn(attn_case(5, 2, 4, 64, "bf16", page, 1111, [300, 1, 0, 129, 257], seed=page))


@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 1200, 1201, 5000])
@pytest.mark.parametrize("prefix,own", [(90, [3, 0, 40, 90]), (1200, [0, 1, 100, 101, 99, 600, -1, 1300])])
def test_attn_window(window, prefix, own):
    run_attn(attn_case(len(own), 2, 4, 64, "f16", 16, prefix, own, seed=window), window=window)


@pytest.mark.parametrize("rows,prefix", [(1, 6000), (40, 3000), (70, 2100), (130, 1500)])
@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 128)])
def test_attn_batches(rows, prefix, dt, d):
    own = [(7 * i) % 50 for i in range(rows)]
    own[-1] = -1 if rows > 1 else 3
    run_attn(attn_case(rows, 2, 4, d, dt, 64, prefix, own, seed=rows))
    run_attn(attn_case(rows, 2, 4, d, dt, 64, prefix, own, seed=rows), window=1000)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("prefix", [50, 1400])
def test_attn_scales_and_output_types(out, prefix):
    c = attn_case(3, 2, 4, 64, "f16", 16, prefix, [20, 0, 333], spread=4.0)   # sharp rows: one position takes nearly all
    run_attn(c, out_dtype=out, scale=0.5)
    run_attn(c, out_dtype=out, scale=-0.25)
    run_attn(c, out_dtype=out, scale=0.0)


def test_attn_rising_scores():
    """Scores that rise along the prompt: every step raises the running maximum."""
    c = attn_case(48, 1, 4, 64, "f16", 16, 2048, [3] * 48)
    c["q"][:] = 1.0
    ramp = torch.arange(2048, device="cuda").float() / 1024
    c["k"][c["prefix"].long()] = ramp.reshape(-1, 1, 16, 1).half().expand(-1, 1, 16, 64)
    run_attn(c, scale=1.0)


def test_attn_strided_rows_and_wider_tables():
    c = attn_case(4, 2, 4, 64, "f16", 16, 1100, [3, 30, 0, 90])
    big = torch.zeros((4, 3 * 512), device="cuda", dtype=torch.float16)
    big[:, 512:1024] = c["q"].flatten(1)
    c["q"] = big[:, 512:1024].unflatten(1, (8, 64))
    wide = torch.full((6, 20), 10 ** 9, device="cuda", dtype=I32)
    wide[:4, :c["table"].shape[1]] = c["table"]
    c["table"] = wide[:4, :17]
    out = torch.full((4, 600), 7.0, device="cuda", dtype=torch.float16)
    view, lse = out[:, 8:520].unflatten(1, (8, 64)), torch.zeros((4, 8), device="cuda")
    nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], 1100, c["table"], c["length"], out=view, lse=lse,
                   work=nb.prefix_attn_work(c["q"], c["k"], 1100, c["table"]))
    check_attn(c, view, lse, 0, None, "f16")
    assert (out[:, :8] == 7.0).all() and (out[:, 520:] == 7.0).all()


@pytest.mark.parametrize("prefix", [60, 1500])
def test_attn_bad_pages_and_lengths(prefix):
    c = attn_case(3, 2, 4, 64, "f16", 16, prefix, [40, 33, 48])
    c["table"][1, 1] = c["k"].shape[0]
    c["table"][2, 0] = -1
    if prefix > 1000:
        c["prefix"][70] = 2 ** 31 - 1
    run_attn(c, status_want=1)
    c = attn_case(3, 2, 4, 64, "f16", 16, prefix, [40, 33, 48])
    c["length"][2] = 10 ** 9
    run_attn(c, status_want=2)


@pytest.mark.parametrize("dt,d", [("f16", 64), ("bf16", 128)])
def test_attn_bad_pages_of_a_prompt_for_many_rows(dt, d):
    c = attn_case(9, 2, 4, d, dt, 16, 700, [3, 0, 40, 1, 2, 5, 16, 17, 0])
    for j, bad in ((0, -1), (8, c["k"].shape[0]), (9, 2 ** 31 - 1), (43, -2 ** 31)):   # the first, two in a tile, the last
        c["prefix"][j] = bad
    run_attn(c, status_want=1)
    run_attn(c, status_want=1, window=500)


@pytest.mark.parametrize("prefix", [1, 15, 127, 128, 129, 255, 256, 257, 384, 1023])
@pytest.mark.parametrize("rows,g,d", [(5, 4, 64), (33, 4, 64), (90, 3, 64), (6, 3, 128), (70, 2, 128)])
def test_attn_tile_borders(prefix, rows, g, d):
    c = attn_case(rows, 1, g, d, "f16", 16, prefix, [300] + [i % 3 for i in range(rows - 1)])
    run_attn(c)
    run_attn(c, window=130)


def test_attn_long_prompt_in_many_parts():
    """A prompt of 90,001 positions whose parts are ended by the number of tiles a part holds (its pages repeat); the
    restatement on the device, in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows, kv, d, page, P = 18, 64, 64, 256, 90001
    pages = [torch.randn((7, kv, page, d), generator=gen, device="cuda").half() for _ in range(2)]
    prefix = torch.randint(0, 7, (-(-P // page),), generator=gen, device="cuda", dtype=I32)
    q = torch.randn((rows, kv, d), generator=gen, device="cuda").half()
    out, lse = torch.zeros_like(q), torch.zeros((rows, kv), device="cuda")
    table, length = torch.zeros((rows, 1), dtype=I32, device="cuda"), torch.zeros(rows, dtype=I32, device="cuda")
    nb.prefix_attn(q, *pages, prefix, P, table, length, out=out, lse=lse, work=nb.prefix_attn_work(q, pages[0], P, table))
    for h in range(kv):
        k, v = (p[prefix.long(), h].reshape(-1, d)[:P].double() for p in pages)
        x = q[:, h].double() @ k.T * d ** -0.5
        z = torch.logsumexp(x, 1)
        e = torch.exp(x - z[:, None])
        o, spread = e @ v, e @ v.abs()
        reach = (q[:, h].double().abs() @ k.abs().T).amax(1)
        ds = (d ** -0.5 * reach * (d * 2.0 ** -23 + 2.0 ** -22))[:, None]   # as in check_attn
        tol = spread * (2 * ds + HALF["f16"] + 2.0 ** -21 + P * 2.0 ** -23) + o.abs() * HALF["f16"] + 2.0 ** -25 + P * 2.0 ** -25 * v.abs().max()
        assert ((out[:, h].double() - o).abs() <= tol).all()
        assert ((lse[:, h].double() - z).abs() <= ds[:, 0] + P * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22 * z.abs()).all()


def test_attn_two_calls_at_once():
    """Two streams, each with its own workspace and outputs."""
    cases = [attn_case(40, 2, 4, 64, "f16", 16, 1500, [(13 * i) % 300 for i in range(40)], seed=s) for s in (1, 2)]
    want = [run_attn(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    works = [nb.prefix_attn_work(c["q"], c["k"], 1500, c["table"]) for c in cases]
    outs = [(torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:2], device="cuda")) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st, w, (o, l) in zip(cases, streams, works, outs):
            nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], 1500, c["table"], c["length"], out=o, lse=l, work=w, stream=st)
    torch.cuda.synchronize()
    for (o, l), (wo, wl) in zip(outs, want):
        assert torch.equal(o, wo) and torch.equal(l, wl)


@pytest.mark.parametrize("rows", [2, 7])
def test_attn_offsets_beyond_32_bits(rows):
    """A cache of 2^32 elements and more: the pages used lie at its start, across 2^31 and 2^32, and at its end."""
    kv, page, d = 8, 256, 64
    n_pages = 2 ** 32 // (kv * page * d) + 9
    pages = [torch.empty((n_pages, kv, page, d), device="cuda", dtype=torch.float16) for _ in range(2)]
    used = [0, 2 ** 31 // (kv * page * d) - 1, 2 ** 31 // (kv * page * d), n_pages // 2 + 7, 2 ** 32 // (kv * page * d), n_pages - 1]
    for p in pages:
        for u in used:
            p[u].normal_()
    small = {"q": torch.randn((rows, 32, 64), device="cuda").half(), "prefix": dev([5, 1, 2, 3], I32), "prefix_len": 1000,
             "table": dev(([[4, 0], [0, 4]] * rows)[:rows], I32), "length": dev(([300, 11] * rows)[:rows], I32), "dt": "f16",
             "k": pages[0][used].clone(), "v": pages[1][used].clone()}
    want = run_attn(small)
    at = dev(used, I32)
    big = dict(small, k=pages[0], v=pages[1], prefix=at[small["prefix"].long()], table=at[small["table"].long()])
    out, lse = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    nb.prefix_attn(big["q"], big["k"], big["v"], big["prefix"], 1000, big["table"], big["length"], out=out, lse=lse,
                   work=nb.prefix_attn_work(big["q"], big["k"], 1000, big["table"]))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    k = torch.randn((4, kv, d), device="cuda").half()
    nb.page_write(k, -k, dev([used[-1] * page + 255, used[3] * page, used[4] * page + 3, 5], I32), *pages)
    assert torch.equal(pages[0][used[-1], :, 255], k[0]) and torch.equal(pages[1][used[4], :, 3], -k[2])


def test_attn_same_call_gives_the_same_bits():
    c = attn_case(65, 2, 4, 64, "f16", 16, 1800, [(31 * i) % 400 for i in range(65)])
    a, b = run_attn(c), run_attn(c)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attn_captured_graphs_replay_with_new_lengths():
    """Two graphs of different calls, each with its own workspace, replayed in turn while the buffers change."""
    cases = [attn_case(20, 2, 4, 64, "f16", 16, 1500, [(13 * i) % 200 for i in range(20)], seed=s) for s in (1, 2)]
    graphs = []
    for c in cases:
        c["out"], c["lse"] = torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:2], device="cuda")
        c["work"] = nb.prefix_attn_work(c["q"], c["k"], 1500, c["table"])
        call = lambda c=c: nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], 1500, c["table"], c["length"], out=c["out"],  # noqa: E731
                                          lse=c["lse"], work=c["work"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    for shift in (0, 50):
        for c in cases:
            c["length"].sub_(shift).clamp_(min=0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c in cases:
            check_attn(c, c["out"], c["lse"], 0, None, "f16")


def test_operators_on_another_stream():
    c = attn_case(20, 2, 4, 64, "f16", 16, 1500, [(13 * i) % 200 for i in range(20)])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    run_attn(c, stream=st)
    x = torch.randn((5, 1003), device="cuda")
    u, ids = torch.rand(5, device="cuda"), torch.zeros(5, dtype=I32, device="cuda")
    st.wait_stream(torch.cuda.current_stream())
    nb.sample(x, u, ids=ids, stream=st.cuda_stream)
    st.synchronize()
    assert ids.tolist() == [plain.sample(r, v)[0] for r, v in zip(x.double().cpu().numpy(), u.double().cpu().numpy())]


# ------------------------------------------------------------------------------------------------------------ sample
def run_sample(x, u, t=None, k=None, p=None, m=None):
    """x: a device tensor [n][vocab]; the settings arrays or None."""
    n = x.shape[0]
    f = lambda v, d: None if v is None else dev(np.broadcast_to(v, n).copy(), d)  # noqa: E731
    ids, kept = (torch.full((n,), 99, dtype=I32, device="cuda") for _ in range(2))
    lp = torch.full((n,), 99.0, device="cuda")
    uu, tt, kk, pp, mm = f(u, torch.float32), f(t, torch.float32), f(k, I32), f(p, torch.float32), f(m, torch.float32)
    nb.sample(x, uu, temperature=tt, top_k=kk, top_p=pp, min_p=mm, ids=ids, logprob=lp, kept=kept)
    h = lambda v, d: np.full(n, d) if v is None else v.double().cpu().numpy()  # noqa: E731
    U, T, K, P, M, X = h(uu, 0), h(tt, 1.0), h(kk, 0), h(pp, 1.0), h(mm, 0.0), x.double().cpu().numpy()
    for i in range(n):
        want = plain.sample(X[i], U[i], T[i], int(K[i]), P[i], M[i])
        got = (int(ids[i]), float(lp[i]), int(kept[i]))
        assert (got[0], got[2]) == (want[0], want[2]), (i, got, want, U[i], T[i], K[i], P[i], M[i])
        # computed in 64 bits (the mass to 2^-44 per word) and rounded once to 32
        assert got[1] == want[1] or abs(got[1] - want[1]) <= 2.0 ** -24 * abs(want[1]) + X.shape[1] * 2.0 ** -44 + 1e-12, (i, got, want)
    return ids, lp, kept


def scores(n, vocab, dt, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((n, vocab), generator=g, device="cuda") * scale).to(DT[dt])


FILTERS = [dict(), dict(k=1), dict(k=50), dict(k=7, p=0.8), dict(p=0.9), dict(p=0.35, t=0.6), dict(m=0.05), dict(k=40, p=0.95, m=0.02, t=0.8),
           dict(p=0.999), dict(k=1500), dict(k=1500, p=0.97), dict(t=0.0), dict(k=300, m=0.3), dict(p=0.5, m=0.001, t=1.7)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 500, 1003, 4099, 40001, 97496])
@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_sample_filters(vocab, dt, f):
    x = scores(4, vocab, dt, vocab + f)
    run_sample(x, np.random.default_rng(f).random(4), **FILTERS[f])


@pytest.mark.parametrize("n,vocab", [(1, 97496), (40, 97496), (150, 20000), (300, 1003), (2, 262144)])
def test_sample_batches_with_settings_per_row(n, vocab):
    rng = np.random.default_rng(n)
    x = scores(n, vocab, "f32", n)
    run_sample(x, rng.random(n), t=rng.choice([0.0, 0.5, 1.0, 1.4], n), k=rng.choice([0, 1, 20, 3000, 10 ** 9, -4], n),
               p=rng.choice([0.0, 0.3, 0.95, 1.0, 1.5, np.nan], n), m=rng.choice([0.0, 0.1, 1.0, 2.0, -1.0, np.nan], n))


@pytest.mark.parametrize("vocab", [5, 1000, 30000])
def test_sample_ties(vocab):
    """Equal scores: kept and walked by id, borders in the middle of them; weights that are whole, so borders are exact."""
    x = torch.zeros((9, vocab), device="cuda")
    x[:, ::2] = -np.log(2.0)                                     # weights 1 and (about) 1/2
    u = np.linspace(0, 0.99999994, 9)
    run_sample(torch.zeros((9, vocab), device="cuda"), u)
    run_sample(torch.zeros((9, vocab), device="cuda"), u, k=max(1, vocab // 3))
    run_sample(torch.zeros((9, vocab), device="cuda"), u, p=0.5)
    run_sample(torch.zeros((9, vocab), device="cuda"), u, m=1.0)
    run_sample(x, u, k=max(1, vocab - vocab // 4))
    run_sample(x, u, p=0.8)
    run_sample(x, u, k=max(1, vocab - vocab // 4), p=0.7)
    z = torch.zeros((2, vocab), device="cuda")
    z[:, 1::2] = -0.0                                            # the two zeros are one score
    run_sample(z, [0.3, 0.8], k=3)
    run_sample(z, [0.3, 0.8], t=0.0)


def test_sample_masked_infinite_and_nan():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    rows = [[-inf] * 6, [nan] * 6, [-inf, 1.0, nan, -inf, -inf, -inf], [low] * 6, [low, low, 3.0, low, 2.0, low], [inf, 0, inf, 1, -inf, nan],
            [1e38, -1e38, low, 3e38, 2.9e38, 0], [nan, -inf, low, nan, low, -inf]]
    x = torch.tensor(rows, device="cuda")
    for f in FILTERS[:8] + [dict(t=0.0), dict(t=1e-30), dict(t=1e30)]:
        for u in (0.0, 0.4, 0.9999):
            run_sample(x, u, **f)
    y = scores(3, 5000, "f32", 9)
    for t in (1e-7, 1e-4, 3e-3, 1e5, 3e30, inf):                 # from the greedy pick to equal shares
        run_sample(y, [0.0, 0.5, 0.999], t=t)
        run_sample(y, [0.0, 0.5, 0.999], t=t, p=0.7)
    for m in (1e-11, 1e-14, 1e-20):                              # below the weights' resolution: kept words count
        run_sample(y, 0.3, m=m, t=0.2)
    big = torch.full((3, 50000), low, device="cuda")             # nearly all masked by the lowest value
    big[:, 40000:40030] = torch.randn((3, 30), device="cuda")
    for f in FILTERS:
        run_sample(big, 0.77, **f)
    far = torch.full((3, 50000), -1e9, device="cuda")            # a second level of search: all but a few in one bin
    far += torch.randn((3, 50000), device="cuda") * 1e6
    far[:, 7] = 5.0
    for k in (2, 100, 5000):
        run_sample(far, 0.5, k=k, t=1e6)
        run_sample(far, 0.5, k=k, p=0.5, t=1e7)
    run_sample(far, 0.5, p=0.5, t=1e9)


def test_sample_nuclei_that_end_anywhere():
    """Flat and steep rows, so that nuclei end in the list, near its end and far below it; borders at p times a sum that the
    32-bit mass only brackets."""
    g = torch.Generator(device="cuda").manual_seed(3)
    rank = torch.arange(60000, device="cuda").float()
    for steep in (0.0, 0.3, 0.7, 1.0, 1.3, 2.0, 4.0):
        x = (-steep * torch.log1p(rank) + 0.01 * torch.randn((6, 60000), generator=g, device="cuda"))[:, torch.randperm(60000, generator=g, device="cuda")]
        for p in (0.01, 0.3, 0.6, 0.9, 0.99, 0.99999):
            run_sample(x, np.array([0.0, 0.2, 0.4, 0.6, 0.8, 0.999]), p=p, m=0.0 if p < 0.9 else 1e-3)


def test_sample_crowded_scores():
    """Scores within a few steps of one another: the search goes down to single values."""
    x = 1.0 + torch.randint(0, 3, (4, 60000), device="cuda") * 2.0 ** -23
    for f in (dict(k=5), dict(k=30000), dict(p=0.4), dict(k=40000, p=0.9), dict(p=0.99, m=0.5)):
        run_sample(x, np.array([0.0, 0.3, 0.6, 0.99]), **f)
    y = scores(3, 60000, "bf16", 5, scale=0.02)
    for f in (dict(k=5), dict(k=30000), dict(p=0.4), dict(k=40000, p=0.9)):
        run_sample(y, 0.41, **f)


def test_sample_uniform_numbers_out_of_range_and_strided_rows():
    x = scores(6, 700, "f32", 1)
    ids = torch.zeros(6, dtype=I32, device="cuda")
    nb.sample(x, dev([-1.0, np.nan, 1.0, 5.0, np.inf, -np.inf], torch.float32), ids=ids)
    X = x.double().cpu().numpy()
    assert ids.tolist() == [plain.sample(X[i], v)[0] for i, v in enumerate([0, 0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0])]
    for dt in ("f32", "bf16"):
        wide = scores(5, 1301, dt, 2)
        run_sample(wide[:, 1:1002], 0.6, p=0.9)
        run_sample(wide[::2, 3:], 0.6, k=9)


def test_sample_frequencies():
    """Equal steps of u give each word its share of the steps, to one step per border."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device="cuda").repeat(20000, 1)
    ids, _, _ = run_sample_fast(x, (np.arange(20000) + 0.5) / 20000)
    w = np.exp(np.array([0.0, 1.0, 2.0, -1.0, 0.5]))
    assert (np.abs(np.bincount(ids, minlength=5) / 20000 - w / w.sum()) <= 2 / 20000).all()


def run_sample_fast(x, u):
    n = x.shape[0]
    ids, kept, lp = (torch.zeros(n, dtype=t, device="cuda") for t in (I32, I32, torch.float32))
    nb.sample(x, dev(u, torch.float32), ids=ids, logprob=lp, kept=kept)
    return ids.cpu().numpy(), lp.cpu().numpy(), kept.cpu().numpy()


# ----------------------------------------------------------------------------------------------------- all together
def test_decode_loop_of_all_operators():
    """Six steps of 20 conversations on one prompt: pages taken, K and V written, attention, a word sampled from scores made of
    the attention's output, its K and V next; one graph, replayed. The attention and the words against the restatement."""
    rng = np.random.default_rng(4)
    n, kv, g, d, page, P, n_pages, width, vocab = 20, 2, 4, 64, 16, 1200, 400, 4, 501
    heads = kv * g
    pages = [torch.full((n_pages, kv, page, d), float("nan"), device="cuda", dtype=torch.float16) for _ in range(2)]
    prefix = dev(rng.permutation(75), I32)
    for p in pages:
        p[:75].normal_()
    emb = dev(rng.standard_normal((vocab, (heads + 2 * kv) * d)), torch.float32)
    head = dev(rng.standard_normal((heads * d, vocab)) * 0.2, torch.float16)
    z = lambda *s, t=I32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    held, add, table = z(n), torch.ones(n, dtype=I32, device="cuda"), torch.full((n, width), -1, dtype=I32, device="cuda")
    held[3], held[17] = -1, 15                                    # a row not in use; one about to open its second page
    table[17, 0] = 399
    pages[0][399].normal_(), pages[1][399].normal_()
    free, nf, start, slots, pos, status = dev(np.arange(75, 399), I32), dev([324], I32), z(n + 1), z(n), z(n), z(2)
    q, ids, u = z(n, heads, d, t=torch.float16), dev(rng.integers(0, vocab, n), I32), z(n, t=torch.float32)
    out, lse, scr = z(n, heads, d, t=torch.float16), z(n, heads, t=torch.float32), z(n, vocab, t=torch.float16)
    temp, tk, tp = torch.full((n,), 0.9, device="cuda"), torch.full((n,), 60, dtype=I32, device="cuda"), torch.full((n,), 0.9, device="cuda")
    kvrow = z(n, 2 * kv * d, t=torch.float32)
    work = nb.prefix_attn_work(q, pages[0], P, table)

    def step():
        e = emb[ids.long()]
        live = torch.cumsum((held >= 0).to(torch.int64), 0) - 1   # the step's rows are those in use, in order
        kvrow.zero_().index_copy_(0, torch.where(held >= 0, live, n - 1), e[:, heads * d:])
        q.copy_(e[:, :heads * d].reshape(n, heads, d))
        nb.page_map(held, add, table, free, nf, page=page, n_pages=n_pages, start=start, length=held, slots=slots, pos=pos,
                    n_free_out=nf, status=status, pos0=P)
        kk = kvrow.unflatten(1, (2, kv, d))
        nb.page_write(kk[:, 0], kk[:, 1], slots, *pages, status=status)
        nb.prefix_attn(q, *pages, prefix, P, table, held, out=out, lse=lse, work=work, status=status)
        scr.copy_(out.flatten(1) @ head)
        nb.sample(scr, u, ids=ids, temperature=temp, top_k=tk, top_p=tp)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.zeros((n, 8), device="cuda", dtype=torch.float16) @ torch.zeros((8, 8), device="cuda", dtype=torch.float16)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(6):
        u.copy_(dev(rng.random(n), torch.float32))
        before = ids.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0]
        assert held.tolist() == [-1 if i == 3 else (16 + k if i == 17 else k + 1) for i in range(n)]
        e = emb[before.long()]
        row = 0
        for i in range(n):
            if i == 3:
                continue
            L = int(held[i]) - 1
            assert int(pos[row]) == P + L and int(slots[row]) == int(table[i, L // page]) * page + L % page
            assert torch.equal(pages[0][int(table[i, L // page]), :, L % page], e[i, heads * d:(heads + kv) * d].reshape(kv, d).half())
            row += 1
        c = {"q": q, "k": pages[0], "v": pages[1], "prefix": prefix, "prefix_len": P, "table": table, "length": held, "dt": "f16"}
        o2, l2 = out.clone(), lse.clone()
        o2[3], l2[3] = 7.0, 7.0
        check_attn(c, o2, l2, 0, None, "f16")
        X, U = scr.double().cpu().numpy(), u.double().cpu().numpy()
        assert ids.tolist() == [plain.sample(X[i], U[i], float(temp[0]), 60, float(tp[0]))[0] for i in range(n)]
    assert int(nf) == 324 - 18 - 1
