"""The serving operators' first calls of a process: captured into a CUDA graph, and from several threads at once; and tables much
wider than the lengths in them."""
import os
import subprocess
import sys
import threading

import pytest

import nunchi_b200 as nb
from test_gpu_serve_ops import attn_case, check_attn, run_attn, run_sample_fast, scores, torch

pytestmark = pytest.mark.gpu
TESTS = os.path.dirname(os.path.abspath(__file__))

CAPTURE = """
import sys
sys.path[:0] = [{tests!r}, {root!r}]
import torch, nunchi_b200 as nb
from test_gpu_serve_ops import attn_case, check_attn, scores, dev, I32
import numpy as np
cases = [attn_case(n, 2, 4, d, dt, 16, p, [5, 0, 33] + [7] * (n - 3), seed=n) for n, d, dt, p in
         ((3, 64, "f16", 40), (3, 128, "bf16", 3000), (40, 64, "f16", 1500), (40, 128, "bf16", 1500))]
for c in cases:
    c["out"], c["lse"] = torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:2], device="cuda")
    c["work"] = nb.prefix_attn_work(c["q"], c["k"], c["prefix_len"], c["table"])
x, u, ids = scores(9, 30011, "f32", 1), torch.rand(9, device="cuda"), torch.zeros(9, dtype=I32, device="cuda")
z = lambda *v: dev(np.array(v), I32)
held, add, nf, status, table = z(0, 20), z(4, 4), z(6), z(0, 0), torch.full((2, 4), -1, dtype=I32, device="cuda")
table[1, :2] = z(6, 7)
start, slots, pos, free = z(0, 0, 0), z(*range(9)), z(*range(9)), z(*range(6))
pages = [torch.zeros((8, 2, 16, 64), device="cuda", dtype=torch.float16) for _ in range(2)]
rows = torch.randn((9, 2, 64), device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    nb.page_map(held, add, table, free, nf, page=16, n_pages=8, start=start, length=held, slots=slots, pos=pos,
                n_free_out=nf, status=status)
    nb.page_write(rows, rows, slots, *pages, status=status)
    for c in cases:
        nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], c["prefix_len"], c["table"], c["length"], out=c["out"], lse=c["lse"], work=c["work"])
    nb.sample(x, u, ids=ids)
g.replay()
torch.cuda.synchronize()
for c in cases:
    check_attn(c, c["out"], c["lse"], 0, None, c["dt"])
want = torch.zeros_like(ids)
nb.sample(x, u, ids=want)
assert torch.equal(ids, want) and held.tolist() == [4, 24] and status.tolist() == [0, 0], (held, status)
assert torch.equal(pages[0][5, :, :4].transpose(0, 1), rows[:4].half()) and torch.equal(pages[1][7, :, 4:8].transpose(0, 1), rows[4:8].half())
print("done")
"""


def test_first_calls_captured():
    r = subprocess.run([sys.executable, "-c", CAPTURE.format(tests=TESTS, root=os.path.dirname(TESTS))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stderr[-3000:]


def test_calls_from_several_threads():
    """Each thread with its own stream, buffers and workspace; the answers are the ones of a call alone."""
    cases = [attn_case(n, 2, 4, 64, "f16", 16, p, [(11 * i) % 90 for i in range(n)], seed=n) for n, p in ((3, 50), (3, 2500), (40, 1500), (9, 1200))]
    alone = [run_attn(c) for c in cases]
    x = scores(20, 30011, "f32", 3)
    u = torch.rand(20, device="cuda")
    words = run_sample_fast(x, u.cpu().numpy())[0]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        try:
            st, c = torch.cuda.Stream(), cases[k]
            with torch.cuda.stream(st):
                out, lse = torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:2], device="cuda")
                ids, ws = torch.zeros(20, dtype=torch.int32, device="cuda"), nb.prefix_attn_work(c["q"], c["k"], c["prefix_len"], c["table"])
                for _ in range(30):
                    nb.prefix_attn(c["q"], c["k"], c["v"], c["prefix"], c["prefix_len"], c["table"], c["length"], out=out, lse=lse, work=ws)
                    nb.sample(x, u, ids=ids)
                try:
                    nb.sample(x, u[:3], ids=ids)
                    failed.append((k, "not refused"))
                except nb.ImiError:
                    pass
            st.synchronize()
            if not (torch.equal(out, alone[k][0]) and torch.equal(lse, alone[k][1]) and (ids.cpu().numpy() == words).all()):
                failed.append((k, "differs"))
        except Exception as e:  # noqa: BLE001
            failed.append((k, repr(e)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("rows,kv,d", [(4, 2, 64), (40, 2, 64), (250, 1, 128)])
def test_attn_tables_much_wider_than_the_lengths_and_mostly_unused_rows(rows, kv, d):
    """Tables of 100,000 positions a row, of which a few hold something (the rest of an entry may be anything), and three rows of
    four not in use: the split between prompt and own positions, which goes by the width, changes no answer."""
    own = [(7 * i) % 90 if i % 4 == 1 else -1 for i in range(rows)]
    for prefix in (60, 1500):
        c = attn_case(rows, kv, 4, d, "f16", 16, prefix, own, seed=rows)
        narrow = run_attn(c)
        wide = torch.full((rows, 6250), -10 ** 9, device="cuda", dtype=torch.int32)
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
        got = run_attn(c)
        check_attn(c, *narrow, 0, None, "f16")
        assert got[0].shape == narrow[0].shape
        run_attn(c, window=70)
