"""The serving operators' refusals on the host: every bad argument is IMI_E_ARG with a message before any device work, and
good ones without a device are IMI_E_NODEV. No GPU needed (the pointers are never followed)."""
import os
import struct
import subprocess

import pytest

import nunchi_b200 as nb

P = 0x10000   # an aligned address that is never read


def call(name, block, good, device=0, **bad):
    a = block.pack(*(v or 0 for v in {**good, **bad}.values()))
    st = getattr(nb.lib(), "imi_cuda_" + name)(device, a, None)
    return st, nb.lib().imi_cuda_error().decode()


MAP = dict(held=P, add=P, n=4, table=P, table_stride=8, width=8, free_pages=P, free_cap=9, n_free=P, page=16, n_pages=40, pos0=0, cap=12,
           start=P, length=P, slots=P, pos=P, n_free_out=P, status=P)
WRITE = dict(k=P, v=P, type=0, row_stride=512, head_stride=64, rows=5, slots=P, n_head_kv=8, head_dim=64, k_pages=P, v_pages=P, page_type=1,
             page=64, n_pages=9, status=None)
ATTN = dict(q=P, type=1, q_stride=2048, rows=4, n_head=32, n_head_kv=8, head_dim=64, k_pages=P, v_pages=P, page=64, n_pages=50, prefix=P,
            prefix_len=1000, table=P, table_stride=9, width=9, length=P, scale=0.125, window=0, out=P, out_type=1, out_stride=2048, lse=P,
            work=P, work_bytes=1 << 30, status=P)
SAMPLE = dict(scores=P, type=0, stride=1000, n=3, vocab=1000, u=P, temperature=P, top_k=P, top_p=P, min_p=P, ids=P, logprob=P, kept=P)


@pytest.mark.parametrize("bad", [
    dict(n=0), dict(n=4097), dict(held=None), dict(add=None), dict(table=None), dict(n_free=None), dict(start=None), dict(length=None),
    dict(n_free_out=None), dict(status=None), dict(slots=None), dict(pos=None), dict(page=0), dict(page=24), dict(page=8), dict(page=512),
    dict(n_pages=0), dict(n_pages=1 << 28), dict(width=0), dict(table_stride=7), dict(cap=-1), dict(free_cap=-1), dict(free_pages=None),
    dict(pos0=-1), dict(pos0=2 ** 31 - 10), dict(held=P + 2), dict(status=P + 1)])
def test_page_map_refuses(bad):
    st, msg = call("page_map", nb._PAGE_MAP, MAP, **bad)
    assert st == 1 and "page_map" in msg


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(page_type=0), dict(page_type=3), dict(type=2), dict(type=-1), dict(n_head_kv=0), dict(head_dim=60), dict(head_dim=0),
    dict(head_dim=264), dict(page=48), dict(n_pages=0), dict(k=None), dict(v=None), dict(slots=None), dict(k_pages=None), dict(v_pages=None),
    dict(row_stride=-1), dict(head_stride=-1), dict(k=P + 2), dict(k_pages=P + 8), dict(slots=P + 2)])
def test_page_write_refuses(bad):
    st, msg = call("page_write", nb._PAGE_WRITE, WRITE, **bad)
    assert st == 1 and "page_write" in msg


@pytest.mark.parametrize("bad", [
    dict(type=0), dict(type=3), dict(out_type=3), dict(out_type=-1), dict(rows=-1), dict(rows=4097), dict(n_head=33), dict(n_head=0),
    dict(n_head_kv=0), dict(n_head=17 * 8), dict(head_dim=96), dict(prefix_len=-1), dict(width=-1), dict(page=100), dict(window=-1),
    dict(n_pages=-1), dict(n_pages=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None), dict(length=None),
    dict(work=None), dict(prefix=None), dict(table=None), dict(k_pages=None), dict(v_pages=None), dict(table_stride=8), dict(q_stride=2040),
    dict(q_stride=2052), dict(out_stride=2040), dict(out_stride=2050), dict(q=P + 8), dict(k_pages=P + 2), dict(out=P + 4), dict(work=P + 8),
    dict(lse=P + 2), dict(work_bytes=100), dict(prefix_len=2 ** 31 - 1)])
def test_prefix_attn_refuses(bad):
    st, msg = call("prefix_attn", nb._PREFIX_ATTN, ATTN, **bad)
    assert st == 1 and "prefix_attn" in msg


def test_prefix_attn_work():
    w = nb.lib().imi_cuda_prefix_attn_work
    assert w(64, 32, 8, 64, 1000, 20, 64) > 0 and w(0, 32, 8, 64, 0, 0, 16) > 0
    for bad in ((-1, 32, 8, 64, 0, 1, 16), (1, 31, 8, 64, 0, 1, 16), (1, 32, 8, 80, 0, 1, 16), (1, 32, 8, 64, -1, 1, 16), (1, 32, 8, 64, 0, 1, 17)):
        assert w(*bad) == 0
    # the workspace of the largest batch serves every smaller one of the same heads
    for prefix in (0, 1, 100, 5000, 100000):
        sizes = [w(r, 32, 8, 64, prefix, 20, 64) for r in range(0, 300)]
        assert all(x <= sizes[-1] for x in sizes)
    for rows in (1, 4, 5, 33, 300):
        sizes = [w(rows, 32, 8, 64, p, 20, 64) for p in range(0, 200000, 997)]
        assert sizes == sorted(sizes)


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(n=65536), dict(vocab=0), dict(vocab=262145, stride=300000), dict(type=3), dict(scores=None), dict(u=None), dict(ids=None),
    dict(stride=999), dict(scores=P + 2), dict(top_k=P + 1), dict(kept=P + 2)])
def test_sample_refuses(bad):
    st, msg = call("sample", nb._SAMPLE, SAMPLE, **bad)
    assert st == 1 and "sample" in msg


def test_null_argument_blocks():
    for f in ("page_map", "page_write", "prefix_attn", "sample"):
        assert getattr(nb.lib(), "imi_cuda_" + f)(0, None, None) == 1


def test_no_such_device():
    for name, block, good in (("page_map", nb._PAGE_MAP, MAP), ("page_write", nb._PAGE_WRITE, WRITE), ("prefix_attn", nb._PREFIX_ATTN, ATTN),
                              ("sample", nb._SAMPLE, SAMPLE)):
        for device in (-1, 4096):
            assert call(name, block, good, device)[0] == 8


def test_argument_blocks_match_the_header(tmp_path):
    """The blocks that the Python binding packs are laid out as the C compiler lays the header's out: every field at its place."""
    names = {"page_map": (nb._PAGE_MAP, MAP), "page_write": (nb._PAGE_WRITE, WRITE), "prefix_attn": (nb._PREFIX_ATTN, ATTN), "sample": (nb._SAMPLE, SAMPLE)}
    src = '#include "imi_cuda.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void) {\n'
    for n, (_, good) in names.items():
        src += f'printf("%zu", sizeof(imi_cuda_{n}_args));\n'
        src += "".join(f'printf(" %zu", offsetof(imi_cuda_{n}_args, {f}));\n' for f in good) + 'puts("");\n'
    c, exe = tmp_path / "t.c", tmp_path / "t"
    c.write_text(src + "return 0; }\n")
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", inc, str(c), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (n, (block, good)) in zip(lines, names.items()):
        size, *offsets = map(int, line.split())
        assert block.size == size, n
        fmt, at = block.format[1:-2], []
        for k in range(len(fmt)):
            at.append(struct.calcsize("@" + fmt[:k] + "0" + fmt[k]))
        assert at == offsets, n


def test_python_refuses_a_strided_workspace():
    torch = pytest.importorskip("torch")
    pages = [torch.zeros(4, 1, 16, 64, dtype=torch.float16) for _ in range(2)]
    q, out = (torch.zeros(1, 4, 64, dtype=torch.float16) for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    call = lambda work: nb.prefix_attn(q, *pages, i32(0), 16, i32(1, 2)[None], i32(5), out=out, work=work)
    with pytest.raises(nb.ImiError, match="contiguous"):
        call(torch.zeros(1 << 20, dtype=torch.uint8)[::2])
    with pytest.raises(nb.ImiError, match="device arrays"):
        call(torch.zeros(1 << 20, dtype=torch.uint8))
