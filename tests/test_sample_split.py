"""How sampling cuts its rows over the CTAs of a cluster (tests/sample_check.cu over sample_split in serve.h): every CTA has words,
about as many as the others, its loads stay aligned, and its parts hold them. No GPU needed."""
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
NW, TILE, SLICE, VOCAB = 16, 128, 32768, 262144


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    if not (os.path.exists(NVCC) or shutil.which("nvcc")):
        pytest.skip("nvcc not found")
    exe = str(tmp_path_factory.mktemp("split") / "sample_check")
    r = subprocess.run([NVCC if os.path.exists(NVCC) else "nvcc", "-std=c++17", "-x", "cu", os.path.join(ROOT, "tests", "sample_check.cu"),
                        "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

    def of(n, lo, hi, step):
        out = subprocess.run([exe, *map(str, (n, lo, hi, step))], capture_output=True, text=True, check=True).stdout
        return np.array([x.split() for x in out.splitlines()], int).T
    return of


@pytest.mark.parametrize("n", [1, 5, 11, 12, 24, 40, 64, 96, 65535])
@pytest.mark.parametrize("lo,hi,step", [(1, 20000, 1), (16001, VOCAB, 37), (VOCAB - 100, VOCAB, 1)])
def test_every_cta_has_its_share(split, n, lo, hi, step):
    v, ctas, seg, share, _ = split(n, lo, hi, step)
    last = v - (ctas - 1) * share
    assert (last > 0).all() and (last <= share).all()                # all words, and no CTA without
    assert (share - last < 4 * ctas).all()                           # as many as the others, to a load each
    assert (share % 4 == 0).all() and (seg % TILE == 0).all() and (seg * NW >= share).all()
    assert (share <= SLICE).all() and (seg * NW <= SLICE).all()
    assert np.isin(ctas, (1, 2, 4, 8)).all()
    # a row goes to c CTAs only with more than c / 2 x 2,048 words: more than 1,024 each, less the rounding by fours. Their lanes (four
    # words each) are more than a nucleus's list asks of a CTA, about 384 / c
    m = ctas > 1
    assert (last[m] > 1024 - 4 * ctas[m]).all() and (last[m] // 4 >= 384 // ctas[m]).all()


@pytest.mark.parametrize("n", [1, 12, 24, 48, 96])
def test_a_nucleus_s_list_is_bounded_by_threads_that_have_words(split, n):
    """The maximum that bounds the list is one that the last CTA has, and of words in any order about 500 are above it, well within
    the list's 768: over 200 random rows of some sizes, by the layout's own threads."""
    v, ctas, seg, share, rank = split(n, 769, 20000, 13)
    last = v - (ctas - 1) * share
    lanes = last // seg * 32 + np.minimum(32, -(-(last % seg) // 4))
    assert (rank >= 1).all() and (rank < lanes).all()
    rng = np.random.default_rng(n)
    for i in rng.choice(v.size, 8, replace=False):
        listed = []
        for _ in range(200):
            x, floor = rng.random(v[i]), 1.0
            for r in range(ctas[i]):
                part = x[r * share[i]:(r + 1) * share[i]]
                at = np.arange(part.size)
                top = np.zeros(16 * 32)
                np.maximum.at(top, at // seg[i] * 32 + at % seg[i] % TILE // 4, part)
                floor = min(floor, np.sort(top)[-rank[i]])
            listed.append((x >= floor).sum())
        # the r-th maximum's place varies by about sqrt(r): the lowest of up to 8 CTAs' lists a third more than one's
        assert 300 < np.mean(listed) < 640 and np.max(listed) <= 768, (v[i], np.mean(listed), np.max(listed))
    assert (split(n, 1, 768, 1)[4] == 512).all()
