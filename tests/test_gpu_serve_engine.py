"""Sampling inside the engine (imi_cuda_sample_states, imi_cuda_sampled) and a conversation's memory handed to the paged operators
(imi_cuda_state_kv), on the small synthetic models; the words against the sampling restated in 64 bits on the engine's own
scores (tests/serve_plain.py)."""
import numpy as np
import pytest

import nunchi_b200 as nb
import serve_plain as plain
from nunchi_b200 import synth

pytestmark = pytest.mark.gpu


def one(x, i):
    return x if np.isscalar(x) else x[i]


def want(state, u, t=1.0, k=0, p=1.0, m=0.0):
    f = np.float32   # the settings as the engine receives them
    return plain.sample(state.logits.astype(np.float64), float(f(u)), float(f(t)), k, float(f(p)), float(f(m)))


@pytest.fixture(scope="module")
def engine(tiny_path):
    e = nb.Engine(tiny_path, n_ctx=256, max_batch=16)
    yield e
    e.close()


def read(engine, n, words=5, seed=3):
    states = [engine.new_state() for _ in range(n)]
    for i, s in enumerate(states):
        s.step_batch(synth.random_ids(words + i % 3, engine.n_vocab, seed + i))
    return states


@pytest.mark.parametrize("n", [1, 2, 9, 16])
def test_sample_states_from_the_latest_scores(engine, n):
    states, rng = read(engine, n), np.random.default_rng(n)
    t, k = rng.choice([0.0, 0.7, 1.0], n).astype(np.float32), rng.choice([0, 5, 200], n).astype(np.int32)
    p, m = rng.choice([0.5, 0.9, 1.0], n).astype(np.float32), rng.choice([0.0, 0.05], n).astype(np.float32)
    u = rng.random(n).astype(np.float32)
    ids, lp, kept = nb.sample_states(states, u, t, k, p, m)
    for i, s in enumerate(states):
        w = want(s, u[i], t[i], int(k[i]), p[i], m[i])
        assert (ids[i], kept[i]) == (w[0], w[2]) and abs(lp[i] - w[1]) <= 2.0 ** -23 * abs(w[1]) + 1e-9
        assert s.argmax()[0] == ids[i]                            # the word is the conversation's last pick
    assert [want(s, 0.25)[0] for s in states] == nb.sample_states(states, 0.25)[0].tolist()


@pytest.mark.parametrize("n,steps", [(1, 5), (2, 70), (11, 6)])
def test_sampled_steps_match_steps_and_samples_one_by_one(engine, n, steps):
    rng = np.random.default_rng(steps)
    u = rng.random((steps, n)).astype(np.float32)
    first = rng.integers(0, engine.n_vocab, n)
    a, b = read(engine, n), read(engine, n)
    ids, lp = nb.sampled(a, steps, u, tokens=first, temperature=0.8, top_k=40, top_p=0.9)
    tok = first
    for k in range(steps):
        nb.step_multi(b, tok)
        got, l, _ = nb.sample_states(b, u[k], 0.8, 40, 0.9)
        assert got.tolist() == ids[k].tolist() and np.array_equal(l, lp[k])
        assert got.tolist() == [want(s, u[k, i], 0.8, 40, 0.9)[0] for i, s in enumerate(b)]
        tok = got
    assert [s.pos for s in a] == [s.pos for s in b]
    more, _ = nb.sampled(a, 2, u[:2], temperature=0.5)           # goes on from the last word
    nb.step_multi(b, tok)
    assert nb.sample_states(b, u[0], 0.5)[0].tolist() == more[0].tolist()


def test_temperature_zero_is_greedy(engine):
    a, b = read(engine, 3), read(engine, 3)
    ids, lp = nb.sampled(a, 12, np.full((12, 3), 0.7, np.float32), tokens=[1, 2, 3], temperature=0.0)
    assert np.array_equal(ids, nb.greedy(b, 12, tokens=[1, 2, 3])) and (lp == 0).all()
    assert np.array_equal(nb.greedy(a, 3), nb.greedy(b, 3))


def test_sampling_refusals(engine):
    a, b = read(engine, 2)
    with pytest.raises(nb.ImiError, match="twice"):
        nb.sample_states([a, a], 0.5)
    with pytest.raises(nb.ImiError, match="token out of range"):
        nb.sampled([a, b], 2, np.zeros((2, 2), np.float32), tokens=[0, engine.n_vocab])
    with pytest.raises(nb.ImiError, match="uniform"):
        nb.sampled([a, b], 2, np.zeros((3, 2), np.float32))
    with pytest.raises(nb.ContextFull):
        nb.sampled([a, b], 256, np.zeros((256, 2), np.float32))
    other = nb.Engine(synth.cached_gguf("tiny"), n_ctx=32)
    s = other.new_state()
    with pytest.raises(nb.ImiError, match="another engine"):
        nb.sample_states([a, s], 0.5)
    s.close()
    other.close()
    assert nb.lib().imi_cuda_sample_states(None, 1, None, None, None, None, None, None, None, None) == 1
    assert nb.lib().imi_cuda_sampled(nb._handles([a]), 1, None, 0, nb._ptr(np.zeros(1, np.float32)), None, None, None, None, None, None) == 1
    with pytest.raises(nb.ImiError, match="layer"):
        a.kv(engine.n_attn)


def test_a_prompt_read_by_the_engine_becomes_shared_pages(engine):
    """A prompt's keys and values of every attention layer, from the engine's memory into pages, are the checkpoint's, and
    attention over these pages for several conversations is the restatement's."""
    torch = pytest.importorskip("torch")
    s = engine.new_state()
    s.step_batch(synth.random_ids(77, engine.n_vocab, 9), want_logits=False)
    img = s.unpack()
    page, n_pages, kv, d = 16, 40, engine.n_head_kv, engine.head_dim
    torch.cuda.synchronize()
    i32 = lambda x: torch.as_tensor(np.asarray(x, np.int32)).to("cuda")  # noqa: E731
    held, add, table = i32([0]), i32([77]), torch.full((1, 8), -1, dtype=torch.int32, device="cuda")
    free, nf, status = i32(np.random.default_rng(1).permutation(n_pages)), i32([n_pages]), i32([0, 0])
    start, slots, pos = i32([0, 0]), i32(np.zeros(77)), i32(np.zeros(77))
    nb.page_map(held, add, table, free, nf, page=page, n_pages=n_pages, start=start, length=held, slots=slots, pos=pos, n_free_out=nf,
                status=status)
    assert held.tolist() == [77] and pos.tolist() == list(range(77))
    for layer in range(engine.n_attn):
        k, v = (torch.as_tensor(x, device="cuda") for x in s.kv(layer))
        assert np.array_equal(k.reshape(77, -1).view(torch.int16).cpu().numpy().view(np.uint16), img["k"][layer])
        assert np.array_equal(v.reshape(77, -1).view(torch.int16).cpu().numpy().view(np.uint16), img["v"][layer])
        pages = [torch.full((n_pages, kv, page, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
        nb.page_write(k, v, slots, *pages, status=status)
        prefix = table[0].contiguous()
        rows = torch.cat([pages[0][int(prefix[p // page]), :, p % page][None] for p in range(77)])
        assert torch.equal(rows, k)
        q = torch.randn((5, engine.n_head, d), device="cuda").half()
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device="cuda")
        own = torch.zeros((5, 1), dtype=torch.int32, device="cuda")
        nb.prefix_attn(q, *pages, prefix, 77, own, i32(np.zeros(5)), out=out, lse=lse, work=nb.prefix_attn_work(q, pages[0], 77, own),
                       status=status)
        h = lambda t: t.double().cpu().numpy()  # noqa: E731
        for i, (o, z, spread, reach, seen) in enumerate(plain.attn(h(q), h(pages[0]), h(pages[1]), h(prefix).astype(int), 77,
                                                                   np.zeros((5, 1), int), np.zeros(5, int), d ** -0.5, 0)):
            # as in test_gpu_serve_ops.py: the scores' error, P's rounding to fp16 (2^-11, and 2^-25 of the largest below its
            # normal range), the output's rounding
            ds = (d ** -0.5 * reach * (d * 2.0 ** -23 + 2.0 ** -22))[:, None]
            tol = spread * (2 * ds + 2.0 ** -11 + 2.0 ** -21 + seen * 2.0 ** -23) + np.abs(o) * 2.0 ** -11 + 2.0 ** -25 + \
                seen * 2.0 ** -25 * np.abs(h(v)).max()
            assert (np.abs(h(out)[i] - o) <= tol).all()
    assert status.tolist() == [0, 0]
    s.close()
