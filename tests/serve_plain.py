"""The serving operators restated on the host in 64 bits (numpy), from their definitions in include/imi_cuda.h: what
tests/test_gpu_serve_ops.py compares the device's answers with."""
import numpy as np


def page_map(held, add, table, free, n_free, page, n_pages, pos0, cap):
    """(table, start, length, slots, pos, n_free_out, status) of imi_cuda_page_map."""
    held, add, table, free = (np.array(x, np.int64) for x in (held, add, table, free))
    n, width = table.shape
    code = 0
    used = held >= 0
    for i in range(n):
        if used[i] and add[i] < 0:
            code = max(code, 5)
        if used[i] and held[i] + max(add[i], 0) > width * page:
            code = max(code, 2)
    a = np.where(used, np.maximum(add, 0), 0)
    need = np.where(used, -(-(held + a) // page) - -(-held // page), 0)
    if a.sum() > cap:
        code = max(code, 3)
    if n_free < 0 or n_free > free.size or need.sum() > n_free:
        code = max(code, 4)
    slots, pos = np.full(cap, -1), np.full(cap, -1)
    if code:
        return table, np.zeros(n + 1, np.int64), np.where(used, held, -1), slots, pos, n_free, code
    start = np.concatenate(([0], np.cumsum(a)))
    left = n_free
    for i in range(n):
        for c in range(-(-held[i] // page), -(-(held[i] + a[i]) // page)) if used[i] else ():
            left -= 1
            table[i, c] = free[left]
        for t in range(a[i]):
            p = held[i] + t
            pg = table[i, p // page]
            pos[start[i] + t] = pos0 + p
            if 0 <= pg < n_pages:
                slots[start[i] + t] = pg * page + p % page
            else:
                code = 1
        for c in range(-(-held[i] // page), -(-(held[i] + a[i]) // page)) if used[i] else ():
            code = max(code, 0 if 0 <= table[i, c] < n_pages else 1)
    return table, start, np.where(used, held + a, -1), slots, pos, left, code


def attn(q, k_pages, v_pages, prefix, prefix_len, table, length, scale, window):
    """(out, lse, spread, reach, seen) per row: the attention in 64 bits; spread = softmax . |V|, reach = the largest sum of
    |q_i K_i| and seen = the number of positions (what error bounds are made of). Rows not in use: None."""
    n_pages, kv, page, d = k_pages.shape
    n, heads, _ = q.shape
    g = heads // kv
    res = []
    for i in range(n):
        L = int(length[i])
        if L < 0:
            res.append(None)
            continue
        L = min(L, table.shape[1] * page)
        at = [(int(prefix[j // page]), j % page) for j in range(prefix_len)] + \
             [(int(table[i, j // page]), j % page) for j in range(L)]
        if window:
            at = at[-window:]
        at = [x for x in at if 0 <= x[0] < n_pages]
        if not at:
            res.append((np.zeros((heads, d)), np.full(heads, -np.inf), np.zeros((heads, d)), np.zeros(heads), 0))
            continue
        pg, of = (np.array(x) for x in zip(*at))
        K, V = k_pages[pg, :, of, :], v_pages[pg, :, of, :]     # [positions][kv][d]
        K, V = np.repeat(K, g, 1), np.repeat(V, g, 1)
        s = np.einsum("hd,phd->hp", q[i], K) * scale
        reach = np.einsum("hd,phd->hp", np.abs(q[i]), np.abs(K)).max(1)
        m = s.max(1, keepdims=True)
        e = np.exp(s - m)
        z = e.sum(1, keepdims=True)
        res.append((np.einsum("hp,phd->hd", e / z, V), (m + np.log(z))[:, 0], np.einsum("hp,phd->hd", e / z, np.abs(V)), reach, len(at)))
    return res


def sample(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(id, logprob, kept) of one row x (64-bit values of the scores)."""
    words = np.flatnonzero(x > -np.inf)                        # NaN is not
    if words.size == 0:
        return -1, -np.inf, 0
    words = words[np.argsort(-x[words], kind="stable")]
    if not t > 0:
        return int(words[0]), 0.0, 1
    top = x[words[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[words] == top, 1.0, np.exp(-(top - x[words]) / t))
    n = words.size
    if 0 < k < n:
        n = k
    if p <= 0:
        n = 1
    elif p < 1:
        before = np.concatenate(([0.0], np.cumsum(w[:n])[:-1]))
        n = max(1, int((before < p * w[:n].sum()).sum()))
    if m > 0:
        n = max(1, int((w[:n] >= min(m, 1.0)).sum()))
    words, w = words[:n], w[:n]
    o = np.argsort(words)
    words, w = words[o], w[o]
    c = np.cumsum(w)
    j = int((c <= u * c[-1]).sum())
    return int(words[j]), float(np.log(w[j] / c[-1])), n
