"""Ends of the range of sampled decoding over caches in pages: draws that fall on a drafted token, rows without a number at any
temperature, values next to f32's ends, outputs between the rows of inputs, scores far from zero, prompts, tables with gaps.
The plain forms and their tolerances are those of test_pages_gpu, with eps = 2^-24 (half a step of f32) and 2^-11 (of f16)."""

import numpy as np
import pytest

import wavo_amd as wa
from test_pages_gpu import NONE, Cache, append, attend, expect, norm_tolerance, probs, rope_table, rows_of, same_words, sample, softmax, turned
from test_tree_gpu import EPS, EPS16, attend_tolerance, bits, trees

pytestmark = pytest.mark.gpu

# ------------------------------------------------------------------------------------------- draws of a child's token


def walk(p, q, tokens, parent, u, vocab):
    """One sequence, in 64 bits: picks, the nodes of the walk, and how often a draw fell on a child's token."""
    picks, path, number, falls = np.full(len(tokens), NONE, np.uint32), [0], float(u[0]), 0
    at, start, w, total = 0, 1, p[0].astype(np.float64), 1.0
    while True:
        for i in range(start, len(tokens)):
            if parent[i] != at or not total > 0 or tokens[i] >= vocab:
                continue
            x = tokens[i]
            if float(u[i]) * (1.0 if q is None else float(q[at, x])) * total < w[x]:
                picks[at] = x
                path.append(i)
                at, w, total = i, p[i].astype(np.float64), 1.0
            elif q is None:
                total -= w[x]
                w[x] = 0
            else:
                w = np.maximum(w / total - q[at].astype(np.float64), 0)
                total = w.sum()
        if not w.sum() > 0:
            w = p[at].astype(np.float64)
        c = np.cumsum(w)
        place = number * c[-1]
        over = np.flatnonzero((c > place) & (w > 0))
        if not len(over):
            return picks, path, falls
        picks[at] = x = over[0]
        child = [i for i in range(at + 1, len(tokens)) if parent[i] == at and tokens[i] == x]
        if not child:
            return picks, path, falls
        falls += 1
        number = (place - (c[x] - w[x])) / w[x]
        at, start, w, total = child[0], child[0] + 1, p[child[0]].astype(np.float64), 1.0
        path.append(at)


def full_tree(levels, spread=3):
    """Parents and who sees whom where every node but the last level's has `spread` children."""
    parents = [0]
    first, end = 0, 1
    for _ in range(levels):
        parents += [i for i in range(first, end) for _ in range(spread)]
        first, end = end, len(parents)
    seen = np.eye(len(parents), dtype=bool)
    for i in range(1, len(parents)):
        seen[i] |= seen[parents[i]]
    return np.array(parents), seen


@pytest.mark.parametrize("kind", ["rejected", "untested", "drafts"])
def test_draws_of_a_childs_token_go_on_there(gpu, kind):
    """Children that are all that is wanted and of which none is accepted, as sums are rounded: the draw takes one of them all the
    same, and the walk that wh_tree_accept takes does not end in a node without a pick."""
    rng = np.random.default_rng({"rejected": 1, "untested": 2, "drafts": 3}[kind])
    vocab, want = 3, 24
    parents, seen = full_tree(3)
    rows = len(parents)
    found = []
    for _ in range(20000):
        x = rng.standard_normal((rows, vocab))
        if kind == "untested":  # (the last child's share is less than the others' roundings)
            x[:, 2] -= rng.uniform(15, 18)
        p, q = softmax(x), None
        tokens = np.zeros(rows, np.uint32)
        for i in range(1, rows, 3):
            tokens[i:i + 3] = np.arange(3) if kind == "untested" else rng.permutation(3)
        u = rng.random(rows).astype(np.float32)
        u[rng.random(rows) < 0.8] = np.float32(1 - 2.0**-24)
        u[0] = rng.random() if kind != "untested" else np.float32(1 - 2.0**-24)
        if kind == "drafts":  # (rows that do not sum to 1: most rejections leave nothing)
            q, p = softmax(rng.standard_normal((rows, vocab))), p * np.float32(2.0**-6)
        if walk(p, q, tokens, parents, u, vocab)[2]:
            found.append((p, q, tokens, u))
        if len(found) == want:
            break
    assert len(found) >= 8
    p, tokens, u = (np.stack([f[i] for f in found]) for i in (0, 2, 3))
    q = np.stack([f[1] for f in found]) if kind == "drafts" else None
    batch = len(found)
    mask = bits(np.broadcast_to(seen, (batch, rows, rows)))
    got = sample(gpu, p, q, tokens, u, vocab, mask)
    paths = []
    for b in range(batch):
        picks, path, _ = walk(p[b], None if q is None else q[b], tokens[b], parents, u[b], vocab)
        assert np.array_equal(got[b], picks), f"sequence {b}"
        paths.append(path)
    up = lambda a: gpu.upload(np.ascontiguousarray(a))  # noqa: E731
    keep = [up(np.zeros(batch, np.int32)), up(tokens), up(mask), up(got)]
    path, kept, nxt, n_out = (up(np.full(s, -9, np.int32)) for s in ((batch, rows), batch, batch, batch))
    gpu.tree_accept(wa.Tree(batch, rows, keep[0], None, keep[1], keep[2], mask[0].size), keep[3], None, None, 0, 0, None, 0, 0, 0, 100, 0, path,
                    kept, nxt, n_out)
    assert np.all(gpu.read(nxt, (batch,), np.uint32) < vocab)
    path, kept = gpu.read(path, (batch, rows), np.int32), gpu.read(kept, (batch,), np.int32)
    assert [path[b, :kept[b]].tolist() for b in range(batch)] == paths


def test_tokens_after_such_a_draw_have_the_targets_distribution(gpu):
    """20000 roots whose children are hardly ever accepted: what is drawn after the child that the first draw fell on."""
    rng = np.random.default_rng(4)
    batch, rows, vocab = 20000, 3, 4
    p, q = np.zeros((batch, rows, vocab), np.float32), np.full((batch, rows, vocab), 0.25, np.float32)
    p[:, 0] = np.float32([0.4, 0.3, 0.2, 0.1]) * np.float32(2.0**-10)
    p[:, 1:] = np.float32([0.1, 0.4, 0.2, 0.3])
    tokens = np.broadcast_to(np.uint32([0, 0, 1]), (batch, rows))
    seen = np.eye(rows, dtype=bool)[None].repeat(batch, 0)
    seen[:, :, 0] = True
    got = sample(gpu, p, q, tokens, rng.random((batch, rows)).astype(np.float32), vocab, bits(seen))
    for node in (1, 2):
        there = got[got[:, 0] == node - 1, node]
        assert len(there) > 4000
        share, want = np.bincount(there, minlength=vocab)[:vocab] / len(there), p[0, 1]
        assert np.all(np.abs(share - want) <= 5 * np.sqrt(want * (1 - want) / len(there))), share


@pytest.mark.parametrize("drafts", [True, False])
def test_second_tokens_have_the_targets_distribution(gpu, drafts):
    """20000 trees of two levels: the tokens after accepted children, within 5 standard deviations."""
    rng = np.random.default_rng(5)
    batch, vocab = 20000, 6
    parents, seen = full_tree(2)
    rows = len(parents)
    p = np.broadcast_to(np.float32([0.05, 0.3, 0.1, 0.25, 0.1, 0.2]), (batch, rows, vocab)).copy()
    p[:, 1:] = np.float32([0.2, 0.05, 0.25, 0.1, 0.3, 0.1])
    q = np.broadcast_to(np.float32([0.3, 0.05, 0.1, 0.05, 0.4, 0.1]), (batch, rows, vocab)).copy()
    tokens = rng.choice(vocab, (batch, rows), p=q[0, 0].astype(np.float64) / q[0, 0].sum(dtype=np.float64)).astype(np.uint32)
    got = sample(gpu, p, q if drafts else None, tokens, rng.random((batch, rows)).astype(np.float32), vocab, bits(seen[None].repeat(batch, 0)))
    second = got[:, 1:4][got[:, 1:4] != NONE]
    assert len(second) > 5000 and (got[:, 4:] != NONE).any(1).sum() > 1000
    share, want = np.bincount(second, minlength=vocab) / len(second), p[0, 1]
    assert np.all(np.abs(share - want) <= 5 * np.sqrt(want * (1 - want) / len(second))), share


# ------------------------------------------------------------------------------------------- probabilities


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [37, 5000, 70001])
def test_probs_without_a_number_at_any_temperature(gpu, half, vocab):
    """NaN and plus infinity, wherever they stand, are not taken for a row's maximum at a temperature of zero, either."""
    l = np.random.default_rng(vocab).standard_normal((10, vocab)).astype(np.float16 if half else np.float32)
    l[0, 0] = l[1, vocab - 1] = l[2, vocab // 2] = np.nan
    l[3, 5] = l[4, vocab - 1] = np.inf
    l[5] = np.nan
    l[6] = -np.inf
    l[7] = -np.inf
    l[7, vocab // 3] = np.nan
    l[8] = -np.inf
    l[8, vocab - 2] = -60000
    for t in (0.0, -1.0, np.nan, 1.0):
        got = probs(gpu, l, 10, 1, vocab, [t] * 10)
        for r in (0, 1, 2, 3, 4, 5, 7):
            assert np.all(np.isnan(got[r])), f"row {r} at {t}"
        assert np.all(got[6] == 0)
        assert got[8, vocab - 2] == 1 and got[8].sum() == 1
        if t != 1:
            assert got[9, l[9].argmax()] == 1 and got[9].sum() == 1


@pytest.mark.parametrize("vocab", [100, 70001])
def test_probs_of_the_largest_values(gpu, vocab):
    """Logits up to f32's ends over the largest temperatures: the exponents' difference is wider than f32, and its factor less than
    f32's smallest normal number (which leaves 2^-22 of it at 1.44 / 3.4e38)."""
    rng = np.random.default_rng(vocab)
    most = np.finfo(np.float32).max
    l = rng.standard_normal((4, vocab)).astype(np.float32)
    l[0, ::3] = -most
    l[1] = most * rng.choice([-1, -0.5, 0, 0.25, 1], vocab).astype(np.float32)
    l[2] = l[1] * np.float32(0.3)
    l[3, 1::2] = -np.inf
    l[3, ::4] = -most
    for t in (np.inf, most, np.float32(2e38), np.float32(1e38), np.float32(1e37)):
        got = probs(gpu, l, 4, 1, vocab, [t] * 4)
        x = l.astype(np.float64)
        with np.errstate(invalid="ignore"):
            z = np.where(np.isneginf(x), -np.inf, (x - x.max(1, keepdims=True)) / np.float64(t))
        want = np.exp(z)
        want /= want.sum(1, keepdims=True)
        size = np.abs(np.where(np.isfinite(z), z, 0)) * 1.4427
        rel = (size + (want * size).sum(1, keepdims=True)) * (3 * EPS + 2.0**-22) + 2.0**-21 + (vocab / 1024 + 30) * EPS + 2.0**-20 * (t == np.inf)
        err = np.abs(got - want)
        assert np.all(err <= want * rel + 1e-37), f"temperature {t}: {np.max(err / (want * rel + 1e-37)):.3g} of what is allowed"


# ------------------------------------------------------------------------------------------- norms


@pytest.mark.parametrize("hd", [8, 40, 64, 128, 256])
@pytest.mark.parametrize("in_place", [False, True])
def test_head_norm_of_values_whose_squares_leave_f32(gpu, hd, in_place):
    """Heads of the largest and of the smallest numbers among ordinary ones: their norm is of f32's range, and so is the result."""
    rng = np.random.default_rng(hd)
    heads, g, rows = 6, 2, 5
    x = rows_of(rng, 1, rows, heads, g, hd, False)
    hx = x[0].reshape(rows, heads + 2 * g, hd)
    hx[0, 1] *= np.float32(1e25)
    hx[0, 7] *= np.float32(1e-25)
    hx[1, :6] *= np.float32(2.0)**rng.integers(-120, 120, 6).astype(np.float32)[:, None]
    hx[2, 0] = rng.choice([-1, 1], hd) * np.finfo(np.float32).max
    hx[2, 6] = rng.integers(-100, 100, hd) * np.float32(2.0**-149)
    hx[2, 7] = np.float32(2.0**-149)
    hx[3, 2, 1:] *= np.float32(1e-30)  # (one large value)
    for eps in (0.0, 1e-6, 1e-38):
        gain, table = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32), rope_table(20, hd)
        keep = [gpu.upload(a) for a in (gain, table, np.array([7], np.int32), x)]
        y = keep[3] if in_place else gpu.buffer(x.size)
        gpu.head_norm(wa.Tree(1, rows, keep[2]), wa.Heads(heads, g, hd, keep[0], keep[0], eps, keep[1], 20, hd), keep[3], x.shape[-1], y, x.shape[-1])
        got = gpu.read(y, hx.shape)
        want = turned(hx[:, :heads + g], gain, eps, table, hd, False, 7 + np.arange(rows))
        err = np.abs(got[:, :heads + g] - want)
        assert np.all(err <= norm_tolerance(hx[:, :heads + g], gain, hd)), f"eps {eps}: {err.max()}"
        assert np.array_equal(got[:, heads + g:], hx[:, heads + g:])


def test_rows_between_each_other(gpu):
    """Outputs whose rows lie in the gaps of their inputs' overlap nothing: the results of buffers of their own."""
    rng = np.random.default_rng(6)
    rows, heads, g, hd = 9, 4, 2, 64
    d = (heads + 2 * g) * hd
    x = rows_of(rng, 1, rows, heads, g, hd, False)[0]
    n, table = gpu.upload(np.array([3], np.int32)), gpu.upload(rope_table(20, hd))
    h, t = wa.Heads(heads, g, hd, table=table, positions=20, rot=hd), wa.Tree(1, rows, n)
    alone, xb = gpu.buffer(rows * d), gpu.upload(x)
    gpu.head_norm(t, h, xb, d, alone, d)
    want = gpu.read(alone, (rows, d))
    both = gpu.upload(np.concatenate([x, np.full((rows, 2 * d), 7, np.float32)], 1))
    gpu.head_norm(t, h, both, 3 * d, both.ptr + 4 * d, 3 * d)
    got = gpu.read(both, (rows, 3, d))
    assert np.array_equal(got[:, 0], x) and np.array_equal(got[:, 1], want) and np.all(got[:, 2] == 7)
    # Queries into the rows of another stride: their own rows' gaps, every second one left.
    cache = Cache(rng, wa.F16, 32, g, hd, 1, 1)
    both = gpu.upload(np.concatenate([x, np.full((rows, d), 7, np.float32)], 1))
    q = both.ptr
    gpu.page_append(t, h, q, q + 4 * heads * hd, q + 4 * (heads + g) * hd, 2 * d, cache.device(gpu), qo=q + 4 * d, qo_stride=2 * d)
    got = gpu.read(both, (rows, 2, d))
    assert np.array_equal(got[:, 0], x) and np.array_equal(got[:, 1, :heads * hd], want[:, :heads * hd]) and np.all(got[:, 1, heads * hd:] == 7)
    # Keys and values side by side.
    kv = gpu.upload(np.full((rows, 2 * g * hd + 2), 7, np.float32))
    gpu.page_read(t, wa.Pages(cache.pool_buffer, cache.pages, cache.table_buffer, 1, 1, 32, wa.F16, g, hd), kv, kv.ptr + 4 * g * hd, 2 * g * hd + 2)
    got = gpu.read(kv, (rows, 2 * g * hd + 2))
    assert np.array_equal(got[:, :g * hd], want[:, heads * hd:(heads + g) * hd].astype(np.float16))
    assert np.array_equal(got[:, g * hd:2 * g * hd], x[:, (heads + g) * hd:].astype(np.float16)) and np.all(got[:, 2 * g * hd:] == 7)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_lengths_out_count_rows_whatever_became_of_them(gpu, type):
    """Missing pages, path entries of no row, lengths outside the table: n_out counts rows up to the table's positions, and a
    position that nothing was stored to keeps its words."""
    rng = np.random.default_rng(8)
    batch, rows, g, hd = 5, 12, 1, 32
    cache = Cache(rng, type, 32, g, hd, batch, 2)
    cache.table[0, 0] = -1
    n, count = [3, 30, 70, -4, 60], [12, 5, 12, 3, 12]
    path = np.tile(np.arange(rows, dtype=np.int32), (batch, 1))
    path[1, 2], path[3, 0] = -1, rows
    before = cache.pool.copy()
    x = rows_of(rng, batch, rows, 1, g, hd, True)
    _, n_out = append(gpu, cache, x, 1, n, None, path, count, q=False)
    assert n_out.tolist() == [15, 35, 64, 3, 64] == expect(cache, x, 1, n, count, path)
    same_words(cache, cache.read_back(gpu))
    after = Cache.__new__(Cache)
    after.__dict__.update(cache.__dict__)
    after.pool = before
    for b, j in ((1, 32), (3, 0)):
        assert np.array_equal(cache.load(b, j), after.load(b, j), equal_nan=True)


# ------------------------------------------------------------------------------------------- attention


def check_rows(got, cache, x, heads, n, seen, exact_scores=False, nodes=True):
    """All rows of a sequence's head at once, with the worst case of their error as test_pages_gpu.check_attend has it.  exact_scores:
    scores are sums of whole numbers below 2^24, without a rounding: what is left of the exponents' are three of those (of at most
    2^4 digits), and the exponential's and the weights' 2^-20."""
    batch, rows = x.shape[:2]
    hd, g = cache.hd, cache.kv_heads
    p16 = got.dtype == np.float16 and x.dtype == np.float16
    for b in range(batch):
        kept = [z for z in (cache.load(b, j) for j in range(n[b])) if z is not None]
        kv = x[b, :, heads * hd:(heads + 2 * g) * hd].astype(np.float16).astype(np.float64).reshape(rows, 2, g, hd)
        both = np.concatenate([np.stack(kept) if kept else np.zeros((0, 2, g, hd)), kv])
        sees = np.concatenate([np.ones((rows, len(kept)), bool), seen[b] if nodes else np.zeros((rows, rows), bool)], 1)
        for h in range(heads):
            q = x[b, :, h * hd:(h + 1) * hd].astype(np.float64)
            kk, vv = both[:, 0, h // (heads // g)], both[:, 1, h // (heads // g)]
            s = np.where(sees, q @ kk.T / np.sqrt(hd), -np.inf)
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max(1, keepdims=True))
                want = np.where(sees.any(1)[:, None], p @ vv / p.sum(1, keepdims=True), 0)
            size = np.abs(vv).max()
            if exact_scores:
                d = 2.0**4 * 3 * EPS + 2.0**-20
                tol = np.full((rows, 1), (2 * d + 2 * len(both) * EPS) * size)
            else:
                tol = np.array([[attend_tolerance(y, kk, vv, hd)] for y in q])
            tol = tol + len(both) * 2.0**-32 * max(1, size)
            if p16:
                tol = tol + (2 * EPS16 + EPS16**2 + len(both) * 2.0**-35 * max(1, size)) * size
            if got.dtype == np.float16:
                tol = tol + EPS16 * np.abs(want) + 2.0**-25
            err = np.abs(got[b, :, h * hd:(h + 1) * hd].astype(np.float64) - want)
            assert np.all(err <= tol), f"sequence {b} head {h}: {err.max():.3e}, {np.max(err / tol):.2f} of what is allowed"


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16,out16", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("heads,rows,page,cols", [(2, 4, 32, 10), (4, 13, 32, 10), (4, 13, 256, 9), (1, 3, 256, 10)])
def test_attend_scores_far_from_zero(gpu, type, in16, out16, heads, rows, page, cols):
    """Scores of some 1e6 whose differences decide: whole numbers, so that they are exact, above and below zero, in few and many row
    tiles, and over tables that are shared out and joined."""
    rng = np.random.default_rng(heads + rows + page)
    batch, g, hd = 2, 1, 64
    cache = Cache(rng, type, page, g, hd, batch, cols)
    n = [cols * page, cols * page - 77]
    cache.fill(rng, n)
    for b in range(batch):
        for j in range(n[b]):
            pg, tile, p = cache.place(b, j)
            w = cache.pool[pg, :, tile]
            key = np.zeros(hd)
            key[0], key[1] = (28, 24)[int(j % 97 == 5)], 4 * rng.integers(-8, 8)
            if type == wa.F16:
                w.view(np.float16)[:, cache.at[0][0][p]] = key
                continue
            w.view(np.float16)[:, 2 * 4 * hd + cache.factor[p]] = 4
            word, shift = (y[p] for y in cache.at[0])
            for i in range(hd):
                w[0, word[i]] = (w[0, word[i]] & ~np.uint32(15 << shift[i])) | np.uint32(int(key[i]) // 4 + 8) << np.uint32(shift[i])
    x = rows_of(rng, batch, rows, heads, g, hd, in16)
    x[..., :(heads + g) * hd] = 0
    x[..., :heads * hd:hd] = 61440 * rng.choice([-1, 1], (batch, rows, heads))
    x[..., 1:heads * hd:hd] = rng.integers(-2, 3, (batch, rows, heads))
    x[..., heads * hd] = 28
    x[..., heads * hd + 1] = 4 * rng.integers(-8, 8, (batch, rows))
    _, seen = trees(rng, batch, rows)
    got = attend(gpu, cache, x, heads, n, None, seen, out16)
    check_rows(got, cache, x, heads, n, seen, True)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16", [False, True])
def test_attend_prompts(gpu, type, in16):
    """The most rows there are, each seeing itself and those before it, with and without positions in pages before them."""
    rng = np.random.default_rng(7)
    batch, rows, heads, g, hd = 2, 1024, 4, 2, 64
    cache = Cache(rng, type, 64, g, hd, batch, 2)
    n = [0, 77]
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, g, hd, in16)
    x[..., :heads * hd] *= 2
    seen = np.tril(np.ones((rows, rows), bool))[None].repeat(batch, 0)
    check_rows(attend(gpu, cache, x, heads, n, None, seen, in16), cache, x, heads, n, seen)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("cols", [3, 70])
def test_tables_wider_than_their_columns(gpu, type, cols):
    """Tables inside wider rows: what stands beside them are pages of nobody."""
    rng = np.random.default_rng(cols)
    batch, rows, heads, g, hd, page = 3, 4, 2, 1, 32, 32
    cache = Cache(rng, type, page, g, hd, batch, cols)
    n = [cols * page - 4, 40, 7]
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, g, hd, True)
    _, seen = trees(rng, batch, rows)
    xb, mb, nb = gpu.upload(x), gpu.upload(bits(seen)), gpu.upload(np.array(n, np.int32))
    t = wa.Tree(batch, rows, nb, None, None, mb, rows)
    got = []
    for more in (0, 5):
        pages = cache.device(gpu)
        wide = np.concatenate([cache.table, np.tile(cache.table[:1, :1], (batch, more))], 1).astype(np.int32)
        tb, o, k, v = gpu.upload(wide), gpu.buffer(batch * rows * heads * hd), gpu.buffer(batch * rows * g * hd), gpu.buffer(batch * rows * g * hd)
        pages = wa.Pages(cache.pool_buffer, cache.pages, tb, cols, cols + more, page, type, g, hd)
        at = xb.ptr + 2 * heads * hd
        gpu.page_attend(t, xb, at, at + 2 * g * hd, x.shape[-1], pages, o, heads, in16=True)
        gpu.page_append(t, wa.Heads(heads, g, hd), None, at, at + 2 * g * hd, x.shape[-1], pages, in16=True)
        gpu.page_read(t, pages, k, v, g * hd)
        got.append([gpu.read(o, (batch, rows, heads * hd)), cache.read_back(gpu), gpu.read(k, (batch, rows, g * hd)), gpu.read(v, (batch, rows, g * hd))])
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(*got))
    check_rows(got[0][0], cache, x, heads, n, seen)
