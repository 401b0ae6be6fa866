"""Decoding with drafted tokens on the device (wh_tree_attend, wh_logit_rules, wh_tree_accept) against plain
64-bit numpy forms of their definitions, and a run of them together: a small decoder that drafts tokens and
has to give the tokens of one that does not.

Tolerances are worst cases of the arithmetic, with eps = 2^-24 (half a step of f32) and 2^-11 (half a step of
f16): see attend_tolerance and the rules' tests."""

import numpy as np
import pytest

import wavo_amd as wa

pytestmark = pytest.mark.gpu

EPS, EPS16 = 2.0**-24, 2.0**-11
NONE = 0xFFFFFFFF


# ------------------------------------------------------------------------------------------- plain forms


def bits(seen):
    """[batch][rows][rows] truth values as the masks' words."""
    b, r, _ = seen.shape
    wide = np.zeros((b, r, 32 * ((r + 31) // 32)), bool)
    wide[:, :, :r] = seen
    return np.ascontiguousarray(np.packbits(wide, axis=-1, bitorder="little").view(np.uint32))


def trees(rng, batch, rows, spread=5):
    """Parents of random trees and who sees whom."""
    parents = np.zeros((batch, rows), np.int64)
    seen = np.zeros((batch, rows, rows), bool)
    for i in range(rows):
        if i:
            parents[:, i] = rng.integers(max(0, i - spread), i, batch)
            seen[:, i] = seen[np.arange(batch), parents[:, i]]
        seen[:, i, i] = True
    return parents, seen


def half(x):
    with np.errstate(over="ignore"):
        return x.astype(np.float16)


def cache_words(k, v):
    """Keys and values [cols][d] in wh_pack's layout: pair i of position j at word i * cols + j, then V by position."""
    cols, d = k.shape
    kt = half(k).reshape(cols, d // 2, 2).transpose(1, 0, 2)
    return np.concatenate([np.ascontiguousarray(kt).reshape(-1), half(v).reshape(-1)]).view(np.uint32)


def plain_attend(q, k, v, seen, n, kc, vc, heads, kv_heads, hd):
    """One sequence: q [rows][heads * hd], k and v [rows][kv_heads * hd] (or None), seen [rows][rows], the cache's first
    n positions kc and vc; the outputs and their worst error for f32 rows (see attend_tolerance)."""
    rows = len(q)
    out, tol = np.zeros((rows, heads * hd)), np.zeros((rows, heads * hd))
    for i in range(rows):
        nodes = [j for j in range(rows) if k is not None and seen[i, j]]
        if not n and not nodes:
            continue
        keys = np.concatenate([kc[:n].astype(np.float64)] + [half(k[j:j + 1]).astype(np.float64) for j in nodes])
        vals = np.concatenate([vc[:n].astype(np.float64)] + [half(v[j:j + 1]).astype(np.float64) for j in nodes])
        for h in range(heads):
            at, of = slice(h * hd, (h + 1) * hd), h // (heads // kv_heads)
            kk, vv = keys[:, of * hd:(of + 1) * hd], vals[:, of * hd:(of + 1) * hd]
            x = q[i, at].astype(np.float64)
            s = kk @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            out[i, at] = p @ vv / p.sum()
            tol[i, at] = attend_tolerance(x, kk, vv, hd)
    return out, tol


def attend_tolerance(x, kk, vv, hd):
    """A score is a sum of hd products in f32 (hd + 2 roundings of at most A = max_j sum |q||k| / sqrt(hd)); splitting q
    into two f16 parts leaves 2^-22 of an element, or 2^-24 of the row's largest where that is more (B); the scaling, the
    maximum's subtraction and the exponential's argument add 10 roundings of 2A, the exponential and the two parts of a
    weight 2^-20.  A weight so off by a factor 1 + d moves the mean of the values by at most 2 d max|v|; the sums over n
    keys add 2 n roundings."""
    a = np.max(np.abs(kk) @ np.abs(x)) / np.sqrt(hd)
    b = np.max(np.abs(kk).sum(1)) * np.abs(x).max() / np.sqrt(hd)
    d = a * (hd + 22) * EPS + a * 2.0**-22 + b * EPS + 2.0**-20
    return (2 * d + 2 * len(kk) * EPS) * np.abs(vv).max() + 1e-30


def attend(gpu, q, k, v, seen, n, count, kc, vc, heads, kv_heads, hd, in16=False, out16=False, mask=None, mask_stride=None,
           shared_cache=False, gap=0, stride_more=0, before=7.0):
    """wh_tree_attend over numpy arrays; q, k, v [batch][rows][...] laid side by side in rows `stride_more` longer."""
    batch, rows = q.shape[:2]
    dt = np.float16 if in16 else np.float32
    parts = [q] + ([k, v] if k is not None else [])
    x = np.concatenate(parts + [np.full((batch, rows, stride_more), np.nan)], 2).astype(dt)
    stride = x.shape[2]
    xb = gpu.upload(x)
    size = x.itemsize
    cols = kc.shape[1]
    words = [np.concatenate([cache_words(kc[b], vc[b]), np.full(gap, 0x7E007E00, np.uint32)]) for b in range(len(kc))]
    kvb = gpu.upload(np.concatenate(words))
    nb = gpu.upload(np.asarray(n, np.int32))
    cb = None if count is None else gpu.upload(np.asarray(count, np.int32))
    if mask is None and seen is not None:
        mask = bits(seen)
    mb = None if mask is None else gpu.upload(mask)
    ob = gpu.upload(np.full((batch, rows, heads * hd), before, np.float16 if out16 else np.float32))
    t = wa.Tree(batch, rows, nb, cb, None, mb, (mask[0].size if mask is not None else 0) if mask_stride is None else mask_stride)
    kp = None if k is None else xb.ptr + size * heads * hd
    vp = None if k is None else xb.ptr + size * (heads + kv_heads) * hd
    gpu.tree_attend(t, xb, kp, vp, stride, kvb, 0 if shared_cache else len(words[0]), cols, ob, heads, kv_heads, hd, in16, out16)
    return gpu.read(ob, (batch, rows, heads * hd), np.float16 if out16 else np.float32)


def check_attend(got, q, k, v, seen, n, count, kc, vc, heads, kv_heads, hd, in16, out16, before=7.0):
    batch, rows = q.shape[:2]
    cols = kc.shape[1]
    for b in range(batch):
        c = rows if count is None else min(max(count[b], 0), rows)
        nn = min(max(n[b], 0), cols)
        kb = None if k is None or seen is None else k[b][:c]
        vb = None if kb is None else v[b][:c]
        s = None if seen is None else seen[b][:c, :c]
        src = b if len(kc) > 1 else 0
        want, tol = plain_attend(q[b][:c], kb, vb, s, nn, kc[src], vc[src], heads, kv_heads, hd)
        if out16:  # the weights are rounded to f16 (their largest is at least 2^-1 of the type's normal range), and the output
            finite = lambda x: np.abs(x[np.isfinite(x)]).max(initial=0).astype(np.float64)  # noqa: E731  (of what may be seen)
            vmax = max(finite(vc[src][:nn]), 0 if vb is None else finite(vb))
            tol = tol + (EPS16 + (nn + rows) * 2.0**-25) * vmax + EPS16 * np.abs(want) + 2.0**-25
        err = np.abs(got[b][:c].astype(np.float64) - want)
        assert np.all(np.isfinite(got[b][:c])), f"sequence {b}"
        assert np.all(err <= tol), f"sequence {b}: error {err.max():.3e}, {np.max(err / tol):.2f} of what is allowed"
        assert np.all(got[b][c:] == before), f"sequence {b}: rows past its {c} nodes written"


def case(seed, batch, rows, heads, kv_heads, hd, cols, in16=False, spread=5):
    rng = np.random.default_rng(seed)
    dt = np.float16 if in16 else np.float32
    q = (2 * rng.standard_normal((batch, rows, heads * hd))).astype(dt)
    k, v = (rng.standard_normal((batch, rows, kv_heads * hd)).astype(dt) for _ in range(2))
    kc, vc = (half(rng.standard_normal((batch, cols, kv_heads * hd))) for _ in range(2))
    return rng, q, k, v, trees(rng, batch, rows, spread)[1], kc, vc


# ------------------------------------------------------------------------------------------- attention

# batch, rows, heads, key heads, head size, cols, n of each sequence
SHAPES = [
    (1, 1, 1, 1, 4, 1, [0]),
    (1, 1, 1, 1, 4, 1, [1]),
    (1, 1, 4, 4, 64, 64, [37]),
    (2, 7, 3, 3, 36, 41, [41, 0]),
    (3, 16, 4, 2, 40, 129, [1, 64, 129]),
    (1, 17, 20, 20, 64, 448, [391]),
    (2, 33, 6, 2, 100, 300, [255, 300]),
    (4, 5, 8, 1, 128, 701, [700, 63, 65, 1]),
    (1, 64, 2, 2, 64, 1500, [1500]),
    (2, 65, 2, 1, 80, 515, [512, 513]),
    (1, 100, 3, 1, 64, 70, [5]),
    (1, 3, 2, 2, 128, 9000, [8999]),
    (1, 40, 16, 1, 64, 2500, [2345]),
    (70, 2, 1, 1, 64, 30, list(range(30)) + list(range(30)) + list(range(10))),
]


@pytest.mark.parametrize("in16,out16", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_attend(gpu, shape, in16, out16):
    batch, rows, heads, kv_heads, hd, cols, n = shape
    rng, q, k, v, seen, kc, vc = case(1, batch, rows, heads, kv_heads, hd, cols, in16)
    got = attend(gpu, q, k, v, seen, n, None, kc, vc, heads, kv_heads, hd, in16, out16)
    check_attend(got, q, k, v, seen, n, None, kc, vc, heads, kv_heads, hd, in16, out16)


# Many rows of the smallest heads, and of caches shorter than a load: several row blocks of the kernel for few rows.
NARROW = [(3, 70, 2, 2, 4, 333, [333, 0, 200]), (2, 70, 3, 1, 64, 3, [3, 2]), (2, 41, 2, 2, 128, 2, [1, 2]), (1, 90, 1, 1, 4, 1, [1]),
          (1, 75, 2, 1, 8, 5, [5]), (2, 70, 1, 1, 12, 4, [4, 3])]


@pytest.mark.parametrize("in16,out16", [(False, False), (True, True)])
@pytest.mark.parametrize("shape", NARROW, ids=lambda s: "x".join(str(x) for x in s[:6]))
def test_attend_narrow(gpu, shape, in16, out16):
    test_attend(gpu, shape, in16, out16)


@pytest.mark.parametrize("rows", [2, 70])
def test_attend_splits_of_very_different_scores(gpu, rows):
    """A long cache whose thirds have scores near -1e34, 0 and 1e34, with the large ones first, last and in the middle:
    shares of a row that are joined across wavefronts and workgroups, one of which carries all of it."""
    batch, heads, hd, cols = 3, 1, 64, 6000
    rng, q, _, _, _, kc, vc = case(9, batch, rows, heads, heads, hd, cols)
    q[:] = 0
    q[:, :, 0] = 1e33
    kc[:, :, 0] = 0
    n = [6000, 5999, 5000]
    for b, top in enumerate((0, 2000, 4000)):
        kc[b, (np.arange(2000) + top + 2000) % 6000, 0] = -8
        kc[b, top:top + 2000:7, 0] = 8
    got = attend(gpu, q, None, None, None, n, None, kc, vc, heads, heads, hd)
    for b, top in enumerate((0, 2000, 4000)):  # equal scores there, and weights of zero everywhere else
        vals = vc[b, top:min(top + 2000, n[b]):7].astype(np.float64)
        assert np.all(np.abs(got[b] - vals.mean(0)) <= (2 * len(vals) * EPS + 2.0**-20) * np.abs(vals).max())


@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 4, 64), (6, 2, 128), (2, 1, 40)])
def test_attend_ragged_any_mask_and_masked_garbage(gpu, heads, kv_heads, hd, in16):
    """Counts from none to all, masks that are no trees (rows that see nothing, later nodes, not themselves), lengths
    past both ends, and NaN and infinities wherever nobody looks: cache places past n, nodes past the count, rows'
    ends, mask bits past the count, and nodes that only some see."""
    batch, rows, cols = 6, 37, 200
    rng, q, k, v, _, kc, vc = case(2, batch, rows, heads, kv_heads, hd, cols, in16)
    n, count = [0, 200, -5, 1000, 130, 0], [37, 36, 20, 1, 0, 1000]
    seen = rng.random((batch, rows, rows)) < 0.3
    seen[0, 3] = seen[0, 36] = False  # (n = 0: nothing at all)
    for b in range(batch):
        nn, c = min(max(n[b], 0), cols), min(max(count[b], 0), rows)
        for x in (kc, vc):
            x[b, nn:] = np.resize([np.nan, np.inf, -np.inf, 65504], x[b, nn:].shape)
        for x in (k, v):
            x[b, c:] = np.nan
        if c > 20:  # a node that nobody sees
            k[b, 20], v[b, 20] = np.inf, np.nan
            seen[b, :, 20] = False
    got = attend(gpu, q, k, v, seen, n, count, kc, vc, heads, kv_heads, hd, in16, in16, gap=13, stride_more=6)
    check_attend(got, q, k, v, seen, n, count, kc, vc, heads, kv_heads, hd, in16, in16)
    assert not got[0, 3].any() and not got[0, 36].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("in16", [False, True])
def test_attend_bad_node_stays_on_its_path(gpu, bad, in16):
    """A node whose value (or key) is not finite spoils the rows that see it, and no other."""
    batch, rows, heads, hd, cols = 2, 30, 3, 64, 100
    rng, q, k, v, seen, kc, vc = case(3, batch, rows, heads, heads, hd, cols, in16)
    n = [77, 0]
    clean = attend(gpu, q, k, v, seen, n, None, kc, vc, heads, heads, hd, in16, in16)
    v[:, 4, 5] = bad
    k[:, 9, 2] = np.nan
    got = attend(gpu, q, k, v, seen, n, None, kc, vc, heads, heads, hd, in16, in16)
    for b in range(batch):
        for i in range(rows):
            spoiled = np.zeros(heads * hd, bool)
            spoiled[5] = seen[b, i, 4]
            spoiled[:hd] |= seen[b, i, 9]
            assert np.array_equal(got[b, i, ~spoiled], clean[b, i, ~spoiled])
            assert not np.isfinite(got[b, i, spoiled]).any()


@pytest.mark.parametrize("rows,hd", [(13, 64), (20, 64), (9, 128), (40, 64), (40, 128)])
@pytest.mark.parametrize("what", [np.nan, np.inf, 1e30, -3.0])
def test_attend_rows_past_the_count_change_nothing(gpu, rows, hd, what):
    """Whatever stands in the queries, keys and values of nodes past the count: the same bits."""
    batch, heads, cols = 2, 3, 300
    _, q, k, v, seen, kc, vc = case(14, batch, rows, heads, heads, hd, cols)
    n, count = [290, 0], [rows // 2, rows - 1]
    want = attend(gpu, q, k, v, seen, n, count, kc, vc, heads, heads, hd)
    for b in range(batch):
        for x in (q, k, v):
            x[b, count[b]:] = what
    assert np.array_equal(attend(gpu, q, k, v, seen, n, count, kc, vc, heads, heads, hd), want)


@pytest.mark.parametrize("rows", [1, 13, 70])
def test_attend_cache_alone(gpu, rows):
    """No mask, or no nodes' keys: cross attention, one cache for all sequences or one each."""
    batch, heads, hd, cols = 3, 5, 64, 333
    _, q, k, v, seen, kc, vc = case(4, batch, rows, heads, heads, hd, cols)
    n, count = [333, 0, 290], [rows, rows, max(1, rows // 2)]
    a = attend(gpu, q, None, None, None, n, count, kc, vc, heads, heads, hd)
    check_attend(a, q, None, None, None, n, count, kc, vc, heads, heads, hd, False, False)
    assert not a[1].any()
    b = attend(gpu, q, None, None, seen, n, count, kc, vc, heads, heads, hd)
    c = attend(gpu, q, k, v, None, n, count, kc, vc, heads, heads, hd)
    assert np.array_equal(a, b) and np.array_equal(a, c)
    one = attend(gpu, q, None, None, None, n, count, kc[:1], vc[:1], heads, heads, hd, shared_cache=True)
    check_attend(one, q, None, None, None, n, count, kc[:1], vc[:1], heads, heads, hd, False, False)


@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("batch,rows,heads,kv_heads,hd,cols", [(3, 1, 4, 4, 64, 3000), (2, 25, 8, 2, 128, 5000), (4, 61, 6, 6, 64, 448), (2, 9, 3, 3, 100, 1500)])
def test_attend_repeats_itself(gpu, batch, rows, heads, kv_heads, hd, cols, in16):
    """The same call gives the same bits, with splits and without, whatever ran on the device before it."""
    _, q, k, v, seen, kc, vc = case(16, batch, rows, heads, kv_heads, hd, cols, in16)
    n = [cols - 3 * b for b in range(batch)]
    want = attend(gpu, q, k, v, seen, n, None, kc, vc, heads, kv_heads, hd, in16, in16)
    for turn in range(6):
        if turn % 2:
            attend(gpu, -q, v, k, seen, n[::-1], None, vc, kc, heads, kv_heads, hd, in16, in16)
        assert np.array_equal(attend(gpu, q, k, v, seen, n, None, kc, vc, heads, kv_heads, hd, in16, in16), want)


def test_attend_one_tree_for_all(gpu):
    batch, rows, heads, hd, cols = 4, 21, 4, 64, 90
    _, q, k, v, seen, kc, vc = case(5, batch, rows, heads, heads, hd, cols)
    n = [90, 3, 0, 64]
    seen[:] = seen[0]
    got = attend(gpu, q, k, v, seen, n, None, kc, vc, heads, heads, hd, mask=bits(seen[:1]), mask_stride=0)
    check_attend(got, q, k, v, seen, n, None, kc, vc, heads, heads, hd, False, False)
    assert np.array_equal(got, attend(gpu, q, k, v, seen, n, None, kc, vc, heads, heads, hd))


@pytest.mark.parametrize("in16", [False, True])
def test_attend_large_and_small_queries(gpu, in16):
    """Scores from far below to far above the softmax's range, queries near both ends of f16, f32 ones past it."""
    batch, rows, heads, hd, cols = 1, 24, 2, 64, 150
    _, q, k, v, seen, kc, vc = case(6, batch, rows, heads, heads, hd, cols, in16)
    scale = np.array([1e-6, 1e-3, 1, 30, 1000, 20000])[np.arange(rows) % 6][None, :, None]
    q = (q * scale / 4).astype(q.dtype)
    if not in16:
        q[0, 5] *= 1e4
        q[0, 11] *= 1e-30
    got = attend(gpu, q, k, v, seen, [131], None, kc, vc, heads, heads, hd, in16, False)
    # Only rows whose scores' own rounding leaves their order certain can be held to the bound; a row of zeros to its mean.
    want, tol = plain_attend(q[0], k[0], v[0], seen[0], 131, kc[0], vc[0], heads, heads, hd)
    err = np.abs(got[0].astype(np.float64) - want)
    assert np.all(np.isfinite(got)) and np.all(err <= tol), np.max(err / tol)


def test_attend_equal_keys_give_the_mean(gpu):
    batch, rows, heads, hd, cols = 1, 3, 1, 64, 1000
    _, q, k, v, seen, kc, vc = case(7, batch, rows, heads, heads, hd, cols)
    kc[:] = 0
    got = attend(gpu, q, k, v, None, [1000], None, kc, vc, heads, heads, hd)
    want = vc[0].astype(np.float64).mean(0)
    assert np.all(np.abs(got[0] - want) <= 2 * 1000 * EPS * np.abs(vc[0]).max())


@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("rows,heads,hd", [(1, 8, 64), (20, 8, 64), (7, 4, 128), (5, 4, 100), (40, 4, 128)])
def test_attend_caches_of_many_positions(gpu, rows, heads, hd, in16):
    """Caches past what the chip keeps (300 MB), of which a few positions are there: the split of a long one, the loads past
    the chip's caches."""
    n, d = 700, heads * hd
    cols = 75_000_003 // d
    _, q, k, v, seen, kc, vc = case(15, 1, rows, heads, heads, hd, n, in16)
    kv = gpu.buffer(cols * d)
    gpu.zero(kv)
    gpu.pack(gpu.upload(np.concatenate([kc[0], vc[0]], 1).astype(np.float32)), 0, 2 * d, kv, n, d, cols, 0)
    x = gpu.upload(np.concatenate([q, k, v], 2))
    size = 2 if in16 else 4
    o = gpu.buffer(rows * d)
    t = wa.Tree(1, rows, gpu.upload(np.array([n], np.int32)), None, None, gpu.upload(bits(seen)), 0)
    gpu.tree_attend(t, x, x.ptr + size * d, x.ptr + 2 * size * d, 3 * d, kv, cols * d, cols, o, heads, heads, hd, in16, in16)
    got = gpu.read(o, (1, rows, d), np.float16 if in16 else np.float32)
    kv.free()
    check_attend(got, q, k, v, seen, [n], None, kc, vc, heads, heads, hd, in16, in16)


def test_attend_offsets_past_32_bits(gpu):
    """A cache of 2^31 words and more to its values (17 GB): keys of zeros but for the last ones, which are large."""
    heads, hd, cols, rows, last = 8, 128, (1 << 22) + 3, 2, 50
    d = heads * hd
    rng = np.random.default_rng(8)
    kv = gpu.buffer(cols * d)
    gpu.zero(kv)
    k, v = rng.standard_normal((2, last, d)).astype(np.float32)
    xb = gpu.upload(np.concatenate([k, v], 1))
    gpu.pack(xb, 0, 2 * d, kv, last, d, cols, cols - last)
    q = (6 * rng.standard_normal((1, rows, d))).astype(np.float32)
    qb, nb, ob = gpu.upload(q), gpu.upload(np.array([cols], np.int32)), gpu.buffer(rows * d)
    gpu.tree_attend(wa.Tree(1, rows, nb), qb, None, None, d, kv, cols * d, cols, ob, heads, heads, hd)
    got = gpu.read(ob, (rows, d)).astype(np.float64)
    kv.free()
    for i in range(rows):
        for h in range(heads):
            at = slice(h * hd, (h + 1) * hd)
            s = half(k[:, at]).astype(np.float64) @ q[0, i, at].astype(np.float64) / np.sqrt(hd)
            p, zero = np.exp(s - s.max()), (cols - last) * np.exp(-s.max())
            want = p @ half(v[:, at]).astype(np.float64) / (p.sum() + zero)
            tol = attend_tolerance(q[0, i, at].astype(np.float64), half(k[:, at]).astype(np.float64), half(v[:, at]).astype(np.float64), hd)
            # The zeros' 4 million equal terms are summed in f32 as well: 2 sqrt(n) roundings where they carry all of it.
            tol += 2 * cols * EPS * zero / (p.sum() + zero) * np.abs(want).max()
            assert np.all(np.abs(got[i, at] - want) <= tol)


# ---------------------------------------------------------------------------------------- logit rules


def plain_rules(x, text, penalty, bias, allow, dt):
    """One row in `dt` arithmetic: the ids' counts in `text`, then penalties, biases (a dict), allowed ids."""
    x = x.astype(dt)
    if penalty is not None:
        r, f, p = (dt(y) for y in penalty)
        ids, times = np.unique(np.asarray(text, np.int64), return_counts=True)
        keep = ids < len(x)
        ids, c = ids[keep], times[keep].astype(dt)
        t = x[ids]
        with np.errstate(invalid="ignore"):
            x[ids] = (np.where(t > 0, t / r, t * r) - f * c) - p
    for i, y in bias.items():
        if i < len(x):
            x[i] = x[i] + dt(y)
    if allow is not None:
        x[~allow] = -np.inf
    return x


def rules_case(seed, batch, rows, vocab, history, biases, f16):
    rng = np.random.default_rng(seed)
    c = {"n": rng.integers(0, history + 1, batch), "count": rng.integers((rows + 1) // 2, rows + 1, batch)}
    c["history"] = rng.integers(0, vocab, (batch, history)) // rng.integers(1, 50, (batch, history))
    c["tokens"] = rng.integers(0, vocab, (batch, rows)) // 3
    c["seen"] = trees(rng, batch, rows)[1]
    c["penalty"] = np.stack([rng.uniform(0.8, 1.6, batch), rng.uniform(-0.3, 0.6, batch), rng.uniform(-0.3, 0.6, batch)], 1).astype(np.float32)
    lens = rng.integers(0, biases + 1, batch)
    c["start"] = np.concatenate([[0], np.cumsum(lens)])
    c["bias_id"], c["bias"] = rng.integers(0, vocab, c["start"][-1] + 1) // 2, rng.normal(0, 3, c["start"][-1] + 1).astype(np.float32)
    c["allow"] = rng.random((batch * rows, vocab)) < rng.choice([0.02, 0.5, 1.0], (batch * rows, 1))
    c["logits"] = (4 * rng.standard_normal((batch * rows, vocab))).astype(np.float16 if f16 else np.float32)
    return c


def run_rules(gpu, c, f16, ld_more=0, penalty=True, bias=True, allow=True, history=True, mask=True, out="new", pick=True,
              logprob=True, from_=0, count=True):
    batch, rows = c["seen"].shape[:2]
    total, vocab = c["logits"].shape
    ld, dt = vocab + ld_more, np.float16 if f16 else np.float32
    x = np.full((total, ld), 3.0, dt)
    x[:, :vocab] = c["logits"]
    xb = gpu.upload(x)
    ob = xb if out == "same" else gpu.upload(np.full((total, ld), 5.0, dt)) if out == "new" else None
    words = (vocab + 31) // 32
    wide = np.ones((total, 32 * words), bool)
    wide[:, :vocab] = c["allow"]
    up = lambda a, dt: gpu.upload(np.ascontiguousarray(a, dt))  # noqa: E731
    keep = [up(c["n"], np.int32), up(c["count"], np.int32), up(c["tokens"], np.uint32), gpu.upload(bits(c["seen"])),
            up(c["penalty"], np.float32), up(c["history"], np.uint32), up(c["start"], np.int32), up(c["bias_id"], np.uint32),
            up(c["bias"], np.float32), gpu.upload(np.packbits(wide, axis=-1, bitorder="little"))]
    nb, cb, tb, mb, pb, hb, sb, ib, vb, ab = keep
    t = wa.Tree(batch, rows, nb, cb if count else None, tb, mb if mask else None, bits(c["seen"])[0].size)
    r = wa.Rules(pb if penalty else None, hb if history else None, c["history"].shape[1] if history else 0, from_, sb if bias else None,
                 ib, vb, len(c["bias"]), ab if allow else None)
    kb, lb = gpu.upload(np.full(total, 77, np.uint32)), gpu.upload(np.full(total, 77, np.float32))
    gpu.logit_rules(t, r, xb, ob, vocab, ld, f16, kb if pick else None, lb if logprob else None)
    o = gpu.read(ob, (total, ld), dt) if ob is not None else None
    return o, gpu.read(kb, (total,), np.uint32), gpu.read(lb, (total,))


def check_rules(c, f16, o, pick, logprob, ld_more=0, penalty=True, bias=True, allow=True, history=True, mask=True, out="new",
                from_=0, count=True):
    batch, rows = c["seen"].shape[:2]
    vocab = c["logits"].shape[1]
    for b in range(batch):
        n = min(max(int(c["n"][b]), 0), c["history"].shape[1])
        there = min(int(c["count"][b]), rows) if count else rows
        biases = {}
        if bias:
            for e in range(max(c["start"][b], 0), min(c["start"][b + 1], len(c["bias"]))):
                biases[int(c["bias_id"][e])] = c["bias"][e]
        for i in range(rows):
            row = b * rows + i
            if i >= there:
                assert pick[row] == 77 and logprob[row] == 77
                if o is not None:
                    assert np.array_equal(o[row, :vocab], c["logits"][row] if out == "same" else np.full(vocab, 5, o.dtype))
                continue
            text = list(c["history"][b, from_:n]) if history else []
            if mask:
                text += [c["tokens"][b, j] for j in range(there) if c["seen"][b, i, j]]
            args = (text, c["penalty"][b] if penalty else None, biases, c["allow"][row] if allow else None)
            x = plain_rules(c["logits"][row], *args, np.float32)
            if o is not None:  # the same sums and products, each rounded once: the same numbers
                assert np.array_equal(o[row, :vocab], half(x) if f16 else x, equal_nan=True), f"row {row}"
                assert np.all(o[row, vocab:] == (3.0 if out == "same" else 5.0))
            with np.errstate(invalid="ignore"):
                best = np.where(np.isnan(x), -np.inf, x)
            want = int(best.argmax()) if best.max() > -np.inf else NONE
            assert pick[row] == want, f"row {row}: {pick[row]} for {want}"
            # And in 64 bits: five roundings of what an id's value is made of.
            y = plain_rules(c["logits"][row], *args, np.float64)
            if np.isnan(x).any():
                assert np.isnan(logprob[row])
            elif want == NONE:
                assert logprob[row] == -np.inf
            elif np.isfinite(best.max()):
                fine = np.isfinite(y)
                made = np.abs(c["logits"][row].astype(np.float64)) * 1.7 + 20 + 0.6 * len(text)
                assert np.all(np.abs(x[fine] - y[fine]) <= 5 * EPS * made[fine])
                rest = np.exp(x[fine].astype(np.float64) - np.float64(x[want])).sum() - 1
                # a term is off by its argument's rounding (at most 104 * 2^-23, past which it is 0) and its own 2^-21
                tol = (104 * 2.0**-23 + 2.0**-21 + 64 * EPS) * rest / (1 + rest) + 2.0**-22 * np.log1p(rest) + 1e-30
                assert abs(logprob[row] + np.log1p(rest)) <= tol, f"row {row}"


RULES = [(1, 1, 1, 1, 0), (1, 1, 33, 3, 5), (2, 5, 1000, 20, 30), (1, 3, 4096, 10, 4), (3, 1, 4097, 300, 100), (2, 33, 5000, 64, 10),
         (1, 70, 12289, 700, 400), (1, 2, 51866, 448, 100), (5, 9, 8191, 5, 1)]
CROWDED = [(2, 300, 2500, 100, 1900), (1, 1024, 700, 30, 5), (1, 130, 2049, 9000, 3000)]  # nodes and listed ids past 64 in a run of ids


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("shape", RULES, ids=lambda s: "x".join(str(x) for x in s))
def test_rules(gpu, shape, f16):
    for seed, ld_more, out in ((1, 0, "new"), (2, 1, "same"), (3, 38, "none")):
        c = rules_case(seed, *shape, f16)
        check_rules(c, f16, *run_rules(gpu, c, f16, ld_more, out=out), ld_more, out=out)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("shape", CROWDED, ids=lambda s: "x".join(str(x) for x in s))
def test_rules_crowded(gpu, shape, f16):
    c = rules_case(11, *shape, f16)
    check_rules(c, f16, *run_rules(gpu, c, f16), out="new")


def test_rules_infinite_biases_past_the_vocabulary(gpu):
    """Ids from vocab on, inside the last run of ids: infinite biases and penalties there must not reach the sums."""
    batch, rows, vocab = 2, 3, 2050
    c = rules_case(12, batch, rows, vocab, 20, 0, False)
    c["start"] = np.array([0, 2, 4])
    c["bias_id"], c["bias"] = np.array([2050, 4095, 2051, 3000]), np.array([np.inf, np.nan, np.inf, np.inf], np.float32)
    c["history"][:, :3] = [2050, 4095, 2060]
    c["n"][:] = 20
    c["tokens"][:] = 2055
    c["penalty"][:] = [0.0, -np.inf, np.nan]
    c["history"][:, 3:] = 2070
    got = run_rules(gpu, c, False, penalty=True)
    check_rules(c, False, *got)
    assert np.isfinite(got[2][got[2] != 77]).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("off", ["penalty", "bias", "allow", "history", "mask", "count", "all"])
def test_rules_left_out(gpu, off, f16):
    c = rules_case(4, 3, 6, 9001, 40, 20, f16)
    on = {x: off not in (x, "all") for x in ("penalty", "bias", "allow", "history", "mask", "count")}
    check_rules(c, f16, *run_rules(gpu, c, f16, **on), **on)
    on["from_"] = 13
    check_rules(c, f16, *run_rules(gpu, c, f16, **on), **on)


@pytest.mark.parametrize("f16", [False, True])
def test_rules_odd_values(gpu, f16):
    """Ties (the first one), rows with nothing left, NaN and infinities in allowed and in masked places, ids and lengths
    past their ends, one id many times in text and biases."""
    batch, rows, vocab = 4, 6, 9000
    c = rules_case(5, batch, rows, vocab, 50, 40, f16)
    c["n"], c["count"] = np.array([1000, -3, 50, 20]), np.array([6, 6, 1000, 0])
    c["history"][0] = 17
    c["history"][2, :10] = [vocab, vocab + 1, 0x7FFFFFFF, 0xFFFFFFFF, 0xFFFFFFFE, 4095, 4096, 8191, 8192, 8999]
    c["tokens"][1] = 8999
    c["tokens"][0, :2] = [0xFFFFFFFF, 9000]
    c["bias_id"][c["start"][1]:c["start"][2]] = 4097
    c["bias_id"][c["start"][2]:c["start"][2] + 2] = [0xFFFFFFFF, 9000]
    c["allow"][:] |= np.random.default_rng(6).random(c["allow"].shape) < 0.4
    x = c["logits"]
    x[0, [5000, 100, 8000]] = 60000  # (three equal maxima)
    c["allow"][0, [5000, 100, 8000]] = True
    c["allow"][1] = False
    x[2] = -np.inf
    x[3, 50], x[3, 51] = np.nan, np.inf
    c["allow"][3, 50:52] = False
    x[4, 7], c["allow"][4, 7] = np.nan, True
    x[5, 9], c["allow"][5, 9] = np.inf, True
    x[6] = -60000
    c["allow"][7] = np.arange(vocab) == 8999
    x[8] = np.nan
    check_rules(c, f16, *run_rules(gpu, c, f16))
    _, pick, lp = run_rules(gpu, c, f16)
    assert pick[1] == NONE and lp[1] == -np.inf and pick[8] == NONE
    assert pick[7] == 8999 and lp[7] == 0
    assert np.isnan(lp[4]) and np.isnan(lp[5]) and pick[5] == 9


def test_rules_outputs_alone(gpu):
    """Each output by itself gives what they give together."""
    c = rules_case(7, 2, 4, 6000, 30, 10, False)
    o, pick, lp = run_rules(gpu, c, False)
    a, p, l = run_rules(gpu, c, False, pick=False, logprob=False)
    assert np.array_equal(a, o) and np.all(p == 77) and np.all(l == 77)
    a, p, l = run_rules(gpu, c, False, out="none", logprob=False)
    assert np.array_equal(p, pick) and np.all(l == 77)
    a, p, l = run_rules(gpu, c, False, out="none", pick=False)
    assert np.array_equal(l, lp) and np.all(p == 77)


# ------------------------------------------------------------------------------------------- the kept path


def plain_accept(parents, tokens, picks, count, n, room):
    """One sequence's walk: the kept nodes and the token after them."""
    path, node = [], 0 if count else None
    while node is not None and len(path) < room:
        path.append(node)
        node = next((i for i in range(node + 1, count) if parents[i] == node and tokens[i] == picks[node] and picks[node] != NONE), None)
    return path, (picks[path[-1]] if path else tokens[0]) if count else None


def run_accept(gpu, seed, batch, rows, layers, d, cols, in16, n=None, count=None, history_more=0, in_place=False, move=True,
               history=True, stride_more=0, vocab=4):
    rng = np.random.default_rng(seed)
    parents, seen = trees(rng, batch, rows, 1 if vocab == 1 else 3)
    tokens, picks = rng.integers(0, vocab, (2, batch, rows)).astype(np.uint32)
    picks[0, rows // 2] = NONE
    n = rng.integers(0, cols + 1, batch) if n is None else np.asarray(n)
    count = rng.integers(0, rows + 1, batch) if count is None else np.asarray(count)
    dt = np.float16 if in16 else np.float32
    x = (300 * rng.standard_normal((layers, batch, rows, 2 * d + stride_more))).astype(dt)
    if not in16:
        x.reshape(-1)[:: max(1, x.size // 50)] = 1e6  # past f16's range: infinity, as wh_pack has it
    words = 0x3C003C00 + rng.integers(0, 99, (layers, batch, cols * d)).astype(np.uint32)
    hcols = cols + history_more
    text = rng.integers(0, 99, (batch, hcols)).astype(np.uint32)
    up = lambda a, t: gpu.upload(np.ascontiguousarray(a, t))  # noqa: E731
    xb, kvb, hb = gpu.upload(x), gpu.upload(words), gpu.upload(text)
    nb, cb, tb, pb, mb = up(n, np.int32), up(count, np.int32), up(tokens, np.uint32), up(picks, np.uint32), gpu.upload(bits(seen))
    path, kept, nxt, n_out = (gpu.upload(np.full(s, 55, np.uint32)) for s in ((batch, rows), batch, batch, batch))
    if in_place:
        n_out = nb
    stride = x.shape[3]
    t = wa.Tree(batch, rows, nb, cb, tb, mb, bits(seen)[0].size)
    gpu.tree_accept(t, pb, xb, xb.ptr + x.itemsize * d, stride, batch * rows * stride, kvb if move else None, cols * d,
                    batch * cols * d, layers, cols, d, path, kept, nxt, n_out, hb if history else None, hcols, in16)
    got = {"path": gpu.read(path, (batch, rows), np.int32), "kept": gpu.read(kept, (batch,), np.int32),
           "next": gpu.read(nxt, (batch,), np.uint32), "n": gpu.read(n_out, (batch,), np.int32),
           "text": gpu.read(hb, text.shape, np.uint32), "kv": gpu.read(kvb, words.shape, np.uint32)}
    lengths = []
    for b in range(batch):
        nn, c = min(max(n[b], 0), cols), min(max(count[b], 0), rows)
        p, after = plain_accept(parents[b], tokens[b], picks[b], c, nn, max(0, min(cols, hcols if history else cols) - nn))
        lengths.append(len(p))
        assert got["path"][b].tolist() == p + [-1] * (rows - len(p)), f"sequence {b}"
        assert got["kept"][b] == len(p) and got["n"][b] == nn + len(p)
        assert got["next"][b] == (55 if after is None else after)
        if history:
            text[b, nn:nn + len(p)] = tokens[b, p]
        if move and p:
            for l in range(layers):
                k, v = half(x[l, b, p, :d]), half(x[l, b, p, d:2 * d])
                w = words[l, b].view(np.float16)
                w[:cols * d].reshape(d // 2, cols, 2)[:, nn:nn + len(p)] = k.reshape(len(p), d // 2, 2).transpose(1, 0, 2)
                w[cols * d:].reshape(cols, d)[nn:nn + len(p)] = v
    assert np.array_equal(got["text"], text)
    assert np.array_equal(got["kv"], words)
    return lengths


ACCEPT = [(1, 1, 1, 2, 1), (1, 1, 3, 64, 5), (5, 7, 2, 130, 40), (3, 33, 1, 600, 100), (2, 64, 4, 256, 448), (2, 200, 2, 34, 33), (1, 1024, 1, 8, 2000)]


@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("shape", ACCEPT, ids=lambda s: "x".join(str(x) for x in s))
def test_accept(gpu, shape, in16):
    batch, rows, layers, d, cols = shape
    for seed in range(3):
        run_accept(gpu, seed, *shape, in16, stride_more=2 * seed)
    # Long paths (chains of one token), no room, room for a part, nothing there.
    assert max(run_accept(gpu, 9, *shape, in16, n=[0] * batch, count=[rows] * batch, vocab=1)) >= min(cols, rows // 2 + 1)
    run_accept(gpu, 10, *shape, in16, n=[cols] * batch, count=[rows] * batch, vocab=1)
    run_accept(gpu, 11, *shape, in16, n=[max(0, cols - 2)] * batch, count=[rows + 5] * batch, vocab=1)
    run_accept(gpu, 12, *shape, in16, n=[-7] * batch, count=[-1] * batch)


@pytest.mark.parametrize("in_place", [False, True])
def test_accept_forms(gpu, in_place):
    shape = (6, 30, 3, 96, 64)
    run_accept(gpu, 1, *shape, False, in_place=in_place)
    run_accept(gpu, 2, *shape, False, in_place=in_place, move=False)
    run_accept(gpu, 3, *shape, False, in_place=in_place, history=False)
    run_accept(gpu, 4, *shape, False, in_place=in_place, history_more=-9, vocab=1)
    run_accept(gpu, 5, *shape, True, in_place=in_place, history_more=9, vocab=1)
    run_accept(gpu, 6, *shape, False, in_place=in_place, move=False, history=False)


def test_accept_root_alone_in_place(gpu):
    """Steps without drafts: the next tokens take the roots' place, their lengths grow, the texts get what they were."""
    batch, steps = 5, 3
    picks = np.arange(100, 100 + batch * steps, dtype=np.uint32).reshape(steps, batch)
    tokens, n = gpu.upload(np.arange(batch, dtype=np.uint32)), gpu.upload(np.array([0, 1, 2, 8, 9], np.int32))
    mask, text = gpu.upload(np.ones((batch, 1), np.uint32)), gpu.upload(np.full((batch, 10), 7, np.uint32))
    path, kept = gpu.buffer(batch), gpu.buffer(batch)
    for p in picks:
        pb = gpu.upload(p)
        gpu.tree_accept(wa.Tree(batch, 1, n, None, tokens, mask, 1), pb, None, None, 0, 0, None, 0, 0, 0, 10, 0, path, kept, tokens, n,
                        text, 10)
    got = gpu.read(text, (batch, 10), np.uint32)
    for b, first in enumerate((0, 1, 2, 8, 9)):
        made = [b, *picks[:, b].tolist()]
        room = min(steps, 10 - first)
        assert got[b].tolist() == [7] * first + made[:room] + [7] * (10 - first - room)
        assert gpu.read(n, (batch,), np.int32)[b] == first + room
        assert gpu.read(tokens, (batch,), np.uint32)[b] == made[room]


def test_accept_one_tree_for_all(gpu):
    """mask_stride 0, and two children with one token: the first counts."""
    batch, rows = 3, 6
    parents = [0, 0, 0, 1, 2, 4]
    seen = np.zeros((1, rows, rows), bool)
    for i in range(rows):
        seen[0, i, i] = True
        if i:
            seen[0, i] |= seen[0, parents[i]]
    tokens = np.array([[9, 5, 5, 6, 6, 7]] * 3, np.uint32)
    picks = np.array([[5, 6, 6, 8, 7, 3], [4, 6, 6, 8, 7, 3], [5, 7, 6, 8, 7, 3]], np.uint32)
    want = [([0, 1, 3], 8), ([0], 4), ([0, 1], 7)]
    tb, pb, mb, nb = gpu.upload(tokens), gpu.upload(picks), gpu.upload(bits(seen)), gpu.upload(np.zeros(batch, np.int32))
    path, kept, nxt, out = (gpu.buffer(n) for n in (batch * rows, batch, batch, batch))
    gpu.tree_accept(wa.Tree(batch, rows, nb, None, tb, mb, 0), pb, None, None, 0, 0, None, 0, 0, 0, 10, 0, path, kept, nxt, out)
    p = gpu.read(path, (batch, rows), np.int32)
    for b, (nodes, after) in enumerate(want):
        assert p[b].tolist() == nodes + [-1] * (rows - len(nodes))
    assert gpu.read(nxt, (batch,), np.uint32).tolist() == [after for _, after in want]
    assert gpu.read(out, (batch,), np.int32).tolist() == [3, 1, 2]


# -------------------------------------------------------------------------------------- together, recorded


class Decoder:
    """A decoder of two attention layers over the framework's ops, for a batch of trees: embedding rows, [q | k | v]
    projections, attention over the caches and the tree, output projections, logits, the rules and the kept path."""

    def __init__(self, gpu, batch, rows, heads=4, kv_heads=2, hd=32, vocab=160, cols=90, layers=2, seed=0):
        rng = np.random.default_rng(seed)
        self.gpu, self.batch, self.rows, self.heads, self.kv_heads, self.hd = gpu, batch, rows, heads, kv_heads, hd
        self.vocab, self.cols, self.layers, self.d = vocab, cols, layers, heads * hd
        d, dk = self.d, kv_heads * hd
        lin = lambda n, k, s: gpu.linear([((s * rng.standard_normal((n, k))).astype(np.float32).tobytes(), wa.F32, k, n)])  # noqa: E731
        self.embed = lin(vocab, d, 1.0)
        self.qkv = [lin(d + 2 * dk, d, 2.0 / np.sqrt(d)) for _ in range(layers)]
        self.proj = [lin(d, d, 1.0 / np.sqrt(d)) for _ in range(layers)]
        self.head = lin(vocab, d, 3.0 / np.sqrt(d))
        self.pos = gpu.upload((0.5 * rng.standard_normal((cols + rows, d))).astype(np.float32))
        self.stride = d + 2 * dk
        assert self.qkv[0].width == self.stride and self.head.width == vocab
        m = batch * rows
        self.x, self.rowsb = gpu.buffer(m * d), gpu.buffer(layers * m * self.stride)
        self.o, self.logits = gpu.buffer(m * d), gpu.buffer(m * vocab)
        self.kv = gpu.buffer(layers * batch * cols * dk)
        self.kv_words, self.dk = cols * dk, dk
        z = lambda *s: gpu.upload(np.zeros(s, np.int32))  # noqa: E731
        self.n, self.count, self.tokens, self.mask = z(batch), z(batch), z(batch, rows), z(batch, rows, (rows + 31) // 32)
        self.pick, self.path, self.kept, self.next = z(batch, rows), z(batch, rows), z(batch), z(batch)
        self.history = z(batch, cols)
        self.penalty = gpu.upload(np.array([[1.2, 0.1, 0.05]] * batch, np.float32))
        self.start = gpu.upload(np.arange(batch + 1, dtype=np.int32))
        self.bias_id, self.bias = gpu.upload(np.arange(batch, dtype=np.int32)), gpu.upload(np.full(batch, 0.5, np.float32))
        allow = np.ones((m, 32 * ((vocab + 31) // 32)), bool)
        allow[:, 3:vocab:17] = False
        self.allow = gpu.upload(np.packbits(allow, axis=-1, bitorder="little"))
        gpu.zero(self.kv)

    def tree(self):
        return wa.Tree(self.batch, self.rows, self.n, self.count, self.tokens, self.mask, self.rows * ((self.rows + 31) // 32))

    def embeddings(self, depths):
        for r in range(self.batch * self.rows):
            self.gpu.embed(self.embed, self.pos, self.x.ptr + 4 * r * self.d, self.tokens, r, int(depths.reshape(-1)[r]) * self.d)

    def step(self):
        """Everything after the embeddings: queued, nothing waited for."""
        g, m, t = self.gpu, self.batch * self.rows, self.tree()
        for l in range(self.layers):
            at = self.rowsb.ptr + 4 * l * m * self.stride
            g.gemm(self.x, self.qkv[l], at, m, wa.BIAS)
            g.tree_attend(t, at, at + 4 * self.d, at + 4 * (self.d + self.dk), self.stride,
                          self.kv.ptr + 4 * l * self.batch * self.kv_words, self.kv_words, self.cols, self.o, self.heads,
                          self.kv_heads, self.hd)
            g.gemm(self.o, self.proj[l], self.x, m, wa.RESIDUAL, 1.0)
        g.gemm(self.x, self.head, self.logits, m, wa.BIAS)
        g.logit_rules(t, wa.Rules(self.penalty, self.history, self.cols, 0, self.start, self.bias_id, self.bias, self.batch, self.allow),
                      self.logits, self.logits, self.vocab, self.vocab, pick=self.pick)
        g.tree_accept(t, self.pick, self.rowsb.ptr + 4 * self.d, self.rowsb.ptr + 4 * (self.d + self.dk), self.stride,
                      m * self.stride, self.kv, self.kv_words, self.batch * self.kv_words, self.layers, self.cols, self.dk,
                      self.path, self.kept, self.next, self.n, self.history, self.cols)

    def generate(self, rng, want, drafts, record=False):
        """Tokens of every sequence up to `want`, drafting from `drafts` (what the undrafted decoder gave) with mistakes.
        The replays of a recorded step have the device's lengths, trees and texts of their time."""
        g, batch, rows = self.gpu, self.batch, self.rows
        g.write(self.n, np.zeros(batch, np.int32))
        root = np.arange(batch) + 20
        text = [[] for _ in range(batch)]
        steps, recorded = 0, None
        while min(len(x) for x in text) < want:
            parents, seen = trees(rng, batch, rows, 4)
            tokens, count = np.zeros((batch, rows), np.int64), np.zeros(batch, np.int64)
            depth = seen.sum(2) - 1
            for b in range(batch):
                tokens[b, 0] = root[b]
                count[b] = 0 if len(text[b]) >= want else rng.integers((rows + 1) // 2, rows + 1)
                for i in range(1, rows):
                    at = len(text[b]) + depth[b, i]
                    right = drafts is not None and at < len(drafts[b]) and rng.random() < 0.6
                    tokens[b, i] = drafts[b][at] if right else rng.integers(0, self.vocab)
            g.write(self.tokens, tokens.astype(np.uint32))
            g.write(self.count, count.astype(np.int32))
            g.write(self.mask, bits(seen))
            self.embeddings(np.array([[len(text[b]) + depth[b, i] for i in range(rows)] for b in range(batch)]))
            if record and recorded is None and steps == 1:
                g.record_begin()
                self.step()
                recorded = g.record_end()
            if recorded is None:
                self.step()
            else:
                recorded.replay()
            kept, path, nxt = g.read(self.kept, (batch,), np.int32), g.read(self.path, (batch, rows), np.int32), g.read(self.next, (batch,), np.uint32)
            for b in range(batch):
                text[b] += [int(tokens[b, i]) for i in path[b, :kept[b]]]
                if count[b]:
                    root[b] = nxt[b]
            steps += 1
        assert np.array_equal(g.read(self.n, (batch,), np.int32), [len(x) for x in text])
        assert all(g.read(self.history, (batch, self.cols), np.uint32)[b, :len(text[b])].tolist() == text[b] for b in range(batch))
        return [x[:want] for x in text], steps


@pytest.mark.parametrize("record", [False, True])
def test_drafted_decoding_gives_the_same_tokens(gpu, record):
    """Trees of drafted tokens, right and wrong ones, against one token per step: the same texts in fewer steps.  The
    two differ by rounding alone (rows of other batch sizes), so the seed's texts have no ties at that level."""
    want, _ = Decoder(gpu, 3, 1).generate(np.random.default_rng(1), 40, None)
    got, steps = Decoder(gpu, 3, 11).generate(np.random.default_rng(2), 40, want, record)
    assert got == want
    assert steps < 30
    assert len(set(want[0])) > 10  # (the penalties keep it from repeating itself)


def test_recorded_passes_share_the_scratch(gpu):
    """Two passes recorded on one context, of sizes whose partial results overlap in its scratch, replayed in turn with
    other lengths, other rows and eager work between: every replay equals the eager call."""
    rng = np.random.default_rng(3)
    sets = []
    for batch, rows, heads, hd, cols in ((2, 9, 4, 64, 3000), (1, 20, 8, 128, 700)):
        d = heads * hd
        q = gpu.upload(rng.standard_normal((batch, rows, 3 * d)).astype(np.float32))
        kv = gpu.upload(half(rng.standard_normal((batch, 2 * cols * d))))
        n, mask = gpu.upload(np.array([cols - 7] * batch, np.int32)), gpu.upload(bits(trees(rng, batch, rows)[1]))
        o, logits, pick = gpu.buffer(batch * rows * d), gpu.upload(rng.standard_normal((batch * rows, 9000)).astype(np.float32)), gpu.buffer(batch * rows)
        t = wa.Tree(batch, rows, n, None, None, mask, rows * ((rows + 31) // 32))

        def call(t=t, q=q, kv=kv, o=o, logits=logits, pick=pick, d=d, cols=cols, heads=heads, hd=hd):
            gpu.tree_attend(t, q, q.ptr + 4 * d, q.ptr + 8 * d, 3 * d, kv, cols * d, cols, o, heads, heads, hd)
            gpu.logit_rules(t, wa.Rules(), logits, None, 9000, 9000, pick=pick)

        sets.append((call, batch, rows, d, cols, n, q, o, pick))
    for s in sets:
        s[0]()
    passes = []
    for s in sets:
        gpu.record_begin()
        s[0]()
        passes.append(gpu.record_end())
    for turn in range(4):
        for s, p in zip(sets, passes):
            call, batch, rows, d, cols, n, q, o, pick = s
            gpu.write(n, np.array([max(0, cols - 700 * turn)] * batch, np.int32))
            gpu.write(q, rng.standard_normal((batch, rows, 3 * d)).astype(np.float32))
            call()
            want = gpu.read(o, (batch, rows, d)), gpu.read(pick, (batch * rows,), np.uint32)
            gpu.zero(o)
            gpu.zero(pick)
            p.replay()
            if turn % 2:
                sets[0][0]()  # eager work behind it
            assert np.array_equal(gpu.read(o, (batch, rows, d)), want[0])
            assert np.array_equal(gpu.read(pick, (batch * rows,), np.uint32), want[1])
    for p in passes:
        p.free()


def test_rules_calls_in_a_row(gpu):
    """Small calls whose last workgroup joins the parts, many behind each other over the same scratch, with other rows and
    row counts each: a part read before it is there, or one of an earlier call, gives another pick."""
    batch, rows, vocab, sets, calls = 3, 4, 30011, 5, 60
    rng = np.random.default_rng(13)
    x = (3 * rng.standard_normal((sets, batch * rows, vocab))).astype(np.float32)
    count = rng.integers(1, rows + 1, (sets, batch)).astype(np.int32)
    xb, cb, nb = [gpu.upload(a) for a in x], [gpu.upload(a) for a in count], gpu.upload(np.zeros(batch, np.int32))
    pick, logprob = gpu.upload(np.full((calls, batch * rows), 77, np.uint32)), gpu.upload(np.full((calls, batch * rows), 77, np.float32))
    for i in range(calls):
        gpu.logit_rules(wa.Tree(batch, rows, nb, cb[i % sets]), wa.Rules(), xb[i % sets], None, vocab, vocab,
                        pick=pick.ptr + 4 * i * batch * rows, logprob=logprob.ptr + 4 * i * batch * rows)
    p, l = gpu.read(pick, (calls, batch, rows), np.uint32), gpu.read(logprob, (calls, batch, rows))
    y = x.astype(np.float64)
    there = np.arange(rows) < count[:, :, None]
    best = np.where(there, x.argmax(2).reshape(sets, batch, rows), 77)
    total = -np.log(np.exp(y - y.max(2, keepdims=True)).sum(2)).reshape(sets, batch, rows)
    for i in range(calls):
        assert np.array_equal(p[i], best[i % sets])
        # (as in check_rules, with rest / (1 + rest) < 1 and a log1p below 16)
        assert np.all(np.abs(l[i] - np.where(there[i % sets], total[i % sets], 77)) <= 104 * 2.0**-23 + 2.0**-21 + 64 * EPS + 2.0**-18)


@pytest.mark.parametrize("batch,rows,vocab", [(3, 4, 30011), (1, 20, 9000), (5, 1, 51866), (2, 64, 4097), (60, 3, 20000)])
@pytest.mark.parametrize("shift", [0, 1, -1])
def test_rules_picks_in_the_tokens_place(gpu, batch, rows, vocab, shift):
    """Picks written over the tokens that the penalties count (or a place off them): those of picks of their own.  Rows of
    one sequence in several workgroups must have read their tokens before the first of them is through."""
    c = rules_case(15, batch, rows, vocab, 40, 10, False)
    c["count"][:] = rows
    total = batch * rows
    x, n, mask = gpu.upload(c["logits"]), gpu.upload(c["n"].astype(np.int32)), gpu.upload(bits(c["seen"]))
    penalty, text = gpu.upload(c["penalty"]), gpu.upload(c["history"].astype(np.uint32))
    rules = wa.Rules(penalty, text, c["history"].shape[1])
    tokens = np.full(total + 2, 5, np.uint32)
    tokens[1:total + 1] = c["tokens"].reshape(-1)
    tb, own, logprob = gpu.upload(tokens), gpu.buffer(total), gpu.buffer(total)
    tree = wa.Tree(batch, rows, n, None, tb.ptr + 4, mask, rows * ((rows + 31) // 32))
    gpu.logit_rules(tree, rules, x, None, vocab, vocab, pick=own, logprob=logprob)
    want, prob = gpu.read(own, (total,), np.uint32), gpu.read(logprob, (total,))
    for _ in range(5):
        gpu.write(tb, tokens)
        gpu.logit_rules(tree, rules, x, None, vocab, vocab, pick=tb.ptr + 4 + 4 * shift, logprob=logprob)
        got = gpu.read(tb, (total + 2,), np.uint32)
        assert np.array_equal(got[1 + shift:1 + shift + total], want)
        assert got[:1 + shift].tolist() == tokens[:1 + shift].tolist()
        assert got[1 + shift + total:].tolist() == tokens[1 + shift + total:].tolist()
        assert np.array_equal(gpu.read(logprob, (total,)), prob)


def test_two_contexts(gpu):
    """The same calls queued on two contexts (streams) at once, without waits between."""
    other = wa.Gpu(0)
    try:
        rng = np.random.default_rng(4)
        batch, rows, heads, hd, cols = 2, 12, 4, 64, 2000
        d = heads * hd
        q = rng.standard_normal((batch, rows, 3 * d)).astype(np.float32)
        kv, n, mask = half(rng.standard_normal((batch, 2 * cols * d))), np.array([cols, 900], np.int32), bits(trees(rng, batch, rows)[1])
        logits = rng.standard_normal((batch * rows, 20000)).astype(np.float32)
        got = {}
        sets = []
        for g in (gpu, other):
            b = [g.upload(x) for x in (q, kv, n, mask, logits)] + [g.buffer(batch * rows * d), g.buffer(batch * rows)]
            sets.append((g, b, wa.Tree(batch, rows, b[2], None, None, b[3], rows)))
        for _ in range(5):
            for g, b, t in sets:
                g.tree_attend(t, b[0], b[0].ptr + 4 * d, b[0].ptr + 8 * d, 3 * d, b[1], cols * d, cols, b[5], heads, heads, hd)
                g.logit_rules(t, wa.Rules(), b[4], None, 20000, 20000, pick=b[6])
        got = [(g.read(b[5], (batch, rows, d)), g.read(b[6], (batch * rows,), np.uint32)) for g, b, t in sets]
        assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
        assert np.array_equal(got[0][1], logits.argmax(1))
    finally:
        other.close()


def test_refused_calls_leave_the_context_usable(gpu):
    c = rules_case(8, 1, 2, 100, 5, 3, False)
    with pytest.raises(wa.WavoError) as e:
        gpu.tree_attend(wa.Tree(1, 2, None), 1 << 20, None, None, 64, 1 << 20, 64, 1, 1 << 20, 1, 1, 64)
    assert e.value.code == wa.EARG
    check_rules(c, False, *run_rules(gpu, c, False))


def test_recording_needs_the_scratch_first(gpu):
    """As every op with scratch: a first call inside a recording that would have to grow it is refused."""
    other = wa.Gpu(0)
    try:
        x, p, n = other.buffer(5000), other.buffer(1), other.upload(np.zeros(1, np.int32))
        t = wa.Tree(1, 1, n)
        other.record_begin()
        with pytest.raises(wa.WavoError) as e:
            other.logit_rules(t, wa.Rules(), x, None, 5000, 5000, pick=p)
        assert "recording" in str(e.value)
        other.record_end().free()
        other.zero(x)
        other.logit_rules(t, wa.Rules(), x, None, 5000, 5000, pick=p)
        assert other.read(p, (1,), np.uint32)[0] == 0
    finally:
        other.close()
