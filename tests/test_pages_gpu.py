"""Sampled decoding over caches in pages on the device (wh_head_norm, wh_page_append, wh_page_read, wh_page_attend,
wh_logit_probs, wh_tree_sample) against plain 64-bit numpy forms of their definitions.

Tolerances are worst cases of the arithmetic, with eps = 2^-24 (half a step of f32) and 2^-11 (half a step of f16).  What is
stored in pages is compared word for word: its keys are computed in 64 bits, whose last bits cross a border of f16 or of 4
bits for one value in 1e10."""

import numpy as np
import pytest

import wavo_amd as wa
from test_tree_gpu import EPS, EPS16, attend_tolerance, bits, half, trees

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
TILE = 32

# ------------------------------------------------------------------------------------------- plain forms


def turned(x, gain, eps, table, rot, pairs, position):
    """Heads x [rows][heads][hd] of positions [rows], in 64 bits."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * gain.astype(np.float64)
    if table is not None:
        t = table.astype(np.float64)[np.clip(position, 0, len(table) - 1)][:, None]
        cos, sin = t[..., :rot // 2], t[..., rot // 2:]
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
        a, b = x[..., i], x[..., j]
        y = x.copy()
        y[..., i], y[..., j] = a * cos - b * sin, b * cos + a * sin
        x = y
    return x


def rope_table(positions, rot):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def quantized(x):
    """f16 values [..., 32 c] in 4 bits: nibbles and factors [..., c]."""
    x = x.astype(np.float16).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", divide="ignore"):
        size = np.abs(x).max(-1)
        d = (np.where((x == size[..., None]).any(-1), size, -size) / -8).astype(np.float16) + np.float16(0)  # (no zero below zero)
        w = d.astype(np.float64)[..., None]
        nib = np.where(w == 0, 8, np.clip(np.floor(x / np.where(w == 0, 1, w) + 8.5), 0, 15))
    odd = ~np.isfinite(x).all(-1)
    d[odd] = np.nan
    return np.where(odd[..., None], 0, nib).astype(np.uint32), d


class Cache:
    """Caches of `batch` sequences in pages, on the host: values by position, and the pool's words."""

    def __init__(self, rng, type, page, kv_heads, hd, batch, cols, spare=2, shared=False):
        self.type, self.page, self.kv_heads, self.hd, self.cols = type, page, kv_heads, hd, cols
        self.pages = (1 if shared else batch) * cols + spare
        self.table = rng.permutation(self.pages)[:self.pages - spare].reshape(-1, cols).astype(np.int32)
        self.tiles = page // TILE
        self.words = 9 * hd if type == wa.Q4_0 else 32 * hd
        # Every bit pattern, infinities and NaN among them, where nothing was stored.
        self.pool = rng.integers(0, 2**32, (self.pages, kv_heads, self.tiles, self.words), dtype=np.uint32)
        z = hd // 32
        p, d = np.arange(TILE)[:, None], np.arange(hd)[None, :]
        g = p % 16 // 4
        k = (16 * (d % 32 // 8) + p % 16, 2 * (d // 32) + p // 16, d % 8 + 0 * p)  # lane, word, element
        v = (16 * g + d % 32 // 2, 2 * (d // 32) + d % 2 + 0 * p, 4 * (p // 16) + p % 4 + 0 * d)
        self.factor = (g * z + np.arange(z)[None, :]) * 8 + 4 * (p // 16) + p % 4  # [32][z]
        self.at = []
        for lane, t, e in (k, v):
            if type == wa.Q4_0:
                whole = 2 * z // 4 * 4
                word = np.where(t < whole, t // 4 * 256 + lane * 4 + t % 4, whole * 64 + lane * 2 + t - whole)
                self.at.append((word, 4 * (e // 2 + 4 * (e % 2))))
            else:
                self.at.append(((t * 64 + lane) * 8 + e, None))

    def place(self, b, j):
        """Page (or None), tile and position of position j of sequence b."""
        page = int(self.table[b if len(self.table) > 1 else 0, j // self.page])
        return (page if 0 <= page < self.pages else None), j % self.page // TILE, j % TILE

    def store(self, b, j, k, v):
        """f16 values [kv_heads][hd] at position j of sequence b, as the device has to."""
        page, tile, p = self.place(b, j)
        if page is None:
            return
        for which, x in enumerate((k, v)):
            words = self.pool[page, :, tile]
            if self.type == wa.F16:
                words.view(np.float16)[:, self.at[which][0][p] + which * 32 * self.hd] = x
                continue
            first = which * (4 * self.hd + self.hd // 2)
            nib, d = quantized(x)
            word, shift = (y[p] for y in self.at[which])
            fine = np.repeat(np.isfinite(d), 32, -1)  # (nibbles beside a NaN factor: any)
            for h in range(self.kv_heads):
                w = words[h, first:first + 4 * self.hd]
                for i in range(self.hd):
                    if fine[h, i]:
                        w[word[i]] = (w[word[i]] & ~np.uint32(15 << shift[i])) | nib[h].reshape(-1)[i] << np.uint32(shift[i])
                words[h].view(np.float16)[2 * (first + 4 * self.hd) + self.factor[p]] = d[h]

    def load(self, b, j):
        """The values that position j stands for, [2][kv_heads][hd] in 64 bits; None where no page is there."""
        page, tile, p = self.place(b, j)
        if page is None:
            return None
        out = []
        for which in range(2):
            words = self.pool[page, :, tile]
            if self.type == wa.F16:
                out.append(words.view(np.float16)[:, self.at[which][0][p] + which * 32 * self.hd].astype(np.float64))
                continue
            first = which * (4 * self.hd + self.hd // 2)
            word, shift = (y[p] for y in self.at[which])
            nib = words[:, first + word] >> shift.astype(np.uint32) & 15
            d = words.view(np.float16)[:, 2 * (first + 4 * self.hd) + self.factor[p]].astype(np.float64)
            out.append((nib.astype(np.float64) - 8) * np.repeat(d, 32, -1))
        return np.stack(out)

    def device(self, gpu):
        self.pool_buffer, self.table_buffer = gpu.upload(self.pool), gpu.upload(self.table)
        return wa.Pages(self.pool_buffer, self.pages, self.table_buffer, self.cols, 0 if len(self.table) == 1 else self.cols, self.page,
                        self.type, self.kv_heads, self.hd)

    def read_back(self, gpu):
        return gpu.read(self.pool_buffer, self.pool.shape, np.uint32)

    def fill(self, rng, n, scale=1.0):
        """Values at the first n[b] positions, straight into the words: any nibbles and plausible factors, or halfs."""
        for b, nn in enumerate(n):
            for j in range(min(max(int(nn), 0), self.cols * self.page)):
                page, tile, p = self.place(b, j)
                if page is None:
                    continue
                w = self.pool[page, :, tile]
                for which in range(2):
                    if self.type == wa.F16:
                        w.view(np.float16)[:, self.at[which][0][p] + which * 32 * self.hd] = scale * rng.standard_normal((self.kv_heads, self.hd))
                    else:
                        first = which * (4 * self.hd + self.hd // 2)
                        d = rng.choice([-0.25, 0.25], (self.kv_heads, self.hd // 32)) * np.exp(0.3 * rng.standard_normal((self.kv_heads, self.hd // 32)))
                        w.view(np.float16)[:, 2 * (first + 4 * self.hd) + self.factor[p]] = scale * d


def same_words(cache, got):
    bad = np.argwhere(got != cache.pool)
    assert not len(bad), f"{len(bad)} words differ, the first at {bad[0]}: {got[tuple(bad[0])]:#x} for {cache.pool[tuple(bad[0])]:#x}"


def rows_of(rng, batch, rows, heads, kv_heads, hd, in16, more=0):
    x = rng.standard_normal((batch, rows, (heads + 2 * kv_heads) * hd + more)).astype(np.float16 if in16 else np.float32)
    return x


# ------------------------------------------------------------------------------------------- norms and rotation


def norm_tolerance(x, gain, hd):
    """The squares' sum has hd + 2 roundings, which the square root halves; quotient, gain and rotation 10 more of values up
    to sqrt(2) times the head's largest."""
    size = np.abs(x).max(-1, keepdims=True).astype(np.float64)
    if gain is not None:
        size = np.sqrt(hd) * np.abs(gain).max()
    return 2 * size * (hd / 2 + 12) * EPS


@pytest.mark.parametrize("heads,kv_heads,hd,rot,pairs,norm", [
    (1, 1, 8, 8, False, True), (3, 1, 40, 40, False, True), (5, 5, 40, 16, True, True), (20, 20, 64, 64, False, True), (8, 2, 64, 64, True, False),
    (32, 8, 128, 128, False, True), (6, 3, 128, 32, False, False), (4, 2, 80, 40, False, True), (4, 4, 96, 96, True, True), (2, 1, 256, 256, False, True),
    (2, 2, 256, 64, True, True), (9, 3, 64, 0, False, True), (7, 7, 48, 0, False, False), (1, 1, 200, 200, False, True)])
@pytest.mark.parametrize("in16,out16", [(False, False), (True, True), (False, True)])
def test_head_norm(gpu, heads, kv_heads, hd, rot, pairs, norm, in16, out16):
    rng = np.random.default_rng(heads * 1000 + hd + rot)
    batch, rows, more = 3, 5, 2
    x = rows_of(rng, batch, rows, heads, kv_heads, hd, in16, more)
    x[1, 1] *= 1e-3
    x[2, 0] = 0
    d, stride = (heads + 2 * kv_heads) * hd, x.shape[-1]
    gq, gk = ((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2))
    table = rope_table(50, rot) if rot else None
    n, count = np.array([0, 44, 17], np.int32), np.array([5, 4, 2], np.int32)
    _, seen = trees(rng, batch, rows)
    for tree in (False, True):
        mask = bits(seen)
        y = gpu.upload(np.full((batch, rows, d + 4), 7, np.float16 if out16 else np.float32))
        keep = [None if z is None else gpu.upload(z) for z in (gq, gk, table, n, count, mask, x)]
        t = wa.Tree(batch, rows, keep[3], keep[4], None, keep[5] if tree else None, mask[0].size)
        gpu.head_norm(t, wa.Heads(heads, kv_heads, hd, keep[0], keep[1], 1e-6, keep[2], 50 if rot else 0, rot, pairs), keep[6], stride, y, d + 4,
                      in16, out16)
        got = gpu.read(y, (batch, rows, d + 4), np.float16 if out16 else np.float32)
        assert np.all(got[..., d:] == 7)
        for b in range(batch):
            c = count[b]
            assert np.all(got[b, c:] == 7)
            depth = seen[b, :c, :c].sum(1) - 1 if tree else np.arange(c)
            hx = x[b, :c, :d].reshape(c, -1, hd)
            for part, gain in ((slice(0, heads), gq), (slice(heads, heads + kv_heads), gk)):
                want = turned(hx[:, part], gain, 1e-6, table, rot, pairs, n[b] + depth)
                tol = norm_tolerance(hx[:, part], gain, hd)
                if out16:
                    tol = tol + EPS16 * np.abs(want) + 2.0**-25
                err = np.abs(got[b, :c, :d].reshape(c, -1, hd)[:, part] - want)
                assert np.all(err <= tol), f"{np.max(err / tol):.2f} of what is allowed"
            with np.errstate(over="ignore"):
                assert np.array_equal(got[b, :c, (heads + kv_heads) * hd:d], x[b, :c, (heads + kv_heads) * hd:d].astype(got.dtype))


def test_head_norm_in_place_keeps_values_and_gaps(gpu):
    rng = np.random.default_rng(3)
    for in16 in (False, True):
        x = rows_of(rng, 2, 7, 6, 2, 64, in16, 6)
        gain, table, n = (gpu.upload(a) for a in (np.ones(64, np.float32), rope_table(300, 64), np.array([290, 0], np.int32)))
        heads = wa.Heads(6, 2, 64, gain, gain, 0.0, table, 300, 64)
        a, b = gpu.upload(x), gpu.upload(x)
        gpu.head_norm(wa.Tree(2, 7, n), heads, a, x.shape[-1], b, x.shape[-1], in16, in16)
        gpu.head_norm(wa.Tree(2, 7, n), heads, a, x.shape[-1], a, x.shape[-1], in16, in16)
        one, two = gpu.read(a, x.shape, x.dtype), gpu.read(b, x.shape, x.dtype)
        assert np.array_equal(one, two)
        assert np.array_equal(one[..., 8 * 64:], x[..., 8 * 64:])


def test_head_norm_deep_trees_and_many_rows(gpu):
    """Depths by masks of many words; a head of its own norm only; no gains for keys."""
    rng = np.random.default_rng(4)
    rows, hd = 1024, 32
    _, seen = trees(rng, 1, rows, 3)
    x = rows_of(rng, 1, rows, 1, 1, hd, False)
    table, gain = rope_table(1200, hd), np.ones(hd, np.float32)
    keep = [gpu.upload(a) for a in (x, table, gain, np.array([100], np.int32), bits(seen))]
    y = gpu.buffer(x.size)
    gpu.head_norm(wa.Tree(1, rows, keep[3], None, None, keep[4], 0), wa.Heads(1, 1, hd, keep[2], None, 1e-6, keep[1], 1200, hd), keep[0], 3 * hd, y, 3 * hd)
    got = gpu.read(y, x.shape)[0].reshape(rows, 3, hd)
    pos = 100 + seen[0].sum(1) - 1
    hx = x[0].reshape(rows, 3, hd)
    for h, g in ((0, gain), (1, None)):
        want = turned(hx[:, h:h + 1], g, 1e-6, table, hd, False, pos)[:, 0]
        assert np.all(np.abs(got[:, h] - want) <= norm_tolerance(hx[:, h], g, hd))


# ------------------------------------------------------------------------------------------- appending and reading


def append(gpu, cache, x, heads, n, count=None, path=None, kept=None, gq=None, gk=None, table=None, rot=0, pairs=False, q=True, out16=None):
    """wh_page_append over numpy rows [q | k | v]; (queries or None, n_out)."""
    batch, rows = x.shape[:2]
    hd, g, in16 = cache.hd, cache.kv_heads, x.dtype == np.float16
    out16 = in16 if out16 is None else out16
    pages = cache.device(gpu)
    xb = gpu.upload(x)
    up = lambda a, t: None if a is None else gpu.upload(np.asarray(a, t))  # noqa: E731
    nb, cb, pb, kb = up(n, np.int32), up(count, np.int32), up(path, np.int32), up(kept, np.int32)
    h = wa.Heads(heads, g, hd, up(gq, np.float32), up(gk, np.float32), 1e-6, up(table, np.float32), 0 if table is None else len(table), rot, pairs)
    qo = gpu.upload(np.full((batch, rows, heads * hd), 7, np.float16 if out16 else np.float32)) if q else None
    no = gpu.upload(np.full(batch, -5, np.int32))
    gpu.page_append(wa.Tree(batch, rows, nb, cb), h, xb if q else None, xb.ptr + x.itemsize * heads * hd, xb.ptr + x.itemsize * (heads + g) * hd,
                    x.shape[-1], pages, pb, kb, qo, heads * hd, no, in16, out16)
    return (gpu.read(qo, (batch, rows, heads * hd), np.float16 if out16 else np.float32) if q else None), gpu.read(no, (batch,), np.int32)


def expect(cache, x, heads, n, count, path=None, gk=None, table=None, rot=0, pairs=False):
    """The same on the host: the cache's words, and n_out."""
    batch, rows = x.shape[:2]
    hd, g, room = cache.hd, cache.kv_heads, cache.cols * cache.page
    out = []
    for b in range(batch):
        nn, c = min(max(int(n[b]), 0), room), min(max(int(count[b]), 0), rows)
        end = min(nn + c, room)
        out.append(end)
        for i in range(end - nn):
            r = i if path is None else int(path[b][i])
            if not 0 <= r < rows:
                continue
            kv = x[b, r, heads * hd:(heads + 2 * g) * hd].reshape(2 * g, hd)
            with np.errstate(over="ignore"):
                k = turned(kv[None, :g], gk, 1e-6, table, rot, pairs, np.array([nn + i]))[0].astype(np.float32).astype(np.float16)
                cache.store(b, nn + i, k, kv[g:].astype(np.float16))
    return out


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,hd,page,rot,pairs,norm", [
    (2, 1, 32, 32, 32, False, True), (6, 3, 64, 64, 64, False, True), (4, 4, 64, 32, 16, True, False), (3, 3, 96, 128, 96, False, True), (3, 1, 96, 32, 48, False, True),
    (4, 2, 96, 32, 96, True, True), (8, 2, 128, 256, 128, False, True), (5, 5, 128, 32, 64, False, False), (2, 2, 128, 64, 8, False, True), (1, 1, 128, 32, 0, False, False)])
def test_append(gpu, type, in16, heads, kv_heads, hd, page, rot, pairs, norm):
    rng = np.random.default_rng(hd + page + rot)
    batch, rows, cols = 5, 70, 256 // page + 1
    cache = Cache(rng, type, page, kv_heads, hd, batch, cols)
    n = [0, 31, 33, cols * page - 40, cols * page]  # (the last two have less room than rows, and none)
    count = [70, 1, 70, 70, 3]
    x = rows_of(rng, batch, rows, heads, kv_heads, hd, in16, 2)
    gq, gk = ((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) if norm else None for _ in range(2))
    table = rope_table(300, rot) if rot else None
    q, n_out = append(gpu, cache, x, heads, n, count, gq=gq, gk=gk, table=table, rot=rot, pairs=pairs)
    want = expect(cache, x, heads, n, count, gk=gk, table=table, rot=rot, pairs=pairs)
    assert n_out.tolist() == want
    same_words(cache, cache.read_back(gpu))
    for b in range(batch):
        c = count[b]
        assert np.all(q[b, c:] == 7)
        hx = x[b, :c, :heads * hd].reshape(c, heads, hd)
        w = turned(hx, gq, 1e-6, table, rot, pairs, min(n[b], cols * page) + np.arange(c))
        tol = norm_tolerance(hx, gq, hd) + (EPS16 * np.abs(w) + 2.0**-25 if in16 else 0)
        assert np.all(np.abs(q[b, :c].reshape(c, heads, hd) - w) <= tol)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_token_by_token_as_at_once(gpu, type):
    """A page filled position by position holds the words of one filled in one call, and all tokens before it stay."""
    rng = np.random.default_rng(8)
    heads = hd = 64
    cache = Cache(rng, type, 32, 2, hd, 1, 3)
    x = rows_of(rng, 1, 67, heads, 2, hd, False)
    gain, table = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32), rope_table(100, hd)
    start = cache.pool.copy()
    append(gpu, cache, x, heads, [5], gk=gain, gq=gain, table=table, rot=hd)
    once = cache.read_back(gpu)
    cache.pool = start
    pages = cache.device(gpu)
    keep = [gpu.upload(a) for a in (gain, table, x)]
    h = wa.Heads(heads, 2, hd, None, keep[0], 1e-6, keep[1], 100, hd)
    for i in range(67):
        n = gpu.upload(np.array([5 + i], np.int32))
        row = keep[2].ptr + 4 * (i * x.shape[-1] + heads * hd)
        gpu.page_append(wa.Tree(1, 1, n), h, None, row, row + 4 * 2 * hd, x.shape[-1], pages)
    assert np.array_equal(once, cache.read_back(gpu))


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_append_of_a_path(gpu, type):
    rng = np.random.default_rng(9)
    batch, rows, heads, g, hd = 6, 40, 2, 2, 64
    cache = Cache(rng, type, 32, g, hd, batch, 2)
    cache.table[1, 1] = -1          # pages that are not there
    cache.table[2, 0] = cache.pages
    n, kept = [3, 25, 10, 40, 0, 60], [4, 20, 9, 100, 0, 30]
    path = np.full((batch, rows), -1, np.int32)
    for b in range(batch):
        c = min(kept[b], rows)
        path[b, :c] = np.sort(rng.permutation(rows)[:c])
    path[0, 2] = rows       # entries of no row: nothing stored there
    path[3, 5] = -7
    x = rows_of(rng, batch, rows, heads, g, hd, True)
    _, n_out = append(gpu, cache, x, heads, n, None, path, kept, q=False)
    assert n_out.tolist() == expect(cache, x, heads, n, kept, path)
    same_words(cache, cache.read_back(gpu))


def test_4_bits_of_odd_blocks(gpu):
    """Zeros, borders between nibbles, equal magnitudes of both signs, the smallest numbers, and numbers that are not finite."""
    rng = np.random.default_rng(10)
    hd, rows = 128, 64
    cache = Cache(rng, wa.Q4_0, 64, 1, hd, 1, 1)
    x = rng.standard_normal((rows, 3, hd))
    x[0] = 0
    x[1] = -0.0
    x[2] = rng.choice([-1, 1], (3, hd))
    x[3] = rng.integers(-16, 17, (3, hd)) / 16  # every border of d = 1 / 8
    x[4] = rng.integers(-16, 17, (3, hd)) * 3 / 16
    x[5] = rng.integers(-16, 17, (3, hd)) * 2.0**-24
    x[6] = rng.integers(-3, 4, (3, hd)) * 2.0**-24
    x[7] = 65504 * rng.choice([-1, 1, 0.5, 0.4375], (3, hd))
    x[8] = rng.integers(-1023, 1024, (3, hd)) * 2.0**-20
    for i in range(9, 40):
        x[i] = rng.integers(-2048, 2049, (3, hd)) * 2.0**rng.integers(-14, 4)
        x[i, :, ::32] = rng.integers(1024, 2048, (3, 4)) / 64.0 * rng.choice([-1, 1])
        x[i, :, 1::32] = x[i, :, ::32] * (2 * rng.integers(-8, 9, (3, 4)) + 1) / 16  # at borders, where f16 holds them
    x = x.astype(np.float16).reshape(1, rows, 3 * hd)
    append(gpu, cache, x, 1, [0], q=False)
    expect(cache, x, 1, [0], [rows])
    same_words(cache, cache.read_back(gpu))
    # A number that is not finite takes the 32 values that it stands among, and nothing else.
    y = x.copy()
    y[0, 50, hd + 5], y[0, 51, 2 * hd + 40], y[0, 52, hd + 127], y[0, 53, 2 * hd] = np.inf, np.nan, -np.inf, -np.nan
    append(gpu, cache, y, 1, [0], q=False)
    k, v, n = gpu.upload(np.zeros((rows, hd), np.float32)), gpu.upload(np.zeros((rows, hd), np.float32)), gpu.upload(np.zeros(1, np.int32))
    gpu.page_read(wa.Tree(1, rows, n), wa.Pages(cache.pool_buffer, cache.pages, cache.table_buffer, 1, 1, 64, wa.Q4_0, 1, hd), k, v, hd)
    got = np.stack([gpu.read(k, (rows, hd)), gpu.read(v, (rows, hd))])
    want = np.stack([cache.load(0, j)[:, 0] for j in range(rows)], 1)
    want[0, 50, :32] = want[1, 51, 32:64] = want[0, 52, 96:] = want[1, 53, :32] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("hd,g,page,out16", [(32, 3, 32, False), (64, 2, 128, True), (96, 1, 64, False), (128, 2, 32, True)])
def test_read(gpu, type, hd, g, page, out16):
    rng = np.random.default_rng(hd + page)
    batch, rows, cols = 4, 50, 3
    cache = Cache(rng, type, page, g, hd, batch, cols)
    cache.table[2, 1] = -1
    cache.fill(rng, [cols * page] * batch)
    n, count = [0, 31, page - 3, cols * page - 7], [50, 3, 50, 50]
    dt = np.float16 if out16 else np.float32
    kb, vb = (gpu.upload(np.full((batch, rows, g * hd + 2), 7, dt)) for _ in range(2))
    nb, cb = (gpu.upload(np.array(a, np.int32)) for a in (n, count))
    gpu.page_read(wa.Tree(batch, rows, nb, cb), cache.device(gpu), kb, vb, g * hd + 2, out16)
    got = np.stack([gpu.read(a, (batch, rows, g * hd + 2), dt) for a in (kb, vb)])
    want = np.full(got.shape, 7, dt)
    for b in range(batch):
        for i in range(count[b]):
            at = cache.load(b, n[b] + i) if n[b] + i < cols * page else None
            want[:, b, i, :g * hd] = 0 if at is None else at.reshape(2, -1)
    assert np.array_equal(got, want)


# ------------------------------------------------------------------------------------------- attention


def attend(gpu, cache, x, heads, n, count=None, seen=None, out16=False, nodes=True, mask=None, before=7.0):
    batch, rows = x.shape[:2]
    hd, g, in16 = cache.hd, cache.kv_heads, x.dtype == np.float16
    xb, nb = gpu.upload(x), gpu.upload(np.asarray(n, np.int32))
    cb = None if count is None else gpu.upload(np.asarray(count, np.int32))
    mask = bits(seen) if mask is None and seen is not None else mask
    mb = None if mask is None else gpu.upload(mask)
    ob = gpu.upload(np.full((batch, rows, heads * hd), before, np.float16 if out16 else np.float32))
    k, v = (xb.ptr + x.itemsize * y * hd if nodes else None for y in (heads, heads + g))
    t = wa.Tree(batch, rows, nb, cb, None, mb, 0 if mask is None else mask[0].size)
    gpu.page_attend(t, xb, k, v, x.shape[-1], cache.device(gpu), ob, heads, in16, out16)
    return gpu.read(ob, (batch, rows, heads * hd), np.float16 if out16 else np.float32)


def check_attend(got, cache, x, heads, n, count=None, seen=None, nodes=True, before=7.0):
    """Softmax over the positions of pages that are there and the seen nodes, row by row, with a worst case of its error: that of
    caches that are not in pages, and, of p * d in two f16 parts or (f16 rows and outputs) p and V (of 4 bits) rounded to f16: 2^-11
    each of the values' size, and 2^-25 at most where they are subnormal, of weights whose largest is at least 2^10 (less the
    power of two of V's largest factor, which is below the largest value)."""
    batch, rows = x.shape[:2]
    hd, g, room = cache.hd, cache.kv_heads, cache.cols * cache.page
    p16 = got.dtype == np.float16 and x.dtype == np.float16
    for b in range(batch):
        c = rows if count is None else min(max(int(count[b]), 0), rows)
        nn = min(max(int(n[b]), 0), room)
        kept = [z for z in (cache.load(b, j) for j in range(nn)) if z is not None]
        kept = np.stack(kept) if kept else np.zeros((0, 2, g, hd))
        kv = x[b, :c, heads * hd:(heads + 2 * g) * hd].astype(np.float16).astype(np.float64).reshape(c, 2, g, hd)
        for i in range(c):
            sees = [j for j in range(c) if nodes and seen is not None and seen[b, i, j]]
            both = np.concatenate([kept, kv[sees]])
            for h in range(heads):
                row = got[b, i, h * hd:(h + 1) * hd].astype(np.float64)
                if not len(both):
                    assert np.all(row == 0)
                    continue
                q = x[b, i, h * hd:(h + 1) * hd].astype(np.float64)
                kk, vv = both[:, 0, h // (heads // g)], both[:, 1, h // (heads // g)]
                s = kk @ q / np.sqrt(hd)
                p = np.exp(s - s.max())
                want = p @ vv / p.sum()
                size = np.abs(vv).max()
                tol = attend_tolerance(q, kk, vv, hd) + len(both) * 2.0**-32 * max(1, size)
                if p16:
                    tol += (2 * EPS16 + EPS16**2 + len(both) * 2.0**-35 * max(1, size)) * size
                if got.dtype == np.float16:
                    tol = tol + EPS16 * np.abs(want) + 2.0**-25
                err = np.abs(row - want)
                assert np.all(err <= tol), f"sequence {b} node {i} head {h}: {err.max():.3e}, {np.max(err / tol):.2f} of what is allowed"
        assert np.all(got[b, c:] == before), f"sequence {b}: rows past its {c} nodes written"


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16,out16", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("heads,kv_heads,hd,rows,page,cols,n", [
    (1, 1, 64, 1, 32, 1, [0, 1, 32]), (2, 2, 32, 3, 32, 3, [31, 33, 96]), (4, 2, 96, 5, 64, 2, [65, 0, 128]), (8, 2, 128, 6, 32, 6, [170, 191, 5]),
    (3, 3, 64, 33, 128, 1, [100, 64, 7]), (6, 1, 128, 9, 256, 1, [250, 3, 129]), (2, 1, 64, 40, 64, 2, [90, 31, 0])])
def test_attend(gpu, type, in16, out16, heads, kv_heads, hd, rows, page, cols, n):
    rng = np.random.default_rng(heads + hd + rows + page)
    batch = 3
    cache = Cache(rng, type, page, kv_heads, hd, batch, cols)
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, kv_heads, hd, in16, 2)
    x[..., :heads * hd] *= 2
    _, seen = trees(rng, batch, rows)
    count = [rows, (rows + 1) // 2, rows]
    check_attend(attend(gpu, cache, x, heads, n, count, seen, out16), cache, x, heads, n, count, seen)
    # Cross attention: the pages alone.
    check_attend(attend(gpu, cache, x, heads, n, count, None, out16, nodes=False), cache, x, heads, n, count, None, nodes=False)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_attend_masks_that_leave_nothing_and_nodes_that_are_not_finite(gpu, type):
    """Any bits for masks; rows that see nothing get zeros; what nobody sees may hold anything."""
    rng = np.random.default_rng(20)
    batch, rows, heads, g, hd = 2, 70, 4, 2, 64
    cache = Cache(rng, type, 32, g, hd, batch, 4)
    n = [0, 50]
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, g, hd, False)
    seen = rng.random((batch, rows, rows)) < 0.1
    seen[:, 5] = seen[:, 37] = False
    odd = [7, 40, 69]
    seen[:, :, odd] = False
    for i, value in zip(odd, (np.nan, np.inf, 1e30)):
        x[:, i, heads * hd:] = value
    x[0, 8, :heads * hd] = np.nan  # a query of its own trouble
    count = [70, 66]
    mask = bits(seen)
    mask[..., -1] |= np.uint32(0xFFFFFFC0)  # bits of nodes that are not there
    got = attend(gpu, cache, x, heads, n, count, seen, mask=mask)
    got[0, 8], x[0, 8, :heads * hd] = 7, 0
    assert np.all(np.isfinite(got))
    keep = got[0, 8].copy()
    one = attend(gpu, cache, np.where(np.isfinite(x), x, 0), heads, n, count, seen, mask=mask)
    one[0, 8] = keep
    assert np.array_equal(got, one)  # whatever stood in them
    x = np.where(np.isfinite(x), x, 0)
    got = attend(gpu, cache, x, heads, n, count, seen, mask=mask)
    check_attend(got, cache, x, heads, n, count, seen)
    # Seen infinities of V reach the rows that see them, and no others.
    y = x.copy()
    y[1, 9, (heads + g) * hd:] = np.inf
    seen[1, 10, 9] = True
    see = seen[1, :, 9]
    got2 = attend(gpu, cache, y, heads, n, count, seen)
    assert np.all(np.isinf(got2[1, :66][see[:66]]) | np.isnan(got2[1, :66][see[:66]]))
    assert np.array_equal(got2[1, :66][~see[:66]], got[1, :66][~see[:66]])


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_attend_pages_that_are_not_there(gpu, type):
    rng = np.random.default_rng(21)
    batch, rows, heads, g, hd, page, cols = 3, 2, 4, 2, 128, 32, 40
    cache = Cache(rng, type, page, g, hd, batch, cols)
    n = [cols * page, 700, 40]
    cache.table[0, [0, 1, 2, 9, 17, 18, 39]] = -1
    cache.table[0, 20] = cache.pages
    cache.table[1, :30] = -2**31  # none at all
    cache.table[2, 1] = 2**31 - 1
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, g, hd, True)
    _, seen = trees(rng, batch, rows)
    got = attend(gpu, cache, x, heads, n, None, seen, True)
    check_attend(got, cache, x, heads, n, None, seen)
    got = attend(gpu, cache, x, heads, n, None, None, True, nodes=False)
    assert np.all(got[1] == 0)
    check_attend(got, cache, x, heads, n, None, None, nodes=False)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16", [False, True])
def test_attend_long_caches_in_splits(gpu, type, in16):
    """Few rows over long tables: workgroups share a sequence's tiles, of which some have none; one table for all."""
    rng = np.random.default_rng(22)
    batch, rows, heads, g, hd, page, cols = 3, 2, 2, 1, 64, 64, 64
    cache = Cache(rng, type, page, g, hd, batch, cols, shared=True)
    n = [cols * page, 1, 2500]
    cache.fill(rng, [cols * page])
    x = rows_of(rng, batch, rows, heads, g, hd, in16)
    x[..., :heads * hd] *= 3
    _, seen = trees(rng, batch, rows)
    check_attend(attend(gpu, cache, x, heads, n, [2, 0, 1], seen, in16), cache, x, heads, n, [2, 0, 1], seen)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("in16,out16", [(False, False), (True, True), (True, False)])
@pytest.mark.parametrize("heads,kv_heads,hd,rows", [(2, 1, 64, 33), (3, 3, 32, 20), (2, 1, 96, 30), (2, 2, 128, 64), (6, 2, 128, 5)])
def test_attend_long_caches_shared_out(gpu, type, in16, out16, heads, kv_heads, hd, rows):
    """Blocks of all sizes over tables that are shared out: sequences of nothing, of little, of no nodes, pages that are not there."""
    rng = np.random.default_rng(heads + hd + rows)
    batch, page, cols = 6, 256, 9
    cache = Cache(rng, type, page, kv_heads, hd, batch, cols)
    n, count = [cols * page, 0, 1500, 700, 33, 2000], [rows, rows, (rows + 1) // 2, 0, 1, rows]
    cache.table[0, [0, 3, 4, 8]] = -1
    cache.table[5] = cache.pages
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, kv_heads, hd, in16, 2)
    x[..., :heads * hd] *= 2
    _, seen = trees(rng, batch, rows)
    seen[0, rows // 2] = False
    check_attend(attend(gpu, cache, x, heads, n, count, seen, out16), cache, x, heads, n, count, seen)
    got = attend(gpu, cache, x, heads, n, count, None, out16, nodes=False)
    assert np.all(got[5] == 0)
    check_attend(got, cache, x, heads, n, count, None, nodes=False)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("batch,few", [(64, False), (65, False), (150, False), (200, True)])
def test_attend_many_sequences_shared_out(gpu, type, batch, few):
    """More sequences than are looked at together; those with something to do few and far between."""
    rng = np.random.default_rng(batch)
    rows, heads, g, hd, page, cols = 3, 2, 1, 32, 128, 18
    cache = Cache(rng, type, page, g, hd, batch, cols, shared=True)
    n = np.where(rng.random(batch) < 0.7, rng.integers(0, 100, batch), rng.integers(0, cols * page + 1, batch))
    count = np.where(rng.random(batch) < (0.02 if few else 0.7), rng.integers(1, rows + 1, batch), 0)
    count[-1] = 2
    cache.fill(rng, [cols * page])
    x = rows_of(rng, batch, rows, heads, g, hd, True)
    _, seen = trees(rng, batch, rows)
    check_attend(attend(gpu, cache, x, heads, n, count, seen, True), cache, x, heads, n, count, seen)
    none = attend(gpu, cache, x, heads, n, np.zeros(batch), seen, True)
    assert np.all(none == 7)


def test_attend_recorded_passes_share_the_scratch(gpu):
    """Two passes whose parts overlap in the scratch, replayed in turn with other lengths, and eager work between."""
    rng = np.random.default_rng(26)
    sets = []
    for type, batch, rows, heads, g, hd in ((wa.Q4_0, 3, 5, 4, 2, 64), (wa.F16, 2, 40, 2, 1, 128)):
        cache = Cache(rng, type, 256, g, hd, batch, 10)
        cache.fill(rng, [2560] * batch)
        pages, n = cache.device(gpu), gpu.upload(np.array([2500] * batch, np.int32))
        x, mask = gpu.upload(rows_of(rng, batch, rows, heads, g, hd, False)), gpu.upload(bits(trees(rng, batch, rows)[1]))
        o, t = gpu.buffer(batch * rows * heads * hd), wa.Tree(batch, rows, n, None, None, mask, rows * ((rows + 31) // 32))

        def call(t=t, x=x, pages=pages, o=o, heads=heads, g=g, hd=hd):
            gpu.page_attend(t, x, x.ptr + 4 * heads * hd, x.ptr + 4 * (heads + g) * hd, (heads + 2 * g) * hd, pages, o, heads)

        sets.append((call, n, batch, o, batch * rows * heads * hd, cache, mask))
    for s in sets:
        s[0]()
    passes = []
    for s in sets:
        gpu.record_begin()
        s[0]()
        passes.append(gpu.record_end())
    for turn in range(4):
        for (call, n, batch, o, size, *_), p in zip(sets, passes):
            gpu.write(n, np.array([2560 - 640 * turn, 100][:batch] + [7] * (batch - 2), np.int32))
            call()
            want = gpu.read(o, (size,))
            gpu.zero(o)
            p.replay()
            if turn % 2:
                sets[0][0]()
            assert np.array_equal(gpu.read(o, (size,)), want)
    for p in passes:
        p.free()


@pytest.mark.parametrize("in16", [False, True])
@pytest.mark.parametrize("scale", [1e-4, 30.0, 4000.0, 60000.0])
def test_attend_factors_of_any_size(gpu, in16, scale):
    """V's factors from the smallest to f16's largest, the large ones late, so that what came before is brought to their scale."""
    rng = np.random.default_rng(23)
    batch, rows, heads, g, hd, page, cols = 2, 3, 2, 2, 64, 32, 24
    cache = Cache(rng, wa.Q4_0, page, g, hd, batch, cols)
    n = [cols * page, 300]
    cache.fill(rng, n)
    first = 4 * hd + hd // 2 + 4 * hd
    for b, j in ((0, 5), (0, 300), (0, 767), (1, 40), (1, 299)):
        pg, tile, p = cache.place(b, j)
        cache.pool[pg, :, tile].view(np.float16)[:, 2 * first + cache.factor[p]] = scale * rng.uniform(0.3, 1, (g, hd // 32))
    x = rows_of(rng, batch, rows, heads, g, hd, in16)
    _, seen = trees(rng, batch, rows)
    check_attend(attend(gpu, cache, x, heads, n, None, seen), cache, x, heads, n, None, seen)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("scale", [1e-4, 100.0, 8188.0])
def test_attend_values_of_any_size_in_f16(gpu, type, scale):
    """f16 rows and outputs: values up to f16's largest (8188 times -8 in 4 bits) among ordinary ones, keys as they were."""
    rng = np.random.default_rng(27)
    batch, rows, heads, g, hd, page, cols = 2, 20, 2, 2, 64, 32, 12
    cache = Cache(rng, type, page, g, hd, batch, cols)
    n = [cols * page, 100]
    cache.fill(rng, n)
    for b, j in ((0, 5), (0, 300), (0, 383), (1, 40), (1, 99)):
        pg, tile, p = cache.place(b, j)
        half_words = cache.pool[pg, :, tile].view(np.float16)
        if type == wa.Q4_0:
            half_words[:, 2 * (8 * hd + hd // 2) + cache.factor[p]] = scale * rng.uniform(0.3, 1, (g, hd // 32))
        else:
            half_words[:, cache.at[1][0][p] + 32 * hd] = 8 * scale * rng.uniform(-1, 1, (g, hd))
    x = rows_of(rng, batch, rows, heads, g, hd, True)
    _, seen = trees(rng, batch, rows)
    check_attend(attend(gpu, cache, x, heads, n, None, seen, True), cache, x, heads, n, None, seen)


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
@pytest.mark.parametrize("size", [1e-6, 300.0, 3e4])
def test_attend_scores_far_apart(gpu, type, size):
    rng = np.random.default_rng(24)
    batch, rows, heads, g, hd, page, cols = 2, 4, 4, 2, 64, 32, 10
    cache = Cache(rng, type, page, g, hd, batch, cols)
    n = [320, 100]
    cache.fill(rng, n)
    x = rows_of(rng, batch, rows, heads, g, hd, False)
    x[..., :heads * hd] *= size
    _, seen = trees(rng, batch, rows)
    got = attend(gpu, cache, x, heads, n, None, seen)
    if size < 1e4:
        check_attend(got, cache, x, heads, n, None, seen)
    assert np.all(np.isfinite(got))


def test_attend_repeats_itself_in_recorded_passes(gpu):
    """Append, attention and the next lengths recorded once: replays follow the lengths on the device, with eager calls between."""
    rng = np.random.default_rng(25)
    batch, heads, g, hd, page, cols = 2, 4, 2, 64, 32, 80
    cache = Cache(rng, wa.Q4_0, page, g, hd, batch, cols)
    n0 = [1000, 31]
    cache.fill(rng, n0)
    x = rows_of(rng, batch, 1, heads, g, hd, False)
    table = rope_table(2000, hd)
    pages = cache.device(gpu)
    keep = [gpu.upload(a) for a in (x, table, np.array(n0, np.int32))]
    n1, qo, o = gpu.buffer(batch), gpu.buffer(batch * heads * hd), gpu.buffer(batch * heads * hd)
    h = wa.Heads(heads, g, hd, None, None, 0.0, keep[1], 2000, hd)
    row = x.shape[-1]

    def step():
        gpu.page_append(wa.Tree(batch, 1, keep[2]), h, keep[0], keep[0].ptr + 4 * heads * hd, keep[0].ptr + 4 * (heads + g) * hd, row, pages, qo=qo,
                        qo_stride=heads * hd, n_out=n1)
        gpu.page_attend(wa.Tree(batch, 1, n1), qo, None, None, heads * hd, pages, o, heads)
        gpu.copy(keep[2], n1, 4 * batch)

    eager = []
    for _ in range(4):
        step()
        eager.append(gpu.read(o, (batch, heads * hd)))
    words = cache.read_back(gpu)
    gpu.write(keep[2], np.array(n0, np.int32))
    gpu.write(cache.pool_buffer, cache.pool)
    gpu.record_begin()
    step()
    p = gpu.record_end()
    other = Cache(rng, wa.F16, 32, 1, 32, 1, 1)
    for i in range(4):
        p.replay()
        assert np.array_equal(gpu.read(o, (batch, heads * hd)), eager[i])
        other.fill(rng, [20])
        attend(gpu, other, rows_of(rng, 1, 1, 1, 1, 32, False), 1, [20], None, None, nodes=False)
    assert np.array_equal(gpu.read(keep[2], (batch,), np.int32), np.array(n0) + 4)
    assert np.array_equal(cache.read_back(gpu), words)
    p.free()


# ------------------------------------------------------------------------------------------- probabilities


def probs(gpu, l, batch, rows, vocab, temperature=None, count=None, gap=0, before=7.0):
    ld, out_ld = l.shape[-1], vocab + gap
    keep = [gpu.upload(a) for a in (l, np.zeros(batch, np.int32))]
    tb = None if temperature is None else gpu.upload(np.asarray(temperature, np.float32))
    cb = None if count is None else gpu.upload(np.asarray(count, np.int32))
    y = gpu.upload(np.full((batch * rows, out_ld), before, np.float32))
    gpu.logit_probs(wa.Tree(batch, rows, keep[1], cb), keep[0], y, vocab, ld, out_ld, tb, l.dtype == np.float16)
    return gpu.read(y, (batch * rows, out_ld))


@pytest.mark.parametrize("half_in", [False, True])
@pytest.mark.parametrize("batch,rows,vocab,ld,gap", [(1, 1, 1, 1, 0), (1, 1, 51866, 51904, 38), (2, 3, 1000, 1001, 1), (3, 2, 33, 35, 0), (1, 5, 131071, 131072, 3), (30, 20, 4097, 4097, 0),
                                                     (2, 1, 300007, 300008, 0)])
def test_probs(gpu, half_in, batch, rows, vocab, ld, gap):
    rng = np.random.default_rng(vocab)
    l = (5 * rng.standard_normal((batch * rows, ld))).astype(np.float16 if half_in else np.float32)
    l[:, vocab:] = np.nan  # (past the row)
    l[rng.random(l.shape) < 0.01] = -np.inf
    l[0, 0] = 3
    temperature = rng.uniform(0.1, 2, batch).astype(np.float32)
    count = rng.integers(1, rows + 1, batch)
    got = probs(gpu, l, batch, rows, vocab, temperature, count, gap)
    assert np.all(got[:, vocab:] == 7)
    for r in range(batch * rows):
        b, i = divmod(r, rows)
        if i >= count[b]:
            assert np.all(got[r] == 7)
            continue
        x = l[r, :vocab].astype(np.float64)
        z = (x - x.max()) / np.float64(temperature[b])
        want = np.exp(z)
        total = want.sum()
        # The exponent's argument has three roundings of its size (in binary digits), its power and the quotient 2^-22; the sum of
        # as many terms a thread, then of threads.
        size = np.abs(np.where(np.isfinite(z), z, 0)) * 1.4427
        rel = size * 3 * EPS + 2.0**-21 + (want * size).sum() / total * 3 * EPS + (vocab / 1024 + 30) * EPS
        assert np.all(np.abs(got[r, :vocab] - want / total) <= want / total * rel + 1e-37)


def test_probs_of_odd_rows(gpu):
    """Nothing left, one left, ties at temperature zero, NaN and infinity, temperatures of all kinds."""
    vocab = 5000
    l = np.random.default_rng(1).standard_normal((8, vocab)).astype(np.float32)
    l[0] = -np.inf
    l[1] = -np.inf
    l[1, 4321] = -1e30
    l[2, [70, 4000, 4999]] = 9
    l[3, 17] = np.nan
    l[4, 17] = np.inf
    l[5, [3, 2]] = 50
    got = probs(gpu, l, 8, 1, vocab, [0.7, 0.5, 0, 1, 1, 1e-30, -1, np.nan])
    assert np.all(got[0] == 0)
    assert got[1, 4321] == 1 and got[1].sum() == 1
    assert got[2, 70] == 1 and got[2].sum() == 1
    assert np.all(np.isnan(got[3])) and np.isnan(got[4, 17])
    assert got[5, 2] == got[5, 3] == 0.5 and got[5].sum() == 1
    for r in (6, 7):
        assert got[r, l[r].argmax()] == 1 and got[r].sum() == 1
    assert np.all(probs(gpu, l[:1], 1, 1, vocab, [0.0])[0] == 0)  # nothing left, greedily


def test_probs_of_temperatures_without_end(gpu):
    """All that is left alike, and nothing of what is not."""
    l = np.float32(np.random.default_rng(2).standard_normal((3, 4100)))
    l[:, 100:] = -np.inf
    got = probs(gpu, l, 3, 1, 4100, [np.inf, 3e38, 1e30])
    assert np.all(np.abs(got[:, :100] - 0.01) <= 0.01 * 2.0**-20) and np.all(got[:, 100:] == 0)


# ------------------------------------------------------------------------------------------- verification


def walk(p, q, tokens, parent, u, vocab):
    """One sequence, in 64 bits: picks."""
    rows = len(tokens)
    picks = np.full(rows, NONE, np.uint32)
    at, w, total = 0, p[0].astype(np.float64), 1.0
    for i in range(1, rows):
        if parent[i] != at or not total > 0 or tokens[i] >= vocab:
            continue
        x = tokens[i]
        if float(u[i]) * (1.0 if q is None else float(q[at, x])) * total < w[x]:
            picks[at] = x
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
    over = np.flatnonzero((c > float(u[0]) * c[-1]) & (w > 0))
    picks[at] = over[0] if len(over) else NONE
    return picks


def sample(gpu, p, q, tokens, u, vocab, mask=None, mask_stride=None, count=None, before=5):
    batch, rows, ld = p.shape
    up = lambda a, t: None if a is None else gpu.upload(np.asarray(a, t))  # noqa: E731
    keep = [up(p, np.float32), up(q, np.float32), up(tokens, np.uint32), up(u, np.float32), up(mask, np.uint32), up(count, np.int32),
            up(np.zeros(batch), np.int32)]
    picks = gpu.upload(np.full((batch, rows), before, np.uint32))
    t = wa.Tree(batch, rows, keep[6], keep[5], keep[2], keep[4], 0 if mask is None else mask[0].size if mask_stride is None else mask_stride)
    gpu.tree_sample(t, keep[0], keep[1], vocab, ld, keep[3], picks)
    return gpu.read(picks, (batch, rows), np.uint32)


def softmax(x):
    with np.errstate(under="ignore"):
        e = np.exp(x - x.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def drafted(rng, batch, rows, vocab, ld, peak=4.0, noise=0.7, spread=4):
    """p, q, tokens drawn from q, parents, masks, random numbers."""
    x = peak * rng.standard_normal((batch, rows, ld))
    x[..., vocab:] = -np.inf
    p, q = softmax(x), softmax(x + noise * rng.standard_normal(x.shape))
    p[..., vocab:] = q[..., vocab:] = np.nan
    parents, seen = trees(rng, batch, rows, spread)
    tokens = np.zeros((batch, rows), np.uint32)
    for b in range(batch):
        for i in range(1, rows):
            c = np.cumsum(q[b, parents[b, i], :vocab].astype(np.float64))
            tokens[b, i] = min(np.searchsorted(c, rng.random() * c[-1]), vocab - 1)
    return p, q, tokens, parents, bits(seen), rng.random((batch, rows)).astype(np.float32)


@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("batch,rows,vocab,ld,spread", [(1, 1, 1, 1, 1), (3, 1, 1000, 1001, 1), (9, 12, 7, 7, 4), (8, 33, 50, 64, 3), (5, 24, 3001, 3003, 7), (2, 9, 51866, 51904, 2), (3, 5, 131071, 131072, 4),
                                                        (40, 6, 999, 999, 5), (2, 70, 4, 4, 70)])
def test_sample(gpu, drafts, batch, rows, vocab, ld, spread):
    rng = np.random.default_rng(batch + rows + vocab)
    p, q, tokens, parents, mask, u = drafted(rng, batch, rows, vocab, ld, spread=spread)
    count = rng.integers((rows + 1) // 2, rows + 1, batch)
    got = sample(gpu, p, q if drafts else None, tokens, u, vocab, mask, count=count)
    for b in range(batch):
        c = count[b]
        want = walk(p[b, :c, :vocab], q[b, :c, :vocab] if drafts else None, tokens[b, :c], parents[b], u[b], vocab)
        assert np.array_equal(got[b, :c], want), f"sequence {b}"
        assert np.all(got[b, c:] == 5)


def test_sample_a_chain_without_masks(gpu):
    rng = np.random.default_rng(5)
    p, q, tokens, _, _, u = drafted(rng, 30, 8, 500, 500, spread=1)
    got = sample(gpu, p, q, tokens, u, 500)
    chain = np.arange(8) - 1
    assert all(np.array_equal(got[b], walk(p[b], q[b], tokens[b], chain, u[b], 500)) for b in range(30))
    assert (got != NONE).sum(1).max() > 3


def test_sample_odd_inputs(gpu):
    """Twins, random numbers at their ends, drafts that are what is wanted, tokens past the vocabulary, rows of nothing."""
    rng = np.random.default_rng(6)
    batch, rows, vocab = 12, 5, 300
    p, q, tokens, _, _, u = drafted(rng, batch, rows, vocab, vocab)
    parents = np.zeros((batch, rows), np.int64)
    seen = np.zeros((batch, rows, rows), bool)
    seen[:, :, 0] = True
    seen[:, np.arange(rows), np.arange(rows)] = True
    tokens[0, 1:] = tokens[0, 1]                # four times the same
    u[1], u[2] = 0, np.float32(1) - np.float32(2.0**-24)
    q[3] = p[3]                                 # always accepted
    p[4, 0], q[4, 0] = 0, 1 / vocab             # nothing wanted
    p[5, 0], q[5, 0] = np.float32(0.5 / vocab), np.float32(1.0 / vocab)  # nothing left after a rejection: from p
    u[5, 1:] = 0.9
    tokens[6, 1:3] = vocab, NONE                # passed over
    p[7, 0] = 0
    p[7, 0, 299] = 1
    p[8, 0], q[8, 0] = 1 / 256, 1 / 512         # sums and places without roundings
    p[8, 0, 256:] = 0
    u[8] = 17 / 256
    got = sample(gpu, p, q, tokens, u, vocab, bits(seen))
    for b in range(batch):
        assert np.array_equal(got[b], walk(p[b], q[b], tokens[b], parents[b], u[b], vocab)), f"sequence {b}"
    assert got[4, 0] == NONE
    none = sample(gpu, p, None, tokens, u, vocab, bits(seen))
    for b in range(batch):
        assert np.array_equal(none[b], walk(p[b], None, tokens[b], parents[b], u[b], vocab)), f"sequence {b}"


@pytest.mark.parametrize("drafts", [True, False])
def test_sampled_tokens_have_the_targets_distribution(gpu, drafts):
    """20000 roots of three children over 6 ids: the first token's frequencies are p's, within 5 standard deviations."""
    rng = np.random.default_rng(7)
    batch, rows, vocab = 20000, 4, 6
    p = np.broadcast_to(np.float32([0.05, 0.3, 0.1, 0.25, 0.1, 0.2]), (batch, rows, vocab)).copy()
    q = np.broadcast_to(np.float32([0.3, 0.05, 0.1, 0.05, 0.4, 0.1]), (batch, rows, vocab)).copy()
    tokens = rng.choice(vocab, (batch, rows), p=q[0, 0].astype(np.float64) / q[0, 0].sum(dtype=np.float64)).astype(np.uint32)
    seen = np.eye(rows, dtype=bool)[None].repeat(batch, 0)
    seen[:, :, 0] = True
    got = sample(gpu, p, q if drafts else None, tokens, rng.random((batch, rows)).astype(np.float32), vocab, bits(seen))
    share = np.bincount(got[:, 0], minlength=vocab) / batch
    assert np.all(np.abs(share - p[0, 0]) <= 5 * np.sqrt(p[0, 0] * (1 - p[0, 0]) / batch)), share


# ------------------------------------------------------------------------------------------- calls beside each other


def long_call(gpu, cache, rng, rows=3, heads=4):
    """page_attend over a table that is shared out, as a call of its own and its output."""
    batch, g, hd = len(cache.table), cache.kv_heads, cache.hd
    x, mask = gpu.upload(rows_of(rng, batch, rows, heads, g, hd, True)), gpu.upload(bits(trees(rng, batch, rows)[1]))
    n, o, pages = gpu.upload(np.array([2400, 1700][:batch], np.int32)), gpu.buffer(batch * rows * heads * hd // 2), cache.device(gpu)
    t = wa.Tree(batch, rows, n, None, None, mask, rows * ((rows + 31) // 32))
    call = lambda: gpu.page_attend(t, x, x.ptr + 2 * heads * hd, x.ptr + 2 * (heads + g) * hd, (heads + 2 * g) * hd, pages, o, heads, True, True)  # noqa: E731
    return call, lambda: gpu.read(o, (batch, rows, heads * hd), np.float16)


def test_two_contexts_at_once(gpu):
    """Calls queued on two contexts in turn, each with parts of its own: what each gives by itself."""
    rng = np.random.default_rng(30)
    caches = [Cache(rng, type, 128, 2, 64, 2, 20) for type in (wa.Q4_0, wa.F16)]
    for c in caches:
        c.fill(rng, [2560, 2560])
    other = wa.Gpu(0)
    try:
        sides = [long_call(g, c, np.random.default_rng(31)) for g, c in zip((gpu, other), caches)]
        want = []
        for call, result in sides:
            call()
            want.append(result())
        for _ in range(20):
            for call, _result in sides:
                call()
        for (_call, result), w in zip(sides, want):
            assert np.array_equal(result(), w)
    finally:
        del sides
        other.close()


def test_recording_does_not_grow_the_scratch():
    """A call that needs parts, recorded on a context that has never made it: refused, and the context goes on."""
    rng = np.random.default_rng(32)
    cache = Cache(rng, wa.Q4_0, 256, 2, 64, 1, 10)
    cache.fill(rng, [2560])
    fresh = wa.Gpu(0)
    try:
        call, result = long_call(fresh, cache, rng)
        fresh.record_begin()
        with pytest.raises(wa.WavoError, match="record"):
            call()
        fresh.record_end().free()
        call()
        want = result()
        fresh.record_begin()
        call()
        p = fresh.record_end()
        p.replay()
        assert np.array_equal(result(), want) and np.abs(want).max() > 0
        p.free()
    finally:
        fresh.close()


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_pools_past_4_gib(gpu, type):
    """Pages at a pool's far end: the words, rows and outputs of the same tokens in a pool of two."""
    rng = np.random.default_rng(33)
    heads, g, hd, page, rows = 4, 2, 128, 256, 300
    size = wa.page_bytes(type, page, g, hd)
    many = (5 << 30) // size
    x = gpu.upload(rows_of(rng, 1, rows, heads, g, hd, True))
    n, n1 = gpu.upload(np.array([0], np.int32)), gpu.upload(np.array([rows], np.int32))
    h, stride = wa.Heads(heads, g, hd), (heads + 2 * g) * hd
    got = []
    for pages, table in ((2, [1, 0]), (many, [many - 1, many - 2])):
        pool, tb = gpu.buffer(pages * size // 4), gpu.upload(np.array(table, np.int32))
        p = wa.Pages(pool, pages, tb, 2, 2, page, type, g, hd)
        gpu.page_append(wa.Tree(1, rows, n), h, None, x.ptr + 2 * heads * hd, x.ptr + 2 * (heads + g) * hd, stride, p, in16=True)
        k, v, o = (gpu.buffer(rows * w * hd) for w in (g, g, heads))
        gpu.page_read(wa.Tree(1, rows, n), p, k, v, g * hd)
        gpu.page_attend(wa.Tree(1, rows, n1), x, None, None, stride, p, o, heads, in16=True)
        got.append([gpu.read(a, (rows, w * hd)) for a, w in ((k, g), (v, g), (o, heads))])
        del pool, p
    assert all(np.array_equal(a, b) and np.abs(a).max() > 0 for a, b in zip(*got))


def test_sample_large_vocabularies(gpu):
    """More ids than single runs of sums hold."""
    rng = np.random.default_rng(34)
    for vocab, draft in ((300007, True), (524289, False)):
        p, q, tokens, parents, mask, u = drafted(rng, 3, 4, vocab, vocab)
        got = sample(gpu, p, q if draft else None, tokens, u, vocab, mask)
        for b in range(3):
            assert np.array_equal(got[b], walk(p[b], q[b] if draft else None, tokens[b], parents[b], u[b], vocab))


# ------------------------------------------------------------------------------------------- all of them


class Sampler:
    """A decoder of two attention layers whose caches lie in pages: embeddings, [q | k | v] projections, norms and rotation,
    attention, output projections, logits, their rules and probabilities, verification, and the kept path into the pages."""

    def __init__(self, gpu, type, batch, rows, temperature, heads=4, kv_heads=2, hd=32, vocab=160, page=32, cols=4, layers=2, seed=0):
        rng = np.random.default_rng(seed)
        self.gpu, self.batch, self.rows, self.heads, self.kv_heads, self.hd = gpu, batch, rows, heads, kv_heads, hd
        self.vocab, self.layers, self.room = vocab, layers, page * cols
        d, dk, m = heads * hd, kv_heads * hd, batch * rows
        self.d, self.dk, self.stride = d, dk, d + 2 * dk
        lin = lambda n, k, s: gpu.linear([((s * rng.standard_normal((n, k))).astype(np.float32).tobytes(), wa.F32, k, n)])  # noqa: E731
        up = lambda a, t: gpu.upload(np.asarray(a, t))  # noqa: E731
        self.embed, self.none = lin(vocab, d, 1.0), up(np.zeros(d), np.float32)
        self.qkv = [lin(self.stride, d, 2.0 / np.sqrt(d)) for _ in range(layers)]
        self.proj = [lin(d, d, 1.0 / np.sqrt(d)) for _ in range(layers)]
        self.head = lin(vocab, d, 3.0 / np.sqrt(d))
        gains = [up(1.5 + 0.2 * rng.standard_normal(hd), np.float32) for _ in range(2)]
        self.table = up(rope_table(self.room, hd), np.float32)
        self.norms = wa.Heads(heads, kv_heads, hd, gains[0], gains[1], 1e-6, self.table, self.room, hd)
        pages = batch * cols + 1
        self.pages = []
        for _ in range(layers):
            pool = gpu.upload(rng.integers(0, 2**32, (pages, wa.page_bytes(type, page, kv_heads, hd) // 4), dtype=np.uint32))
            self.pages.append(wa.Pages(pool, pages, up(rng.permutation(pages)[:batch * cols], np.int32), cols, cols, page, type, kv_heads, hd))
        self.x, self.raw = gpu.buffer(m * d), [gpu.buffer(m * self.stride) for _ in range(layers)]
        self.turned, self.o, self.logits, self.probs = gpu.buffer(m * self.stride), gpu.buffer(m * d), gpu.buffer(m * vocab), gpu.buffer(m * vocab)
        z = lambda *s: up(np.zeros(s), np.int32)  # noqa: E731
        self.n, self.n1, self.count, self.tokens, self.mask = z(batch), z(batch), z(batch), z(batch, rows), z(batch, rows, (rows + 31) // 32)
        self.pick, self.path, self.kept, self.next, self.history = z(batch, rows), z(batch, rows), z(batch), z(batch), z(batch, self.room)
        self.penalty, self.temperature = up([[1.2, 0.1, 0.05]] * batch, np.float32), up([temperature] * batch, np.float32)
        self.u, self.q = gpu.buffer(m), gpu.buffer(m * vocab)
        self.draws = temperature > 0

    def tree(self):
        return wa.Tree(self.batch, self.rows, self.n, self.count, self.tokens, self.mask, self.rows * ((self.rows + 31) // 32))

    def step(self):
        g, m, t, rules = self.gpu, self.batch * self.rows, self.tree(), wa.Rules(self.penalty, self.history, self.room)
        for r in range(m):
            g.embed(self.embed, self.none, self.x.ptr + 4 * r * self.d, self.tokens, r, 0)
        for l in range(self.layers):
            g.gemm(self.x, self.qkv[l], self.raw[l], m, wa.BIAS)
            g.head_norm(t, self.norms, self.raw[l], self.stride, self.turned, self.stride)
            g.page_attend(t, self.turned, self.turned.ptr + 4 * self.d, self.turned.ptr + 4 * (self.d + self.dk), self.stride, self.pages[l], self.o,
                          self.heads)
            g.gemm(self.o, self.proj[l], self.x, m, wa.RESIDUAL, 1.0)
        g.gemm(self.x, self.head, self.logits, m, wa.BIAS)
        g.logit_rules(t, rules, self.logits, self.logits, self.vocab, self.vocab)
        g.logit_probs(t, self.logits, self.probs, self.vocab, self.vocab, self.vocab, self.temperature)
        g.tree_sample(t, self.probs, self.q if self.draws else None, self.vocab, self.vocab, self.u, self.pick)
        g.tree_accept(t, self.pick, None, None, 0, 0, None, 0, 0, 0, self.room, 0, self.path, self.kept, self.next, self.n1, self.history, self.room)
        for l in range(self.layers):
            k = self.raw[l].ptr + 4 * self.d
            g.page_append(t, self.norms, None, k, k + 4 * self.dk, self.stride, self.pages[l], self.path, self.kept)
        g.copy(self.n, self.n1, 4 * self.batch)

    def generate(self, rng, want, drafts=None, record=False):
        """Texts of `want` tokens, with draft trees of right (from `drafts`) and wrong tokens, or of those drawn from random rows."""
        g, batch, rows, vocab = self.gpu, self.batch, self.rows, self.vocab
        g.write(self.n, np.zeros(batch, np.int32))
        root, text = np.arange(batch) + 20, [[] for _ in range(batch)]
        steps, recorded = 0, None
        while min(len(x) for x in text) < want:
            parents, seen = trees(rng, batch, rows, 4)
            tokens, count, depth = np.zeros((batch, rows), np.uint32), np.zeros(batch, np.int32), seen.sum(2) - 1
            q = softmax(3 * rng.standard_normal((batch, rows, vocab)))
            for b in range(batch):
                tokens[b, 0], count[b] = root[b], 0 if len(text[b]) >= want else rng.integers((rows + 1) // 2, rows + 1)
                for i in range(1, rows):
                    at = len(text[b]) + depth[b, i]
                    c = np.cumsum(q[b, parents[b, i]].astype(np.float64))
                    x = min(np.searchsorted(c, rng.random() * c[-1]), vocab - 1)
                    tokens[b, i] = drafts[b][at] if drafts is not None and at < len(drafts[b]) and rng.random() < 0.6 else x
            g.write(self.tokens, tokens)
            g.write(self.count, count)
            g.write(self.mask, bits(seen))
            g.write(self.u, rng.random((batch, rows)).astype(np.float32))
            g.write(self.q, q)
            if record and steps == 1:
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
        return [x[:want] for x in text], steps


@pytest.mark.parametrize("record", [False, True])
def test_drafted_decoding_over_pages_gives_the_same_tokens(gpu, record):
    """At temperature zero, over pages of f16: trees of drafts, right and wrong ones, against one token per step.  The two differ by
    rounding alone (rows of other batch sizes, f32 norms for 64 bits'), so the seed's texts have no ties at that level."""
    want, _ = Sampler(gpu, wa.F16, 3, 1, 0.0).generate(np.random.default_rng(1), 40)
    got, steps = Sampler(gpu, wa.F16, 3, 11, 0.0).generate(np.random.default_rng(2), 40, want, record)
    assert got == want
    assert steps < 30
    assert len(set(want[0])) > 10


@pytest.mark.parametrize("type", [wa.Q4_0, wa.F16])
def test_sampled_decoding_over_pages_repeats_itself(gpu, type):
    """The same random numbers and drafts: the same texts, recorded or not."""
    texts = [Sampler(gpu, type, 3, 9, 0.8).generate(np.random.default_rng(3), 30, None, record)[0] for record in (False, False, True)]
    assert texts[0] == texts[1] == texts[2]
    assert len(set(texts[0][0])) > 10
